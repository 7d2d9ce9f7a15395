// Host-only check of the norm, 8-bit and decaying-attention part of the C++ header: sizes, and
// arguments that are refused or have nothing to do before anything is launched.  Built and run
// by tests/test_layer_hpp_cpu.py.
#include "fufft/fufft.hpp"

using namespace fufft::layer;

int main()
{
   if(padded(129) != 256 || code_bytes(3, 129) != 768) return 1;
   uint8_t* const at = reinterpret_cast<uint8_t*>(0x10000000);
   const auto floats = [&](int64_t i) { return reinterpret_cast<float*>(at + i * 0x1000000); };
   const Rows8 none, a{at, floats(1)}, b{at + 0x2000000, floats(3)};
   const Matrix x{at + 0x4000000, Type::BF16, 4, 64}, narrow{at + 0x4000000, Type::BF16, 4, 64, 32};
   const MutableMatrix out{at + 0x5000000, Type::F32, 4, 8}, over{a.codes, Type::F32, 4, 8};
   if(quantize(x, none) != FUFFT_ERR_INVALID || quantize(narrow, a) != FUFFT_ERR_INVALID) return 2;
   if(quantize(x, {at + 1, floats(1)}) != FUFFT_ERR_ALIGN || dequantize(a, over) != FUFFT_ERR_INVALID) return 3;
   if(matmul(a, none, out, 64) != FUFFT_ERR_INVALID || matmul(a, b, over, 64) != FUFFT_ERR_INVALID) return 4;
   if(matmul(a, b, out, 131072) != FUFFT_ERR_UNSUPPORTED) return 5;
   if(matmul(a, b, {nullptr, Type::F32, 0, 8}, 64) != FUFFT_OK) return 6;
   Norm n;
   if(rms_norm(x, n, Type::F32) != FUFFT_ERR_INVALID) return 7;                     // nothing to write
   n.out = {at + 0x6000000};
   if(rms_norm(x, n, Type::F16) != FUFFT_ERR_INVALID) return 8;                     // neither x's type nor fp32
   n.total = {at + 0x6000000};
   if(rms_norm(x, n, Type::BF16) != FUFFT_ERR_INVALID) return 9;                    // two outputs at one place
   if(rms_norm({nullptr, Type::BF16, 0, 64}, n, Type::BF16) != FUFFT_OK) return 10;
   const MutableMatrix dx{at + 0x7000000, Type::BF16, 4, 64};
   if(rms_norm_grad(x, {at + 0x8000000, Type::F32, 3, 64}, {}, nullptr, 1e-6f, dx, nullptr, nullptr, 0) != FUFFT_ERR_INVALID)
      return 11;
   if(rms_norm_grad(x, {at + 0x8000000, Type::F32, 4, 64}, {}, nullptr, 1e-6f, dx, floats(9), nullptr, 0) != FUFFT_ERR_INVALID)
      return 12;
   Decay d{2, 5, 3, 8, 8, Type::BF16, floats(10)};
   const fufft_strides side{120, 24, 8};
   const Heads q{at + 0xb000000, side}, k{at + 0xc000000, side}, v{at + 0xd000000, side};
   const MutableHeads y{at + 0xe000000, side}, onto{at + 0xb000000, side}, z{at + 0xf000000, side};
   if(attention(d, q, k, v, onto) != FUFFT_ERR_INVALID) return 13;
   d.splits = 4;
   if(attention(d, q, k, v, y) != FUFFT_ERR_INVALID) return 14;                     // splits without their space
   d.splits = 0;
   if(attention_grad(d, q, q, k, v, y, y, z) != FUFFT_ERR_INVALID) return 15;       // two gradients at one place
   if(step(d, q, k, v, y, floats(16), 1) != FUFFT_ERR_INVALID) return 16;           // two sequences, one state
   d.dk = 129;
   if(attention(d, q, k, v, y) == FUFFT_OK) return 17;
   d.dk    = 8;
   d.batch = 0;
   if(attention(d, q, k, v, y) != FUFFT_OK || step(d, q, k, v, y, floats(16), 1) != FUFFT_OK) return 18;
   return 0;
}
