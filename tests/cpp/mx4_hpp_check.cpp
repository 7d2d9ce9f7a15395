// Host-only check of the 4-bit part of the C++ header: sizes, and arguments that are refused
// before anything is launched.  Built and run by tests/test_mx4_cpu.py.
#include "fufft/fufft.hpp"

using namespace fufft::mx4;

int main()
{
   if(padded(129) != 256 || code_bytes(3, 129) != 384 || scale_bytes(3, 129) != 24) return 1;
   uint8_t* const at = reinterpret_cast<uint8_t*>(0x10000000);
   const Blocks none, b{at, at + 0x1000000}, d{at + 0x2000000, at + 0x3000000};
   const Matrix x{at + 0x4000000, Type::BF16, 4, 64}, narrow{at + 0x4000000, Type::BF16, 4, 64, 32};
   const MutableMatrix out{at + 0x5000000, Type::F32, 4, 8}, over{b.codes, Type::F32, 4, 8};
   if(quantize(x, none) != FUFFT_ERR_INVALID || quantize(narrow, b) != FUFFT_ERR_INVALID) return 2;
   if(quantize(x, {at + 1, at + 0x1000000}) != FUFFT_ERR_ALIGN) return 3;
   if(dequantize(b, over) != FUFFT_ERR_INVALID) return 4;
   if(matmul(b, none, out, 64) != FUFFT_ERR_INVALID || matmul(b, d, over, 64) != FUFFT_ERR_INVALID) return 5;
   if(linear({at + 0x4000000, Type::BF16, 3, 64}, b, out) != FUFFT_ERR_INVALID) return 6;
   if(matmul(b, d, {nullptr, Type::F32, 0, 8}, 64) != FUFFT_OK) return 7;
   const int32_t* const ints = reinterpret_cast<const int32_t*>(at + 0x6000000);
   Cache c{b, 8, 16, 64, ints, 4, ints + 4096, 2};
   if(write(c, x, nullptr) != FUFFT_ERR_INVALID || write(c, {at, Type::F32, 4, 63}, nullptr) != FUFFT_ERR_INVALID) return 8;
   c.page = 12;
   if(read(c, at + 0x5000000, Type::F32, 10) != FUFFT_ERR_INVALID) return 9;
   c.page = 16;
   if(conv(c, at + 0x7000000, Type::F32, 10, at + 0x5000000, Type::BF16) != FUFFT_ERR_INVALID) return 10;
   c.batch = 0;
   if(read(c, nullptr, Type::F32, 10) != FUFFT_OK) return 11;
   return 0;
}
