// Internal interface between the entry points of the norm, 8-bit and decaying-attention
// calls (layer_capi.hip) and their kernels (norm.hip, i8_matmul.hip, decay.hip).
#pragma once

#include "mx4_internal.hpp"

namespace fufft {
namespace layer {

using mx4::grid_ok;
using mx4::kTooLarge;
using mx4::padded;
using mx4::T_BF16;
using mx4::T_F16;
using mx4::T_F32;

struct NormParams {
   const void*  x;
   const void*  residual;    // or NULL
   void*        total;       // or NULL
   const float* weight;      // or NULL
   void*        out;         // or NULL
   int8_t*      codes;       // rows x padded(k), or NULL
   float*       scales;
   int64_t      ldx, ldr, ldt, ldo, rows, k;
   float        eps;
   int          type, sum_type;
};
hipError_t launch_rms_norm(const NormParams& p, hipStream_t s);
hipError_t launch_i8_quantize(const NormParams& p, hipStream_t s);   // x, codes, scales, ldx, rows, k, type

struct NormGradParams {
   const void*  dy;
   const void*  h;
   const void*  dtotal;      // or NULL
   const float* weight;      // or NULL
   void*        dx;
   float*       dweight;     // or NULL
   float*       work;        // splits x k
   int64_t      ldy, ldh, ldt, ldx, rows, k, splits;
   float        eps;
   int          type, sum_type, dx_type;
};
hipError_t launch_rms_norm_grad(const NormGradParams& p, hipStream_t s);

hipError_t launch_i8_dequantize(const int8_t* codes, const float* scales, void* out, int type, int64_t ld, int64_t rows,
                                int64_t k, hipStream_t s);

constexpr int64_t kLongestI8 = 131071;     // 128 * 128 * 131072 leaves 32 bits

struct I8Params {
   const int8_t* a;          // m x padded(k)
   const int8_t* b;          // n x padded(k)
   const float*  a_scales;
   const float*  b_scales;
   const float*  bias;       // or NULL
   void*         out;        // m x n, leading dimension ld
   int64_t       ld, m, n, k;
   int           type;
};
hipError_t launch_i8_matmul(const I8Params& p, hipStream_t s);

}  // namespace layer
}  // namespace fufft
