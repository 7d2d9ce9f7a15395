// Products with microscaled 4-bit operands on the matrix cores.
//
//   matmul: out[i][j] = bias[j] + sum_k x[i][k] w[j][k], both in blocks;
//   linear: the same with x in fp32, bf16 or fp16 as it is.
//
// The scaled product instruction takes 4-bit operands whole: in the 16 x 16 x 128
// form a lane gives one block, 16 bytes of codes and their scale byte, of row
// lane % 16 and block lane / 16; in the 32 x 32 x 64 form row lane % 32 and block
// lane / 32.  Products and sums are fp32.
#include "mx4_device.hpp"
#include "mx4_internal.hpp"

namespace fufft {
namespace mx4 {

namespace {

typedef int    i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ inline i32x8 operand4(u32x4 c)
{
   return i32x8{(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
}

// ---- few rows: operands straight from memory, K split over the wavefronts ----------
//
// A workgroup computes 16 MT rows of x times 16 NT rows of w.  Its wavefronts take
// the groups of 128 values in turn, and their sums are joined in LDS in the order
// of the wavefronts.

// The rows of x as the w operand meets them: a value in bf16 is one, in fp16 two, in
// fp32 three bf16 parts (8, 11 and 24 significant bits at 8 a part, cut off rather than
// rounded, so that no part overflows).  The parts add up to the value exactly but for
// bits below 2^-133, so the product is that of the values themselves.
template<class T> struct PartsOf;
template<> struct PartsOf<bf16>  { static constexpr int value = 1; };
template<> struct PartsOf<f16>   { static constexpr int value = 2; };
template<> struct PartsOf<float> { static constexpr int value = 3; };

template<class T, int PARTS = PartsOf<T>::value>
__device__ inline void split8(const float (&v)[8], bf16x8 (&part)[PARTS])
{
#pragma unroll
   for(int i = 0; i < 8; i++) {
      float left = v[i];
#pragma unroll
      for(int q = 0; q < PARTS; q++) {
         const float b = __uint_as_float(__float_as_uint(left) & 0xffff0000u);
         part[q][i] = __builtin_bit_cast(bf16, (uint16_t)(__float_as_uint(left) >> 16));
         if(q + 1 < PARTS) left = magnitude(left) == 0x7f800000u ? 0.0f : left - b;   // all of an infinity is in one part
      }
   }
}

__device__ inline bf16x8 decode8_bf16(uint32_t c, float p)
{
   const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, p, 0);
   const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, p, 1);
   const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, p, 2);
   const bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, p, 3);
   return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// wavefronts of a workgroup with so many 16 x 16 tiles: their sums fill at most 64 KiB of LDS
constexpr int most_waves(int tiles) { return tiles >= 16 ? 4 : tiles >= 4 ? 8 : 16; }

// the sums of all wavefronts, joined, and stored: acc[mt][nt] holds rows
// 4 (lane / 16) + r of w and row lane % 16 of x
template<class O, int MT, int NT>
__device__ inline void join_and_store(const MatmulParams& p, f32x4 (&acc)[MT][NT], float* join, int waves, int64_t m0,
                                      int64_t n0)
{
   constexpr int COLS = 16 * NT, ROWS = 16 * MT;
   const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
   for(int a = 0; a < MT; a++)
#pragma unroll
      for(int b = 0; b < NT; b++)
         *reinterpret_cast<f32x4*>(join + (wave * ROWS + a * 16 + (lane & 15)) * COLS + b * 16 + (lane >> 4) * 4) =
            acc[a][b];
   __syncthreads();
   O* out = static_cast<O*>(p.out);
   for(int i = threadIdx.x; i < ROWS * COLS; i += waves * 64) {
      const int64_t m = m0 + i / COLS, n = n0 + i % COLS;
      if(m >= p.m || n >= p.n) continue;
      float v = 0.0f;
      for(int w = 0; w < waves; w++) v += join[w * ROWS * COLS + i];
      if(p.bias) v += p.bias[n];
      out[m * p.ld + n] = (O)v;
   }
}

template<class O, int MT, int NT>
__global__ void __launch_bounds__(64 * most_waves(MT * NT))
matmul_rows(MatmulParams p, int64_t groups, int waves)
{
   extern __shared__ float join[];
   const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
   const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
   const uint8_t* xc[MT];
   const uint8_t* xs[MT];
   const uint8_t* wc[NT];
   const uint8_t* ws[NT];
#pragma unroll
   for(int a = 0; a < MT; a++) {         // rows beyond the last read the last one
      int64_t r = m0 + a * 16 + (lane & 15);
      r = r < p.m ? r : p.m - 1;
      xc[a] = static_cast<const uint8_t*>(p.x) + r * groups * 64 + (lane >> 4) * 16;
      xs[a] = p.x_scales + r * groups * 4 + (lane >> 4);
   }
#pragma unroll
   for(int b = 0; b < NT; b++) {
      int64_t r = n0 + b * 16 + (lane & 15);
      r = r < p.n ? r : p.n - 1;
      wc[b] = p.w + r * groups * 64 + (lane >> 4) * 16;
      ws[b] = p.w_scales + r * groups * 4 + (lane >> 4);
   }
   f32x4 acc[MT][NT] = {};
#pragma unroll 1
   for(int64_t g = wave; g < groups; g += waves) {
      u32x4 x[MT], w[NT];
      int sx[MT], sw[NT];
#pragma unroll
      for(int b = 0; b < NT; b++) {
         w[b] = *reinterpret_cast<const u32x4*>(wc[b] + g * 64);
         sw[b] = ws[b][g * 4];
      }
#pragma unroll
      for(int a = 0; a < MT; a++) {
         x[a] = *reinterpret_cast<const u32x4*>(xc[a] + g * 64);
         sx[a] = xs[a][g * 4];
      }
#pragma unroll
      for(int a = 0; a < MT; a++)
#pragma unroll
         for(int b = 0; b < NT; b++)
            acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand4(w[b]), operand4(x[a]), acc[a][b], 4, 4,
                                                                         0, sw[b], 0, sx[a]);
   }
   join_and_store<O, MT, NT>(p, acc, join, waves, m0, n0);
}

// The block that a lane reads holds its 8 values of each of four products, so
// product t takes values 8 t .. 8 t + 7 of the four blocks of a group.
template<class T, class O, int MT, int NT>
__global__ void __launch_bounds__(64 * most_waves(MT * NT))
linear_rows(MatmulParams p, int64_t groups, int waves)
{
   constexpr int PARTS = PartsOf<T>::value;
   extern __shared__ float join[];
   const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
   const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
   const int64_t k0 = (lane >> 4) * 32;
   const T* x[MT];
   const uint8_t* wc[NT];
   const uint8_t* ws[NT];
#pragma unroll
   for(int a = 0; a < MT; a++) {
      int64_t r = m0 + a * 16 + (lane & 15);
      r = r < p.m ? r : p.m - 1;
      x[a] = static_cast<const T*>(p.x) + r * p.ldx;
   }
#pragma unroll
   for(int b = 0; b < NT; b++) {
      int64_t r = n0 + b * 16 + (lane & 15);
      r = r < p.n ? r : p.n - 1;
      wc[b] = p.w + r * groups * 64 + (lane >> 4) * 16;
      ws[b] = p.w_scales + r * groups * 4 + (lane >> 4);
   }
   f32x4 acc[MT][NT] = {};
#pragma unroll 1
   for(int64_t g = wave; g < groups; g += waves) {
      u32x4 w[NT];
      float sw[NT];
#pragma unroll
      for(int b = 0; b < NT; b++) {
         w[b] = *reinterpret_cast<const u32x4*>(wc[b] + g * 64);
         sw[b] = scale_operand(ws[b][g * 4]);
      }
#pragma unroll
      for(int t = 0; t < 4; t++) {
         bf16x8 part[MT][PARTS];
         const int64_t k = g * 128 + k0 + t * 8;
#pragma unroll
         for(int a = 0; a < MT; a++) {
            float v[8];
            if(k + 8 <= p.k) {
               load8(x[a] + k, v);
            } else {
#pragma unroll
               for(int i = 0; i < 8; i++) v[i] = k + i < p.k ? to_float(x[a][k + i]) : 0.0f;
            }
            split8<T>(v, part[a]);
         }
#pragma unroll
         for(int b = 0; b < NT; b++) {
            const bf16x8 v = decode8_bf16(w[b][t], sw[b]);
#pragma unroll
            for(int a = 0; a < MT; a++)
#pragma unroll
               for(int q = 0; q < PARTS; q++)
                  acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, part[a][q], acc[a][b], 0, 0, 0);
         }
      }
   }
   join_and_store<O, MT, NT>(p, acc, join, waves, m0, n0);
}

int wavefronts(int64_t groups, int most)
{
   int w = 1;
   while(w < most && w * 2 <= groups) w *= 2;
   return w;
}

template<class O, int MT, int NT>
hipError_t rows_shape(const MatmulParams& p, hipStream_t s)
{
   const int64_t groups = padded(p.k) / kGroup;
   const int waves = wavefronts(groups, most_waves(MT * NT));
   const int64_t gx = (p.n + 16 * NT - 1) / (16 * NT), gy = (p.m + 16 * MT - 1) / (16 * MT);
   if(gx > 0x7fffffff || gy > 65535) return hipErrorInvalidValue;
   matmul_rows<O, MT, NT><<<dim3((unsigned)gx, (unsigned)gy), waves * 64, (size_t)waves * MT * NT * 1024, s>>>(
      p, groups, waves);
   return hipGetLastError();
}

template<class O>
hipError_t matmul_typed(const MatmulParams& p, hipStream_t s)
{
   if(p.m <= 16) return rows_shape<O, 1, 1>(p, s);
   if(p.m <= 32) return rows_shape<O, 2, 1>(p, s);
   return rows_shape<O, 4, 4>(p, s);
}

template<class T, class O, int MT, int NT>
hipError_t linear_shape(const MatmulParams& p, hipStream_t s)
{
   const int64_t groups = padded(p.k) / kGroup;
   const int waves = wavefronts(groups, most_waves(MT * NT));
   const int64_t gx = (p.n + 16 * NT - 1) / (16 * NT), gy = (p.m + 16 * MT - 1) / (16 * MT);
   if(gx > 0x7fffffff || gy > 65535) return hipErrorInvalidValue;
   linear_rows<T, O, MT, NT><<<dim3((unsigned)gx, (unsigned)gy), waves * 64, (size_t)waves * MT * NT * 1024, s>>>(
      p, groups, waves);
   return hipGetLastError();
}

template<class T, class O>
hipError_t linear_typed(const MatmulParams& p, hipStream_t s)
{
   if(p.m <= 16) return linear_shape<T, O, 1, 1>(p, s);
   if(p.m <= 32) return linear_shape<T, O, 2, 1>(p, s);
   return linear_shape<T, O, 4, 1>(p, s);
}

template<class T>
hipError_t linear_out(const MatmulParams& p, hipStream_t s)
{
   switch(p.type) {
      case T_F32:  return linear_typed<T, float>(p, s);
      case T_BF16: return linear_typed<T, bf16>(p, s);
      default:     return linear_typed<T, f16>(p, s);
   }
}

}  // namespace

hipError_t launch_matmul(const MatmulParams& p, hipStream_t s)
{
   if(p.m <= 0 || p.n <= 0) return hipSuccess;
   switch(p.type) {
      case T_F32:  return matmul_typed<float>(p, s);
      case T_BF16: return matmul_typed<bf16>(p, s);
      default:     return matmul_typed<f16>(p, s);
   }
}

hipError_t launch_linear(const MatmulParams& p, hipStream_t s)
{
   if(p.m <= 0 || p.n <= 0) return hipSuccess;
   switch(p.x_type) {
      case T_F32:  return linear_out<float>(p, s);
      case T_BF16: return linear_out<bf16>(p, s);
      default:     return linear_out<f16>(p, s);
   }
}

}  // namespace mx4
}  // namespace fufft
