// Device code shared by the kernels on microscaled 4-bit blocks (mx4): element
// types, the block's scale and codes, and the way back to values.
//
// A block is 32 consecutive values of a row.  Its scale byte s stands for
// 2^(s - 127) (255: NaN), its codes for 0, .5, 1, 1.5, 2, 3, 4, 6 and their
// negatives; a value is the product.  Rows are padded to whole groups of 128
// values (64 bytes of codes, 4 scale bytes) with zero codes, so a row of either
// array starts aligned and every product reads whole groups.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fufft {
namespace mx4 {

constexpr int kBlock = 32;    // values per scale
constexpr int kGroup = 128;   // values per padding unit of a row

typedef __bf16   bf16;
typedef _Float16 f16;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float    f32x2 __attribute__((ext_vector_type(2)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16   bf16x2 __attribute__((ext_vector_type(2)));

template<class T> __device__ inline float to_float(T v) { return (float)v; }

// eight consecutive elements, at the element type's alignment (the global loads
// and stores of gfx950 take any alignment at their full width)
template<class T>
__device__ inline void load8(const T* p, float (&v)[8])
{
   struct __attribute__((packed, aligned(sizeof(T)))) V { T e[8]; };
   const V t = *reinterpret_cast<const V*>(p);
#pragma unroll
   for(int i = 0; i < 8; i++) v[i] = to_float(t.e[i]);
}
template<class T>
__device__ inline void store8(T* p, const float (&v)[8])
{
   struct __attribute__((packed, aligned(sizeof(T)))) V { T e[8]; };
   V t;
#pragma unroll
   for(int i = 0; i < 8; i++) t.e[i] = (T)v[i];
   *reinterpret_cast<V*>(p) = t;
}

template<int CTRL>
__device__ inline uint32_t dpp(uint32_t v)
{
   return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kQuadSwap1 = 0xb1;    // lane ^ 1
constexpr int kQuadSwap2 = 0x4e;    // lane ^ 2
constexpr int kRowLeft4  = 0x104;   // lane + 4 of the 16
constexpr int kRowLeft8  = 0x108;   // lane + 8 of the 16

__device__ inline uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ inline uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The block's scale byte from the bits of its largest magnitude (which order as
// the magnitudes do, NaN above infinity).  `fit`: the smallest power of two p
// with top <= 6 p, so nothing saturates; otherwise the power of two below top,
// over 4, and magnitudes above 6 p saturate.  A power below 2^-127 becomes that.
__device__ inline uint32_t scale_byte(uint32_t top, bool fit)
{
   if(top >= 0x7f800000u) return 255u;
   const int e = (int)(top >> 23) - 2 + ((fit && (top & 0x7fffffu) > 0x400000u) ? 1 : 0);
   return e < 0 ? 0u : (uint32_t)e;
}

// 2^(s - 127) as the scaled conversions and products take it: they read the
// exponent field alone, 0 there as 2^-127 and 255 as NaN
__device__ inline float scale_operand(uint32_t s) { return __uint_as_float(s << 23); }

// Eight values to eight codes, nearest, ties to the even code, at most 6.
__device__ inline uint32_t encode8(const float (&v)[8], uint32_t s)
{
   if(s == 255u) return 0u;
   const float p = scale_operand(s);
   uint32_t c = 0;
   c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], p, 0);
   c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], p, 1);
   c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], p, 2);
   c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], p, 3);
   return c;
}

// One value to its code with a given random byte r: the neighbour above if the
// distance to the one below, in steps, plus (r + 1/2) / 256 reaches 1.  a, t, and
// t - low are exact (a power of two, a halving and a difference of neighbours);
// where a underflows no r rounds it up.
__device__ inline uint32_t encode_random(float v, float inverse, uint32_t r)
{
   const float a = __uint_as_float(magnitude(v)) * inverse;
   const float t = a >= 4.0f ? a * 0.5f : a >= 2.0f ? a : a * 2.0f;
   const float low = floorf(t);
   const uint32_t up = (t - low) >= 1.0f - ((float)r + 0.5f) * (1.0f / 256.0f) ? 1u : 0u;
   uint32_t c = (uint32_t)low + up + (a >= 4.0f ? 4u : a >= 2.0f ? 2u : 0u);
   c = c > 7u ? 7u : c;
   return c | ((__float_as_uint(v) >> 28) & 8u);
}
// The same for values of 16-bit types by the conversion to the nearest, in half the
// instructions.  With p the power of two below a (1 at least, 4 at most, so that a step
// is p / 2), c = a + p ((r + 1/2) / 512 - 1/4 + 2^-22) is half a step below a plus that
// share of a step, so the nearest code to c is the one to take, but where c falls
// below the power of two under a, past which the steps are finer: c is at least that.
// The 2^-22 p decides ties upwards; a has 11 bits, so c is exact and nothing else lies
// that near a tie.  (r, K: the share is exact in fp32 too.)
__device__ inline float dithered(float v, float inverse, float r)
{
   const float a = __uint_as_float(magnitude(v)) * inverse;
   const float below = __uint_as_float(__float_as_uint(a) & 0x7f800000u);
   const float p = __builtin_amdgcn_fmed3f(below, 1.0f, 4.0f);
   const float share = fmaf(r, 1.0f / 512.0f, 1.0f / 1024.0f - 0.25f + 0x1p-22f);
   const float c = fmaxf(fmaf(p, share, a), below);
   return __uint_as_float((__float_as_uint(v) & 0x80000000u) | __float_as_uint(c));
}

// eight values with their random bytes; 16 bits: the values are of a 16-bit type
template<bool BITS16>
__device__ inline uint32_t encode8_random(const float (&v)[8], uint32_t s, const uint32_t (&r)[8])
{
   if(s == 255u) return 0u;
   const float inverse = __uint_as_float((254u - s) << 23);   // 2^(127 - s); s <= 253 here
   uint32_t c = 0;
   if constexpr(BITS16) {
      float d[8];
#pragma unroll
      for(int i = 0; i < 8; i++) d[i] = dithered(v[i], inverse, (float)r[i]);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, d[0], d[1], 1.0f, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, d[2], d[3], 1.0f, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, d[4], d[5], 1.0f, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, d[6], d[7], 1.0f, 3);
   } else {
#pragma unroll
      for(int i = 0; i < 8; i++) c |= encode_random(v[i], inverse, r[i]) << (4 * i);
   }
   return c;
}

// eight codes back to values (exact; NaN for scale 255)
__device__ inline void decode8(uint32_t c, uint32_t s, float (&v)[8])
{
   const float p = scale_operand(s);
   const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, p, 0);
   const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, p, 1);
   const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, p, 2);
   const f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, p, 3);
   v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
   v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
}

}  // namespace mx4
}  // namespace fufft
