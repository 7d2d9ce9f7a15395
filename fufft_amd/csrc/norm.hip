// Root-mean-square norm with the residual's sum and 8-bit rows, its gradients, and the way
// to 8-bit rows and back.
//
//   h = x + residual      r = 1 / sqrt(mean(h^2) + eps)      y = h r w
//   8 bits: scale = max|y| / 127, code = the integer nearest to 127 y / max|y|, ties to even
//   dx = r (w dy - n mean(w dy n)) + dtotal,   n = r h;      dw = sum over rows of dy n
//
// Rows are held in registers between reading and writing, by 4 lanes to 16 wavefronts,
// so that each byte crosses memory once: every call here is bound by its bytes.
#include "layer_internal.hpp"
#include "mx4_device.hpp"

namespace fufft {
namespace layer {

namespace {

using mx4::bf16;
using mx4::dpp;
using mx4::f16;
using mx4::load8;
using mx4::magnitude;
using mx4::store8;
using mx4::u32x2;
using mx4::umax;

// eight consecutive elements as they are in memory, at the element's alignment
template<class T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T e[8]; };

// of a row of k elements from `col` on, zeros beyond its end
template<class T>
__device__ inline Eight<T> fetch8(const T* row, int64_t col, int64_t k)
{
   if(col + 8 <= k) return *reinterpret_cast<const Eight<T>*>(row + col);
   Eight<T> v;
#pragma unroll
   for(int i = 0; i < 8; i++) v.e[i] = col + i < k ? row[col + i] : (T)0.0f;
   return v;
}
// the same where k is a multiple of 8: no branch, the row's first eight in place of those that are not there
template<class T>
__device__ inline Eight<T> fetch8_whole(const T* row, int64_t col, int64_t k)
{
   return *reinterpret_cast<const Eight<T>*>(row + (col < k ? col : 0));
}
// past: beyond the L2, of 16-bit elements
template<class T>
__device__ inline void put8(T* row, int64_t col, int64_t k, const float (&v)[8], bool past = false)
{
   if(col + 8 <= k) {
      if(sizeof(T) == 2 && past) {
         typedef uint32_t V __attribute__((ext_vector_type(2 * sizeof(T)), aligned(sizeof(T))));
         Eight<T> t;
#pragma unroll
         for(int i = 0; i < 8; i++) t.e[i] = (T)v[i];
         __builtin_nontemporal_store(__builtin_bit_cast(V, t), reinterpret_cast<V*>(row + col));
      } else {
         store8<T>(row + col, v);
      }
   } else {
#pragma unroll
      for(int i = 0; i < 8; i++)
         if(col + i < k) row[col + i] = (T)v[i];
   }
}

__device__ inline void put_codes(int8_t* to, u32x2 c, bool past)
{
   if(past) __builtin_nontemporal_store(c, reinterpret_cast<u32x2*>(to));
   else     *reinterpret_cast<u32x2*>(to) = c;
}

// ---- sums and maxima over the lanes of a row ----------------------------------------

constexpr int kHalfMirror = 0x141, kMirror = 0x140;     // within 8 and 16 lanes

__device__ inline float lane_value(float v, int lane)
{
   return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
// over 16 lanes by DPP, the same in all of them
__device__ inline float sum16(float v)
{
   v += __uint_as_float(dpp<mx4::kQuadSwap1>(__float_as_uint(v)));
   v += __uint_as_float(dpp<mx4::kQuadSwap2>(__float_as_uint(v)));
   v += __uint_as_float(dpp<kHalfMirror>(__float_as_uint(v)));
   return v + __uint_as_float(dpp<kMirror>(__float_as_uint(v)));
}
__device__ inline uint32_t max16(uint32_t v)
{
   v = umax(v, dpp<mx4::kQuadSwap1>(v));
   v = umax(v, dpp<mx4::kQuadSwap2>(v));
   v = umax(v, dpp<kHalfMirror>(v));
   return umax(v, dpp<kMirror>(v));
}
__device__ inline float sum4(float v)
{
   v += __uint_as_float(dpp<mx4::kQuadSwap1>(__float_as_uint(v)));
   return v + __uint_as_float(dpp<mx4::kQuadSwap2>(__float_as_uint(v)));
}
__device__ inline uint32_t max4(uint32_t v)
{
   v = umax(v, dpp<mx4::kQuadSwap1>(v));
   return umax(v, dpp<mx4::kQuadSwap2>(v));
}
// over the wavefront: the four sixteens
__device__ inline float wave_sum(float v)
{
   v = sum16(v);
   return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
__device__ inline uint32_t wave_max(uint32_t v)
{
   v = max16(v);
   const uint32_t a = umax(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
   return umax(a, umax(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// Over the LANES lanes of a row, several rows a workgroup.  `turn` counts the uses of the exchange between
// wavefronts, which has two sides so that one barrier a use is enough; all rows of a workgroup
// come to it alike.
template<int LANES>
__device__ inline float row_sum(float v, uint32_t (&side)[2][16], int& turn)
{
   if constexpr(LANES == 4) return sum4(v);
   if constexpr(LANES == 16) return sum16(v);
   v = wave_sum(v);
   if constexpr(LANES == 64) return v;
   uint32_t* const at = side[turn++ & 1];
   if((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = __float_as_uint(v);
   __syncthreads();
   float s = 0.0f;
#pragma unroll
   for(int w = 0; w < LANES / 64; w++) s += __uint_as_float(at[threadIdx.x / LANES * (LANES / 64) + w]);
   return s;
}
// three sums in one exchange, up to 4 wavefronts
template<int LANES>
__device__ inline void row_sums(float (&v)[3], uint32_t (&side)[2][16], int& turn)
{
   static_assert(LANES > 64 && LANES <= 256, "");
   __shared__ float more[2][3][16];
   const int t = turn++ & 1, first = threadIdx.x / LANES * (LANES / 64);
#pragma unroll
   for(int i = 0; i < 3; i++) {
      v[i] = wave_sum(v[i]);
      if((threadIdx.x & 63) == 0) more[t][i][threadIdx.x >> 6] = v[i];
   }
   __syncthreads();
#pragma unroll
   for(int i = 0; i < 3; i++) {
      v[i] = 0.0f;
#pragma unroll
      for(int w = 0; w < LANES / 64; w++) v[i] += more[t][i][first + w];
   }
}
template<int LANES>
__device__ inline uint32_t row_max(uint32_t v, uint32_t (&side)[2][16], int& turn)
{
   if constexpr(LANES == 4) return max4(v);
   if constexpr(LANES == 16) return max16(v);
   v = wave_max(v);
   if constexpr(LANES == 64) return v;
   uint32_t* const at = side[turn++ & 1];
   if((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
   __syncthreads();
   uint32_t m = 0;
#pragma unroll
   for(int w = 0; w < LANES / 64; w++) m = umax(m, at[threadIdx.x / LANES * (LANES / 64) + w]);
   return m;
}

// Factors of a row: n = h * c * r.  c is 1 but where squares of h leave fp32's range, upwards, or
// downwards with an eps that does not hide it: the sum is then taken again of h * c.
struct Factors {
   float c, r;
};
__device__ inline float squares(const float (&h)[8], float c)
{
   float ss = 0.0f;
#pragma unroll
   for(int i = 0; i < 8; i++) ss = __builtin_fmaf(h[i] * c, h[i] * c, ss);
   return ss;
}
// part(c): the lane's share of the sum of (h c)^2
template<int LANES, int ROWS, class F>
__device__ inline Factors factors_from(F part, int64_t k, float eps, uint32_t (&side)[2][16], int& turn)
{
   constexpr float DOWN = 0x1p-80f, UP = 0x1p+80f;
   if constexpr(ROWS > 1 && LANES > 64) {
      // rows that share barriers cannot go back for another sum: all three in one exchange
      float sums[3] = {part(1.0f), part(DOWN), part(UP)};
      row_sums<LANES>(sums, side, turn);
      const bool large = !(sums[0] < __builtin_inff()), small = sums[0] < 0x1p-60f && eps < 0x1p-60f;
      const float c = large ? DOWN : small ? UP : 1.0f, ss = large ? sums[1] : small ? sums[2] : sums[0];
      return {c, 1.0f / sqrtf(ss / (float)k + (eps * c) * c)};
   } else {
      float c = 1.0f, ss = row_sum<LANES>(part(c), side, turn);
      const bool large = !(ss < __builtin_inff()), small = ss < 0x1p-60f && eps < 0x1p-60f;
      if(large || small) {                 // the same in all lanes of the row
         c = large ? DOWN : UP;
         ss = row_sum<LANES>(part(c), side, turn);
      }
      return {c, 1.0f / sqrtf(ss / (float)k + (eps * c) * c)};
   }
}
template<int LANES, int ROWS, int V>
__device__ inline Factors factors_of(const float (&h)[V][8], int64_t k, float eps, uint32_t (&side)[2][16], int& turn)
{
   return factors_from<LANES, ROWS>([&](float c) {
      float ss = 0.0f;
#pragma unroll
      for(int v = 0; v < V; v++) ss += squares(h[v], c);
      return ss;
   }, k, eps, side, turn);
}

// ---- eight bits ---------------------------------------------------------------------------

// What makes codes of a row's values: y * up * inv is 127 y / max|y| to within 2^-22 of
// itself.  up lifts rows whose reciprocal would overflow.
struct Step {
   float  up, inv;
   double top;        // max|y| * up
};
__device__ inline Step step_of(uint32_t top_bits)
{
   const float top = __uint_as_float(top_bits), up = top < 0x1p-100f ? 0x1p+100f : 1.0f;
   return {up, top_bits ? 127.0f / (top * up) : 0.0f, (double)(top * up)};
}
// Eight codes.  Where the product is so near to half-way between two integers that its own
// error could decide, the exact comparison does: 254 |y| against (2 m + 1) max|y|, which
// fp64 holds.  (Half of a row's largest magnitude is half-way: 16-bit rows meet it.)
__device__ inline u32x2 codes8(const float (&y)[8], const Step& s)
{
   // 1.5 * 2^23 more rounds to an integer, whose byte is the last one of the sum
   constexpr float ROUND = 0x1.8p23f;
   uint32_t n[8];
   float    q[8], off = 0.0f;
#pragma unroll
   for(int i = 0; i < 8; i++) {
      q[i] = y[i] * s.up * s.inv;
      const float sum = q[i] + ROUND;
      n[i] = __float_as_uint(sum);
      off = fmaxf(off, fabsf(q[i] - (sum - ROUND)));
   }
   const bool near = off > 0.49997f;
   if(near) {
#pragma unroll
      for(int i = 0; i < 8; i++) {
         const float a = fabsf(q[i]), low = floorf(a);
         if(fabsf(a - low - 0.5f) < 0.00004f) {
            const int    m = (int)low;
            const double twice = 254.0 * (double)fabsf(y[i] * s.up), half = (double)(2 * m + 1) * s.top;
            const int    c = twice > half || (twice == half && (m & 1)) ? m + 1 : m;
            n[i] = (uint32_t)(q[i] < 0.0f ? -c : c);
         }
      }
   }
   u32x2 w;
#pragma unroll
   for(int i = 0; i < 2; i++)
      w[i] = __builtin_amdgcn_perm(n[4 * i + 1], n[4 * i], 0x0c0c0400) | __builtin_amdgcn_perm(n[4 * i + 3], n[4 * i + 2], 0x04000c0c);
   return w;
}

// ---- the norm, and rows to 8 bits (NORM false: y = x) -----------------------------------
//
// LANES lanes have a row, V vectors of 8 elements each; a workgroup of 256 has 64 rows at 4 lanes, 16 at 16, 4 at 64.
// 8192 x 4096 in bf16: norm 21.7 us (6.2 TB/s), with an fp32 residual, total and 8-bit rows 69 (5.3), rows to 8 bits
// 20 (5.0); a torch copy runs at 5.3.
template<class X, class S, int LANES, int V, bool NORM>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES, LANES == 1024 && !NORM ? 8 : 1)     // two rows a CU
norm_rows(NormParams p, int64_t kp, bool past)
{
   __shared__ uint32_t side[2][16];
   constexpr int PER = LANES < 256 ? 256 / LANES : 1;
   const int lane = threadIdx.x % LANES;
   const int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
   if(row >= p.rows) return;                     // all lanes of a row, which meet no barrier where rows share a workgroup
   const X* const x = static_cast<const X*>(p.x) + row * p.ldx;
   int turn = 0;
   float h[V][8];
   {
      Eight<X> a[V];
#pragma unroll
      for(int v = 0; v < V; v++) a[v] = fetch8<X>(x, (int64_t)(v * LANES + lane) * 8, p.k);
      if(NORM && p.residual) {
         const S* const res = static_cast<const S*>(p.residual) + row * p.ldr;
         Eight<S> b[V];
#pragma unroll
         for(int v = 0; v < V; v++) b[v] = fetch8<S>(res, (int64_t)(v * LANES + lane) * 8, p.k);
#pragma unroll
         for(int v = 0; v < V; v++)
#pragma unroll
            for(int i = 0; i < 8; i++) h[v][i] = (float)a[v].e[i] + (float)b[v].e[i];
      } else {
#pragma unroll
         for(int v = 0; v < V; v++)
#pragma unroll
            for(int i = 0; i < 8; i++) h[v][i] = (float)a[v].e[i];
      }
   }
   if constexpr(NORM) {
      const Factors f = factors_of<LANES, PER, V>(h, p.k, p.eps, side, turn);
      S* const total = p.total ? static_cast<S*>(p.total) + row * p.ldt : nullptr;
      X* const out = p.out ? static_cast<X*>(p.out) + row * p.ldo : nullptr;
#pragma unroll
      for(int v = 0; v < V; v++) {
         const int64_t col = (int64_t)(v * LANES + lane) * 8;
         if(total) put8<S>(total, col, p.k, h[v]);
         Eight<float> w;
         if(p.weight) w = fetch8<float>(p.weight, col, p.k);
#pragma unroll
         for(int i = 0; i < 8; i++) {
            h[v][i] = h[v][i] * f.c * f.r;
            if(p.weight) h[v][i] *= w.e[i];
         }
         if(out) put8<X>(out, col, p.k, h[v], past);
      }
      if(!p.codes) return;
   }
   uint32_t top = 0;
#pragma unroll
   for(int v = 0; v < V; v++)
#pragma unroll
      for(int i = 0; i < 8; i++) top = umax(top, magnitude(h[v][i]));      // values beyond the end are zeros
   top = row_max<LANES>(top, side, turn);
   const bool finite = top < 0x7f800000u;
   if(lane == 0) p.scales[row] = finite ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
   const Step step = step_of(finite ? top : 0);
   int8_t* const codes = p.codes + row * kp;
#pragma unroll
   for(int v = 0; v < V; v++) {
      const int64_t col = (int64_t)(v * LANES + lane) * 8;
      if(col >= kp) break;
      u32x2 c = {0, 0};
      if(finite) c = codes8(h[v], step);
      put_codes(codes + col, c, past);
   }
}

// Rows too long for registers (32768 values in bf16 still fit: 4.6 TB/s): 1024 lanes go over their row once for the sum of squares, once for the
// largest magnitude where codes are asked for, once to write.  What a lane writes it has read itself, in
// the same trip, so total may still be residual and out x.
template<class X, class S, bool NORM>
__global__ void __launch_bounds__(1024)
norm_long(NormParams p, int64_t kp, bool past)
{
   __shared__ uint32_t side[2][16];
   const int64_t row = blockIdx.x;
   const X* const x = static_cast<const X*>(p.x) + row * p.ldx;
   const S* const res = NORM && p.residual ? static_cast<const S*>(p.residual) + row * p.ldr : nullptr;
   int turn = 0;
   auto sums = [&](int64_t col, float (&h)[8]) {
      const Eight<X> a = fetch8<X>(x, col, p.k);
#pragma unroll
      for(int i = 0; i < 8; i++) h[i] = (float)a.e[i];
      if(res) {
         const Eight<S> b = fetch8<S>(res, col, p.k);
#pragma unroll
         for(int i = 0; i < 8; i++) h[i] += (float)b.e[i];
      }
   };
   Factors f{1.0f, 1.0f};
   if constexpr(NORM)
      f = factors_from<1024, 1>([&](float c) {
         float ss = 0.0f;
         for(int64_t col = threadIdx.x * 8; col < p.k; col += 8192) {
            float h[8];
            sums(col, h);
            ss += squares(h, c);
         }
         return ss;
      }, p.k, p.eps, side, turn);
   auto normed = [&](int64_t col, float (&h)[8]) {
      if(!NORM) return;
      Eight<float> w;
      if(p.weight) w = fetch8<float>(p.weight, col, p.k);
#pragma unroll
      for(int i = 0; i < 8; i++) {
         h[i] = h[i] * f.c * f.r;
         if(p.weight) h[i] *= w.e[i];
      }
   };
   uint32_t top = 0;
   if(!NORM || p.codes) {
      for(int64_t col = threadIdx.x * 8; col < p.k; col += 8192) {
         float h[8];
         sums(col, h);
         normed(col, h);
#pragma unroll
         for(int i = 0; i < 8; i++) top = umax(top, magnitude(h[i]));
      }
      top = row_max<1024>(top, side, turn);
   }
   const bool finite = top < 0x7f800000u;
   const Step step = step_of(finite ? top : 0);
   if(p.codes && threadIdx.x == 0) p.scales[row] = finite ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
   for(int64_t col = threadIdx.x * 8; col < kp; col += 8192) {
      float h[8];
      sums(col, h);                                // zeros from k on
      if(NORM && p.total) put8<S>(static_cast<S*>(p.total) + row * p.ldt, col, p.k, h);
      normed(col, h);
      if(NORM && p.out) put8<X>(static_cast<X*>(p.out) + row * p.ldo, col, p.k, h, past);
      if(!p.codes) continue;
      u32x2 c = {0, 0};
      if(finite) c = codes8(h, step);
      put_codes(p.codes + row * kp + col, c, past);
   }
}

// one lane, eight values; a row of lanes as long as a padded row (8192 x 4096 to bf16 15.9 us, 6.3 TB/s)
template<class O>
__global__ void __launch_bounds__(256)
dequantize_rows(const int8_t* codes, const float* scales, O* out, int64_t ld, int64_t first, int64_t rows, int64_t k,
                int64_t kp, bool past)
{
   const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = kp / 8;
   const int64_t row = first + i / per, col = i % per * 8;
   if(row >= rows || col >= k) return;
   const u32x2 c = *reinterpret_cast<const u32x2*>(codes + row * kp + col);
   const float s = scales[row];
   float v[8];
#pragma unroll
   for(int j = 0; j < 8; j++) v[j] = (float)(int8_t)(c[j / 4] >> (8 * (j % 4))) * s;
   put8<O>(out + row * ld, col, k, v, past);
}

// ---- the norm's gradients ----------------------------------------------------------------
//
// Workgroup i of `groups` has PER rows from PER i on, then every PER groups'th, and the sums of its rows' part of
// dweight in registers; the next row's values are on their way while one is summed (not with V > 1, which
// has no registers for it).  8 elements a lane: more wavefronts to a row wait for each other, but as many
// more loads are on their way (8192 x 4096 in bf16 with its dtotal 68 us; with 256 lanes of 16 elements 79).  V > 1 is
// for widths in whole eights.  What is left are the waits for the two exchanges of a row: wavefronts wait 70 % of their time.
constexpr int kGradBlock = 512;

template<class D, class S, class O, int LANES, int V>
__global__ void __launch_bounds__(LANES < kGradBlock ? kGradBlock : LANES)
norm_grad_rows(NormGradParams p, int64_t groups)
{
   __shared__ uint32_t side[2][16];
   constexpr int PER = LANES < kGradBlock ? kGradBlock / LANES : 1;
   const int lane = threadIdx.x % LANES, mine = threadIdx.x / LANES;
   const int64_t step = groups * PER;
   int turn = 0;
   Eight<D> dy[V];
   Eight<S> hh[V], dt[V];
   // rows beyond the last read that one
   auto fetch = [&](int64_t row) {
      const int64_t r = row < p.rows ? row : p.rows - 1;
#pragma unroll
      for(int v = 0; v < V; v++) {
         const int64_t col = (int64_t)(v * LANES + lane) * 8;
         const D* const y = static_cast<const D*>(p.dy) + r * p.ldy;
         const S* const x = static_cast<const S*>(p.h) + r * p.ldh;
         const S* const t = static_cast<const S*>(p.dtotal) + r * p.ldt;
         dy[v] = V > 1 ? fetch8_whole<D>(y, col, p.k) : fetch8<D>(y, col, p.k);
         hh[v] = V > 1 ? fetch8_whole<S>(x, col, p.k) : fetch8<S>(x, col, p.k);
         if(V == 1 && p.dtotal) dt[v] = fetch8<S>(t, col, p.k);
      }
   };
   float dw[V][8] = {};
   int64_t row0 = (int64_t)blockIdx.x * PER;
   if(V == 1) fetch(row0 + mine);
   for(; row0 < p.rows; row0 += step) {
      const int64_t row = row0 + mine;
      const bool there = row < p.rows;
      if(V > 1) fetch(row);
      float g[V][8], h[V][8], through[8];
#pragma unroll
      for(int v = 0; v < V; v++)
#pragma unroll
         for(int i = 0; i < 8; i++) {
            const bool in = there && (V == 1 || (v * LANES + lane) * 8 < p.k);
            g[v][i] = in ? (float)dy[v].e[i] : 0.0f;
            h[v][i] = in ? (float)hh[v].e[i] : 0.0f;
            if(V == 1) through[i] = p.dtotal ? (float)dt[0].e[i] : 0.0f;
         }
      if(V == 1) fetch(row + step);
      auto add_through = [&](int v, int64_t r, float (&o)[8]) {
         if(V > 1) {                                           // read only now: no registers to hold it
            Eight<S> t{};
            if(p.dtotal) t = fetch8_whole<S>(static_cast<const S*>(p.dtotal) + r * p.ldt, (int64_t)(v * LANES + lane) * 8, p.k);
#pragma unroll
            for(int i = 0; i < 8; i++) through[i] = (float)t.e[i];
         }
#pragma unroll
         for(int i = 0; i < 8; i++) o[i] += through[i];
      };
      const Factors f = factors_of<LANES, PER, V>(h, p.k, p.eps, side, turn);
      float mean = 0.0f;
#pragma unroll
      for(int v = 0; v < V; v++) {
         const int64_t col = (int64_t)(v * LANES + lane) * 8;
         Eight<float> w;
         if(p.weight) w = V > 1 ? fetch8_whole<float>(p.weight, col, p.k) : fetch8<float>(p.weight, col, p.k);
#pragma unroll
         for(int i = 0; i < 8; i++) {
            h[v][i] = h[v][i] * f.c * f.r;
            dw[v][i] = __builtin_fmaf(g[v][i], there ? h[v][i] : 0.0f, dw[v][i]);
            if(p.weight) g[v][i] *= w.e[i];
            mean = __builtin_fmaf(g[v][i], h[v][i], mean);
         }
      }
      mean = row_sum<LANES>(mean, side, turn) / (float)p.k;
      if(!there) continue;
      O* const dx = static_cast<O*>(p.dx) + row * p.ldx;
#pragma unroll
      for(int v = 0; v < V; v++) {
         float o[8];
#pragma unroll
         for(int i = 0; i < 8; i++) o[i] = __builtin_fmaf(-h[v][i], mean, g[v][i]) * f.r * f.c;
         add_through(v, row, o);
         const int64_t col = (int64_t)(v * LANES + lane) * 8;
         if(V == 1) put8<O>(dx, col, p.k, o);
         else if(col < p.k) store8<O>(dx + col, o);
      }
   }
   if(!p.dweight) return;
   float* const work = p.work + (int64_t)blockIdx.x * p.k;
   if constexpr(PER > 1) {
      // the rows' sums, in their order
      __shared__ float join[PER][V * LANES * 8];
#pragma unroll
      for(int v = 0; v < V; v++)
#pragma unroll
         for(int i = 0; i < 8; i++) join[mine][(v * 8 + i) * LANES + lane] = dw[v][i];
      __syncthreads();
      for(int i = threadIdx.x; i < V * 8 * LANES; i += kGradBlock) {
         const int64_t col = (int64_t)(i / (8 * LANES) * LANES + i % LANES) * 8 + i / LANES % 8;
         float s = 0.0f;
#pragma unroll
         for(int w = 0; w < PER; w++) s += join[w][i];
         if(col < p.k) work[col] = s;
      }
   } else {
#pragma unroll
      for(int v = 0; v < V; v++) {
         const int64_t col = (int64_t)(v * LANES + lane) * 8;
         if(V == 1) put8<float>(work, col, p.k, dw[v]);
         else if(col < p.k) store8<float>(work + col, dw[v]);
      }
   }
}

// Rows too long for registers: three trips over a row by 1024 lanes; dweight's sums are in the workgroup's
// row of the workspace, every element in the hands of one lane.  2048 x 32768 in bf16 296 us.
template<class D, class S, class O>
__global__ void __launch_bounds__(1024)
norm_grad_long(NormGradParams p, int64_t groups)
{
   __shared__ uint32_t side[2][16];
   int turn = 0;
   float* const work = p.dweight ? p.work + (int64_t)blockIdx.x * p.k : nullptr;
   for(int64_t row = blockIdx.x; row < p.rows; row += groups) {
      const D* const dy = static_cast<const D*>(p.dy) + row * p.ldy;
      const S* const hh = static_cast<const S*>(p.h) + row * p.ldh;
      const Factors f = factors_from<1024, 1>([&](float c) {
         float ss = 0.0f;
         for(int64_t col = threadIdx.x * 8; col < p.k; col += 8192) {
            const Eight<S> a = fetch8<S>(hh, col, p.k);
            float h[8];
#pragma unroll
            for(int i = 0; i < 8; i++) h[i] = (float)a.e[i];
            ss += squares(h, c);
         }
         return ss;
      }, p.k, p.eps, side, turn);
      // n into h, w dy into g, dy into plain
      auto values = [&](int64_t col, float (&h)[8], float (&g)[8], float (&plain)[8]) {
         const Eight<S> a = fetch8<S>(hh, col, p.k);
         const Eight<D> b = fetch8<D>(dy, col, p.k);
         Eight<float> w;
         if(p.weight) w = fetch8<float>(p.weight, col, p.k);
#pragma unroll
         for(int i = 0; i < 8; i++) {
            h[i] = (float)a.e[i] * f.c * f.r;
            plain[i] = (float)b.e[i];
            g[i] = p.weight ? plain[i] * w.e[i] : plain[i];
         }
      };
      float mean = 0.0f;
      for(int64_t col = threadIdx.x * 8; col < p.k; col += 8192) {
         float h[8], g[8], plain[8];
         values(col, h, g, plain);
#pragma unroll
         for(int i = 0; i < 8; i++) mean += g[i] * h[i];
      }
      mean = row_sum<1024>(mean, side, turn) / (float)p.k;
      const S* const dt = p.dtotal ? static_cast<const S*>(p.dtotal) + row * p.ldt : nullptr;
      for(int64_t col = threadIdx.x * 8; col < p.k; col += 8192) {
         float h[8], g[8], plain[8];
         values(col, h, g, plain);
         Eight<S> t;
         if(dt) t = fetch8<S>(dt, col, p.k);
         if(work) {
            float sum[8];
            const Eight<float> before = fetch8<float>(work, col, p.k);
#pragma unroll
            for(int i = 0; i < 8; i++) sum[i] = (row == blockIdx.x ? 0.0f : before.e[i]) + plain[i] * h[i];
            put8<float>(work, col, p.k, sum);
         }
#pragma unroll
         for(int i = 0; i < 8; i++) g[i] = __builtin_fmaf(-h[i], mean, g[i]) * f.r * f.c + (dt ? (float)t.e[i] : 0.0f);
         put8<O>(static_cast<O*>(p.dx) + row * p.ldx, col, p.k, g);
      }
   }
}

// dweight = the sum of `splits` rows of k: 32 columns a workgroup, 32 runs of rows, joined in order; 512 x 4096 4.5 us
__global__ void __launch_bounds__(1024)
join_weight(const float* work, float* dweight, int64_t splits, int64_t k)
{
   __shared__ float part[32][33];
   const int c = threadIdx.x % 32, g = threadIdx.x / 32;
   const int64_t col = (int64_t)blockIdx.x * 32 + c;
   float s = 0.0f;
   if(col < k)
#pragma unroll 8
      for(int64_t r = g; r < splits; r += 32) s += work[r * k + col];
   part[g][c] = s;
   __syncthreads();
   if(g == 0 && col < k) {
      s = 0.0f;
#pragma unroll
      for(int i = 0; i < 32; i++) s += part[i][c];
      dweight[col] = s;
   }
}

// ---- launches --------------------------------------------------------------------------------

// Results of half the L2s' 32 MiB and more are written past them, where they do not take the place of what comes in (8192 x 4096
// in bf16: norm 27 / 21.7 us, back from 8 bits 16.5 / 15.9, residual, 8 bits and back 91 / 86; 2048 x 4096: norm 8.3 /
// 6.6, but 8-bit rows and their way back 22.6 / 23.2).  Not so: fp32 results, whose lanes write two pieces (back from 8 bits 34
// / 46.6), the gradients (67.5 / 69.2); and loads gain nothing.
bool past_l2(int64_t bytes) { return bytes >= (int64_t)16 << 20; }
template<class X>
int64_t result_bytes(const NormParams& p)
{
   return (p.out ? p.rows * p.k * (int64_t)sizeof(X) : 0) + (p.codes ? p.rows * padded(p.k) : 0);
}

template<class X, class S, int LANES, int V, bool NORM>
hipError_t norm_shape(const NormParams& p, hipStream_t s)
{
   constexpr int PER = LANES < 256 ? 256 / LANES : 1, BLOCK = LANES < 256 ? 256 : LANES;
   const int64_t groups = (p.rows + PER - 1) / PER;
   if(!grid_ok(groups, BLOCK)) return kTooLarge;
   norm_rows<X, S, LANES, V, NORM><<<(unsigned)groups, BLOCK, 0, s>>>(p, padded(p.k), past_l2(result_bytes<X>(p)));
   return hipGetLastError();
}

// the lanes and vectors for a width
template<class X, class S, bool NORM>
hipError_t norm_typed(const NormParams& p, hipStream_t s)
{
   if constexpr(NORM)                                        // 16 lanes write the padding of a row of codes too
      if(p.k <= 32 && !p.codes) return norm_shape<X, S, 4, 1, NORM>(p, s);
   if(p.k <= 128)   return norm_shape<X, S, 16, 1, NORM>(p, s);
   if(p.k <= 512)   return norm_shape<X, S, 64, 1, NORM>(p, s);
   if(p.k <= 1024)  return norm_shape<X, S, 64, 2, NORM>(p, s);
   if(p.k <= 2048)  return norm_shape<X, S, 256, 1, NORM>(p, s);
   if(p.k <= 4096)  return norm_shape<X, S, 256, 2, NORM>(p, s);
   if(p.k <= 8192)  return norm_shape<X, S, 256, 4, NORM>(p, s);
   if(p.k <= 16384) return norm_shape<X, S, 1024, 2, NORM>(p, s);
   if(p.k <= 32768) return norm_shape<X, S, 1024, 4, NORM>(p, s);
   if(!grid_ok(p.rows, 1024)) return kTooLarge;
   norm_long<X, S, NORM><<<(unsigned)p.rows, 1024, 0, s>>>(p, padded(p.k), past_l2(result_bytes<X>(p)));
   return hipGetLastError();
}

template<class O>
hipError_t dequantize_typed(const int8_t* codes, const float* scales, void* out, int64_t ld, int64_t rows, int64_t k,
                            hipStream_t s)
{
   const int64_t kp = padded(k), per = kp / 8;
   const int64_t most = (int64_t)1 << 31;               // lanes of a launch, whole rows of them
   const int64_t each = most / per > 0 ? most / per : 1;
   if(!grid_ok((per + 255) / 256, 256)) return kTooLarge;
   for(int64_t first = 0; first < rows; first += each) {
      const int64_t n = rows - first < each ? rows - first : each;
      dequantize_rows<O><<<(unsigned)((n * per + 255) / 256), 256, 0, s>>>(codes, scales, static_cast<O*>(out), ld, first,
                                                                          first + n, k, kp, past_l2(rows * k * (int64_t)sizeof(O)));
      const hipError_t e = hipGetLastError();
      if(e != hipSuccess) return e;
   }
   return hipSuccess;
}

// LANES 0: the kernel of long rows
template<class D, class S, class O, int LANES, int V>
hipError_t grad_shape(const NormGradParams& p, hipStream_t s)
{
   constexpr int PER = LANES == 0 || LANES >= kGradBlock ? 1 : kGradBlock / (LANES ? LANES : 1), BLOCK = LANES < kGradBlock ? kGradBlock : LANES;
   int64_t groups = (p.rows + PER - 1) / PER;
   if(p.dweight) groups = groups < p.splits ? groups : p.splits;
   if(groups > 2048) groups = 2048;
   if(groups > 0) {                                     // no rows: dweight is zero
      if constexpr(LANES == 0) norm_grad_long<D, S, O><<<(unsigned)groups, 1024, 0, s>>>(p, groups);
      else                     norm_grad_rows<D, S, O, LANES, V><<<(unsigned)groups, BLOCK, 0, s>>>(p, groups);
      const hipError_t e = hipGetLastError();
      if(e != hipSuccess) return e;
   }
   if(!p.dweight) return hipSuccess;
   if(!grid_ok((p.k + 31) / 32, 1024)) return kTooLarge;
   join_weight<<<(unsigned)((p.k + 31) / 32), 1024, 0, s>>>(p.work, p.dweight, groups, p.k);
   return hipGetLastError();
}

template<class D, class S, class O>
hipError_t grad_typed(const NormGradParams& p, hipStream_t s)
{
   if(p.k <= 32)    return grad_shape<D, S, O, 4, 1>(p, s);
   if(p.k <= 128)   return grad_shape<D, S, O, 16, 1>(p, s);
   if(p.k <= 512)   return grad_shape<D, S, O, 64, 1>(p, s);
   if(p.k <= 1024)  return grad_shape<D, S, O, 128, 1>(p, s);
   if(p.k <= 2048)  return grad_shape<D, S, O, 256, 1>(p, s);
   if(p.k <= 4096)  return grad_shape<D, S, O, 512, 1>(p, s);
   if(p.k <= 8192)  return grad_shape<D, S, O, 1024, 1>(p, s);
   if(p.k <= 16384 && p.k % 8 == 0) return grad_shape<D, S, O, 1024, 2>(p, s);
   return grad_shape<D, S, O, 0, 0>(p, s);
}

}  // namespace

hipError_t launch_rms_norm(const NormParams& p, hipStream_t s)
{
   const bool wide = p.sum_type == T_F32;
   switch(p.type) {
      case T_F32:  return norm_typed<float, float, true>(p, s);
      case T_BF16: return wide ? norm_typed<bf16, float, true>(p, s) : norm_typed<bf16, bf16, true>(p, s);
      default:     return wide ? norm_typed<f16, float, true>(p, s) : norm_typed<f16, f16, true>(p, s);
   }
}

hipError_t launch_i8_quantize(const NormParams& p, hipStream_t s)
{
   switch(p.type) {
      case T_F32:  return norm_typed<float, float, false>(p, s);
      case T_BF16: return norm_typed<bf16, bf16, false>(p, s);
      default:     return norm_typed<f16, f16, false>(p, s);
   }
}

hipError_t launch_i8_dequantize(const int8_t* codes, const float* scales, void* out, int type, int64_t ld, int64_t rows,
                                int64_t k, hipStream_t s)
{
   switch(type) {
      case T_F32:  return dequantize_typed<float>(codes, scales, out, ld, rows, k, s);
      case T_BF16: return dequantize_typed<bf16>(codes, scales, out, ld, rows, k, s);
      default:     return dequantize_typed<f16>(codes, scales, out, ld, rows, k, s);
   }
}

hipError_t launch_rms_norm_grad(const NormGradParams& p, hipStream_t s)
{
   const bool wide = p.sum_type == T_F32, wide_out = p.dx_type == T_F32;
   switch(p.type) {
      case T_F32: return grad_typed<float, float, float>(p, s);
      case T_BF16:
         if(!wide) return grad_typed<bf16, bf16, bf16>(p, s);
         return wide_out ? grad_typed<bf16, float, float>(p, s) : grad_typed<bf16, float, bf16>(p, s);
      default:
         if(!wide) return grad_typed<f16, f16, f16>(p, s);
         return wide_out ? grad_typed<f16, float, float>(p, s) : grad_typed<f16, float, f16>(p, s);
   }
}

}  // namespace layer
}  // namespace fufft
