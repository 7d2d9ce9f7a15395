// Microscaled 4-bit blocks: rows of values to blocks along the rows, along the
// columns, or both from one reading, and back.  The format and the rounding are
// in mx4_device.hpp.
#include "mx4_device.hpp"
#include "mx4_internal.hpp"

namespace fufft {
namespace mx4 {

namespace {

constexpr int kLanes = 256;

// v[8] of row `row` from column `col` on, zeros beyond k
template<class T>
__device__ inline void load_row8(const T* x, int64_t ld, int64_t row, int64_t col, int64_t k, float (&v)[8])
{
   const T* p = x + row * ld + col;
   if(col + 8 <= k) {
      load8(p, v);
   } else {
#pragma unroll
      for(int i = 0; i < 8; i++) v[i] = col + i < k ? to_float(p[i]) : 0.0f;
   }
}
__device__ inline void load_rand8(const uint8_t* rand, int64_t row, int64_t col, int64_t k, uint32_t (&r)[8])
{
   const uint8_t* p = rand + row * k + col;
   if(col + 8 <= k) {
      struct __attribute__((packed, aligned(1))) V { uint32_t e[2]; };
      const V t = *reinterpret_cast<const V*>(p);
#pragma unroll
      for(int i = 0; i < 8; i++) r[i] = (t.e[i / 4] >> (8 * (i % 4))) & 255u;
   } else {
#pragma unroll
      for(int i = 0; i < 8; i++) r[i] = col + i < k ? p[i] : 0u;
   }
}

// Blocks along rows.  A lane holds 8 consecutive values, four lanes a block, and
// 16 lanes a group of 128, whose four scale bytes go out as one word.  A
// workgroup has 2^lr lanes to a row and 256 >> lr rows at a time, ROWS of them
// per lane in flight.
template<class T, bool RAND, int ROWS>
__global__ void __launch_bounds__(kLanes)
quantize_rows(QuantizeParams p, int64_t kp, int lr)
{
   const T* x = static_cast<const T*>(p.x);
   const int lane = threadIdx.x & ((1 << lr) - 1);
   const int64_t col = ((int64_t)blockIdx.x << (lr + 3)) + lane * 8;
   const int per = kLanes >> lr;
   const int64_t row0 = ((int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y) * (per * ROWS) + (threadIdx.x >> lr);
   float v[ROWS][8];
   uint32_t r[ROWS][8];
   int64_t to[ROWS];
#pragma unroll
   for(int u = 0; u < ROWS; u++) {
      const int64_t row = row0 + u * per;
      const bool in = row < p.rows && col < kp;
      to[u] = in ? (p.slots ? p.slots[row] : row) : -1;
#pragma unroll
      for(int i = 0; i < 8; i++) v[u][i] = 0.0f;
      if(in && col < p.k) load_row8(x, p.ld, row, col, p.k, v[u]);
      if constexpr(RAND) {
#pragma unroll
         for(int i = 0; i < 8; i++) r[u][i] = 0;
         if(in && col < p.k) load_rand8(p.rand, row, col, p.k, r[u]);
      }
   }
#pragma unroll
   for(int u = 0; u < ROWS; u++) {
      uint32_t top = 0;
#pragma unroll
      for(int i = 0; i < 8; i++) top = umax(top, magnitude(v[u][i]));
      top = umax(top, dpp<kQuadSwap1>(top));
      top = umax(top, dpp<kQuadSwap2>(top));
      const uint32_t s = scale_byte(top, p.fit != 0);
      uint32_t word = s | (dpp<kRowLeft4>(s) << 8);
      word |= dpp<kRowLeft8>(word) << 16;
      uint32_t c;
      if constexpr(RAND) c = encode8_random(v[u], s, r[u]);
      else               c = encode8(v[u], s);
      if(to[u] >= 0 && to[u] < p.slot_count) {
         *reinterpret_cast<uint32_t*>(p.codes + to[u] * (kp / 2) + col / 2) = c;
         if((lane & 15) == 0) *reinterpret_cast<uint32_t*>(p.scales + to[u] * (kp / kBlock) + col / kBlock) = word;
      }
   }
}

// Blocks along columns, and along rows too where p.codes is given, from one
// reading: a workgroup takes 128 rows x 128 columns.  The rows' part is the
// kernel above; the values (and random bytes) then wait in LDS in their own
// type, and each lane takes two neighbouring columns of 32 rows: 16 bytes of
// codes a column, four lanes a group of 128 rows.  The pair of columns (row,
// pair) lies at slot pair ^ 16 (row / 32), so that the four lanes of a group read
// different banks.
template<class T> struct Pair { T a, b; };

template<class T, bool RAND>
__global__ void __launch_bounds__(kLanes)
quantize_both(QuantizeParams p, int64_t kp, int64_t rowsp)
{
   __shared__ Pair<T> tile[128 * 64];
   __shared__ Pair<uint8_t> rtile[RAND ? 128 * 64 : 1];
   const T* x = static_cast<const T*>(p.x);
   const int64_t c0 = (int64_t)blockIdx.x * 128;
   const int64_t r0 = ((int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y) * 128;
   if(r0 >= rowsp) return;
   const bool fit = p.fit != 0;
   const int lane = threadIdx.x & 15;
   const int64_t col = c0 + lane * 8;
#pragma unroll 2
   for(int u = 0; u < 8; u++) {
      const int lrow = u * 16 + (threadIdx.x >> 4);
      const int64_t row = r0 + lrow;
      float v[8] = {};
      uint32_t r[8] = {};
      if(row < p.rows && col < p.k) {
         load_row8(x, p.ld, row, col, p.k, v);
         if constexpr(RAND) load_rand8(p.rand, row, col, p.k, r);
      }
#pragma unroll
      for(int i = 0; i < 4; i++) {
         const int at = lrow * 64 + ((lane * 4 + i) ^ ((lrow >> 5) << 4));
         tile[at] = Pair<T>{(T)v[2 * i], (T)v[2 * i + 1]};
         if constexpr(RAND) rtile[at] = Pair<uint8_t>{(uint8_t)r[2 * i], (uint8_t)r[2 * i + 1]};
      }
      if(p.codes) {
         uint32_t top = 0;
#pragma unroll
         for(int i = 0; i < 8; i++) top = umax(top, magnitude(v[i]));
         top = umax(top, dpp<kQuadSwap1>(top));
         top = umax(top, dpp<kQuadSwap2>(top));
         const uint32_t s = scale_byte(top, fit);
         uint32_t word = s | (dpp<kRowLeft4>(s) << 8);
         word |= dpp<kRowLeft8>(word) << 16;
         uint32_t c;
         if constexpr(RAND) c = encode8_random(v, s, r);
         else               c = encode8(v, s);
         if(row < p.rows) {
            *reinterpret_cast<uint32_t*>(p.codes + row * (kp / 2) + col / 2) = c;
            if(lane == 0) *reinterpret_cast<uint32_t*>(p.scales + row * (kp / kBlock) + col / kBlock) = word;
         }
      }
   }
   __syncthreads();
   const int blk = threadIdx.x & 3, pair = threadIdx.x >> 2;
   const int base = blk * 32 * 64 + (pair ^ (blk << 4));
   uint32_t top[2] = {0, 0};
#pragma unroll
   for(int i = 0; i < 32; i++) {
      const Pair<T> t = tile[base + i * 64];
      top[0] = umax(top[0], magnitude(to_float(t.a)));
      top[1] = umax(top[1], magnitude(to_float(t.b)));
   }
#pragma unroll
   for(int h = 0; h < 2; h++) {
      const uint32_t s = scale_byte(top[h], fit);
      uint32_t word = s | (dpp<kQuadSwap1>(s) << 8);     // right at the group's lane 0, which alone stores it
      word |= dpp<kQuadSwap2>(word) << 16;
      u32x4 c;
#pragma unroll
      for(int q = 0; q < 4; q++) {
         float v[8];
         uint32_t r[8];
#pragma unroll
         for(int i = 0; i < 8; i++) {
            const int at = base + (q * 8 + i) * 64;
            v[i] = to_float(h ? tile[at].b : tile[at].a);
            if constexpr(RAND) r[i] = h ? rtile[at].b : rtile[at].a;
         }
         if constexpr(RAND) c[q] = encode8_random(v, s, r);
         else               c[q] = encode8(v, s);
      }
      const int64_t tcol = c0 + pair * 2 + h;
      if(tcol < p.k) {
         *reinterpret_cast<u32x4*>(p.codes_t + tcol * (rowsp / 2) + r0 / 2 + blk * 16) = c;
         if(blk == 0) *reinterpret_cast<uint32_t*>(p.scales_t + tcol * (rowsp / kBlock) + r0 / kBlock) = word;
      }
   }
}

// Blocks back to values: 8 codes a lane.
template<class T, int ROWS>
__global__ void __launch_bounds__(kLanes)
dequantize_rows(DequantizeParams p, int64_t kp, int lr)
{
   T* out = static_cast<T*>(p.out);
   const int lane = threadIdx.x & ((1 << lr) - 1);
   const int64_t col = ((int64_t)blockIdx.x << (lr + 3)) + lane * 8;
   if(col >= p.k) return;
   const int per = kLanes >> lr;
   const int64_t row0 = ((int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y) * (per * ROWS) + (threadIdx.x >> lr);
   uint32_t c[ROWS], s[ROWS];
#pragma unroll
   for(int u = 0; u < ROWS; u++) {
      const int64_t row = row0 + u * per;
      c[u] = s[u] = 0;
      if(row < p.rows) {
         c[u] = *reinterpret_cast<const uint32_t*>(p.codes + row * (kp / 2) + col / 2);
         s[u] = p.scales[row * (kp / kBlock) + col / kBlock];
      }
   }
#pragma unroll
   for(int u = 0; u < ROWS; u++) {
      const int64_t row = row0 + u * per;
      if(row >= p.rows) break;
      float v[8];
      decode8(c[u], s[u], v);
      T* o = out + row * p.ld + col;
      if(col + 8 <= p.k) {
         store8(o, v);
      } else {
#pragma unroll
         for(int i = 0; i < 8; i++)
            if(col + i < p.k) o[i] = (T)v[i];
      }
   }
}

// lanes to a row (a power of two, 16 .. 256) for kp values, as a logarithm
int lanes_log(int64_t kp)
{
   int lr = 4;
   while(lr < 8 && ((int64_t)8 << lr) < kp) lr++;
   return lr;
}

// a grid of gx columns and `tiles` rows of tiles, the latter over y and z (each at most 65535)
bool make_grid(int64_t gx, int64_t tiles, dim3* g)
{
   const int64_t gy = tiles < 65535 ? tiles : 65535, gz = (tiles + gy - 1) / gy;
   if(gx > 0x7fffffff || gz > 65535) return false;
   *g = dim3((unsigned)gx, (unsigned)gy, (unsigned)gz);
   return true;
}

template<class T, bool RAND>
hipError_t quantize_typed(const QuantizeParams& p, hipStream_t s)
{
   const int64_t kp = padded(p.k);
   dim3 g;
   if(p.codes_t) {
      const int64_t rowsp = padded(p.rows);
      if(!make_grid(kp / 128, rowsp / 128, &g)) return hipErrorInvalidValue;
      quantize_both<T, RAND><<<g, kLanes, 0, s>>>(p, kp, rowsp);
   } else {
      constexpr int ROWS = 4;
      const int lr = lanes_log(kp);
      const int64_t per = (kLanes >> lr) * ROWS;
      if(!make_grid((kp / 8 + (1 << lr) - 1) >> lr, (p.rows + per - 1) / per, &g)) return hipErrorInvalidValue;
      quantize_rows<T, RAND, ROWS><<<g, kLanes, 0, s>>>(p, kp, lr);
   }
   return hipGetLastError();
}

template<class T>
hipError_t dequantize_typed(const DequantizeParams& p, hipStream_t s)
{
   constexpr int ROWS = 4;
   const int64_t kp = padded(p.k);
   const int lr = lanes_log(kp);
   const int64_t per = (kLanes >> lr) * ROWS;
   dim3 g;
   if(!make_grid((kp / 8 + (1 << lr) - 1) >> lr, (p.rows + per - 1) / per, &g)) return hipErrorInvalidValue;
   dequantize_rows<T, ROWS><<<g, kLanes, 0, s>>>(p, kp, lr);
   return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize(const QuantizeParams& p, hipStream_t s)
{
   if(p.rows <= 0 || p.k <= 0) return hipSuccess;
   switch(p.type) {
      case T_F32:  return p.rand ? quantize_typed<float, true>(p, s) : quantize_typed<float, false>(p, s);
      case T_BF16: return p.rand ? quantize_typed<bf16, true>(p, s) : quantize_typed<bf16, false>(p, s);
      default:     return p.rand ? quantize_typed<f16, true>(p, s) : quantize_typed<f16, false>(p, s);
   }
}

hipError_t launch_dequantize(const DequantizeParams& p, hipStream_t s)
{
   if(p.rows <= 0 || p.k <= 0) return hipSuccess;
   switch(p.type) {
      case T_F32:  return dequantize_typed<float>(p, s);
      case T_BF16: return dequantize_typed<bf16>(p, s);
      default:     return dequantize_typed<f16>(p, s);
   }
}

}  // namespace mx4
}  // namespace fufft
