// Microscaled 4-bit blocks: rows of values to blocks along the rows, along the
// columns, or both from one reading, and back.  The format and the rounding are
// in mx4_device.hpp.
#include "mx4_device.hpp"
#include "mx4_internal.hpp"

namespace fufft {
namespace mx4 {

namespace {

constexpr int kLanes = 256;

// eight consecutive elements, as they are in memory
template<class T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T e[8]; };
struct __attribute__((packed, aligned(1))) Bytes8 { uint32_t e[2]; };

// of row `row` from column `col` on, zeros beyond k
template<class T>
__device__ inline Eight<T> load_row8(const T* x, int64_t ld, int64_t row, int64_t col, int64_t k)
{
   const T* p = x + row * ld + col;
   if(col + 8 <= k) return *reinterpret_cast<const Eight<T>*>(p);
   Eight<T> v;
#pragma unroll
   for(int i = 0; i < 8; i++) v.e[i] = col + i < k ? p[i] : (T)0.0f;
   return v;
}
__device__ inline u32x2 load_rand8(const uint8_t* rand, int64_t row, int64_t col, int64_t k)
{
   const uint8_t* p = rand + row * k + col;
   if(col + 8 <= k) {
      const Bytes8 t = *reinterpret_cast<const Bytes8*>(p);
      return u32x2{t.e[0], t.e[1]};
   }
   u32x2 r = {0, 0};
#pragma unroll
   for(int i = 0; i < 8; i++)
      if(col + i < k) r[i / 4] |= (uint32_t)p[i] << (8 * (i % 4));
   return r;
}

template<class T, bool RAND>
__device__ inline uint32_t encode(const float (&v)[8], uint32_t s, const uint32_t (&r)[8])
{
   if constexpr(RAND) return encode8_random<sizeof(T) == 2>(v, s, r);
   else               return encode8(v, s);
}

// A block's part of a row, 8 values a lane, four lanes a block: the lane's codes, and the
// group's four scale bytes as one word, right in the first of the group's 16 lanes.
template<class T, bool RAND>
__device__ inline void encode_row8(const Eight<T>& x, u32x2 r, bool fit, uint32_t* codes, uint32_t* word)
{
   float v[8];
   uint32_t top = 0;
#pragma unroll
   for(int i = 0; i < 8; i++) {
      v[i] = to_float(x.e[i]);
      top = umax(top, magnitude(v[i]));
   }
   top = umax(top, dpp<kQuadSwap1>(top));
   top = umax(top, dpp<kQuadSwap2>(top));
   const uint32_t s = scale_byte(top, fit);
   *word = s | (dpp<kRowLeft4>(s) << 8);
   *word |= dpp<kRowLeft8>(*word) << 16;
   uint32_t b[8];
#pragma unroll
   for(int i = 0; i < 8; i++) b[i] = (r[i / 4] >> (8 * (i % 4))) & 255u;
   *codes = encode<T, RAND>(v, s, b);
}

// Blocks along rows: 16 lanes a group of 128 values.  A workgroup has 2^lr lanes to a
// row and 256 >> lr rows at a time, ROWS of them per lane in flight.  Bound by its bytes:
// 8192 x 4096 in bf16 15.7 us, 5.4 TB/s (the best copy of large arrays 6.7, torch's 5.0), with random
// bytes 22 to 25; in fp32 27.5, with random bytes 35.
template<class T, bool RAND, int ROWS>
__global__ void __launch_bounds__(kLanes)
quantize_rows(QuantizeParams p, int64_t kp, int lr)
{
   const T* x = static_cast<const T*>(p.x);
   const int lane = threadIdx.x & ((1 << lr) - 1);
   const int64_t col = ((int64_t)blockIdx.x << (lr + 3)) + lane * 8;
   const int per = kLanes >> lr;
   const int64_t row0 = ((int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y) * (per * ROWS) + (threadIdx.x >> lr);
   Eight<T> v[ROWS];
   u32x2 r[ROWS];
   int64_t to[ROWS];
   // a workgroup whose rows and columns are all there has its loads in straight code
   const bool whole = row0 - (threadIdx.x >> lr) + per * ROWS <= p.rows && col - lane * 8 + (8 << lr) <= p.k;
   if(whole) {
#pragma unroll
      for(int u = 0; u < ROWS; u++) {
         const int64_t row = row0 + u * per;
         v[u] = *reinterpret_cast<const Eight<T>*>(x + row * p.ld + col);
         if constexpr(RAND) {
            const Bytes8 t = *reinterpret_cast<const Bytes8*>(p.rand + row * p.k + col);
            r[u] = u32x2{t.e[0], t.e[1]};
         }
         to[u] = p.slots ? p.slots[row] : row;
      }
   } else {
#pragma unroll
      for(int u = 0; u < ROWS; u++) {
         const int64_t row = row0 + u * per;
         const bool in = row < p.rows && col < kp;
         to[u] = in ? (p.slots ? p.slots[row] : row) : -1;
         v[u] = {};
         r[u] = u32x2{0, 0};
         if(in && col < p.k) {
            v[u] = load_row8(x, p.ld, row, col, p.k);
            if constexpr(RAND) r[u] = load_rand8(p.rand, row, col, p.k);
         }
      }
   }
#pragma unroll
   for(int u = 0; u < ROWS; u++) {
      uint32_t c, word;
      encode_row8<T, RAND>(v[u], r[u], p.fit != 0, &c, &word);
      if(to[u] >= 0 && to[u] < p.slot_count) {
         *reinterpret_cast<uint32_t*>(p.codes + to[u] * (kp / 2) + col / 2) = c;
         if((lane & 15) == 0) *reinterpret_cast<uint32_t*>(p.scales + to[u] * (kp / kBlock) + col / kBlock) = word;
      }
   }
}

// eight 16-bit elements without the first n (1 .. 7), zeros behind
template<class T>
__device__ inline Eight<T> drop_first(const Eight<T>& v, int n)
{
   struct Halves { uint64_t lo, hi; } h = __builtin_bit_cast(Halves, v);
   const int bits = 16 * n;
   if(bits >= 64) {
      h.lo = h.hi >> (bits - 64);
      h.hi = 0;
   } else {
      h.lo = (h.lo >> bits) | (h.hi << (64 - bits));
      h.hi >>= bits;
   }
   return __builtin_bit_cast(Eight<T>, h);
}

// Blocks along columns, and along rows too where p.codes is given, from one
// reading: a workgroup takes 128 rows x 128 columns, a lane 8 values of 8 rows.  The
// values (and random bytes) wait in LDS in their own type, and each lane takes two
// neighbouring columns of 32 rows: 16 bytes of codes a column, four lanes a group of
// 128 rows.  The pair of columns (row, pair) lies at slot pair ^ 16 (row / 32), so that
// the four lanes of a group read different banks.  8192 x 4096 in bf16 34 us to the nearest (VALU
// instructions 35 % of the cycles, waiting 47 % of the wavefronts' time), 44 with random bytes
// (VALU 63 %), where the bytes are 15 and 20.
template<class T> struct alignas(2 * sizeof(T)) Pair { T a, b; };

template<class T, bool RAND>
__global__ void __launch_bounds__(kLanes)
quantize_both(QuantizeParams p, int64_t kp, int64_t rowsp)
{
   __shared__ alignas(16) Pair<T> tile[128 * 64];
   __shared__ alignas(16) uint16_t rtile[RAND ? 128 * 64 : 8];
   const T* x = static_cast<const T*>(p.x);
   const int64_t c0 = (int64_t)blockIdx.x * 128;
   const int64_t r0 = ((int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y) * 128;
   if(r0 >= rowsp) return;
   const bool fit = p.fit != 0;
   const int lane = threadIdx.x & 15, first = threadIdx.x >> 4;
   const int64_t col = c0 + lane * 8;
   Eight<T> v[8];
   u32x2 r[8];
   if(p.k % 8 == 0 || c0 + 128 <= p.k || (sizeof(T) == 2 && p.k >= 8)) {
      // whole pieces of eight: all loads ahead, beyond the matrix from its last row or piece
      // (777 x 520, fp16 with random bytes: 13.6 us with a branch around each piece, 8.4 so).
      // A piece that the last column cuts is the row's last eight values, the earlier
      // ones shifted out.
      const int64_t c = col + 8 <= p.k ? col : p.k - 8;
      const int drop = col < p.k ? (int)(col - c) : 0;
#pragma unroll
      for(int u = 0; u < 8; u++) {
         const int64_t row = r0 + u * 16 + first, at = row < p.rows ? row : p.rows - 1;
         v[u] = *reinterpret_cast<const Eight<T>*>(x + at * p.ld + c);
         r[u] = u32x2{0, 0};
         if constexpr(RAND) {
            const Bytes8 t = *reinterpret_cast<const Bytes8*>(p.rand + at * p.k + c);
            r[u] = u32x2{t.e[0], t.e[1]};
         }
      }
#pragma unroll
      for(int u = 0; u < 8; u++)
         if(r0 + u * 16 + first >= p.rows || col >= p.k) v[u] = {};
      if constexpr(sizeof(T) == 2) {
         if(p.k % 8 != 0 && c0 + 128 > p.k) {
#pragma unroll
            for(int u = 0; u < 8; u++) {
               if(!drop) break;
               v[u] = drop_first(v[u], drop);
               const uint64_t b = (((uint64_t)r[u][1] << 32) | r[u][0]) >> (8 * drop);
               r[u] = u32x2{(uint32_t)b, (uint32_t)(b >> 32)};
            }
         }
      }
   } else {
#pragma unroll
      for(int u = 0; u < 8; u++) {
         const int64_t row = r0 + u * 16 + first;
         v[u] = {};
         r[u] = u32x2{0, 0};
         if(row < p.rows && col < p.k) {
            v[u] = load_row8(x, p.ld, row, col, p.k);
            if constexpr(RAND) r[u] = load_rand8(p.rand, row, col, p.k);
         }
      }
   }
#pragma unroll
   for(int u = 0; u < 8; u++) {
      const int lrow = u * 16 + first, at = lrow * 64 + ((lane * 4) ^ ((lrow >> 5) << 4));
      struct alignas(16) Whole { T e[8]; };
      *reinterpret_cast<Whole*>(&tile[at]) = __builtin_bit_cast(Whole, v[u]);
      if constexpr(RAND) *reinterpret_cast<u32x2*>(&rtile[at]) = r[u];
      if(p.codes) {
         const int64_t row = r0 + lrow;
         uint32_t c, word;
         encode_row8<T, RAND>(v[u], r[u], fit, &c, &word);
         if(row < p.rows) {
            *reinterpret_cast<uint32_t*>(p.codes + row * (kp / 2) + col / 2) = c;
            if(lane == 0) *reinterpret_cast<uint32_t*>(p.scales + row * (kp / kBlock) + col / kBlock) = word;
         }
      }
   }
   __syncthreads();
   const int blk = threadIdx.x & 3, pair = threadIdx.x >> 2;
   const int base = blk * 32 * 64 + (pair ^ (blk << 4));
   Pair<T> t[32];
   uint32_t b[RAND ? 32 : 1] = {};                    // the random bytes of both columns
   uint32_t top[2] = {0, 0};
#pragma unroll
   for(int i = 0; i < 32; i++) {
      t[i] = tile[base + i * 64];
      if constexpr(RAND) b[i] = rtile[base + i * 64];
      top[0] = umax(top[0], magnitude(to_float(t[i].a)));
      top[1] = umax(top[1], magnitude(to_float(t[i].b)));
   }
#pragma unroll
   for(int h = 0; h < 2; h++) {
      const uint32_t s = scale_byte(top[h], fit);
      uint32_t word = s | (dpp<kQuadSwap1>(s) << 8);     // right at the group's lane 0, which alone stores it
      word |= dpp<kQuadSwap2>(word) << 16;
      u32x4 c;
#pragma unroll
      for(int q = 0; q < 4; q++) {
         float w[8];
         uint32_t rr[8];
#pragma unroll
         for(int i = 0; i < 8; i++) {
            w[i] = to_float(h ? t[q * 8 + i].b : t[q * 8 + i].a);
            rr[i] = (b[RAND ? q * 8 + i : 0] >> (8 * h)) & 255u;
         }
         c[q] = encode<T, RAND>(w, s, rr);
      }
      const int64_t tcol = c0 + pair * 2 + h;
      if(tcol < p.k) {
         *reinterpret_cast<u32x4*>(p.codes_t + tcol * (rowsp / 2) + r0 / 2 + blk * 16) = c;
         if(blk == 0) *reinterpret_cast<uint32_t*>(p.scales_t + tcol * (rowsp / kBlock) + r0 / kBlock) = word;
      }
   }
}

// Blocks back to values: 8 codes a lane, bound by the values' bytes (8192 x 4096 to bf16 13.7
// us, 6.2 TB/s with the codes from the last-level cache).
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
   if(!grid_ok(gx, kLanes) || gz > 65535) return false;
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
      if(!make_grid(kp / 128, rowsp / 128, &g)) return kTooLarge;
      quantize_both<T, RAND><<<g, kLanes, 0, s>>>(p, kp, rowsp);
   } else {
      constexpr int ROWS = 4;
      const int lr = lanes_log(kp);
      const int64_t per = (kLanes >> lr) * ROWS;
      if(!make_grid((kp / 8 + (1 << lr) - 1) >> lr, (p.rows + per - 1) / per, &g)) return kTooLarge;
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
   if(!make_grid((kp / 8 + (1 << lr) - 1) >> lr, (p.rows + per - 1) / per, &g)) return kTooLarge;
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
