// Products with microscaled 4-bit operands on the matrix cores.
//
//   matmul: out[i][j] = bias[j] + sum_k x[i][k] w[j][k], both in blocks;
//   linear: the same with x in fp32, bf16 or fp16 as it is.
//
// The scaled product instruction takes 4-bit operands whole: in the 16 x 16 x 128
// form a lane gives one block, 16 bytes of codes and their scale byte, of row
// lane % 16 and block lane / 16; in the 32 x 32 x 64 form row lane % 32 and block
// lane / 32.  Products and sums are fp32.
#include "fufft_internal.hpp"
#include "mx4_device.hpp"
#include "mx4_internal.hpp"

#include <type_traits>

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

// ---- many rows: tiles staged in LDS ---------------------------------------------------
//
// A workgroup of WM x WN wavefronts computes BM x BN results, a wavefront FM x FN
// products of 32 x 32 x 64.  K goes by slabs of 256 values: BM + BN rows of 128 bytes
// and, for two slabs at a time, of 16 scale bytes.  Two slabs are in LDS, one read, one
// on its way there: straight from memory, so that no register waits for it.  The
// loads write lane after lane, 8 rows of 8 chunks of 16 bytes; which chunk a lane
// fetches is free, and slot c of row r gets chunk c ^ (r % 8) ^ (r / 8 % 2), so that
// the lanes of a product, which read one chunk of 32 rows, meet all banks.
//
// Block 2 t + lane / 32 of a slab takes part in product t: both its halves' scales are
// bytes 0 and 2 (t = 0, 1) of a word shifted by 8 (lane / 32), and where K ends with
// half a slab, products 2 and 3 are left out.
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kFlags = 0x00020000;     // raw buffer, 32-bit elements

__device__ inline __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t bytes)
{
   const int64_t most = 0xfffffff0;
   return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)(uint32_t)(bytes < most ? bytes : most), kFlags);
}

typedef __attribute__((address_space(3))) void lds_void;

// 16 bytes a lane from buffer offset voff + soff to LDS at `to` + 16 lane
__device__ inline void fetch16(__amdgpu_buffer_rsrc_t r, uint8_t* to, uint32_t voff, uint32_t soff)
{
   __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)to, 16, (int)voff, (int)soff, 0, 0);
}

// Tile of workgroup `id` of tm x tn.  Workgroups go to the 8 XCDs in turn; each XCD,
// with an L2 of its own, gets a run of tiles, and a run goes through strips of 8
// tiles along m, so that the tiles that an XCD works on share rows.
__device__ inline void tile_of(uint32_t id, uint32_t tm, uint32_t tn, uint32_t* m, uint32_t* n)
{
   const uint32_t total = tm * tn, each = total / 8, more = total % 8, xcd = id % 8;
   const uint32_t i = xcd * each + (xcd < more ? xcd : more) + id / 8;
   const uint32_t strip = i / (8 * tn), in = i - strip * 8 * tn;
   const uint32_t high = tm - strip * 8 < 8 ? tm - strip * 8 : 8;
   *m = strip * 8 + in % high;
   *n = in / high;
}

template<class O, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN)
matmul_tiles(MatmulParams p, uint32_t groups, uint32_t tm, uint32_t tn)
{
   constexpr int WAVES = WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;
   constexpr int ROWS = BM + BN, SLAB = ROWS * 128, SCALES = ROWS * 16;
   constexpr int JOBS = ROWS / 8 / WAVES;                     // fetches of 8 rows a wavefront and slab
   extern __shared__ uint8_t lds[];
   uint8_t* const scale_lds = lds + 2 * SLAB;
   const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
   const int half = lane >> 5;
   uint32_t ti, tj;
   tile_of(blockIdx.x, tm, tn, &ti, &tj);
   const int64_t m0 = (int64_t)ti * BM, n0 = (int64_t)tj * BN;
   const int ml = (int)(p.m - m0 < BM ? p.m - m0 : BM), nl = (int)(p.n - n0 < BN ? p.n - n0 : BN);
   const uint32_t row_bytes = groups * 64, srow_bytes = groups * 4;
   const __amdgpu_buffer_rsrc_t rx = buffer(static_cast<const uint8_t*>(p.x) + m0 * row_bytes, (int64_t)ml * row_bytes);
   const __amdgpu_buffer_rsrc_t rw = buffer(p.w + n0 * row_bytes, (int64_t)nl * row_bytes);
   const __amdgpu_buffer_rsrc_t rsx = buffer(p.x_scales + m0 * srow_bytes, (int64_t)ml * srow_bytes);
   const __amdgpu_buffer_rsrc_t rsw = buffer(p.w_scales + n0 * srow_bytes, (int64_t)nl * srow_bytes);

   // job j of this wavefront: rows 8 (wave JOBS + j) .. + 7 of the slab, x's rows first.  Rows
   // beyond the matrix fetch its last one.
   uint32_t voff[JOBS], back[2];               // back: from chunk 4 .. 7 to 0 .. 3, by the row's turn
   for(int j = 0; j < 2; j++) back[j] = (((lane & 7) ^ (lane >> 3) ^ j) & 4) * 16;
#pragma unroll
   for(int j = 0; j < JOBS; j++) {
      const int r8 = wave * JOBS + j, row = r8 * 8 + (lane >> 3);
      const int in = row < BM ? (row < ml ? row : ml - 1) : (row - BM < nl ? row - BM : nl - 1);
      const uint32_t chunk = (lane & 7) ^ (lane >> 3) ^ (r8 & 1);
      voff[j] = (uint32_t)in * row_bytes + chunk * 16;
   }
   const uint32_t slabs = (groups + 1) / 2;
   auto fetch_slab = [&](uint32_t s) {
      uint8_t* const to = lds + (s & 1) * SLAB + wave * JOBS * 1024;
      const bool odd = 2 * s + 2 > groups;                    // half a slab: chunks 4 .. 7 fetch 0 .. 3
#pragma unroll
      for(int j = 0; j < JOBS; j++) {
         const int row = (wave * JOBS + j) * 8;
         const uint32_t v = odd ? voff[j] - back[(wave * JOBS + j) & 1] : voff[j];
         fetch16(row < BM ? rx : rw, to + j * 1024, v, s * 128);
      }
   };
   // the scales of slabs 2 q and 2 q + 1: 64 rows a fetch; beyond the matrix the buffer's end gives zeros
   auto fetch_scales = [&](uint32_t q) {
#pragma unroll
      for(int j = 0; j < (ROWS / 64 + WAVES - 1) / WAVES; j++) {
         const int r = (wave + j * WAVES) * 64;
         if(r >= ROWS) break;
         uint8_t* const to = scale_lds + (q & 1) * SCALES + r * 16;
         const uint32_t row = r + lane;
         if(r < BM) fetch16(rsx, to, row * srow_bytes, q * 16);
         else       fetch16(rsw, to, (row - BM) * srow_bytes, q * 16);
      }
   };

   const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
   uint32_t xat[FM], wat[FN];                                  // LDS offsets of this lane's rows
#pragma unroll
   for(int a = 0; a < FM; a++) xat[a] = wm + a * 32 + (lane & 31);
#pragma unroll
   for(int b = 0; b < FN; b++) wat[b] = BM + wn + b * 32 + (lane & 31);
   const uint32_t turn = (lane & 7) ^ ((lane >> 3) & 1);       // the slot's turn of this lane's rows

   f32x16 acc[FM][FN] = {};
   if(slabs) {
      fetch_scales(0);
      fetch_slab(0);
   }
   for(uint32_t s = 0; s < slabs; s++) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if(s + 1 < slabs) {
         if((s & 1) == 0 && s + 2 < slabs) fetch_scales(s / 2 + 1);
         fetch_slab(s + 1);
      }
      const uint8_t* const data = lds + (s & 1) * SLAB;
      const uint8_t* const sc = scale_lds + ((s >> 1) & 1) * SCALES + (s & 1) * 8;
      u32x2 sx[FM], sw[FN];
#pragma unroll
      for(int a = 0; a < FM; a++) sx[a] = *reinterpret_cast<const u32x2*>(sc + xat[a] * 16) >> (uint32_t)(half * 8);
#pragma unroll
      for(int b = 0; b < FN; b++) sw[b] = *reinterpret_cast<const u32x2*>(sc + wat[b] * 16) >> (uint32_t)(half * 8);
      auto step = [&](auto tc) {
         constexpr int t = decltype(tc)::value;
         const uint32_t slot = ((2 * t + half) ^ turn) * 16;
         u32x4 x[FM], w[FN];
#pragma unroll
         for(int b = 0; b < FN; b++) w[b] = *reinterpret_cast<const u32x4*>(data + wat[b] * 128 + slot);
#pragma unroll
         for(int a = 0; a < FM; a++) x[a] = *reinterpret_cast<const u32x4*>(data + xat[a] * 128 + slot);
#pragma unroll
         for(int a = 0; a < FM; a++)
#pragma unroll
            for(int b = 0; b < FN; b++)
               acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand4(x[a]), operand4(w[b]), acc[a][b], 4, 4,
                                                                           (t & 1) * 2, (int)sx[a][t >> 1], (t & 1) * 2,
                                                                           (int)sw[b][t >> 1]);
      };
      step(std::integral_constant<int, 0>());
      step(std::integral_constant<int, 1>());
      if(2 * s + 2 <= groups) {
         step(std::integral_constant<int, 2>());
         step(std::integral_constant<int, 3>());
      }
   }
   // register i of a product: row 8 (i / 4) + 4 half + i % 4 of x, row lane % 32 of w
   O* out = static_cast<O*>(p.out);
#pragma unroll
   for(int b = 0; b < FN; b++) {
      const int j = wn + b * 32 + (lane & 31);
      const float bias = p.bias && j < nl ? p.bias[n0 + j] : 0.0f;
#pragma unroll
      for(int a = 0; a < FM; a++)
#pragma unroll
         for(int i = 0; i < 16; i++) {
            const int r = wm + a * 32 + 8 * (i / 4) + 4 * half + i % 4;
            if(r < ml && j < nl) out[(m0 + r) * p.ld + n0 + j] = (O)(acc[a][b][i] + bias);
         }
   }
}

template<class O, int BM, int BN, int WM, int WN>
hipError_t tiles_shape(const MatmulParams& p, hipStream_t s)
{
   constexpr size_t bytes = (size_t)(BM + BN) * (2 * 128 + 2 * 16);
   const int64_t groups = padded(p.k) / kGroup, tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
   if(tm * tn > 0x7fffffff) return hipErrorInvalidValue;
   static std::atomic<uint64_t> mask{0};
   const hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(&matmul_tiles<O, BM, BN, WM, WN>), bytes, mask);
   if(e != hipSuccess) return e;
   matmul_tiles<O, BM, BN, WM, WN><<<(unsigned)(tm * tn), 64 * WM * WN, bytes, s>>>(p, (uint32_t)groups, (uint32_t)tm,
                                                                                   (uint32_t)tn);
   return hipGetLastError();
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
   // a tile's offsets are 32-bit: 256 rows of k / 2 bytes
   if(p.k <= (int64_t)1 << 24) {
      const int64_t big = ((p.m + 255) / 256) * ((p.n + 255) / 256);
      if(big >= 200) return tiles_shape<O, 256, 256, 2, 4>(p, s);
      if(p.m > 64) return tiles_shape<O, 128, 128, 2, 2>(p, s);
   }
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
