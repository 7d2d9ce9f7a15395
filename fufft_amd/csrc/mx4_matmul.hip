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
// runs of four groups of 128 values in turn, and their sums are joined in LDS in the
// order of the wavefronts.  What bounds these kernels is w's bytes where N is large
// and else the wait for memory, so each wavefront has DEPTH runs on their way.
//
// A load of 16 scale bytes or words of 16 rows takes as long as one of 16 bytes of
// codes a lane.  So the 16 bytes of a row and run come in one load, a word for each of
// the four lanes of a row, and the words go round between those lanes: at 16384 x 16384
// the load of a byte for each block took 57 us where scales left out took 39.

constexpr int kRun = 4;                // groups of 128 values

// A lane's part of a run of 16 rows: its block of every group, and the word that
// holds the four scales of group lane / 16.
struct Run {
   u32x4    c[kRun];
   uint32_t s;
};

__device__ inline void fetch_run(Run& r, const uint8_t* codes, const uint8_t* scales, int64_t first, int groups)
{
   // first: the run's first group; the last group's scales again beyond the last
   const int lane = threadIdx.x & 63, mine = (int)first + (lane >> 4);
#pragma unroll
   for(int g = 0; g < kRun; g++)
      if(g == 0 || first + g < groups) r.c[g] = *reinterpret_cast<const u32x4*>(codes + (first + g) * 64);
   r.s = *reinterpret_cast<const uint32_t*>(scales + (int64_t)(mine < groups ? mine : groups - 1) * 4);
}
// the lane's scale byte of group g of the run, in the low byte
__device__ inline uint32_t run_scale(const Run& r, int g)
{
   const int lane = threadIdx.x & 63;
   return (uint32_t)__builtin_amdgcn_ds_bpermute((g * 16 + (lane & 15)) * 4, (int)r.s) >> ((lane >> 4) * 8);
}

// wavefronts of a workgroup with so many 16 x 16 tiles: their sums fill at most 64 KiB of LDS
constexpr int most_waves(int tiles) { return tiles >= 8 ? 4 : 8; }

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
      if(m >= p.m) break;
      if(n >= p.n) continue;
      float v = 0.0f;
      for(int w = 0; w < waves; w++) v += join[w * ROWS * COLS + i];
      if(p.bias) v += p.bias[n];
      out[m * p.ld + n] = (O)v;
   }
}

// the row that a lane reads for a tile of 16: rows beyond the last read the last one
__device__ inline int64_t row_of(int64_t first, int64_t rows)
{
   const int64_t r = first + (threadIdx.x & 15);
   return r < rows ? r : rows - 1;
}

template<class O, int MT, int NT, int DEPTH>
__global__ void __launch_bounds__(64 * most_waves(MT * NT))
matmul_rows(MatmulParams p, int groups, int waves)
{
   extern __shared__ float join[];
   const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
   const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
   const uint8_t* xc[MT];
   const uint8_t* xs[MT];
   const uint8_t* wc[NT];
   const uint8_t* ws[NT];
#pragma unroll
   for(int a = 0; a < MT; a++) {
      const int64_t r = row_of(m0 + a * 16, p.m);
      xc[a] = static_cast<const uint8_t*>(p.x) + r * groups * 64 + (lane >> 4) * 16;
      xs[a] = p.x_scales + r * groups * 4;
   }
#pragma unroll
   for(int b = 0; b < NT; b++) {
      const int64_t r = row_of(n0 + b * 16, p.n);
      wc[b] = p.w + r * groups * 64 + (lane >> 4) * 16;
      ws[b] = p.w_scales + r * groups * 4;
   }
   Run x[DEPTH][MT], w[DEPTH][NT];
   auto fetch = [&](int d, int64_t g) {
#pragma unroll
      for(int b = 0; b < NT; b++) fetch_run(w[d][b], wc[b], ws[b], g, groups);
#pragma unroll
      for(int a = 0; a < MT; a++) fetch_run(x[d][a], xc[a], xs[a], g, groups);
   };
   f32x4 acc[MT][NT] = {};
   const int step = waves * kRun;
#pragma unroll
   for(int d = 0; d < DEPTH; d++)
      if(wave * kRun + d * step < groups) fetch(d, wave * kRun + d * step);
#pragma unroll 1
   for(int g0 = wave * kRun; g0 < groups; g0 += step * DEPTH) {
#pragma unroll
      for(int d = 0; d < DEPTH; d++) {
         const int g = g0 + d * step;
#pragma unroll
         for(int i = 0; i < kRun; i++) {
            if(g + i >= groups) break;
            uint32_t sw[NT];
#pragma unroll
            for(int b = 0; b < NT; b++) sw[b] = run_scale(w[d][b], i);
#pragma unroll
            for(int a = 0; a < MT; a++) {
               const uint32_t sx = run_scale(x[d][a], i);
#pragma unroll
               for(int b = 0; b < NT; b++)
                  acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand4(w[d][b].c[i]), operand4(x[d][a].c[i]),
                                                                               acc[a][b], 4, 4, 0, (int)sw[b], 0, (int)sx);
            }
         }
         if(g + step * DEPTH < groups) fetch(d, g + step * DEPTH);
      }
   }
   join_and_store<O, MT, NT>(p, acc, join, waves, m0, n0);
}

// The rows of x as the w operand meets them: a value in bf16 is one, in fp16 two, in
// fp32 three bf16 parts (8, 11 and 24 significant bits at 8 a part, cut off rather than
// rounded, so that no part overflows).  The parts add up to the value exactly but for
// bits below 2^-133, so the product is that of the values themselves.
template<class T> struct PartsOf;
template<> struct PartsOf<bf16>  { static constexpr int value = 1; };
template<> struct PartsOf<f16>   { static constexpr int value = 2; };
template<> struct PartsOf<float> { static constexpr int value = 3; };

template<class T, int PARTS = PartsOf<T>::value>
__device__ inline void split8(const T (&v)[8], bf16x8 (&part)[PARTS])
{
#pragma unroll
   for(int i = 0; i < 8; i++) {
      if constexpr(PARTS == 1) {
         part[0][i] = v[i];
      } else {
         float left = to_float(v[i]);
#pragma unroll
         for(int q = 0; q < PARTS; q++) {
            const float b = __uint_as_float(__float_as_uint(left) & 0xffff0000u);
            part[q][i] = __builtin_bit_cast(bf16, (uint16_t)(__float_as_uint(left) >> 16));
            if(q + 1 < PARTS) left = magnitude(left) == 0x7f800000u ? 0.0f : left - b;   // all of an infinity is in one part
         }
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

// The block that a lane reads holds its 8 values of each of four products, so
// product t takes values 8 t .. 8 t + 7 of the four blocks of a group.  (Blocks turned among
// a row's four lanes, so that those read 64 bytes of x in a row: 1 x 8192 x 8192 10.9 / 11.1 us,
// 64 x 8192 x 8192 in bf16 43 / 42, in fp32 89 / 75.)
template<class T, class O, int MT, int NT, int DEPTH>
__global__ void __launch_bounds__(64 * most_waves(MT * NT))
linear_rows(MatmulParams p, int groups, int waves)
{
   constexpr int PARTS = PartsOf<T>::value;
   extern __shared__ float join[];
   const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
   const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
   const int64_t k0 = (lane >> 4) * 32;
   const T* x[MT];
   const uint8_t* wc[NT];
   const uint8_t* ws[NT];
#pragma unroll
   for(int a = 0; a < MT; a++) x[a] = static_cast<const T*>(p.x) + row_of(m0 + a * 16, p.m) * p.ldx + k0;
#pragma unroll
   for(int b = 0; b < NT; b++) {
      const int64_t r = row_of(n0 + b * 16, p.n);
      wc[b] = p.w + r * groups * 64 + (lane >> 4) * 16;
      ws[b] = p.w_scales + r * groups * 4;
   }
   Run w[DEPTH][NT];
   auto fetch = [&](int d, int64_t g) {
#pragma unroll
      for(int b = 0; b < NT; b++) fetch_run(w[d][b], wc[b], ws[b], g, groups);
   };
   f32x4 acc[MT][NT] = {};
   const int step = waves * kRun;
#pragma unroll
   for(int d = 0; d < DEPTH; d++)
      if(wave * kRun + d * step < groups) fetch(d, wave * kRun + d * step);
#pragma unroll 1
   for(int g0 = wave * kRun; g0 < groups; g0 += step * DEPTH) {
#pragma unroll
      for(int d = 0; d < DEPTH; d++) {
         const int64_t first = g0 + d * step;
         struct __attribute__((packed, aligned(sizeof(T)))) Block { T e[4][8]; };
         auto group = [&](int i, const Block (&v)[MT]) {
            float sw[NT];
#pragma unroll
            for(int b = 0; b < NT; b++) sw[b] = scale_operand(run_scale(w[d][b], i) & 255u);
#pragma unroll
            for(int t = 0; t < 4; t++) {
               bf16x8 part[MT][PARTS];
#pragma unroll
               for(int a = 0; a < MT; a++) split8<T>(v[a].e[t], part[a]);
#pragma unroll
               for(int b = 0; b < NT; b++) {
                  const bf16x8 c = decode8_bf16(w[d][b].c[i][t], sw[b]);
#pragma unroll
                  for(int a = 0; a < MT; a++)
#pragma unroll
                     for(int q = 0; q < PARTS; q++)
                        acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c, part[a][q], acc[a][b], 0, 0, 0);
               }
            }
         };
         if((first + kRun) * 128 <= p.k) {
            // whole runs in straight code: x's loads go ahead of the products
#pragma unroll
            for(int i = 0; i < kRun; i++) {
               Block v[MT];
#pragma unroll
               for(int a = 0; a < MT; a++) v[a] = *reinterpret_cast<const Block*>(x[a] + (first + i) * 128);
               group(i, v);
            }
         } else {
            // the last run: whole groups as above, then what is left of x in pieces of eight, beyond
            // its end the last piece again, made zero; single values where K cuts one
#pragma unroll
            for(int i = 0; i < kRun; i++) {
               const int64_t k = (first + i) * 128;
               if(k >= p.k) break;
               Block v[MT];
               if(k + 128 <= p.k) {
#pragma unroll
                  for(int a = 0; a < MT; a++) v[a] = *reinterpret_cast<const Block*>(x[a] + k);
               } else {
                  struct __attribute__((packed, aligned(sizeof(T)))) Eight { T e[8]; };
#pragma unroll
                  for(int t = 0; t < 4; t++) {
                     const int64_t at = k + k0 + t * 8;      // in the row; x[a] starts at k0
#pragma unroll
                     for(int a = 0; a < MT; a++) {
                        const T* const row = x[a] - k0;
                        Eight e;
                        if(p.k % 8 == 0) {
                           e = *reinterpret_cast<const Eight*>(row + (at < p.k ? at : p.k - 8));
                        } else {
#pragma unroll
                           for(int j = 0; j < 8; j++) e.e[j] = row[at + j < p.k ? at + j : p.k - 1];
                        }
#pragma unroll
                        for(int j = 0; j < 8; j++) v[a].e[t][j] = at + j < p.k ? e.e[j] : (T)0.0f;
                     }
                  }
               }
               group(i, v);
            }
         }
         if(first + step * DEPTH < groups) fetch(d, first + step * DEPTH);
      }
   }
   join_and_store<O, MT, NT>(p, acc, join, waves, m0, n0);
}

// ---- many rows: tiles staged in LDS ---------------------------------------------------
//
// A workgroup of WM x WN wavefronts computes BM x BN results, a wavefront FM x FN
// products of 32 x 32 x 64.  K goes by slabs of 256 values: BM + BN rows of 128 bytes.
// Two slabs are in LDS, one read, one on its way there: straight from memory, so
// that no register waits for it.  The loads write lane after lane, 8 rows of 8 chunks
// of 16 bytes; which chunk a lane fetches is free, and slot c of row r gets chunk
// c ^ (r % 8) ^ (r / 8 % 2), so that the lanes of a product, which read one chunk of 32
// rows, meet all banks.
//
// A row's scales lie in one place for all of K, so a slab's are 8 bytes from each of BM +
// BN places.  They come 64 bytes a row at a time, for 8 slabs, through registers (LDS has
// no room for a second set); fetched 16 bytes a row for every two slabs, they were a
// third of all requests to the L2 (8192 x 8192 x 8192: 286 -> 282 us).
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
// with an L2 of its own, gets a run of tiles, and a run goes through strips of 4
// tiles along m, so that the tiles that an XCD works on share rows (8192 x 8192 x 4096:
// tiles in plain order 157 us, strips of 8 147, of 4 145.5).
__device__ inline void tile_of(uint32_t id, uint32_t tm, uint32_t tn, uint32_t* m, uint32_t* n)
{
   const uint32_t total = tm * tn, each = total / 8, more = total % 8, xcd = id % 8;
   const uint32_t i = xcd * each + (xcd < more ? xcd : more) + id / 8;
   const uint32_t strip = i / (4 * tn), in = i - strip * 4 * tn;
   const uint32_t high = tm - strip * 4 < 4 ? tm - strip * 4 : 4;
   *m = strip * 4 + in % high;
   *n = in / high;
}

template<class O, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN)
matmul_tiles(MatmulParams p, uint32_t groups, uint32_t tm, uint32_t tn)
{
   constexpr int WAVES = WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;
   constexpr int ROWS = BM + BN, SLAB = ROWS * 128, SCALES = ROWS * 64;
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
   // the scales of slabs 8 q .. 8 q + 7: 4 lanes a row, ROWS / 4 / WAVES fetches of 16 rows a wavefront; 16-byte
   // part c of row r at slot c ^ (r / 4 % 4).  Beyond the matrix the buffer's end gives zeros.
   constexpr int PARTS = ROWS / 16 / WAVES;
   u32x4 next[PARTS];
   auto load_scales = [&](uint32_t q) {
#pragma unroll
      for(int j = 0; j < PARTS; j++) {
         const int r = (j * WAVES + wave) * 16;
         const uint32_t at = q * 64 + (lane & 3) * 16, row = r + (lane >> 2);
         next[j] = __builtin_bit_cast(u32x4, r < BM ? __builtin_amdgcn_raw_buffer_load_b128(rsx, row * srow_bytes + at, 0, 0)
                                                    : __builtin_amdgcn_raw_buffer_load_b128(rsw, (row - BM) * srow_bytes + at, 0, 0));
      }
   };
   auto keep_scales = [&]() {
#pragma unroll
      for(int j = 0; j < PARTS; j++) {
         const uint32_t row = (j * WAVES + wave) * 16 + (lane >> 2);
         *reinterpret_cast<u32x4*>(scale_lds + row * 64 + ((lane & 3) ^ (row >> 2 & 3)) * 16) = next[j];
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
      load_scales(0);
      fetch_slab(0);
      keep_scales();
   }
   for(uint32_t s = 0; s < slabs; s++) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if((s & 7) == 0 && s) {
         keep_scales();
         __syncthreads();
      }
      if(s + 1 < slabs) fetch_slab(s + 1);
      if((s & 7) == 4 && s + 4 < slabs) load_scales(s / 8 + 1);
      const uint8_t* const data = lds + (s & 1) * SLAB;
      const uint32_t sc = ((s >> 1 & 3) ^ (lane >> 2 & 3)) * 16 + (s & 1) * 8;
      u32x2 sx[FM], sw[FN];
#pragma unroll
      for(int a = 0; a < FM; a++)
         sx[a] = *reinterpret_cast<const u32x2*>(scale_lds + xat[a] * 64 + sc) >> (uint32_t)(half * 8);
#pragma unroll
      for(int b = 0; b < FN; b++)
         sw[b] = *reinterpret_cast<const u32x2*>(scale_lds + wat[b] * 64 + sc) >> (uint32_t)(half * 8);
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
               acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand4(w[b]), operand4(x[a]), acc[a][b], 4, 4,
                                                                           (t & 1) * 2, (int)sw[b][t >> 1], (t & 1) * 2,
                                                                           (int)sx[a][t >> 1]);
      };
      step(std::integral_constant<int, 0>());
      step(std::integral_constant<int, 1>());
      if(2 * s + 2 <= groups) {
         step(std::integral_constant<int, 2>());
         step(std::integral_constant<int, 3>());
      }
   }
   // Register i of a product: row 8 (i / 4) + 4 half + i % 4 of w, row lane % 32 of x.  Each
   // wavefront turns its results in its share of the LDS and stores whole 16-byte
   // pieces of rows.
   constexpr int COLS = FN * 32, PITCH = COLS * (int)sizeof(O) + 16, SHARE = (2 * SLAB + SCALES) / WAVES;
   constexpr int PASS = SHARE / (32 * PITCH) < FM ? SHARE / (32 * PITCH) : FM;    // 32-row parts at a time
   static_assert(PASS > 0 && FM % PASS == 0, "a wavefront's share of the LDS holds whole parts");
   constexpr int PIECE = 16 / (int)sizeof(O), ACROSS = COLS / PIECE, DOWN = 64 / ACROSS;
   struct __attribute__((packed, aligned(sizeof(O)))) Piece { O e[PIECE]; };
   __syncthreads();
   uint8_t* const mine = lds + wave * SHARE;
   O* out = static_cast<O*>(p.out) + m0 * p.ld + n0;
#pragma unroll
   for(int a0 = 0; a0 < FM; a0 += PASS) {
#pragma unroll
      for(int b = 0; b < FN; b++)
#pragma unroll
         for(int q = 0; q < 4; q++) {
            const int j = b * 32 + q * 8 + half * 4;
            float bias[4] = {};
            if(p.bias)
#pragma unroll
               for(int i = 0; i < 4; i++) bias[i] = wn + j + i < nl ? p.bias[n0 + wn + j + i] : 0.0f;
#pragma unroll
            for(int a = a0; a < a0 + PASS; a++) {
               struct alignas(4 * sizeof(O)) Four { O e[4]; } v;
#pragma unroll
               for(int i = 0; i < 4; i++) v.e[i] = (O)(acc[a][b][q * 4 + i] + bias[i]);
               *reinterpret_cast<Four*>(mine + ((a - a0) * 32 + (lane & 31)) * PITCH + j * sizeof(O)) = v;
            }
         }
      __builtin_amdgcn_wave_barrier();
      const int j = wn + (lane % ACROSS) * PIECE;
#pragma unroll 4
      for(int i = 0; i < PASS * 32 / DOWN; i++) {
         const int in = i * DOWN + lane / ACROSS, r = wm + a0 * 32 + in;
         const u32x4 v = *reinterpret_cast<const u32x4*>(mine + in * PITCH + (lane % ACROSS) * 16);
         if(r >= ml) continue;
         const Piece piece = __builtin_bit_cast(Piece, v);
         O* to = out + (int64_t)r * p.ld + j;
         if(j + PIECE <= nl) {
            *reinterpret_cast<Piece*>(to) = piece;
         } else {
#pragma unroll
            for(int e = 0; e < PIECE; e++)
               if(j + e < nl) to[e] = piece.e[e];
         }
      }
      __builtin_amdgcn_wave_barrier();
   }
}

template<class O, int BM, int BN, int WM, int WN>
hipError_t tiles_shape(const MatmulParams& p, hipStream_t s)
{
   constexpr size_t bytes = (size_t)(BM + BN) * (2 * 128 + 64);
   const int64_t groups = padded(p.k) / kGroup, tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
   if(!grid_ok(tm * tn, 64 * WM * WN)) return kTooLarge;
   static std::atomic<uint64_t> mask{0};
   const hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(&matmul_tiles<O, BM, BN, WM, WN>), bytes, mask);
   if(e != hipSuccess) return e;
   matmul_tiles<O, BM, BN, WM, WN><<<(unsigned)(tm * tn), 64 * WM * WN, bytes, s>>>(p, (uint32_t)groups, (uint32_t)tm,
                                                                                   (uint32_t)tn);
   return hipGetLastError();
}

// wavefronts for so many runs: a power of two, `most` at most
int wavefronts(int64_t runs, int most)
{
   int w = 1;
   while(w < most && w < runs) w *= 2;
   return w;
}

template<class O, int MT, int NT, int DEPTH>
hipError_t rows_shape(const MatmulParams& p, hipStream_t s)
{
   const int64_t groups = padded(p.k) / kGroup;
   if(groups > 0x3fffffff) return kTooLarge;
   const int waves = wavefronts((groups + kRun - 1) / kRun, most_waves(MT * NT));
   const int64_t gx = (p.n + 16 * NT - 1) / (16 * NT), gy = (p.m + 16 * MT - 1) / (16 * MT);
   if(!grid_ok(gx, waves * 64) || gy > 65535) return kTooLarge;
   matmul_rows<O, MT, NT, DEPTH><<<dim3((unsigned)gx, (unsigned)gy), waves * 64, (size_t)waves * MT * NT * 1024, s>>>(
      p, (int)groups, waves);
   return hipGetLastError();
}

int64_t tiles(const MatmulParams& p, int64_t rows, int64_t cols)
{
   return ((p.m + rows - 1) / rows) * ((p.n + cols - 1) / cols);
}

// The kernel for a size, on MI355X's 256 CUs; us at m x n x k.
//   Up to 16 rows: 16 rows of w a workgroup, 32 where 16 are more than 256 workgroups (1 x 8192
//     x 8192 11.6 / 9.3).
//   At most 64 tiles of 64 x 64 and k long: the largest of 16 x 16, 32 x 16 and 32 x 32 of
//     at most 256 workgroups, with K split over their wavefronts, against 64 x 64 staged:
//     64 x 512 x 8192 6.7 / 13.6, 32 x 4096 x 4096 5.7 / 8.3, 512 x 512 x 8192 12.4 / 17.1; at
//     64 x 512 x 512 even.
//   Staged tiles: 256 x 256, one a CU, runs at 1.2 times the rate of 128 x 128, two a CU, so
//     the rounds that each needs decide: 4096 x 3200 x 2048 22.2 / 24.3, 8192 x 3200 x 2048
//     41.7 / 43.8, but 2048 x 4096 x 4096 32.9 / 25.6, 8192 x 2560 x 4096 66.5 / 58.7.
//     64 x 64 below 256 tiles of 128 x 128: 1001 x 2000 x 1504 8.3 -> 6.3, 256 x 4096 x 4096
//     14.5 -> 10.3.
template<class O>
hipError_t matmul_typed(const MatmulParams& p, hipStream_t s)
{
   if(p.m <= 16) return p.n > 16 * 256 ? rows_shape<O, 1, 2, 2>(p, s) : rows_shape<O, 1, 1, 2>(p, s);
   const bool far = p.k > (int64_t)1 << 24;           // a staged tile's offsets are 32-bit: 256 rows of k / 2 bytes
   if(p.k >= 2048 || far) {
      if(tiles(p, 16, 16) <= 256) return rows_shape<O, 1, 1, 2>(p, s);
      if(tiles(p, 32, 16) <= 256) return rows_shape<O, 2, 1, 2>(p, s);
      if(tiles(p, 32, 32) <= 256 || far) return rows_shape<O, 2, 2, 2>(p, s);
   }
   const int64_t big = tiles(p, 256, 256), mid = tiles(p, 128, 128);
   if(5 * ((big + 255) / 256) <= 3 * ((mid + 511) / 512)) return tiles_shape<O, 256, 256, 2, 4>(p, s);
   if(mid >= 256) return tiles_shape<O, 128, 128, 2, 2>(p, s);
   return tiles_shape<O, 64, 64, 2, 2>(p, s);
}

// A launch for every 65535 tiles of rows, a grid's end in y.
template<class T, class O, int MT, int NT, int DEPTH>
hipError_t linear_shape(const MatmulParams& p, hipStream_t s)
{
   const int64_t groups = padded(p.k) / kGroup;
   if(groups > 0x3fffffff) return kTooLarge;
   const int waves = wavefronts((groups + kRun - 1) / kRun, most_waves(MT * NT));
   const int64_t gx = (p.n + 16 * NT - 1) / (16 * NT), most = 65535 * 16 * MT;
   if(!grid_ok(gx, waves * 64)) return kTooLarge;
   for(int64_t first = 0; first < p.m; first += most) {
      MatmulParams q = p;
      q.m = p.m - first < most ? p.m - first : most;
      q.x = static_cast<const T*>(p.x) + first * p.ldx;
      q.out = static_cast<O*>(p.out) + first * p.ld;
      const unsigned gy = (unsigned)((q.m + 16 * MT - 1) / (16 * MT));
      linear_rows<T, O, MT, NT, DEPTH><<<dim3((unsigned)gx, gy), waves * 64, (size_t)waves * MT * NT * 1024, s>>>(
         q, (int)groups, waves);
      const hipError_t e = hipGetLastError();
      if(e != hipSuccess) return e;
   }
   return hipSuccess;
}

template<class T, class O>
hipError_t linear_typed(const MatmulParams& p, hipStream_t s)
{
   // 32 rows of w a workgroup share x's loads; 16 where 32 would leave CUs without one (us, 16 / 32
   // rows: 1 x 8192 x 8192 11.6 / 10.8, 13 x 5000 x 2056 5.4 / 4.7, 16 x 16384 x 16384 84 / 58, but 1 x
   // 4096 x 4096 4.1 / 5.7).  Beyond 32 rows of x, more workgroups: 64 rows in one took as long (64 x
   // 8192 x 8192 41 / 43, 64 x 4096 x 4096 19.9 / 19.4) and 48 x 208 x 113 8.5 / 5.8.
   const bool wide = p.n > 16 * 256;
   if(p.m <= 16) return wide ? linear_shape<T, O, 1, 2, 2>(p, s) : linear_shape<T, O, 1, 1, 2>(p, s);
   return wide ? linear_shape<T, O, 2, 2, 1>(p, s) : linear_shape<T, O, 2, 1, 1>(p, s);
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
