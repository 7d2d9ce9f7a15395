// Products of 8-bit rows on the matrix cores:
//
//   out[i][j] = bias[j] + sa[i] sb[j] sum_k a[i][k] b[j][k]
//
// The integer sum is exact in 32 bits.  In the 16 x 16 x 64 product a lane gives 16 bytes
// of row lane % 16 from byte 16 (lane / 16) on, in the 32 x 32 x 32 product of row lane %
// 32 from 16 (lane / 32) on.  Register i of a result: row 4 (lane / 16) + i, or
// 8 (i / 4) + 4 (lane / 32) + i % 4, of the first operand, row lane % 16 or 32 of the second.
// The first operand is b, so that a lane holds neighbours of a row of out.
#include "fufft_internal.hpp"
#include "layer_internal.hpp"
#include "mx4_device.hpp"

#include <type_traits>

namespace fufft {
namespace layer {

namespace {

using mx4::bf16;
using mx4::f16;
using mx4::u32x4;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// The scale of a row of a: a sum times a large one can leave fp32 where its product with the other scale does not,
// so that such a scale is taken 2^-40 times, and the result 2^40 times.  Both are exact: the sum is below 2^31, so that the first
// product stays below 2^119, and it is 2^24 at least, so that no scale of b brings the second one below the normal numbers.
struct RowScale {
   float s, up;
};
__device__ inline RowScale row_scale(float s)
{
   const bool large = fabsf(s) > 0x1p+64f;
   return {large ? s * 0x1p-40f : s, large ? 0x1p+40f : 1.0f};
}
__device__ inline float scaled(int sum, RowScale a, float b) { return (float)sum * a.s * b * a.up; }

// ---- single tokens: rows of b whole, products of four bytes -------------------------------
//
// A wavefront has 4 rows of b and M of a (those that are not there are zeros), the lanes 16 bytes each of 1 KiB
// of every row; the wavefronts of a workgroup share K, and their sums are joined in LDS.  Bound by b's bytes: a load
// is 1 KiB of one row, where the matrix cores' operands are 64 bytes of 16 rows (1 x 8192 x 8192 18.8 us so).
constexpr int kTokenRows = 4;

template<class O, int M, int UNROLL>
__global__ void __launch_bounds__(512)
i8_tokens(I8Params p, int64_t row_bytes)
{
   __shared__ int join[8][kTokenRows * M];
   const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
   const int waves = blockDim.x >> 6;
   const int64_t n0 = (int64_t)blockIdx.x * kTokenRows;
   const int8_t* b[kTokenRows];
#pragma unroll
   for(int r = 0; r < kTokenRows; r++) b[r] = p.b + (n0 + r < p.n ? n0 + r : p.n - 1) * row_bytes;
   int sum[kTokenRows][M] = {};
   const int64_t step = 1024 * UNROLL;
   for(int64_t k = wave * step; k < row_bytes; k += waves * step) {
      i32x4 w[UNROLL][kTokenRows], x[UNROLL][M];
#pragma unroll
      for(int u = 0; u < UNROLL; u++) {
         const int64_t at = k + u * 1024 + lane * 16;
         const bool in = at < row_bytes;
         const int64_t from = in ? at : 0;                  // beyond the end: any bytes of b, times zeros
#pragma unroll
         for(int r = 0; r < kTokenRows; r++) w[u][r] = *reinterpret_cast<const i32x4*>(b[r] + from);
#pragma unroll
         for(int i = 0; i < M; i++) {
            x[u][i] = *reinterpret_cast<const i32x4*>(p.a + (i < p.m ? i : 0) * row_bytes + from);
#pragma unroll
            for(int e = 0; e < 4; e++) x[u][i][e] = in ? x[u][i][e] : 0;
         }
      }
#pragma unroll
      for(int u = 0; u < UNROLL; u++)
#pragma unroll
         for(int i = 0; i < M; i++)
#pragma unroll
            for(int r = 0; r < kTokenRows; r++)
#pragma unroll
               for(int e = 0; e < 4; e++) sum[r][i] = __builtin_amdgcn_sdot4(w[u][r][e], x[u][i][e], sum[r][i], false);
   }
#pragma unroll
   for(int r = 0; r < kTokenRows; r++)
#pragma unroll
      for(int i = 0; i < M; i++) {
         uint32_t v = (uint32_t)sum[r][i];
         v += mx4::dpp<mx4::kQuadSwap1>(v);
         v += mx4::dpp<mx4::kQuadSwap2>(v);
         v += mx4::dpp<0x141>(v);                            // the mirrors within 8 and 16 lanes
         v += mx4::dpp<0x140>(v);
         const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)v, 0) + (uint32_t)__builtin_amdgcn_readlane((int)v, 16) +
                              (uint32_t)__builtin_amdgcn_readlane((int)v, 32) + (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
         if(lane == 0) join[wave][i * kTokenRows + r] = (int)all;
      }
   __syncthreads();
   const int i = threadIdx.x / kTokenRows, r = threadIdx.x % kTokenRows;
   const int64_t n = n0 + r;
   if(threadIdx.x < kTokenRows * M && i < p.m && n < p.n) {
      int total = 0;
      for(int w = 0; w < waves; w++) total += join[w][threadIdx.x];
      float v = row_bytes ? scaled(total, row_scale(p.a_scales[i]), p.b_scales[n]) : 0.0f;
      if(p.bias) v += p.bias[n];
      static_cast<O*>(p.out)[i * p.ld + n] = (O)v;
   }
}

// ---- few rows: operands straight from memory, K split over the wavefronts ----------
//
// A workgroup computes 16 MT rows of a times 16 NT rows of b; its wavefronts take runs of
// 256 bytes in turn, DEPTH of them on their way, and their sums are joined in LDS.  Bound by
// b's bytes, or by the wait for memory where b is small.

constexpr int kRun = 4;                // pieces of 64 bytes, a product each

constexpr int most_waves(int tiles) { return tiles >= 8 ? 4 : 8; }

// the row that a lane reads for a tile of 16: rows beyond the last read the last one
__device__ inline int64_t row_of(int64_t first, int64_t rows)
{
   const int64_t r = first + (threadIdx.x & 15);
   return r < rows ? r : rows - 1;
}

template<class O, int MT, int NT, int DEPTH>
__global__ void __launch_bounds__(64 * most_waves(MT * NT))
i8_rows(I8Params p, int pieces, int waves)
{
   extern __shared__ int join[];
   constexpr int COLS = 16 * NT, ROWS = 16 * MT;
   const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
   const int64_t n0 = (int64_t)blockIdx.x * COLS, m0 = (int64_t)blockIdx.y * ROWS;
   const int8_t* a[MT];
   const int8_t* b[NT];
#pragma unroll
   for(int i = 0; i < MT; i++) a[i] = p.a + row_of(m0 + i * 16, p.m) * pieces * 64 + (lane >> 4) * 16;
#pragma unroll
   for(int j = 0; j < NT; j++) b[j] = p.b + row_of(n0 + j * 16, p.n) * pieces * 64 + (lane >> 4) * 16;
   struct Run { i32x4 c[kRun]; };
   Run x[DEPTH][MT], w[DEPTH][NT];
   // pieces beyond the last are left as they are, and no product takes them
   auto fetch = [&](int d, int64_t first) {
#pragma unroll
      for(int g = 0; g < kRun; g++)
         if(g == 0 || first + g < pieces) {
#pragma unroll
            for(int j = 0; j < NT; j++) w[d][j].c[g] = *reinterpret_cast<const i32x4*>(b[j] + (first + g) * 64);
#pragma unroll
            for(int i = 0; i < MT; i++) x[d][i].c[g] = *reinterpret_cast<const i32x4*>(a[i] + (first + g) * 64);
         }
   };
   i32x4 acc[MT][NT] = {};
   const int step = waves * kRun;
#pragma unroll
   for(int d = 0; d < DEPTH; d++)
      if(wave * kRun + d * step < pieces) fetch(d, wave * kRun + d * step);
#pragma unroll 1
   for(int g0 = wave * kRun; g0 < pieces; g0 += step * DEPTH) {
#pragma unroll
      for(int d = 0; d < DEPTH; d++) {
         const int g = g0 + d * step;
#pragma unroll
         for(int r = 0; r < kRun; r++) {
            if(g + r >= pieces) break;
#pragma unroll
            for(int i = 0; i < MT; i++)
#pragma unroll
               for(int j = 0; j < NT; j++)
                  acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d][j].c[r], x[d][i].c[r], acc[i][j], 0, 0, 0);
         }
         if(g + step * DEPTH < pieces) fetch(d, g + step * DEPTH);
      }
   }
#pragma unroll
   for(int i = 0; i < MT; i++)
#pragma unroll
      for(int j = 0; j < NT; j++)
         *reinterpret_cast<i32x4*>(join + (wave * ROWS + i * 16 + (lane & 15)) * COLS + j * 16 + (lane >> 4) * 4) = acc[i][j];
   __syncthreads();
   O* out = static_cast<O*>(p.out);
   for(int i = threadIdx.x; i < ROWS * COLS; i += waves * 64) {
      const int64_t m = m0 + i / COLS, n = n0 + i % COLS;
      if(m >= p.m) break;
      if(n >= p.n) continue;
      int sum = 0;
      for(int w2 = 0; w2 < waves; w2++) sum += join[w2 * ROWS * COLS + i];
      float v = pieces ? scaled(sum, row_scale(p.a_scales[m]), p.b_scales[n]) : 0.0f;
      if(p.bias) v += p.bias[n];
      out[m * p.ld + n] = (O)v;
   }
}

// ---- many rows: tiles staged in LDS ---------------------------------------------------
//
// A workgroup of WM x WN wavefronts computes BM x BN results, a wavefront FM x FN products
// of 32 x 32.  K goes by slabs of 128 bytes of BM + BN rows.  STAGES slabs are in LDS, one read, the others
// on their way there straight from memory, so that no register waits for them.  The loads
// write lane after lane, 8 rows of 8 chunks of 16 bytes; slot c of row r gets chunk c ^ (r % 8) ^
// (r / 8 % 2), so that the lanes of a product, which read one chunk of 32 rows, meet all banks.
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

// float i of a buffer, 0 beyond its end
__device__ inline float load_float(__amdgpu_buffer_rsrc_t r, int i)
{
   return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, i * 4, 0, 0));
}

// Tile of workgroup `id` of tm x tn.  Workgroups go to the 8 XCDs in turn; each XCD, with
// an L2 of its own, gets a run of tiles, in strips of 4 along m, so that the tiles that an
// XCD works on share rows.
__device__ inline void tile_of(uint32_t id, uint32_t tm, uint32_t tn, uint32_t* m, uint32_t* n)
{
   const uint32_t total = tm * tn, each = total / 8, more = total % 8, xcd = id % 8;
   const uint32_t i = xcd * each + (xcd < more ? xcd : more) + id / 8;
   const uint32_t strip = i / (4 * tn), in = i - strip * 4 * tn;
   const uint32_t high = tm - strip * 4 < 4 ? tm - strip * 4 : 4;
   *m = strip * 4 + in % high;
   *n = in / high;
}

template<class O, int BM, int BN, int WM, int WN, int STAGES>
__global__ void __launch_bounds__(64 * WM * WN)
i8_tiles(I8Params p, uint32_t slabs, uint32_t tm, uint32_t tn)
{
   constexpr int WAVES = WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;
   constexpr int ROWS = BM + BN, SLAB = ROWS * 128;
   constexpr int JOBS = ROWS / 8 / WAVES;                     // fetches of 8 rows a wavefront and slab
   extern __shared__ uint8_t lds[];
   const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
   const int half = lane >> 5;
   uint32_t ti, tj;
   tile_of(blockIdx.x, tm, tn, &ti, &tj);
   const int64_t m0 = (int64_t)ti * BM, n0 = (int64_t)tj * BN;
   const int ml = (int)(p.m - m0 < BM ? p.m - m0 : BM), nl = (int)(p.n - n0 < BN ? p.n - n0 : BN);
   const uint32_t row_bytes = slabs * 128;
   const __amdgpu_buffer_rsrc_t ra = buffer(p.a + m0 * row_bytes, (int64_t)ml * row_bytes);
   const __amdgpu_buffer_rsrc_t rb = buffer(p.b + n0 * row_bytes, (int64_t)nl * row_bytes);

   // job j of this wavefront: rows 8 (wave JOBS + j) .. + 7 of the slab, a's rows first.  Rows
   // beyond the matrix fetch its last one.
   uint32_t voff[JOBS];
#pragma unroll
   for(int j = 0; j < JOBS; j++) {
      const int r8 = wave * JOBS + j, row = r8 * 8 + (lane >> 3);
      const int in = row < BM ? (row < ml ? row : ml - 1) : (row - BM < nl ? row - BM : nl - 1);
      const uint32_t chunk = (lane & 7) ^ (lane >> 3) ^ (r8 & 1);
      voff[j] = (uint32_t)in * row_bytes + chunk * 16;
   }
   // slab s to its place among the STAGES; beyond the last one that again, so that all wavefronts always have the same
   // number of fetches on their way
   auto fetch_slab = [&](uint32_t s) {
      uint8_t* const to = lds + s % STAGES * SLAB + wave * JOBS * 1024;
      const uint32_t from = s < slabs ? s : slabs - 1;
#pragma unroll
      for(int j = 0; j < JOBS; j++) {
         const int row = (wave * JOBS + j) * 8;
         fetch16(row < BM ? ra : rb, to + j * 1024, voff[j], from * 128);
      }
   };
   const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
   uint32_t xat[FM], wat[FN];                                  // LDS offsets of this lane's rows
#pragma unroll
   for(int a = 0; a < FM; a++) xat[a] = wm + a * 32 + (lane & 31);
#pragma unroll
   for(int b = 0; b < FN; b++) wat[b] = BM + wn + b * 32 + (lane & 31);
   const uint32_t turn = (lane & 7) ^ ((lane >> 3) & 1);       // the slot's turn of this lane's rows

   i32x16 acc[FM][FN] = {};
   // Operands of a step of 32 bytes are read while the step before is multiplied, those of a slab's first step under the
   // last one of the slab before: the barrier between slabs, after which one may be read and the other
   // overwritten, stands before that last step's products.
   struct Step {
      i32x4 x[FM], w[FN];
   };
   auto read = [&](Step& to, uint32_t slab, int t) {
      const uint8_t* const data = lds + slab % STAGES * SLAB;
      const uint32_t slot = ((2 * t + half) ^ turn) * 16;
#pragma unroll
      for(int b = 0; b < FN; b++) to.w[b] = *reinterpret_cast<const i32x4*>(data + wat[b] * 128 + slot);
#pragma unroll
      for(int a = 0; a < FM; a++) to.x[a] = *reinterpret_cast<const i32x4*>(data + xat[a] * 128 + slot);
   };
   auto multiply = [&](const Step& f) {
#pragma unroll
      for(int a = 0; a < FM; a++)
#pragma unroll
         for(int b = 0; b < FN; b++) acc[a][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[b], f.x[a], acc[a][b], 0, 0, 0);
   };
   Step even, odd;
   if(slabs) {
#pragma unroll
      for(int i = 0; i < STAGES; i++) fetch_slab(i);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * JOBS) : "memory");
      __syncthreads();
      read(even, 0, 0);
   }
   for(uint32_t s = 0; s < slabs; s++) {
      read(odd, s, 1);
      multiply(even);
      read(even, s, 2);
      multiply(odd);
      read(odd, s, 3);
      multiply(even);
      if(s + 1 < slabs) {
         asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * JOBS) : "memory");
         __syncthreads();
         fetch_slab(s + STAGES);
         read(even, s + 1, 0);
      }
      multiply(odd);
   }
   asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // nothing is on its way to the LDS that the results take
   // scales and bias beyond the matrix, or not given, are zeros
   const __amdgpu_buffer_rsrc_t rsa = buffer(p.a_scales + m0, slabs ? ml * 4 : 0);
   const __amdgpu_buffer_rsrc_t rsb = buffer(p.b_scales + n0, slabs ? nl * 4 : 0);
   const __amdgpu_buffer_rsrc_t rbias = buffer(p.bias + n0, p.bias ? nl * 4 : 0);
   // Each wavefront turns its results in its share of the LDS and stores whole 16-byte pieces of
   // rows.
   constexpr int COLS = FN * 32, PITCH = COLS * (int)sizeof(O) + 16, SHARE = STAGES * SLAB / WAVES;
   constexpr int ROOM = SHARE / (32 * PITCH);
   constexpr int PASS = ROOM >= FM ? FM : ROOM >= 2 && FM % 2 == 0 ? 2 : 1;       // 32-row parts at a time
   static_assert(ROOM > 0 && FM % PASS == 0, "a wavefront's share of the LDS holds whole parts");
   constexpr int PIECE = 16 / (int)sizeof(O), ACROSS = COLS / PIECE, DOWN = 64 / ACROSS;
   struct __attribute__((packed, aligned(sizeof(O)))) Piece { O e[PIECE]; };
   __syncthreads();
   uint8_t* const mine = lds + wave * SHARE;
   O* out = static_cast<O*>(p.out) + m0 * p.ld + n0;
#pragma unroll
   for(int a0 = 0; a0 < FM; a0 += PASS) {
      RowScale sa[PASS];
#pragma unroll
      for(int a = 0; a < PASS; a++) sa[a] = row_scale(load_float(rsa, wm + (a0 + a) * 32 + (lane & 31)));
#pragma unroll
      for(int b = 0; b < FN; b++)
#pragma unroll
         for(int q = 0; q < 4; q++) {
            const int j = b * 32 + q * 8 + half * 4;
            float sb[4], bias[4];
#pragma unroll
            for(int i = 0; i < 4; i++) {
               sb[i] = load_float(rsb, wn + j + i);
               bias[i] = load_float(rbias, wn + j + i);
            }
#pragma unroll
            for(int a = a0; a < a0 + PASS; a++) {
               struct alignas(4 * sizeof(O)) Four { O e[4]; } v;
#pragma unroll
               for(int i = 0; i < 4; i++) v.e[i] = (O)(scaled(acc[a][b][q * 4 + i], sa[a - a0], sb[i]) + bias[i]);
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

template<class O, int BM, int BN, int WM, int WN, int STAGES>
hipError_t tiles_shape(const I8Params& p, hipStream_t s)
{
   constexpr size_t bytes = (size_t)(BM + BN) * 128 * STAGES;
   const int64_t slabs = padded(p.k) / 128, tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
   if(!grid_ok(tm * tn, 64 * WM * WN)) return kTooLarge;
   static std::atomic<uint64_t> mask{0};
   const hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(&i8_tiles<O, BM, BN, WM, WN, STAGES>), bytes, mask);
   if(e != hipSuccess) return e;
   i8_tiles<O, BM, BN, WM, WN, STAGES><<<(unsigned)(tm * tn), 64 * WM * WN, bytes, s>>>(p, (uint32_t)slabs, (uint32_t)tm,
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
hipError_t rows_shape(const I8Params& p, hipStream_t s)
{
   const int64_t pieces = padded(p.k) / 64;
   const int waves = wavefronts((pieces + kRun - 1) / kRun, most_waves(MT * NT));
   const int64_t gx = (p.n + 16 * NT - 1) / (16 * NT), gy = (p.m + 16 * MT - 1) / (16 * MT);
   if(!grid_ok(gx, waves * 64) || gy > 65535) return kTooLarge;
   i8_rows<O, MT, NT, DEPTH><<<dim3((unsigned)gx, (unsigned)gy), waves * 64, (size_t)waves * MT * NT * 1024, s>>>(
      p, (int)pieces, waves);
   return hipGetLastError();
}

template<class O, int M>
hipError_t tokens_shape(const I8Params& p, hipStream_t s)
{
   // K shared until there are 16 wavefronts a CU or each has its last KiB
   const int64_t row_bytes = padded(p.k), groups = (p.n + kTokenRows - 1) / kTokenRows;
   constexpr int UNROLL = M <= 4 ? 2 : 1;
   int waves = 1;
   while(waves < 8 && waves * 1024 * UNROLL < row_bytes && groups * waves < 16 * 256) waves *= 2;
   if(!grid_ok(groups, waves * 64)) return kTooLarge;
   i8_tokens<O, M, UNROLL><<<(unsigned)groups, waves * 64, 0, s>>>(p, row_bytes);
   return hipGetLastError();
}

int64_t tiles(const I8Params& p, int64_t rows, int64_t cols)
{
   return ((p.m + rows - 1) / rows) * ((p.n + cols - 1) / cols);
}

// The kernel for a size, on MI355X's 256 CUs; us at m x n x k.
//   Up to 8 rows: four-byte products, 1 KiB of a row of b a load (16 rows on the matrix cores / so: 1 x 8192 x 8192
//     18.8 / 11.6, 1 x 16384 x 8192 37.4 / 23.6, 8 x 16384 x 8192 37 / 29, 8 x 8192 x 8192 20.4 / 17.7).
//   K split over wavefronts, operands straight from memory, where at most 256 workgroups of 16 or 32 rows by 16
//     columns have all results and K is long, and up to 16 rows by 8192 columns (against 64 x 64 staged: 24 x 4096 x
//     4096 8.4 / 10.7, 100 x 100 x 1024 3.8 / 5.2; 16 rows by 4608, 6144, 8192 columns x K: 2048 5.7, 5.9, 6.1 / 6.7, 6.6, 6.6,
//     4096 8.6, 8.9, 10.1 / 10.0, 10.1, 10.2, 16384 29.8, 31.4, 35.8 / 33.8, 35.1, 38.1, 8192 14.5, 16.7, 20.9 / 16.8, 16.9, 18.5,
//     that last one the only size of them that loses; but 16 x 16384 x 8192 37.2 / 24.9).
//   Staged tiles: 256 x 256, one a CU, against 128 x 128, two a CU, by the rounds that each needs; 64 x 64, four slabs
//     on their way, below 256 tiles of 128 x 128 (128 x 4096 x 4096 10.9 / 21.8, 1001 x 2000 x 1504 9.7 / 12.7; with two
//     slabs 128 x 4096 x 4096 16.8, 64 x 16384 x 8192 48.6 / 27.1).
template<class O>
hipError_t matmul_typed(const I8Params& p, hipStream_t s)
{
   if(p.m <= 1) return tokens_shape<O, 1>(p, s);
   if(p.m <= 2) return tokens_shape<O, 2>(p, s);
   if(p.m <= 4) return tokens_shape<O, 4>(p, s);
   if(p.m <= 8) return tokens_shape<O, 8>(p, s);
   if(p.m <= 16 && p.n <= 16 * 512) return p.n > 16 * 256 ? rows_shape<O, 1, 2, 2>(p, s) : rows_shape<O, 1, 1, 2>(p, s);
   if(p.k >= 1024) {
      if(tiles(p, 16, 16) <= 256) return rows_shape<O, 1, 1, 2>(p, s);
      if(tiles(p, 32, 16) <= 256) return rows_shape<O, 2, 1, 2>(p, s);
   }
   const int64_t big = tiles(p, 256, 256), mid = tiles(p, 128, 128);
   if(5 * ((big + 255) / 256) <= 3 * ((mid + 511) / 512)) return tiles_shape<O, 256, 256, 2, 4, 2>(p, s);
   if(mid >= 256) return tiles_shape<O, 128, 128, 2, 2, 2>(p, s);
   return tiles_shape<O, 64, 64, 2, 2, 4>(p, s);
}

}  // namespace

hipError_t launch_i8_matmul(const I8Params& p, hipStream_t s)
{
   switch(p.type) {
      case T_F32:  return matmul_typed<float>(p, s);
      case T_BF16: return matmul_typed<bf16>(p, s);
      default:     return matmul_typed<f16>(p, s);
   }
}

}  // namespace layer
}  // namespace fufft
