// A paged cache of signals in microscaled 4-bit blocks: reading it back, as token
// rows or as the channel signals the convolutions take, and the convolution's
// single-token form, which reads it in place.  (Writing it is quantize_rows with
// slots, mx4.hip.)
#include "mx4_device.hpp"
#include "mx4_internal.hpp"

#include <type_traits>

namespace fufft {
namespace mx4 {

namespace {

constexpr int kLanes = 256;

// Row of codes and scales that holds token t of a sequence, or -1 where its page
// is none of the cache's.
__device__ inline int64_t cache_row(const CacheParams& c, const int32_t* table, int64_t t)
{
   const int64_t pg = table[t >> c.page_log];
   const int64_t off = t & (((int64_t)1 << c.page_log) - 1);
   return pg >= 0 && pg < c.pages ? (pg << c.page_log) + off : -1;
}

// tokens of sequence b: its length within what the page table can hold
__device__ inline int64_t sequence_length(const CacheParams& c, int64_t b)
{
   const int64_t n = c.lens[b], most = c.width << c.page_log;
   return n < 0 ? 0 : n < most ? n : most;
}

// out[b][t][channel], zeros from each sequence's length on: 8 channels a lane, the tokens of
// this launch from `first` on.
template<class T, int ROWS>
__global__ void __launch_bounds__(kLanes)
read_tokens(CacheParams c, T* out, int64_t first, int64_t length, int64_t cp, int lr)
{
   const int lane = threadIdx.x & ((1 << lr) - 1);
   const int64_t col = ((int64_t)blockIdx.x << (lr + 3)) + lane * 8;
   if(col >= c.channels) return;
   const int per = kLanes >> lr;
   const int64_t t0 = first + (int64_t)blockIdx.y * (per * ROWS) + (threadIdx.x >> lr);
   for(int64_t b = blockIdx.z; b < c.batch; b += gridDim.z) {
      const int64_t n = sequence_length(c, b);
      const int32_t* table = c.table + b * c.width;
      int64_t from[ROWS];
      uint32_t q[ROWS], s[ROWS];
#pragma unroll
      for(int u = 0; u < ROWS; u++) {
         const int64_t t = t0 + u * per;
         from[u] = t < n && t < length ? cache_row(c, table, t) : -1;
      }
#pragma unroll
      for(int u = 0; u < ROWS; u++) {
         q[u] = s[u] = 0;
         if(from[u] >= 0) {
            q[u] = *reinterpret_cast<const uint32_t*>(c.codes + from[u] * (cp / 2) + col / 2);
            s[u] = c.scales[from[u] * (cp / kBlock) + col / kBlock];
         }
      }
#pragma unroll
      for(int u = 0; u < ROWS; u++) {
         const int64_t t = t0 + u * per;
         if(t >= length) break;
         float v[8];
         decode8(q[u], s[u], v);
         T* o = out + (b * length + t) * c.channels + col;
         if(col + 8 <= c.channels) {
            store8(o, v);
         } else {
#pragma unroll
            for(int i = 0; i < 8; i++)
               if(col + i < c.channels) o[i] = (T)v[i];
         }
      }
   }
}

// out[b][channel][t], zeros from each sequence's length on, from token `first` on: tiles of 64 tokens
// x 128 channels turned in LDS, so that codes are read along channels and signals
// written along tokens.  4 x 8192 tokens x 2048 channels in fp32: 63 to 72 us, 268 MB written at
// 3.7 to 4.3 TB/s.
template<class T>
__global__ void __launch_bounds__(kLanes)
read_channels(CacheParams c, T* out, int64_t first, int64_t length, int64_t cp)
{
   __shared__ float tile[128 * 65];
   const int64_t c0 = (int64_t)blockIdx.x * 128, t0 = first + (int64_t)blockIdx.y * 64;
   const int lane = threadIdx.x & 15;
   for(int64_t b = blockIdx.z; b < c.batch; b += gridDim.z) {
      const int64_t n = sequence_length(c, b);
      const int32_t* table = c.table + b * c.width;
      uint32_t q[4], s[4];
#pragma unroll
      for(int u = 0; u < 4; u++) {
         const int64_t t = t0 + u * 16 + (threadIdx.x >> 4);
         const int64_t from = t < n ? cache_row(c, table, t) : -1;
         q[u] = s[u] = 0;
         if(from >= 0) {
            q[u] = *reinterpret_cast<const uint32_t*>(c.codes + from * (cp / 2) + c0 / 2 + lane * 4);
            s[u] = c.scales[from * (cp / kBlock) + c0 / kBlock + lane / 4];
         }
      }
#pragma unroll
      for(int u = 0; u < 4; u++) {
         float v[8];
         decode8(q[u], s[u], v);
#pragma unroll
         for(int i = 0; i < 8; i++) tile[(lane * 8 + i) * 65 + u * 16 + (threadIdx.x >> 4)] = v[i];
      }
      __syncthreads();
      const int64_t t = t0 + (threadIdx.x & 63);
      if(t < length) {
#pragma unroll 8
         for(int i = 0; i < 32; i++) {
            const int ch = i * 4 + (threadIdx.x >> 6);
            if(c0 + ch < c.channels)
               out[(b * c.channels + c0 + ch) * length + t] = (T)tile[ch * 65 + (threadIdx.x & 63)];
         }
      }
      __syncthreads();
   }
}

// out[b][channel] = sum over j < min(len_b, taps) of taps[j][channel] times the
// value of token len_b - 1 - j.  The bytes bound it: 17/32 a token and channel, and the taps,
// which weigh most where few sequences share them.
//
// A wavefront has one token at a time of each of SEQS sequences, CH channels a lane, so that
// pages and rows are scalar work, and reads TAPS taps and their tokens of every
// sequence before it uses them.  A workgroup covers one slice of 64 CH channels and
// one split, taps [split * chunk, ...), its wavefronts taking TAPS taps in turn; their sums are
// joined in LDS, those of the splits by join_splits, both in a fixed order.  The
// workgroups of all sequence groups that read the same taps follow each other on one XCD, whose
// L2 then has them.
template<int CH> struct Codes;
template<> struct Codes<8> { typedef uint32_t type; };
template<> struct Codes<4> { typedef uint16_t type; };

template<int CH>
__device__ inline void decode(uint32_t c, uint32_t s, float (&v)[CH])
{
   const float p = scale_operand(s);
   const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, p, 0);
   const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, p, 1);
   v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
   if constexpr(CH == 8) {
      const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, p, 2);
      const f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, p, 3);
      v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
   }
}

// a row's CH taps without the first `drop` of them, which are another lane's
template<class T, int CH>
__device__ inline void drop_first(T (&e)[CH], int drop)
{
#pragma unroll
   for(int by = CH / 2; by > 0; by /= 2) {
      const bool go = (drop & by) != 0;
#pragma unroll
      for(int i = 0; i < CH; i++) e[i] = go ? (i + by < CH ? e[i + by] : (T)0.0f) : e[i];
   }
}

template<class T, int CH, int SEQS, int TAPS, int WAVES, bool FEW>
__global__ void __launch_bounds__(64 * WAVES)
cache_conv(CacheParams c, const T* taps, uint32_t tap_count, uint32_t chunk, uint32_t cp, uint32_t slices, uint32_t parts,
           uint32_t seq_groups, float* sums)
{
   typedef typename Codes<CH>::type Code;
   struct __attribute__((packed, aligned(sizeof(T)))) Taps { T e[CH]; };
   __shared__ float join[WAVES * 64 * CH];
   const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
   // ids 8 apart run on one XCD: part 8 i + (id % 8) for every group of sequences, then the next i
   const uint32_t set = blockIdx.x / (8 * seq_groups), in = blockIdx.x % (8 * seq_groups);
   const uint32_t part = set * 8 + in % 8;
   if(part >= parts) return;
   const uint32_t split = part / slices, col = part % slices * (64 * CH) + lane * CH;
   const int64_t b0 = (int64_t)(in / 8) * SEQS;
   // tokens and taps count in 32 bits, as lengths do.  Sequence g takes part in taps j < end[g].
   uint32_t n[SEQS], end[SEQS], j_end = 0;
   const uint32_t chunk_end = (split + 1) * chunk < tap_count ? (split + 1) * chunk : tap_count;
#pragma unroll
   for(int g = 0; g < SEQS; g++) {
      n[g] = b0 + g < c.batch && c.pages > 0 ? (uint32_t)sequence_length(c, b0 + g) : 0;
      end[g] = n[g] < chunk_end ? n[g] : chunk_end;
      j_end = end[g] > j_end ? end[g] : j_end;
   }
   const uint32_t pages = c.pages < 0x7fffffff ? (uint32_t)c.pages : 0x7fffffffu, page_mask = (1u << c.page_log) - 1;
   float acc[SEQS][CH] = {};
   // Every load of a step has an address that is good, so that all go out before the first
   // is used: taps past the end are the last one, channels past the end the last ones,
   // a token that is none is row 0 (n > 0 somewhere, so there is a page and a table).
   // A lane that the last channel cuts reads the row's last CH taps and drops the first; a
   // kernel for fewer channels than that (FEW) reads them one by one.  Each is code of its own: a
   // branch at each load would end in a wait for it (51 x 4144 x 2044, fp32 taps: 250 us, 85 so).
   auto steps = [&](auto cut) {
      constexpr bool CUT = decltype(cut)::value;
      const uint32_t channels = (uint32_t)c.channels, at = CUT && col + CH > channels ? channels - CH : col;
      const int drop = CUT && col < channels ? (int)(col - at) : 0;
      const uint32_t code_at = (col < cp ? col : 0) / 2, scale_at = (col < cp ? col : 0) / kBlock;
      for(uint32_t j0 = split * chunk + wave * TAPS; j0 < j_end; j0 += WAVES * TAPS) {
         Taps h[TAPS];
#pragma unroll
         for(int u = 0; u < TAPS; u++) {
            const T* row = taps + (int64_t)(j0 + u < j_end ? j0 + u : j_end - 1) * c.channels;
            if constexpr(FEW) {
#pragma unroll
               for(int i = 0; i < CH; i++) h[u].e[i] = row[col + i < channels ? col + i : channels - 1];
            } else {
               h[u] = *reinterpret_cast<const Taps*>(row + at);
            }
         }
         uint32_t q[SEQS][TAPS], s[SEQS][TAPS];
         bool there[SEQS][TAPS];
#pragma unroll
         for(int g = 0; g < SEQS; g++) {
            const int32_t* table = c.table + (b0 + g < c.batch ? b0 + g : c.batch - 1) * c.width;
#pragma unroll
            for(int u = 0; u < TAPS; u++) {
               const int32_t left = (int32_t)(n[g] - 1 - j0 - u);
               const uint32_t t = left > 0 ? left : 0, pg = (uint32_t)table[t >> c.page_log];
               there[g][u] = j0 + u < end[g] && pg < pages;
               const uint64_t row = ((uint64_t)(pg < pages ? pg : 0) << c.page_log) + (t & page_mask);
               const uint64_t from = row * (cp / 2);
               q[g][u] = *reinterpret_cast<const Code*>(c.codes + from + code_at);
               s[g][u] = (c.scales + (from >> 4))[scale_at];
            }
         }
         if constexpr(CUT) {
#pragma unroll
            for(int u = 0; u < TAPS; u++) drop_first<T, CH>(h[u].e, drop);
         }
#pragma unroll
         for(int g = 0; g < SEQS; g++)
#pragma unroll
            for(int u = 0; u < TAPS; u++) {
               if(!there[g][u]) continue;       // a tap that meets no token may be anything
               float v[CH];
               decode<CH>(q[g][u], s[g][u], v);
#pragma unroll
               for(int i = 0; i < CH; i++) acc[g][i] = fmaf(to_float(h[u].e[i]), v[i], acc[g][i]);
            }
      }
   };
   if(FEW || col - lane * CH + 64 * CH <= c.channels) steps(std::false_type());
   else if constexpr(!FEW)                            steps(std::true_type());
#pragma unroll
   for(int g = 0; g < SEQS; g++) {
      if(b0 + g >= c.batch) break;
      if(g) __syncthreads();
#pragma unroll
      for(int i = 0; i < CH; i++) join[(wave * CH + i) * 64 + lane] = acc[g][i];
      __syncthreads();
      float* to = sums + ((int64_t)split * c.batch + b0 + g) * c.channels;
      for(int k = threadIdx.x; k < 64 * CH; k += 64 * WAVES) {
         const int64_t ch = (int64_t)(col - lane * CH) + k;
         float a = 0.0f;
#pragma unroll
         for(int w = 0; w < WAVES; w++) a += join[(w * CH + k % CH) * 64 + k / CH];
         if(ch < c.channels) to[ch] = a;
      }
   }
}

// The splits' sums, 8 lanes a result, each taking every eighth.
template<class T>
__global__ void __launch_bounds__(kLanes)
join_splits(const float* sums, T* out, int64_t count, int splits)
{
   __shared__ float part[8][32];
   const int lane = threadIdx.x & 31, k0 = threadIdx.x >> 5;
   const int64_t i = (int64_t)blockIdx.x * 32 + lane;
   float a = 0.0f;
   if(i < count) {
#pragma unroll 8
      for(int k = k0; k < splits; k += 8) a += sums[k * count + i];
   }
   part[k0][lane] = a;
   __syncthreads();
   if(k0 == 0 && i < count) {
#pragma unroll
      for(int k = 1; k < 8; k++) a += part[k][lane];
      out[i] = (T)a;
   }
}

// A launch for every 65535 tiles of tokens, a grid's end in y: beyond them a text is long enough that
// a launch more costs nothing (a loop in the kernel costs the others: 4 x 8192 x 2048 to bf16 rows 34 -> 35 us).
template<class T>
hipError_t read_typed(const CacheParams& c, T* out, int64_t length, bool channels_first, hipStream_t s)
{
   constexpr int ROWS = 4;
   const int64_t cp = padded(c.channels);
   const unsigned gz = (unsigned)(c.batch < 65535 ? c.batch : 65535);
   int lr = 4;
   while(lr < 8 && ((int64_t)8 << lr) < cp) lr++;
   const int64_t per = channels_first ? 64 : (kLanes >> lr) * ROWS;
   const int64_t gx = channels_first ? cp / 128 : (cp / 8 + (1 << lr) - 1) >> lr;
   if(!grid_ok(gx, kLanes)) return kTooLarge;
   for(int64_t first = 0; first < length; first += 65535 * per) {
      const int64_t tiles = (length - first + per - 1) / per;
      const dim3 g((unsigned)gx, (unsigned)(tiles < 65535 ? tiles : 65535), gz);
      if(channels_first) read_channels<T><<<g, kLanes, 0, s>>>(c, out, first, length, cp);
      else               read_tokens<T, ROWS><<<g, kLanes, 0, s>>>(c, out, first, length, cp, lr);
      const hipError_t e = hipGetLastError();
      if(e != hipSuccess) return e;
   }
   return hipSuccess;
}

template<class T, int CH, int SEQS, int TAPS, int WAVES, bool FEW = false>
hipError_t conv_shape(const CacheParams& c, const T* taps, int64_t tap_count, float* direct, float* work,
                      int64_t splits, int* used, hipStream_t s)
{
   const int64_t cp = padded(c.channels), slices = (cp + 64 * CH - 1) / (64 * CH);
   if(cp > 0x7fffffff) return kTooLarge;
   const int64_t seq_groups = (c.batch + SEQS - 1) / SEQS, step = WAVES * TAPS;
   // two workgroups a CU, each with one step at least
   int64_t want = (512 + slices * seq_groups - 1) / (slices * seq_groups);
   const int64_t most = (tap_count + step - 1) / step;
   want = want < most ? want : most;
   want = want < splits ? want : splits;
   if(want < 1) want = 1;
   int64_t chunk = ((tap_count + want - 1) / want + step - 1) / step * step;
   if(chunk < step) chunk = step;
   const int64_t parts = slices * (tap_count > 0 ? (tap_count + chunk - 1) / chunk : 1);
   const int64_t sets = (parts + 7) / 8 * 8, most_groups = kMostLanes / (64 * WAVES) / sets;
   if(most_groups < 1 || parts / slices > 0x7fffffff) return kTooLarge;
   const int count = (int)(parts / slices);
   float* sums = count == 1 && direct ? direct : work;
   // one launch, but for so many sequences that its lanes would pass 32 bits: these have one split, so
   // the sums of each launch's sequences lie together
   for(int64_t first = 0; first < seq_groups; first += most_groups) {
      const int64_t groups = seq_groups - first < most_groups ? seq_groups - first : most_groups, b0 = first * SEQS;
      CacheParams q = c;
      q.table += b0 * c.width;
      q.lens += b0;
      if(groups < seq_groups) q.batch = c.batch - b0 < groups * SEQS ? c.batch - b0 : groups * SEQS;
      cache_conv<T, CH, SEQS, TAPS, WAVES, FEW><<<(unsigned)(sets * groups), 64 * WAVES, 0, s>>>(
         q, taps, (uint32_t)tap_count, (uint32_t)chunk, (uint32_t)cp, (uint32_t)slices, (uint32_t)parts, (uint32_t)groups,
         sums + b0 * c.channels);
      const hipError_t e = hipGetLastError();
      if(e != hipSuccess) return e;
   }
   *used = sums == direct ? 0 : count;
   return hipSuccess;
}

template<class T>
hipError_t conv_typed(const CacheParams& c, const T* taps, int64_t tap_count, float* direct, float* work,
                      int64_t splits, int* used, hipStream_t s)
{
   // Few sequences, or few channels: the wait for memory and the taps' bytes are the work, and
   // many wavefronts of one sequence, 4 channels a lane, serve them best (1 x 65536 x 1024, bf16
   // taps: 32 us, 5.3 TB/s; one sequence a group / two or four: 3 x 38104 x 62 20 / 38 us, 7 x 9546
   // x 46 12 / 21, 3 x 30000 x 768 28 / 45, but 8 x 4000 x 1000 23 / 19, 40 x 2000 x 100 21 / 15).
   // More: what scalar work a token costs counts, so 8 channels, and registers for four
   // sequences with 2 taps (24 x 8000 x 4096, fp32 taps: 4 x 2 taps 126 us, 4 x 4 148, 2 x 4 170;
   // 2 x 4000 x 4096 two at a time 21, one 22.5).
   // Fewer channels than a lane may hold have a kernel of their own, as a third loop in each
   // kernel would spill scalars.
   if(c.channels < 8) return conv_shape<T, 4, 1, 8, 16, true>(c, taps, tap_count, direct, work, splits, used, s);
   const int64_t lanes = c.batch * ((padded(c.channels) + 255) / 256);
   if(c.batch == 1 || lanes <= 16) return conv_shape<T, 4, 1, 8, 16>(c, taps, tap_count, direct, work, splits, used, s);
   if(c.batch <= 3) return conv_shape<T, 8, 2, 4, 8>(c, taps, tap_count, direct, work, splits, used, s);
   return conv_shape<T, 8, 4, 2, 8>(c, taps, tap_count, direct, work, splits, used, s);
}

template<class T>
hipError_t join_typed(const float* sums, T* out, int64_t count, int splits, hipStream_t s)
{
   // one launch, but for so many results that its lanes would pass 32 bits: these have one split
   constexpr int64_t most = kMostLanes / kLanes * 32;
   for(int64_t first = 0; first < count; first += most) {
      const int64_t n = count - first < most ? count - first : most;
      join_splits<T><<<(unsigned)((n + 31) / 32), kLanes, 0, s>>>(sums + first, out + first, n, splits);
      const hipError_t e = hipGetLastError();
      if(e != hipSuccess) return e;
   }
   return hipSuccess;
}

}  // namespace

hipError_t launch_cache_read(const CacheParams& c, void* out, int type, int64_t length, bool channels_first,
                             hipStream_t s)
{
   if(c.batch <= 0 || c.channels <= 0 || length <= 0) return hipSuccess;
   switch(type) {
      case T_F32:  return read_typed(c, static_cast<float*>(out), length, channels_first, s);
      case T_BF16: return read_typed(c, static_cast<bf16*>(out), length, channels_first, s);
      default:     return read_typed(c, static_cast<f16*>(out), length, channels_first, s);
   }
}

hipError_t launch_cache_conv(const CacheParams& c, const void* taps, int tap_type, int64_t tap_count, void* out,
                             int out_type, float* work, int64_t splits, hipStream_t s)
{
   if(c.batch <= 0 || c.channels <= 0) return hipSuccess;
   // no token is beyond the page table, nor beyond a 32-bit length
   int64_t most = c.width << c.page_log;
   if(most > 0x7fffffff) most = 0x7fffffff;
   if(tap_count > most) tap_count = most;
   // fp32 results that one workgroup sums need no workspace and no join
   float* direct = out_type == T_F32 ? static_cast<float*>(out) : nullptr;
   int used = 0;
   hipError_t e;
   switch(tap_type) {
      case T_F32:  e = conv_typed(c, static_cast<const float*>(taps), tap_count, direct, work, splits, &used, s); break;
      case T_BF16: e = conv_typed(c, static_cast<const bf16*>(taps), tap_count, direct, work, splits, &used, s); break;
      default:     e = conv_typed(c, static_cast<const f16*>(taps), tap_count, direct, work, splits, &used, s); break;
   }
   if(e != hipSuccess || used == 0) return e;
   switch(out_type) {
      case T_F32:  return join_typed(work, static_cast<float*>(out), c.batch * c.channels, used, s);
      case T_BF16: return join_typed(work, static_cast<bf16*>(out), c.batch * c.channels, used, s);
      default:     return join_typed(work, static_cast<f16*>(out), c.batch * c.channels, used, s);
   }
}

}  // namespace mx4
}  // namespace fufft
