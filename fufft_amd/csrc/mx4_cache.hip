// A paged cache of signals in microscaled 4-bit blocks: reading it back, as token
// rows or as the channel signals the convolutions take, and the convolution's
// single-token form, which reads it in place.  (Writing it is quantize_rows with
// slots, mx4.hip.)
#include "mx4_device.hpp"
#include "mx4_internal.hpp"

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

// out[b][t][channel], zeros from each sequence's length on: 8 channels a lane.
template<class T, int ROWS>
__global__ void __launch_bounds__(kLanes)
read_tokens(CacheParams c, T* out, int64_t length, int64_t cp, int lr)
{
   const int lane = threadIdx.x & ((1 << lr) - 1);
   const int64_t col = ((int64_t)blockIdx.x << (lr + 3)) + lane * 8;
   if(col >= c.channels) return;
   const int per = kLanes >> lr;
   const int64_t t0 = (int64_t)blockIdx.y * (per * ROWS) + (threadIdx.x >> lr);
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

// out[b][channel][t], zeros from each sequence's length on: tiles of 64 tokens x
// 128 channels turned in LDS, so that codes are read along channels and signals
// written along tokens.
template<class T>
__global__ void __launch_bounds__(kLanes)
read_channels(CacheParams c, T* out, int64_t length, int64_t cp)
{
   __shared__ float tile[128 * 65];
   const int64_t c0 = (int64_t)blockIdx.x * 128, t0 = (int64_t)blockIdx.y * 64;
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
// value of token len_b - 1 - j.  8 channels a lane; a workgroup has L = 1 << lr
// lanes to a token and 256 / L runs of TAPS taps at a time, for SEQS sequences
// that share the taps it holds.  It covers taps [y * chunk, (y + 1) * chunk); the
// sums of its runs are joined in LDS, those of the chunks by join_splits, both in
// a fixed order.
template<class T, int SEQS, int TAPS>
__global__ void __launch_bounds__(kLanes)
cache_conv(CacheParams c, const T* taps, int64_t tap_count, int64_t chunk, int64_t cp, int lr, float* sums)
{
   __shared__ float join[kLanes * 8];
   const int lane = threadIdx.x & ((1 << lr) - 1), run = threadIdx.x >> lr, runs = kLanes >> lr;
   const int64_t col = ((int64_t)blockIdx.x << (lr + 3)) + lane * 8;
   const int64_t b0 = (int64_t)blockIdx.z * SEQS;
   const int64_t j_begin = (int64_t)blockIdx.y * chunk;
   int64_t n[SEQS], most = 0;
#pragma unroll
   for(int g = 0; g < SEQS; g++) {
      n[g] = b0 + g < c.batch ? sequence_length(c, b0 + g) : 0;
      most = n[g] > most ? n[g] : most;
   }
   int64_t j_end = j_begin + chunk;
   if(j_end > tap_count) j_end = tap_count;
   if(j_end > most) j_end = most;
   float acc[SEQS][8] = {};
   if(col < c.channels) {
      for(int64_t j0 = j_begin + run * TAPS; j0 < j_end; j0 += (int64_t)runs * TAPS) {
         float h[TAPS][8];
#pragma unroll
         for(int u = 0; u < TAPS; u++) {
#pragma unroll
            for(int i = 0; i < 8; i++) h[u][i] = 0.0f;
            if(j0 + u < j_end) {
               const T* at = taps + (j0 + u) * c.channels + col;
               if(col + 8 <= c.channels) {
                  load8(at, h[u]);
               } else {
#pragma unroll
                  for(int i = 0; i < 8; i++)
                     if(col + i < c.channels) h[u][i] = to_float(at[i]);
               }
            }
         }
#pragma unroll
         for(int g = 0; g < SEQS; g++) {
            if(j0 >= n[g]) continue;
            const int32_t* table = c.table + (b0 + g) * c.width;
            uint32_t q[TAPS], s[TAPS];
            bool there[TAPS];
#pragma unroll
            for(int u = 0; u < TAPS; u++) {
               const int64_t t = n[g] - 1 - j0 - u;
               const int64_t from = t >= 0 && j0 + u < j_end ? cache_row(c, table, t) : -1;
               there[u] = from >= 0;
               q[u] = s[u] = 0;
               if(there[u]) {
                  q[u] = *reinterpret_cast<const uint32_t*>(c.codes + from * (cp / 2) + col / 2);
                  s[u] = c.scales[from * (cp / kBlock) + col / kBlock];
               }
            }
#pragma unroll
            for(int u = 0; u < TAPS; u++) {
               if(!there[u]) continue;       // a tap that meets no token may be anything
               float v[8];
               decode8(q[u], s[u], v);
#pragma unroll
               for(int i = 0; i < 8; i++) acc[g][i] = fmaf(h[u][i], v[i], acc[g][i]);
            }
         }
      }
   }
#pragma unroll
   for(int g = 0; g < SEQS; g++) {
      if(b0 + g >= c.batch) break;
      if(g) __syncthreads();
#pragma unroll
      for(int i = 0; i < 8; i++) join[i * kLanes + threadIdx.x] = acc[g][i];
      __syncthreads();
      float* to = sums + ((int64_t)blockIdx.y * c.batch + b0 + g) * c.channels;
      for(int k = threadIdx.x; k < 8 << lr; k += kLanes) {
         const int64_t ch = ((int64_t)blockIdx.x << (lr + 3)) + k;
         float a = 0.0f;
         for(int r = 0; r < runs; r++) a += join[(k & 7) * kLanes + (r << lr) + (k >> 3)];
         if(ch < c.channels) to[ch] = a;
      }
   }
}

template<class T>
__global__ void __launch_bounds__(kLanes)
join_splits(const float* sums, T* out, int64_t count, int64_t splits)
{
   const int64_t i = (int64_t)blockIdx.x * kLanes + threadIdx.x;
   if(i >= count) return;
   float a = 0.0f;
   for(int64_t k = 0; k < splits; k++) a += sums[k * count + i];
   out[i] = (T)a;
}

template<class T>
hipError_t read_typed(const CacheParams& c, T* out, int64_t length, bool channels_first, hipStream_t s)
{
   const int64_t cp = padded(c.channels);
   const unsigned gz = (unsigned)(c.batch < 65535 ? c.batch : 65535);
   if(channels_first) {
      const int64_t gy = (length + 63) / 64;
      if(gy > 65535 || cp / 128 > 0x7fffffff) return hipErrorInvalidValue;
      read_channels<T><<<dim3((unsigned)(cp / 128), (unsigned)gy, gz), kLanes, 0, s>>>(c, out, length, cp);
   } else {
      constexpr int ROWS = 4;
      int lr = 4;
      while(lr < 8 && ((int64_t)8 << lr) < cp) lr++;
      const int64_t per = (kLanes >> lr) * ROWS, gy = (length + per - 1) / per;
      const int64_t gx = (cp / 8 + (1 << lr) - 1) >> lr;
      if(gy > 65535 || gx > 0x7fffffff) return hipErrorInvalidValue;
      read_tokens<T, ROWS><<<dim3((unsigned)gx, (unsigned)gy, gz), kLanes, 0, s>>>(c, out, length, cp, lr);
   }
   return hipGetLastError();
}

template<class T, int SEQS, int TAPS>
hipError_t conv_shape(const CacheParams& c, const T* taps, int64_t tap_count, float* direct, float* work,
                      int64_t splits, int64_t* used, hipStream_t s)
{
   const int64_t cp = padded(c.channels);
   int lr = 4;
   while(lr < 6 && ((int64_t)8 << lr) < cp) lr++;
   const int64_t gx = (cp / 8 + (1 << lr) - 1) >> lr, gz = (c.batch + SEQS - 1) / SEQS;
   const int64_t step = (int64_t)(kLanes >> lr) * TAPS;
   int64_t want = (2048 + gx * gz - 1) / (gx * gz);
   const int64_t most = (tap_count + step - 1) / step;
   want = want < most ? want : most;
   want = want < splits ? want : splits;
   if(want < 1) want = 1;
   int64_t chunk = ((tap_count + want - 1) / want + step - 1) / step * step;
   if(chunk < step) chunk = step;
   const int64_t gy = tap_count > 0 ? (tap_count + chunk - 1) / chunk : 1;
   if(gx > 0x7fffffff || gy > 65535 || gz > 65535) return hipErrorInvalidValue;
   float* sums = gy == 1 && direct ? direct : work;
   cache_conv<T, SEQS, TAPS><<<dim3((unsigned)gx, (unsigned)gy, (unsigned)gz), kLanes, 0, s>>>(
      c, taps, tap_count, chunk, cp, lr, sums);
   *used = sums == direct ? 0 : gy;
   return hipGetLastError();
}

template<class T>
hipError_t conv_typed(const CacheParams& c, const T* taps, int64_t tap_count, float* direct, float* work,
                      int64_t splits, int64_t* used, hipStream_t s)
{
   if(c.batch == 1) return conv_shape<T, 1, 4>(c, taps, tap_count, direct, work, splits, used, s);
   return conv_shape<T, 2, 4>(c, taps, tap_count, direct, work, splits, used, s);
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
   // no token is beyond the page table
   const int64_t most = c.width << c.page_log;
   if(tap_count > most) tap_count = most;
   // fp32 results that one workgroup sums need no workspace and no join
   float* direct = out_type == T_F32 ? static_cast<float*>(out) : nullptr;
   int64_t used = 0;
   hipError_t e;
   switch(tap_type) {
      case T_F32:  e = conv_typed(c, static_cast<const float*>(taps), tap_count, direct, work, splits, &used, s); break;
      case T_BF16: e = conv_typed(c, static_cast<const bf16*>(taps), tap_count, direct, work, splits, &used, s); break;
      default:     e = conv_typed(c, static_cast<const f16*>(taps), tap_count, direct, work, splits, &used, s); break;
   }
   if(e != hipSuccess || used == 0) return e;
   const int64_t count = c.batch * c.channels, groups = (count + kLanes - 1) / kLanes;
   if(groups > 0x7fffffff) return hipErrorInvalidValue;
   const dim3 g((unsigned)groups);
   switch(out_type) {
      case T_F32:  join_splits<float><<<g, kLanes, 0, s>>>(work, static_cast<float*>(out), count, used); break;
      case T_BF16: join_splits<bf16><<<g, kLanes, 0, s>>>(work, static_cast<bf16*>(out), count, used); break;
      default:     join_splits<f16><<<g, kLanes, 0, s>>>(work, static_cast<f16*>(out), count, used); break;
   }
   return hipGetLastError();
}

}  // namespace mx4
}  // namespace fufft
