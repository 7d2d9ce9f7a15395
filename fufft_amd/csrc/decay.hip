// Linear attention with a decay for each head.  With a = exp(log_decay), of one head:
//
//   S[t] = a S[t-1] + k[t] v[t]^T          out[t] = scale q[t]^T S[t]
//
// Chunks of 64 tokens; with S the state before a chunk of n tokens, tokens counted within it:
//
//   out[t] = a^(t+1) q[t]^T S + sum over s <= t of a^(t-s) (q[t].k[s]) v[s]
//   S'     = a^n S + sum over s of a^(n-1-s) k[s] v[s]^T
//
// The gradients are the same sums in other roles:  dq = the sum with (dout, v, k) for (q, k, v),
// and from the last token back, with D[t] = q[t] dout[t]^T + a D[t+1],  dk[t] = D[t] v[t] is the
// one with (v, dout, q), dv[t] = D[t]^T k[t] the one with (k, q, dout).  A state given to the
// sums from the back meets its first token undecayed, and the state they return is decayed
// once more: `late` is 1 there, and a power of a moves by one.
//
// A workgroup goes through the chunks of a segment of one sequence and head, the state in its
// registers.  Few sequences and heads: the tokens are cut into segments, a first launch makes
// every segment's own part of the state, a second one adds them up in order, and the third
// starts each segment from its state.
#include "decay_internal.hpp"
#include "fufft_internal.hpp"
#include "mx4_device.hpp"

namespace fufft {
namespace layer {

namespace {

using mx4::bf16;
using mx4::f16;
using mx4::f32x4;

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 64, kLanes = 512;

// What the matrix cores take for an input type: bf16 as it is, fp16 and fp32 in fp32.  Every operand
// is 16 bytes a lane: row lane % 16, of each block of the summed index (32 or 16 values)
// the lane / 16-th piece of 8 or 4.  A result of 16 x 16: column lane % 16, rows 4 (lane / 16) ..
// + 3.  So a result is, piece by piece, an operand again whose block of 32 takes rows 4 g .. 4 g + 3 of
// two results (with g = lane / 16), or whose block of 16 takes those of one.
template<class T> struct Cores {
   typedef float E;
   typedef f32x4 Frag;
   static constexpr int PARTS = 1;
   static __device__ inline f32x4 mma(Frag a, Frag b, f32x4 c)
   {
#pragma unroll
      for(int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
      return c;
   }
};
template<> struct Cores<bf16> {
   typedef bf16 E;
   typedef bf16x8 Frag;
   static constexpr int PARTS = 2;       // weighted keys are a sum of two bf16 parts, 16 bits
   static __device__ inline f32x4 mma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

template<class T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T e[8]; };

// Rows of 16-byte slots in LDS, a slot's bytes apart more than they hold: 16 lanes that read one slot of 16
// rows meet all banks, and every address of a lane is one register and a constant.
constexpr int pitch_of(int bytes) { return bytes + 16; }

// `x` as the compiler cannot know it from before: what is derived from it is not kept in registers
// over the chunks
__device__ inline int anew(int x)
{
   asm volatile("" : "+s"(x));
   return x;
}
__device__ inline int anew_lane(int x)
{
   asm volatile("" : "+v"(x));
   return x;
}

// 2^(g2 n), 1 at n = 0 whatever g2 is (-infinity is held as -1e30)
__device__ inline float power(float g2, float n) { return __builtin_amdgcn_exp2f(g2 * n); }

// LDS of a kernel: keys as they are, values by channel, weighted keys by channel, the state by
// value channel; the first and the last are not needed for a segment's own part.
template<class T, int DK, int DV, bool LOCAL> struct Room {
   typedef Cores<T> C;
   static constexpr int E = sizeof(typename C::E);
   static constexpr int TP = pitch_of(kChunk * E), KP = pitch_of(DK * E);       // rows of tokens, of keys' channels
   static constexpr int VALUES = 0, KEYS_T = VALUES + DV * TP, KEYS = KEYS_T + C::PARTS * DK * TP;
   static constexpr int STATE = LOCAL ? KEYS : KEYS + kChunk * KP, FLAGS = LOCAL ? KEYS : STATE + DV * KP;
   static constexpr int BYTES = FLAGS + 16;
};

// where tokens 4 q .. 4 q + 3 are in a row of tokens: in bf16 in block q / 8, of its piece q % 4 the first or
// second half
template<class E>
__device__ inline int tokens_at(int q)
{
   return sizeof(E) == 4 ? q * 16 : ((q >> 3) * 4 + (q & 3)) * 16 + ((q >> 2) & 1) * 8;
}
template<class E>
__device__ inline void put4(uint8_t* to, const float (&v)[4])
{
   if constexpr(sizeof(E) == 4) *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
   else *reinterpret_cast<bf16x4*>(to) = bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
}

template<class T, int DK, int DV, bool LOCAL>
__global__ void __launch_bounds__(kLanes)
decay_chunks(DecayParams p)
{
   typedef Cores<T> C;
   typedef typename C::E E;
   typedef typename C::Frag Frag;
   typedef Room<T, DK, DV, LOCAL> M;
   constexpr int BLOCK = sizeof(E) == 2 ? 32 : 16;             // of the summed index of a product
   constexpr int NK = DK / BLOCK, NS = kChunk / BLOCK;          // blocks of keys' channels, of tokens
   constexpr int KP = M::KP, TP = M::TP;
   constexpr int SA = DK / 64, SB = DV / 32;                   // a wavefront's results of the state; SB of out too
   constexpr int KT = DK / 32, VT = DV / 32;                   // wavefronts that stage keys, values: 4 tokens x 8 channels a lane
   static_assert(KT + VT <= kLanes / 64, "every piece has a lane");
   extern __shared__ uint8_t lds[];
   int* const flags = reinterpret_cast<int*>(lds + M::FLAGS);
   const DecayRole& role = p.role[blockIdx.y];
   const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
   const int row = lane & 15, g = lane >> 4;

   // slices of one segment run on one XCD, whose L2 they share
   const uint32_t id = blockIdx.x, slices = (uint32_t)p.slices;
   const int slice = (int)(id / 8 % slices);
   const int64_t item = (int64_t)(id / (8 * slices)) * 8 + id % 8;
   if(item >= p.items) return;
   const int64_t bh = item % p.pairs, seg = item / p.pairs;
   const int64_t b = bh / p.heads, h = bh % p.heads;
   int64_t len = p.tokens;
   if(p.lens) {
      len = p.lens[b];
      len = len < 0 ? 0 : len > p.tokens ? p.tokens : len;
   }
   const int64_t first = seg * p.segment;
   if(first >= len && seg > 0) return;
   const int64_t left = len - first < p.segment ? len - first : p.segment;      // this segment's tokens
   if(LOCAL && first + left >= len) return;                     // the last segment's part is not asked for
   const int dk = role.dk, dv = role.dv, dv0 = slice * DV;
   if(dv0 >= dv) return;                                       // a role of fewer slices
   const int dvn = dv - dv0 < DV ? dv - dv0 : DV;
   float g2 = p.log_decay[h] * 1.44269504f;
   g2 = g2 < -1e30f ? -1e30f : g2;

   // token t of the segment: t steps from its first one
   const int64_t dir = role.reverse ? -1 : 1, at0 = role.reverse ? len - 1 - first : first;
   auto rows_of = [&](const void* base, const Strides& s) {
      return static_cast<const T*>(base) + b * s.batch + h * s.head + at0 * s.token;
   };
   const T* const q = rows_of(role.q, role.sq);
   const T* const k = rows_of(role.k, role.sk);
   const T* const v = rows_of(role.v, role.sv) + dv0;

   // staging: this lane's tokens and channels
   const bool keys = wave < KT, values = !keys && wave < KT + VT;
   const int piece = keys ? tid : tid - KT * 64;
   const int width = (keys ? DK : DV) / 8, cb = piece % width, tq = piece / width;
   const T* const src = (keys ? k : v) + cb * 8;
   const int64_t step = dir * (keys ? role.sk.token : role.sv.token);
   const int dim = keys ? dk : dvn;
   Eight<T> raw[4];
   auto fetch = [&](int64_t t0) {
      if(!keys && !values) return;
      const int d = anew(dim), n = (int)(left - t0 < kChunk ? left - t0 : kChunk);
      const T* const p0 = src + (t0 + tq * 4) * step;
#pragma unroll
      for(int i = 0; i < 4; i++) {
         raw[i] = Eight<T>{};
         if(d % 8 == 0) {
            if(tq * 4 + i < n && cb * 8 < d) raw[i] = *reinterpret_cast<const Eight<T>*>(p0 + i * step);
         } else if(tq * 4 + i < n) {
#pragma unroll
            for(int j = 0; j < 8; j++)
               if(cb * 8 + j < d) raw[i].e[j] = p0[i * step + j];
         }
      }
   };

   // this wavefront's strip of 16 tokens and half of the values; two wavefronts of a SIMD have 5 of the
   // 8 strips' blocks of scores between them
   const int strip = wave < 4 ? wave : 7 - wave, half = wave >> 2;
   const int v0 = half * (DV / 2), k0 = (wave & 3) * (DK / 4);
   Frag qf[NK];
   auto fetch_q = [&](int64_t t0) {
      constexpr int N = 16 / (int)sizeof(E);
      struct __attribute__((packed, aligned(sizeof(T)))) Piece { T e[N]; };
      const int d = anew(dk);
      const bool there = t0 + strip * 16 + row < left;
      const T* const p0 = q + (t0 + strip * 16 + row) * dir * role.sq.token + g * N;
#pragma unroll
      for(int i = 0; i < NK; i++) {
         const int at = i * BLOCK + g * N;
         Piece x{};
         if(d % N == 0) {
            if(there && at < d) x = *reinterpret_cast<const Piece*>(p0 + i * BLOCK);
         } else if(there) {
#pragma unroll
            for(int j = 0; j < N; j++)
               if(at + j < d) x.e[j] = p0[i * BLOCK + j];
         }
#pragma unroll
         for(int j = 0; j < N; j++) qf[i][j] = (E)x.e[j];
      }
   };

   // weights of scores: a^(t - s), rows s of result i, column t; and of q S at t
   float wt[4][4], wq = 0.0f;
   if constexpr(!LOCAL) {
#pragma unroll
      for(int i = 0; i < 4; i++)
#pragma unroll
         for(int r = 0; r < 4; r++) {
            const int d = (strip - i) * 16 + row - g * 4 - r;
            wt[i][r] = d >= 0 ? power(g2, (float)d) * role.p_scale * role.out_scale : 0.0f;
         }
      wq = power(g2, (float)(strip * 16 + row + 1 - role.late)) * role.out_scale;
   }

   // the state before the segment: keys' channels k0 + 16 a + 4 g + r, value v0 + 16 b + row
   f32x4 S[SA][SB];
   const int64_t count = (int64_t)dk * dv;
   // the elements of a state that this lane has and memory holds
   auto each_state = [&](bool turned, auto body) {
      const int rows = anew(dk), cols = anew(dv);
#pragma unroll
      for(int a = 0; a < SA; a++)
#pragma unroll
         for(int c = 0; c < SB; c++) {
            const int i = k0 + a * 16 + g * 4, j = dv0 + v0 + c * 16 + row;
            const int at = turned ? j * rows + i : i * cols + j, step = turned ? 1 : cols;
#pragma unroll
            for(int r = 0; r < 4; r++) if(j < cols && i + r < rows) body(a, c, r, at + r * step);
         }
   };
   const float* const from = LOCAL ? nullptr
                             : p.segments > 1 ? role.work + (seg * p.pairs + bh) * count
                             : role.state ? role.state + bh * count : nullptr;
#pragma unroll
   for(int a = 0; a < SA; a++)
#pragma unroll
      for(int c = 0; c < SB; c++) S[a][c] = f32x4{};
   if(from) each_state(p.segments > 1 ? false : role.turned, [&](int a, int c, int r, int at) { S[a][c][r] = from[at]; });

   if(left > 0) {
      fetch(0);
      if constexpr(!LOCAL) fetch_q(0);
   }
   if(tid < 2) flags[tid] = 0;
   __syncthreads();
   int side = 0;
   for(int64_t t0 = 0; t0 < left; t0 += kChunk, side ^= 1) {
      const int n = (int)(left - t0 < kChunk ? left - t0 : kChunk);
      // to LDS: values and weighted keys by channel, keys as they are, the state by value
      if(keys) {
         float w[4];
#pragma unroll
         for(int i = 0; i < 4; i++) {
            const int s = tq * 4 + i;
            w[i] = s < n ? power(g2, (float)(n - 1 - s + role.late)) * role.kv_scale : 0.0f;
         }
         uint8_t* const to = lds + M::KEYS_T + cb * 8 * TP + tokens_at<E>(tq);
#pragma unroll
         for(int j = 0; j < 8; j++) {
            float x[4];
#pragma unroll
            for(int i = 0; i < 4; i++) x[i] = (float)raw[i].e[j] * w[i];
            put4<E>(to + j * TP, x);
            if constexpr(C::PARTS == 2) {
               // what bf16 leaves of it; nothing of an infinity
               float y[4];
#pragma unroll
               for(int i = 0; i < 4; i++) {
                  const float whole = (float)(bf16)x[i];
                  y[i] = fabsf(whole) < __builtin_inff() ? x[i] - whole : 0.0f;
               }
               put4<E>(to + (DK + j) * TP, y);
            }
         }
         if constexpr(!LOCAL) {
            uint8_t* const plain = lds + M::KEYS + tq * 4 * KP + cb * 8 * (int)sizeof(E);
#pragma unroll
            for(int i = 0; i < 4; i++) {
               if constexpr(sizeof(E) == 2) {
                  *reinterpret_cast<bf16x8*>(plain + i * KP) = __builtin_bit_cast(bf16x8, raw[i]);
               } else {
#pragma unroll
                  for(int j = 0; j < 2; j++) {
                     const float x[4] = {(float)raw[i].e[4 * j], (float)raw[i].e[4 * j + 1], (float)raw[i].e[4 * j + 2],
                                         (float)raw[i].e[4 * j + 3]};
                     put4<E>(plain + i * KP + j * 16, x);
                  }
               }
            }
         }
      }
      if(values) {
         bool odd = false;
         uint8_t* const to = lds + M::VALUES + cb * 8 * TP + tokens_at<E>(tq);
#pragma unroll
         for(int j = 0; j < 8; j++) {
            float x[4];
#pragma unroll
            for(int i = 0; i < 4; i++) {
               x[i] = (float)raw[i].e[j];
               odd |= !(fabsf(x[i]) < __builtin_inff());
            }
            put4<E>(to + j * TP, x);
         }
         if(odd) flags[side] = 1;
      }
      if constexpr(!LOCAL) {
         uint8_t* const to = lds + M::STATE + (v0 + row) * KP + (k0 + g * 4) * (int)sizeof(E);
#pragma unroll
         for(int a = 0; a < SA; a++)
#pragma unroll
            for(int c = 0; c < SB; c++) {
               const float x[4] = {S[a][c][0], S[a][c][1], S[a][c][2], S[a][c][3]};
               put4<E>(to + c * 16 * KP + a * 16 * (int)sizeof(E), x);
            }
      }
      __syncthreads();
      const bool special = flags[side] != 0;
      if(tid == 0) flags[side ^ 1] = 0;
      auto frag = [&](int base, int pitch, int r, int block) {
         return *reinterpret_cast<const Frag*>(lds + base + (r + row) * pitch + (block * 4 + g) * 16);
      };
      auto value_frag = [&](int c, int sb) { return frag(M::VALUES, TP, v0 + c * 16, sb); };
      const bool more = t0 + kChunk < left;
      if(more) fetch(t0 + kChunk);                              // on its way under the products

      if constexpr(!LOCAL) {
         f32x4 o[SB] = {};
#pragma unroll
         for(int i = 0; i < NK; i++)
#pragma unroll
            for(int c = 0; c < SB; c++)
               o[c] = C::mma(frag(M::STATE, KP, v0 + c * 16, i), qf[i], o[c]);
#pragma unroll
         for(int c = 0; c < SB; c++) o[c] *= wq;
         const int reach = anew_lane(strip * 16 + row - g * 4);      // scores of tokens up to this plus 4 g count
#pragma unroll
         for(int sb = 0; sb < NS; sb++) {
            constexpr int EACH = BLOCK / 16;                    // results to a block
            if(sb * EACH > strip) break;
            f32x4 s[EACH];
#pragma unroll
            for(int e = 0; e < EACH; e++) {
               const int tile = sb * EACH + e;
               f32x4 x = {};
               if(tile <= strip)
#pragma unroll
                  for(int i = 0; i < NK; i++)
                     x = C::mma(frag(M::KEYS, KP, tile * 16, i), qf[i], x);
               // tokens behind t have no part in it, whatever they hold
#pragma unroll
               for(int r = 0; r < 4; r++) s[e][r] = tile * 16 + r <= reach ? x[r] * wt[tile][r] : 0.0f;
            }
            Frag w;
#pragma unroll
            for(int e = 0; e < EACH; e++)
#pragma unroll
               for(int r = 0; r < 4; r++) w[e * 4 + r] = (E)s[e][r];
            if(!special) {
#pragma unroll
               for(int c = 0; c < SB; c++) o[c] = C::mma(value_frag(c, sb), w, o[c]);
            } else {
               // A value that is infinite or NaN times a weight of zero would reach tokens before it.  Such values
               // are left out of the products, and added one by one to the results that they belong to.
#pragma unroll
               for(int c = 0; c < SB; c++) {
                  Frag x = value_frag(c, sb);
#pragma unroll
                  for(int i = 0; i < EACH * 4; i++) x[i] = fabsf((float)x[i]) < __builtin_inff() ? x[i] : (E)0.0f;
                  o[c] = C::mma(x, w, o[c]);
               }
#pragma unroll
               for(int i = 0; i < EACH * 4; i++)
#pragma unroll 1
                  for(int from_g = 0; from_g < 4; from_g++) {
                     const int t1 = sb * BLOCK + (i / 4) * 16 + from_g * 4 + i % 4;
                     const float weight = __shfl((float)w[i], row + from_g * 16);
                     if(t1 > strip * 16 + row) continue;
                     const uint8_t* const at = lds + M::VALUES + (v0 + g * 4) * TP + tokens_at<E>(t1 / 4) + t1 % 4 * (int)sizeof(E);
#pragma unroll
                     for(int c = 0; c < SB; c++)
#pragma unroll
                        for(int r = 0; r < 4; r++) {
                           const float x = (float)*reinterpret_cast<const E*>(at + (c * 16 + r) * TP);
                           if(!(fabsf(x) < __builtin_inff())) o[c][r] += weight * x;
                        }
                  }
            }
         }
         if(more) fetch_q(t0 + kChunk);
         const int t = strip * 16 + row;
         if(t < n) {
            const int d = anew(dvn);
            T* const out = static_cast<T*>(role.o) + b * role.so.batch + h * role.so.head + (at0 + dir * (t0 + t)) * role.so.token + dv0;
            struct __attribute__((packed, aligned(sizeof(T)))) Four { T e[4]; };
#pragma unroll
            for(int c = 0; c < SB; c++) {
               const int j = v0 + c * 16 + g * 4;
               Four x;
#pragma unroll
               for(int r = 0; r < 4; r++) x.e[r] = (T)o[c][r];
               if(d % 4 == 0) {
                  if(j < d) *reinterpret_cast<Four*>(out + j) = x;
               } else {
#pragma unroll
                  for(int r = 0; r < 4; r++)
                     if(j + r < d) out[j + r] = x.e[r];
               }
            }
         }
      }
      // the state behind the chunk
      const float an = power(g2, (float)n);
#pragma unroll
      for(int a = 0; a < SA; a++)
#pragma unroll
         for(int c = 0; c < SB; c++) S[a][c] *= an;
#pragma unroll
      for(int sb = 0; sb < NS; sb++) {
         Frag x[SB];
#pragma unroll
         for(int c = 0; c < SB; c++) x[c] = value_frag(c, sb);
#pragma unroll
         for(int part = 0; part < C::PARTS; part++)
#pragma unroll
            for(int a = 0; a < SA; a++) {
               const Frag w = frag(M::KEYS_T, TP, part * DK + k0 + a * 16, sb);
#pragma unroll
               for(int c = 0; c < SB; c++) S[a][c] = C::mma(w, x[c], S[a][c]);
            }
      }
      __syncthreads();
   }

   float* const to = LOCAL ? role.work + (seg * p.pairs + bh) * count
                     : role.new_state && first + left >= len ? role.new_state + bh * count : nullptr;
   if(!to) return;
   each_state(!LOCAL && role.turned, [&](int a, int c, int r, int at) { to[at] = S[a][c][r]; });
}

// Every segment's part of the state in work becomes the state before that segment.  A lane has one
// element of a state; the parts of eight segments are read ahead of their sums.
__global__ void __launch_bounds__(256)
decay_scan(DecayParams p)
{
   const DecayRole& role = p.role[blockIdx.y];
   const int64_t count = (int64_t)role.dk * role.dv, per = (count + 255) / 256;
   const int64_t bh = blockIdx.x / per, e = blockIdx.x % per * 256 + threadIdx.x;
   if(bh >= p.pairs || e >= count) return;
   const int64_t b = bh / p.heads, h = bh % p.heads;
   int64_t len = p.tokens;
   if(p.lens) {
      len = p.lens[b];
      len = len < 0 ? 0 : len > p.tokens ? p.tokens : len;
   }
   float g2 = p.log_decay[h] * 1.44269504f;
   g2 = g2 < -1e30f ? -1e30f : g2;
   const float a = power(g2, (float)p.segment);                  // every segment but the last is whole
   float s = 0.0f;
   if(role.state) s = role.state[bh * count + (role.turned ? e % role.dv * role.dk + e / role.dv : e)];
   float* const work = role.work + bh * count + e;
   const int64_t pitch = p.pairs * count;
   constexpr int AHEAD = 8;
   for(int64_t seg = 0; seg < p.segments && (seg == 0 || seg * p.segment < len); seg += AHEAD) {
      float part[AHEAD];
#pragma unroll
      for(int i = 0; i < AHEAD; i++) part[i] = (seg + i + 1) * p.segment < len ? work[(seg + i) * pitch] : 0.0f;
#pragma unroll
      for(int i = 0; i < AHEAD; i++) {
         if(seg + i < p.segments && (seg + i == 0 || (seg + i) * p.segment < len)) work[(seg + i) * pitch] = s;
         s = a * s + part[i];
      }
   }
}

// ---- one token ------------------------------------------------------------------------------
//
// A workgroup has 32 values of one sequence and head: 8 lanes of 4 values, 32 rows of the state at a
// time, all of them on their way at once.  Bound by the state's bytes, read and written once.
constexpr int kStepValues = 32, kStepRows = 4;          // 4 x 32 rows: dk up to 128

template<class T>
__global__ void __launch_bounds__(256)
decay_step(StepParams p)
{
   __shared__ float join[4][kStepValues];
   __shared__ int taken;
   struct __attribute__((packed, aligned(4))) Four { float e[4]; };
   const int tid = threadIdx.x, c = tid & 7, r0 = tid >> 3;
   const int64_t b = blockIdx.x / (p.heads * p.slices), rest = blockIdx.x % (p.heads * p.slices);
   const int64_t h = rest / p.slices;
   const int j0 = (int)(rest % p.slices) * kStepValues + c * 4;
   const int64_t slot = p.slots ? p.slots[b] : b;
   const bool inside = slot >= 0 && slot < p.slot_count;
   float* const state = inside ? p.state + (slot * p.heads + h) * p.dk * p.dv : nullptr;
   Four s[kStepRows];
   float kk[kStepRows], qq[kStepRows];
   const T* const q = static_cast<const T*>(p.q) + b * p.sq.batch + h * p.sq.head;
   const T* const k = static_cast<const T*>(p.k) + b * p.sk.batch + h * p.sk.head;
   const T* const v = static_cast<const T*>(p.v) + b * p.sv.batch + h * p.sv.head;
   const bool whole = j0 + 4 <= p.dv;
#pragma unroll
   for(int i = 0; i < kStepRows; i++) {
      const int r = r0 + i * 32;
      s[i] = Four{};
      kk[i] = qq[i] = 0.0f;
      if(inside && r < p.dk) {
         const float* const at = state + r * p.dv + j0;
         if(whole) s[i] = *reinterpret_cast<const Four*>(at);
         else
#pragma unroll
            for(int e = 0; e < 4; e++)
               if(j0 + e < p.dv) s[i].e[e] = at[e];
         kk[i] = (float)k[r];
         qq[i] = (float)q[r];
      }
   }
   float vv[4];
#pragma unroll
   for(int e = 0; e < 4; e++) vv[e] = j0 + e < p.dv ? (float)v[j0 + e] : 0.0f;
   // whether an earlier sequence has the same state
   bool mine = inside;
   if(p.slots) {
      if(tid == 0) taken = 0;
      __syncthreads();
      bool found = false;
      for(int64_t i = tid; i < b; i += 256) found |= p.slots[i] == slot;
      if(found) taken = 1;
      __syncthreads();
      mine = inside && !taken;
   }
   const float a = expf(p.log_decay[h]);
   float acc[4] = {};
#pragma unroll
   for(int i = 0; i < kStepRows; i++) {
#pragma unroll
      for(int e = 0; e < 4; e++) {
         s[i].e[e] = a * s[i].e[e] + kk[i] * vv[e];
         acc[e] += qq[i] * s[i].e[e];
      }
      const int r = r0 + i * 32;
      if(mine && r < p.dk) {
         float* const at = state + r * p.dv + j0;
         if(whole) *reinterpret_cast<Four*>(at) = s[i];
         else
#pragma unroll
            for(int e = 0; e < 4; e++)
               if(j0 + e < p.dv) at[e] = s[i].e[e];
      }
   }
#pragma unroll
   for(int e = 0; e < 4; e++) {
      acc[e] += __shfl_xor(acc[e], 8);
      acc[e] += __shfl_xor(acc[e], 16);
      acc[e] += __shfl_xor(acc[e], 32);
   }
   if((tid & 63) < 8)
#pragma unroll
      for(int e = 0; e < 4; e++) join[tid >> 6][c * 4 + e] = acc[e];
   __syncthreads();
   const int j = (int)(rest % p.slices) * kStepValues + tid;
   if(tid < kStepValues && j < p.dv) {
      const float sum = ((join[0][tid] + join[1][tid]) + join[2][tid]) + join[3][tid];
      static_cast<T*>(p.out)[b * p.so.batch + h * p.so.head + j] = (T)(mine ? sum * p.scale : 0.0f);
   }
}

// ---- launches --------------------------------------------------------------------------------

template<class T, int DK, int DV, bool LOCAL>
hipError_t chunks_shape(DecayParams p, int roles, hipStream_t s)
{
   constexpr int bytes = Room<T, DK, DV, LOCAL>::BYTES;
   static_assert(bytes <= 160 * 1024, "fits the LDS");
   static std::atomic<uint64_t> mask{0};
   const hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(&decay_chunks<T, DK, DV, LOCAL>), bytes, mask);
   if(e != hipSuccess) return e;
   int most = 0;
   for(int r = 0; r < roles; r++) most = p.role[r].dv > most ? p.role[r].dv : most;
   p.slices = (most + DV - 1) / DV;
   p.items = p.pairs * (LOCAL ? p.segments - 1 : p.segments);
   const int64_t groups = (p.items + 7) / 8 * 8 * p.slices;
   if(!grid_ok(groups, kLanes)) return kTooLarge;
   decay_chunks<T, DK, DV, LOCAL><<<dim3((unsigned)groups, (unsigned)roles), kLanes, bytes, s>>>(p);
   return hipGetLastError();
}

template<class T, int DK, int DV>
hipError_t chunks_launches(DecayParams p, int roles, hipStream_t s)
{
   // Segments so that each CU has as many workgroups as fit its LDS, none of fewer than 4 chunks
   const int64_t chunks = (p.tokens + kChunk - 1) / kChunk;
   const int64_t groups = p.pairs * roles * ((p.role[0].dv + DV - 1) / DV);
   const int64_t fit = 256 * (160 * 1024 / Room<T, DK, DV, false>::BYTES);
   int64_t n = fit / (groups > 0 ? groups : 1);
   if(n > p.splits) n = p.splits;
   if(n > chunks / 4) n = chunks / 4;
   if(n < 1) n = 1;
   const int64_t each = chunks > 0 ? (chunks + n - 1) / n : 1;
   p.segment = each * kChunk;
   p.segments = chunks > 0 ? (chunks + each - 1) / each : 1;
   if(p.segments > 1) {
      hipError_t e = chunks_shape<T, DK, DV, true>(p, roles, s);
      if(e != hipSuccess) return e;
      int64_t most = 0;
      for(int r = 0; r < roles; r++) {
         const int64_t per = ((int64_t)p.role[r].dk * p.role[r].dv + 255) / 256;
         most = per > most ? per : most;
      }
      if(!grid_ok(p.pairs * most, 256)) return kTooLarge;
      decay_scan<<<dim3((unsigned)(p.pairs * most), (unsigned)roles), 256, 0, s>>>(p);
      e = hipGetLastError();
      if(e != hipSuccess) return e;
   }
   return chunks_shape<T, DK, DV, false>(p, roles, s);
}

// roles whose keys have the same width
template<class T>
hipError_t decay_typed(const DecayParams& p, int roles, hipStream_t s)
{
   const int dk = p.role[0].dk;
   if constexpr(sizeof(typename Cores<T>::E) == 2) {
      int dv = 0;
      for(int r = 0; r < roles; r++) dv = p.role[r].dv > dv ? p.role[r].dv : dv;
      if(dv > 64) return dk <= 64 ? chunks_launches<T, 64, 128>(p, roles, s) : chunks_launches<T, 128, 128>(p, roles, s);
   }
   return dk <= 64 ? chunks_launches<T, 64, 64>(p, roles, s) : chunks_launches<T, 128, 64>(p, roles, s);
}

hipError_t decay_roles(const DecayParams& p, int roles, hipStream_t s)
{
   switch(p.type) {
      case T_F32:  return decay_typed<float>(p, roles, s);
      case T_BF16: return decay_typed<bf16>(p, roles, s);
      default:     return decay_typed<f16>(p, roles, s);
   }
}

}  // namespace

hipError_t launch_decay(const DecayParams& p, int roles, hipStream_t s)
{
   if(p.pairs <= 0) return hipSuccess;
   // roles of one width run in one launch
   bool same = true;
   for(int r = 1; r < roles; r++) same = same && (p.role[r].dk <= 64) == (p.role[0].dk <= 64) && (p.role[r].dv <= 64) == (p.role[0].dv <= 64);
   if(same) return decay_roles(p, roles, s);
   for(int r = 0; r < roles; r++) {
      DecayParams one = p;
      one.role[0] = p.role[r];
      const hipError_t e = decay_roles(one, 1, s);
      if(e != hipSuccess) return e;
   }
   return hipSuccess;
}

hipError_t launch_decay_step(const StepParams& params, hipStream_t s)
{
   StepParams p = params;
   p.slices = (p.dv + kStepValues - 1) / kStepValues;
   const int64_t groups = p.batch * p.heads * p.slices;
   if(groups <= 0) return hipSuccess;
   if(!grid_ok(groups, 256)) return kTooLarge;
   switch(p.type) {
      case T_F32:  decay_step<float><<<(unsigned)groups, 256, 0, s>>>(p); break;
      case T_BF16: decay_step<bf16><<<(unsigned)groups, 256, 0, s>>>(p); break;
      default:     decay_step<f16><<<(unsigned)groups, 256, 0, s>>>(p); break;
   }
   return hipGetLastError();
}

}  // namespace layer
}  // namespace fufft
