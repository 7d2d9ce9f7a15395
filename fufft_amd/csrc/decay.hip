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

#include <type_traits>

namespace fufft {
namespace layer {

namespace {

using mx4::bf16;
using mx4::f16;
using mx4::f32x4;

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 64, kLanes = 512;

// What the matrix cores take for an input type.  Every operand is 16 bytes a lane: row lane % 16, of each block
// of the summed index (32 or 16 values) the lane / 16-th piece of 8 or 4.  A result of 16 x 16: column lane %
// 16, rows 4 (lane / 16) .. + 3.  So a result is, piece by piece, an operand again whose block of 32 takes rows 4 g .. 4 g + 3
// of two results (with g = lane / 16), or whose block of 16 takes those of one.
//
//   fp32: everything in fp32, whose products run at a sixteenth of the others' rate and bound these kernels.
//   bf16: what becomes an operand again (the state that q meets, weighted scores, weighted keys) is two bf16 parts, 16 bits,
//     so that only the result's own rounding is left (0.00166 of results of Gaussian inputs; with the state and scores rounded
//     to one part 0.00235, and 65536 tokens x 16 heads in 471 us, not 515).
//   fp16: scores in fp16 as they are.  fp16's range would not hold what becomes an operand again, so that
//     and what meets it are sums of two bf16 parts, 16 bits of a value and all 11 of fp16; of the four products the
//     smallest, of both second parts, is left out (2^-16).
//
// Where the state is returned, weighted keys are three bf16 parts in both, fp32's 24 bits (FINE): in the launch whose sums
// become that state, which is the first one where tokens are split (65536 tokens x 16 heads in bf16 with its state: 527 us
// with three parts in both launches, 512 so).
template<class T> struct Cores {
   typedef float E;
   typedef f32x4 Frag, Plain;            // operands in E; of q and k as they are
   static constexpr int KEY_PARTS = 1, FINE_PARTS = 1;       // of weighted keys
   static constexpr int PARTS = 1;       // of values, and of q where it meets the state
   static constexpr int MADE = 1;        // of weights and the state
   static __device__ inline f32x4 mma(Frag a, Frag b, f32x4 c)
   {
#pragma unroll
      for(int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
      return c;
   }
   static __device__ inline f32x4 scores(Plain a, Plain b, f32x4 c) { return mma(a, b, c); }
};
template<> struct Cores<bf16> {
   typedef bf16 E;
   typedef bf16x8 Frag, Plain;
   static constexpr int KEY_PARTS = 2, FINE_PARTS = 3, PARTS = 1, MADE = 2;
   static __device__ inline f32x4 mma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
   static __device__ inline f32x4 scores(Plain a, Plain b, f32x4 c) { return mma(a, b, c); }
};
template<> struct Cores<f16> {
   typedef bf16 E;
   typedef bf16x8 Frag;
   typedef f16x8 Plain;
   static constexpr int KEY_PARTS = 2, FINE_PARTS = 3, PARTS = 2, MADE = 2;
   static __device__ inline f32x4 mma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
   static __device__ inline f32x4 scores(Plain a, Plain b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
// sums of parts, all products but that of both second parts
template<class C, int A, int B>
__device__ inline f32x4 mma_parts(const typename C::Frag (&a)[A], const typename C::Frag (&b)[B], f32x4 c)
{
#pragma unroll
   for(int i = 0; i < A; i++)
#pragma unroll
      for(int j = 0; j < B; j++)
         if(i + j < 2) c = C::mma(a[i], b[j], c);
   return c;
}
// what bf16 leaves of values (NaN of an infinity)
template<int N>
__device__ inline void rest(float (&x)[N])
{
#pragma unroll
   for(int i = 0; i < N; i++) x[i] -= (float)(bf16)x[i];
}

// N neighbours of a row as they are in memory, loaded at the element's alignment.
template<class T, int N> struct Raw {
   static constexpr int WORDS = N * (int)sizeof(T) / 4;
   uint32_t w[WORDS];

   __device__ inline float value(int j) const
   {
      if constexpr(sizeof(T) == 4) {
         return __uint_as_float(w[j]);
      } else if constexpr(std::is_same<T, bf16>::value) {
         return __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
      } else {
         return (float)__builtin_bit_cast(T, (uint16_t)(w[j / 2] >> (j % 2 * 16)));
      }
   }
   // elements from `count` on made zero
   __device__ inline void cut(int count)
   {
#pragma unroll
      for(int j = 0; j < N; j++)
         if(j >= count) {
            if constexpr(sizeof(T) == 4) w[j] = 0u;
            else w[j / 2] &= j % 2 ? 0x0000ffffu : 0xffff0000u;
         }
   }
};
template<class T, int N>
__device__ inline Raw<T, N> raw_at(const T* p)
{
   typedef uint32_t V __attribute__((ext_vector_type(Raw<T, N>::WORDS), aligned(sizeof(T))));
   const V v = *reinterpret_cast<const V*>(p);
   Raw<T, N> x;
#pragma unroll
   for(int i = 0; i < Raw<T, N>::WORDS; i++) x.w[i] = v[i];
   return x;
}
// the same of a row whose elements from `count` on are not there: the first one is read in their place
template<class T, int N>
__device__ inline Raw<T, N> raw_of(const T* p, const T* first, int count)
{
   Raw<T, N> x{};
#pragma unroll
   for(int j = 0; j < N; j++) {
      const T e = *(j == 0 || j < count ? p + j : first);
      if constexpr(sizeof(T) == 4) x.w[j] = __builtin_bit_cast(uint32_t, e);
      else x.w[j / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, e) << (j % 2 * 16);
   }
   return x;
}
// whether one of them is infinite or NaN
template<class T, int N>
__device__ inline bool odd_one(const Raw<T, N> (&x)[8])
{
   if constexpr(sizeof(T) == 2) {
      typedef uint16_t V __attribute__((ext_vector_type(2)));
      V m = {0, 0};
#pragma unroll
      for(int i = 0; i < 8; i++)
#pragma unroll
         for(int j = 0; j < Raw<T, N>::WORDS; j++) m = __builtin_elementwise_max(m, __builtin_bit_cast(V, x[i].w[j] & 0x7fff7fffu));
      constexpr uint16_t LIMIT = std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00;
      return m[0] >= LIMIT || m[1] >= LIMIT;
   } else {
      uint32_t m = 0;
#pragma unroll
      for(int i = 0; i < 8; i++)
#pragma unroll
         for(int j = 0; j < N; j++) m = mx4::umax(m, x[i].w[j] & 0x7fffffffu);
      return m >= 0x7f800000u;
   }
}

// LDS.  Keys as they are and the state: rows of 16-byte slots, a slot further apart than they are long, so that lanes
// that read one slot of 8 rows meet all banks.  By channel, rows of a chunk's tokens: slot s of row r is at
// s ^ turn(r), which does the same for 8 rows that follow each other, as products read them, and for 8 every
// second one, as staging writes them.  (Padded rows there, written 8 bytes a lane, were two thirds of all
// LDS cycles conflicts: 65536 tokens x 16 heads 457 us in the last launch.)
constexpr int pitch_of(int bytes) { return bytes + 16; }
__device__ inline int turn(int row) { return (row & 7) ^ (row >> 3 & 1); }

// `x` as the compiler cannot know it from before: what is derived from it is not kept in registers
// over the chunks
__device__ inline int anew(int x)       // of one value in all lanes
{
   x = __builtin_amdgcn_readfirstlane(x);
   asm volatile("" : "+s"(x));
   return x;
}
__device__ inline int64_t anew(int64_t x)
{
   const uint32_t lo = (uint32_t)anew((int)(uint32_t)x), hi = (uint32_t)anew((int)(uint32_t)(x >> 32));
   return (int64_t)((uint64_t)hi << 32 | lo);
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
template<class T, int DK, int DV, bool LOCAL, bool FINE> struct Room {
   typedef Cores<T> C;
   static constexpr int E = sizeof(typename C::E), KEY_PARTS = FINE ? C::FINE_PARTS : C::KEY_PARTS;
   static constexpr int TP = kChunk * E, KP = pitch_of(DK * E);       // bytes of a row of tokens, of keys' channels
   static constexpr int VALUES = 0, KEYS_T = VALUES + C::PARTS * DV * TP, KEYS = KEYS_T + KEY_PARTS * DK * TP;
   static constexpr int STATE = LOCAL ? KEYS : KEYS + kChunk * KP, FLAGS = LOCAL ? KEYS : STATE + C::MADE * DV * KP;
   static constexpr int BYTES = FLAGS + 16;
};

// The slot of a row of tokens that token t is in, and its bytes in it: in bf16 a slot has tokens 4 g .. 4 g + 3 of
// two 16 tokens, as an operand's block of 32 takes them.
template<class E> __device__ inline int slot_of(int t) { return sizeof(E) == 4 ? t / 4 : t / 32 * 4 + t / 4 % 4; }
template<class E> __device__ inline int in_slot(int t) { return sizeof(E) == 4 ? t % 4 * 4 : (t / 16 % 2 * 4 + t % 4) * 2; }
template<class E>
__device__ inline void put4(uint8_t* to, const float (&v)[4])
{
   if constexpr(sizeof(E) == 4) *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
   else *reinterpret_cast<bf16x4*>(to) = bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
}

template<class T, int DK, int DV, bool LOCAL, bool WHOLE, bool FINE>
__global__ void __launch_bounds__(kLanes)
decay_chunks(DecayParams p)
{
   typedef Cores<T> C;
   typedef typename C::E E;
   typedef typename C::Frag Frag;
   typedef typename C::Plain Plain;
   typedef Room<T, DK, DV, LOCAL, FINE> M;
   constexpr int BLOCK = sizeof(E) == 2 ? 32 : 16;             // of the summed index of a product
   constexpr int EACH = BLOCK / 16;                            // results to a block
   constexpr int NK = DK / BLOCK, NS = kChunk / BLOCK;          // blocks of keys' channels, of tokens
   constexpr int KP = M::KP, TP = M::TP;
   constexpr int SA = DK / 64, SB = DV / 32;                   // a wavefront's results of the state; SB of out too
   constexpr int KJ = DK * 4, VJ = DV * 4;                     // lanes that stage keys, values: 8 tokens x 2 channels each
   static_assert(KJ <= kLanes && VJ <= kLanes, "every piece has a lane");
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
   const int64_t first = seg * (LOCAL ? p.part : p.segment);
   if(first >= len && seg > 0) return;
   const int64_t most = LOCAL ? p.part : p.segment;
   const int left = (int)(len - first < most ? len - first : most);      // this segment's tokens
   // the last part of all is only for the state behind the tokens
   if(LOCAL && first + left >= len && !role.new_state) return;
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
   T* const out = LOCAL ? nullptr : static_cast<T*>(role.o) + b * role.so.batch + h * role.so.head + at0 * role.so.token + dv0;
   const int64_t ostep = dir * role.so.token;

   // Staging: this lane's two channels of 8 tokens of keys and of values, those of one slot of a row of tokens (of two in
   // fp32): token i is st + i of the first four, st + 16 + i - 4 of the others.  Where a token or a channel is not there the
   // segment's first one is read, and what came is cleared on its way to LDS: no load waits for another,
   // and none is beyond the array.
   typedef Raw<T, 2> Pair;
   const bool has_k = wave < KJ / 64, has_v = wave >= (kLanes - VJ) / 64;
   const int pv = tid - (kLanes - VJ);
   const int kc = tid % (DK / 2) * 2, vc = pv % (DV / 2) * 2, kj = tid / (DK / 2), vj = pv / (DV / 2);
   const int kt = kj / 4 * 32 + kj % 4 * 4, vt = vj / 4 * 32 + vj % 4 * 4;
   const int64_t kstep = dir * role.sk.token, vstep = dir * role.sv.token;
   Pair kr[8], vr[8];
   auto token = [](int i) { return i < 4 ? i : i + 12; };
   // where this lane's first token of the segment is; the others are multiples of a step on, which scalar
   // code makes (as products of each lane's they took 16 clocks each)
   const T* const klane = k + kt * kstep + (kc < dk ? kc : 0);
   const T* const vlane = v + vt * vstep + (vc < dvn ? vc : 0);
   auto fetch_pair = [&](Pair& to, const T* at, const T* base, int64_t step, int t, int c, int dim, int n, int t0, int i) {
      const T* const from = t + token(i) < n ? at + (t0 + token(i)) * anew(step) : base;
      if constexpr(WHOLE) to = raw_at<T, 2>(from);
      else                to = raw_of<T, 2>(from, from, anew(dim) - c);
   };
   // tokens i of chunk t0
   auto fetch = [&](int t0, int i) {
      const int n = left - t0 < kChunk ? left - t0 : kChunk;
      if(has_k) fetch_pair(kr[i], klane, k, kstep, kt, kc, dk, n, t0, i);
      if(has_v) fetch_pair(vr[i], vlane, v, vstep, vt, vc, dvn, n, t0, i);
   };
   // clears what is not there
   auto clear = [&](Pair (&x)[8], int t, int c, int dim, int n) {
      const int channels = anew(dim);
#pragma unroll
      for(int i = 0; i < 8; i++) x[i].cut(t + token(i) < n ? channels - c : 0);
   };

   // this wavefront's strip of 16 tokens and half of the values; two wavefronts of a SIMD have 5 of the
   // 8 strips' blocks of scores between them
   const int strip = wave < 4 ? wave : 7 - wave, half = wave >> 2;
   const int v0 = half * (DV / 2), k0 = (wave & 3) * (DK / 4);
   T* const olane = out + (strip * 16 + row) * ostep;
   constexpr int N = 16 / (int)sizeof(E);                       // values of a piece of an operand
   Raw<T, N> qr[NK];
   const int64_t qstep = dir * role.sq.token;
   const T* const qlane = q + (strip * 16 + row) * qstep + g * N;
   auto fetch_q = [&](int t0, int from_block, int to_block) {
      const int channels = anew(dk);
      const bool there = t0 + strip * 16 + row < left;          // else any row: its results are not kept
      const T* const at = there ? qlane + t0 * anew(qstep) : q + g * N;
#pragma unroll
      for(int i = from_block; i < to_block; i++) {
         const int c = i * BLOCK + g * N;
         const T* const from = at + (c < channels ? i * BLOCK : -g * N);
         if constexpr(WHOLE) qr[i] = raw_at<T, N>(from);
         else                qr[i] = raw_of<T, N>(from, from, channels - c);
      }
   };
   auto operand_q = [&](int i) {
      if(dk < DK) qr[i].cut(anew(dk) - i * BLOCK - g * N);
      Plain f;
      if constexpr(sizeof(E) == sizeof(T)) {
         f = __builtin_bit_cast(Plain, qr[i]);
      } else {
#pragma unroll
         for(int j = 0; j < N; j++) f[j] = (E)qr[i].value(j);
      }
      return f;
   };

   // weights of keys on their way into the state; those of tokens that are not there meet zeros
   const int late = role.late;
   const float kv_scale = role.kv_scale;
   float wk[8];
   auto key_weights = [&](int n) {
#pragma unroll
      for(int i = 0; i < 8; i++) {
         const int d = n - 1 - kt - token(i) + late;
         wk[i] = power(g2, (float)(d < 0 ? 0 : d)) * kv_scale;
      }
   };
   key_weights(kChunk);

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
      wq = power(g2, (float)(strip * 16 + row + 1 - late)) * role.out_scale;
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
            for(int r = 0; r < 4; r++)
               if(j < cols && i + r < rows) body(a, c, r, at + r * step);
         }
   };
   const float* const from = LOCAL ? nullptr
                             : p.segments > 1 ? role.work + (first / p.part * p.pairs + bh) * count
                             : role.state ? role.state + bh * count : nullptr;
   float* const behind = LOCAL ? role.work + (seg * p.pairs + bh) * count
                         : role.new_state && first + left >= len ? role.new_state + bh * count : nullptr;
#pragma unroll
   for(int a = 0; a < SA; a++)
#pragma unroll
      for(int c = 0; c < SB; c++) S[a][c] = f32x4{};
   if(from) each_state(p.segments > 1 ? false : role.turned, [&](int a, int c, int r, int at) { S[a][c][r] = from[at]; });

   if(left > 0) {
#pragma unroll
      for(int i = 0; i < 8; i++) fetch(0, i);
      if constexpr(!LOCAL) fetch_q(0, 0, NK);
   }
   if(tid < 2) flags[tid] = 0;
   __syncthreads();
   int side = 0;
   for(int t0 = 0; t0 < left; t0 += kChunk, side ^= 1) {
      const int n = left - t0 < kChunk ? left - t0 : kChunk;
      // to LDS: values and weighted keys by channel, keys as they are, the state by value
      auto put_tokens = [&](int base, int row, int slot, const float (&x)[8]) {
         uint8_t* const to = lds + base + row * TP;
         if constexpr(sizeof(E) == 4) {
            *reinterpret_cast<f32x4*>(to + (slot ^ turn(row)) * 16) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(to + ((slot + 4) ^ turn(row)) * 16) = f32x4{x[4], x[5], x[6], x[7]};
         } else {
            bf16x8 e;
#pragma unroll
            for(int i = 0; i < 8; i++) e[i] = (bf16)x[i];
            *reinterpret_cast<bf16x8*>(to + (slot ^ turn(row)) * 16) = e;
         }
      };
      if(has_v) {
         if(n < kChunk || dvn < DV) clear(vr, vt, vc, dvn, n);
         if(!LOCAL && odd_one(vr)) flags[side] = 1;
         if constexpr(std::is_same<T, bf16>::value) {
#pragma unroll
            for(int j = 0; j < 2; j++) {
               mx4::u32x4 e;
#pragma unroll
               for(int i = 0; i < 4; i++) e[i] = __builtin_amdgcn_perm(vr[2 * i + 1].w[0], vr[2 * i].w[0], j ? 0x07060302 : 0x05040100);
               *reinterpret_cast<mx4::u32x4*>(lds + M::VALUES + (vc + j) * TP + (slot_of<E>(vt) ^ turn(vc + j)) * 16) = e;
            }
         } else {
#pragma unroll
            for(int j = 0; j < 2; j++) {
               float x[8];
#pragma unroll
               for(int i = 0; i < 8; i++) x[i] = vr[i].value(j);
               put_tokens(M::VALUES, vc + j, slot_of<E>(vt), x);
               if constexpr(C::PARTS == 2) {
                  rest(x);
                  put_tokens(M::VALUES + DV * TP, vc + j, slot_of<E>(vt), x);
               }
            }
         }
      }
      if(has_k) {
         if(n < kChunk || dk < DK) clear(kr, kt, kc, dk, n);
         if constexpr(!LOCAL) {
            uint8_t* const plain = lds + M::KEYS + kt * KP + kc * (int)sizeof(E);
#pragma unroll
            for(int i = 0; i < 8; i++) {
               if constexpr(sizeof(E) == 2) *reinterpret_cast<uint32_t*>(plain + token(i) * KP) = kr[i].w[0];
               else *reinterpret_cast<mx4::f32x2*>(plain + token(i) * KP) = mx4::f32x2{kr[i].value(0), kr[i].value(1)};
            }
         }
         if(n < kChunk) key_weights(n);
#pragma unroll
         for(int j = 0; j < 2; j++) {
            float x[8];
#pragma unroll
            for(int i = 0; i < 8; i++) x[i] = kr[i].value(j) * wk[i];
            put_tokens(M::KEYS_T, kc + j, slot_of<E>(kt), x);
#pragma unroll
            for(int part = 1; part < M::KEY_PARTS; part++) {
               rest(x);
               put_tokens(M::KEYS_T + part * DK * TP, kc + j, slot_of<E>(kt), x);
            }
         }
      }
      if constexpr(!LOCAL) {
         uint8_t* const to = lds + M::STATE + (v0 + row) * KP + (k0 + g * 4) * (int)sizeof(E);
#pragma unroll
         for(int a = 0; a < SA; a++)
#pragma unroll
            for(int c = 0; c < SB; c++) {
               float x[4] = {S[a][c][0], S[a][c][1], S[a][c][2], S[a][c][3]};
               put4<E>(to + c * 16 * KP + a * 16 * (int)sizeof(E), x);
               if constexpr(C::MADE == 2) {
                  rest(x);
                  put4<E>(to + (DV + c * 16) * KP + a * 16 * (int)sizeof(E), x);
               }
            }
      }
      Plain qf[NK];
      if constexpr(!LOCAL) {
#pragma unroll
         for(int i = 0; i < NK; i++) qf[i] = operand_q(i);
      }
      __syncthreads();
      const bool special = flags[side] != 0;
      if(tid == 0) flags[side ^ 1] = 0;
      auto key_frag = [&](int r, int block) {
         return *reinterpret_cast<const Plain*>(lds + M::KEYS + (r + row) * KP + (block * 4 + g) * 16);
      };
      auto state_frag = [&](int r, int block) {
         return *reinterpret_cast<const Frag*>(lds + M::STATE + (r + row) * KP + (block * 4 + g) * 16);
      };
      auto token_frag = [&](int base, int r, int block) {       // of a row of tokens, r a multiple of 16
         return *reinterpret_cast<const Frag*>(lds + base + (r + row) * TP + ((block * 4 + g) ^ turn(row)) * 16);
      };
      // The next chunk's loads go out between the products, a few at a time: a CU takes in 9 bytes a clock at most, and
      // a wavefront that issues more than are on their way stands still (all 16 at once: 3600 clocks).
      const int t1 = t0 + kChunk;
      const bool more = t1 < left;
      auto fetch_some = [&](int from, int to) {
         __builtin_amdgcn_sched_barrier(0);
         if(more)
#pragma unroll
            for(int i = from; i < to; i++) fetch(t1, i);
         __builtin_amdgcn_sched_barrier(0);
      };
      if constexpr(LOCAL) fetch_some(0, 8);

      if constexpr(!LOCAL) {
         f32x4 o[SB] = {};
#pragma unroll
         for(int i = 0; i < NK; i++) {
            Frag x[SB][C::MADE], qs[C::PARTS];
#pragma unroll
            for(int c = 0; c < SB; c++)
#pragma unroll
               for(int part = 0; part < C::MADE; part++) x[c][part] = state_frag(part * DV + v0 + c * 16, i);
            if constexpr(C::PARTS == 1) {
               qs[0] = qf[i];
            } else {
#pragma unroll
               for(int j = 0; j < N; j++) {
                  const float whole = (float)qf[i][j];
                  qs[0][j] = (bf16)whole;
                  qs[1][j] = (bf16)(whole - (float)(bf16)whole);
               }
            }
#pragma unroll
            for(int c = 0; c < SB; c++) o[c] = mma_parts<C>(x[c], qs, o[c]);
            fetch_some(i * 4 / NK, (i + 1) * 4 / NK);
         }
#pragma unroll
         for(int c = 0; c < SB; c++) o[c] *= wq;
         const int reach = anew_lane(strip * 16 + row - g * 4);      // scores of tokens up to this plus 4 g count
#pragma unroll
         for(int sb = 0; sb < NS; sb++) {
            fetch_some(4 + sb * 4 / NS, 4 + (sb + 1) * 4 / NS);
            if(sb * EACH > strip) continue;
            f32x4 s[EACH];
            Plain kf[EACH][NK];
            Frag vf[SB][C::PARTS];
#pragma unroll
            for(int e = 0; e < EACH; e++)
#pragma unroll
               for(int i = 0; i < NK; i++) kf[e][i] = key_frag((sb * EACH + e) * 16, i);
#pragma unroll
            for(int c = 0; c < SB; c++)
#pragma unroll
               for(int part = 0; part < C::PARTS; part++) vf[c][part] = token_frag(M::VALUES, part * DV + v0 + c * 16, sb);
#pragma unroll
            for(int e = 0; e < EACH; e++) s[e] = f32x4{};
#pragma unroll
            for(int i = 0; i < NK; i++)
#pragma unroll
               for(int e = 0; e < EACH; e++) s[e] = C::scores(kf[e][i], qf[i], s[e]);
#pragma unroll
            for(int e = 0; e < EACH; e++) {
               const int tile = sb * EACH + e;
#pragma unroll
               for(int r = 0; r < 4; r++) s[e][r] *= wt[tile][r];
               // tokens behind t have no part in it, whatever they hold
               if(tile >= strip)
#pragma unroll
                  for(int r = 0; r < 4; r++) s[e][r] = tile * 16 + r <= reach ? s[e][r] : 0.0f;
            }
            Frag w[C::MADE];
#pragma unroll
            for(int e = 0; e < EACH; e++)
#pragma unroll
               for(int r = 0; r < 4; r++) {
                  w[0][e * 4 + r] = (E)s[e][r];
                  if constexpr(C::MADE == 2) w[1][e * 4 + r] = (E)(s[e][r] - (float)(E)s[e][r]);
               }
            if(!special) {
#pragma unroll
               for(int c = 0; c < SB; c++) o[c] = mma_parts<C>(vf[c], w, o[c]);
            } else {
               // A value that is infinite or NaN times a weight of zero would reach tokens before it.  Such values
               // are left out of the products, and added one by one to the results that they belong to.
#pragma unroll
               for(int c = 0; c < SB; c++) {
#pragma unroll
                  for(int part = 0; part < C::PARTS; part++)
#pragma unroll
                     for(int i = 0; i < EACH * 4; i++)
                        vf[c][part][i] = fabsf((float)vf[c][part][i]) < __builtin_inff() ? vf[c][part][i] : (E)0.0f;
                  o[c] = mma_parts<C>(vf[c], w, o[c]);
               }
#pragma unroll
               for(int i = 0; i < EACH * 4; i++)
#pragma unroll 1
                  for(int from_g = 0; from_g < 4; from_g++) {
                     const int s1 = sb * BLOCK + (i / 4) * 16 + from_g * 4 + i % 4;
                     const float weight = __shfl(s[i / 4][i % 4], row + from_g * 16);
                     if(s1 > strip * 16 + row) continue;
#pragma unroll
                     for(int c = 0; c < SB; c++)
#pragma unroll
                        for(int r = 0; r < 4; r++) {
                           const int channel = v0 + c * 16 + g * 4 + r;
                           const float x = (float)*reinterpret_cast<const E*>(
                              lds + M::VALUES + channel * TP + (slot_of<E>(s1) ^ turn(channel)) * 16 + in_slot<E>(s1));
                           if(!(fabsf(x) < __builtin_inff())) o[c][r] += weight * x;
                        }
                  }
            }
         }
         const int t = strip * 16 + row;
         if(t < n) {
            const int d = anew(dvn);
            T* const to = olane + t0 * anew(ostep);
            struct __attribute__((packed, aligned(sizeof(T)))) Four { T e[4]; };
#pragma unroll
            for(int c = 0; c < SB; c++) {
               const int j = v0 + c * 16 + g * 4;
               Four x;
#pragma unroll
               for(int r = 0; r < 4; r++) x.e[r] = (T)o[c][r];
               if constexpr(WHOLE) {
                  if(j < d) *reinterpret_cast<Four*>(to + j) = x;
               } else {
#pragma unroll
                  for(int r = 0; r < 4; r++)
                     if(j + r < d) to[j + r] = x.e[r];
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
         Frag x[SB][C::PARTS], w[SA][M::KEY_PARTS];
         if constexpr(!LOCAL)
            if(more) fetch_q(t1, sb * NK / NS, (sb + 1) * NK / NS);
#pragma unroll
         for(int c = 0; c < SB; c++)
#pragma unroll
            for(int part = 0; part < C::PARTS; part++) x[c][part] = token_frag(M::VALUES, part * DV + v0 + c * 16, sb);
#pragma unroll
         for(int a = 0; a < SA; a++)
#pragma unroll
            for(int part = 0; part < M::KEY_PARTS; part++) w[a][part] = token_frag(M::KEYS_T, part * DK + k0 + a * 16, sb);
#pragma unroll
         for(int i = 0; i < M::KEY_PARTS; i++)
#pragma unroll
            for(int j = 0; j < C::PARTS; j++)
               if(i + j < M::KEY_PARTS)
#pragma unroll
                  for(int a = 0; a < SA; a++)
#pragma unroll
                     for(int c = 0; c < SB; c++) S[a][c] = C::mma(w[a][i], x[c][j], S[a][c]);
      }
      __syncthreads();
   }

   if(behind) each_state(!LOCAL && role.turned, [&](int a, int c, int r, int at) { behind[at] = S[a][c][r]; });
}

// What every part of the tokens adds to the state, in work, becomes the state before that part.  A lane has one
// element of a state; eight parts are read ahead of their sums.
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
   const float a = power(g2, (float)p.part);                   // of every part but the last
   const int64_t at = bh * count + (role.turned ? e % role.dv * role.dk + e / role.dv : e);
   float s = role.state ? role.state[at] : 0.0f;
   float* const work = role.work + bh * count + e;
   const int64_t pitch = p.pairs * count, last = role.new_state ? len : len - 1;     // parts that end up to there are there
   constexpr int AHEAD = 8;
   for(int64_t seg = 0; seg < p.parts && (seg == 0 || seg * p.part < len); seg += AHEAD) {
      float part[AHEAD];
#pragma unroll
      for(int i = 0; i < AHEAD; i++) {
         const int64_t from = (seg + i) * p.part, to = from + p.part < len ? from + p.part : len;
         part[i] = from < len && to <= last ? work[(seg + i) * pitch] : 0.0f;
      }
#pragma unroll
      for(int i = 0; i < AHEAD; i++) {
         const int64_t from = (seg + i) * p.part;
         if(seg + i < p.parts && (seg + i == 0 || from < len)) work[(seg + i) * pitch] = s;
         if(from < len) s = (from + p.part <= len ? a : power(g2, (float)(len - from))) * s + part[i];
      }
   }
   if(role.new_state) role.new_state[at] = s;
}

// ---- one token ------------------------------------------------------------------------------
//
// A workgroup has 4 LANES values of one sequence and head: LANES lanes of 4 values, 256 / LANES rows of the state at
// a time, all of them on their way at once.  Bound by the state's bytes, read and written once.  Every workgroup
// looks for its slot among those of the earlier sequences, which is nothing beside states of 128 x 128 (128 sequences x 32 heads 79 us without
// slots, 81 with; 4096 x 8 853 / 858) and is felt by small ones of very many sequences (1024 x 8 heads of 16 x 16 15 / 17,
// 4096 x 8 of them 49 / 80, 16384 x 4 of 64 x 64 394 / 588).
constexpr int kStepLanes = 256;

// WHOLE: values in whole fours.  What is not there is read at its row's or column's first place instead, and not written.
template<class T, int LANES, bool WHOLE>
__global__ void __launch_bounds__(kStepLanes)
decay_step(StepParams p)
{
   constexpr int ROWS = kStepLanes / LANES, PASSES = 128 / ROWS;       // dk up to 128
   __shared__ float join[kStepLanes / 64][LANES * 4];
   __shared__ int taken;
   const int tid = threadIdx.x, c = tid % LANES, r0 = tid / LANES;
   const int64_t b = blockIdx.x / (p.heads * p.slices), rest = blockIdx.x % (p.heads * p.slices);
   const int64_t h = rest / p.slices;
   const int first = (int)(rest % p.slices) * LANES * 4, j0 = first + c * 4;
   T* const out = static_cast<T*>(p.out) + b * p.so.batch + h * p.so.head + first;
   const int64_t slot = p.slots ? p.slots[b] : b;
   if(slot < 0 || slot >= p.slot_count) {
      if(tid < LANES * 4 && first + tid < p.dv) out[tid] = (T)0.0f;
      return;
   }
   float* const state = p.state + (slot * p.heads + h) * p.dk * p.dv;
   const T* const q = static_cast<const T*>(p.q) + b * p.sq.batch + h * p.sq.head;
   const T* const k = static_cast<const T*>(p.k) + b * p.sk.batch + h * p.sk.head;
   const T* const v = static_cast<const T*>(p.v) + b * p.sv.batch + h * p.sv.head;
   int at[4];                                              // columns
#pragma unroll
   for(int e = 0; e < 4; e++) at[e] = WHOLE ? (j0 < p.dv ? j0 : 0) + e : j0 + e < p.dv ? j0 + e : 0;
   f32x4 s[PASSES];
   T kk[PASSES], qq[PASSES];
#pragma unroll
   for(int i = 0; i < PASSES; i++) {
      const int r = r0 + i * ROWS < p.dk ? r0 + i * ROWS : 0;
      if constexpr(WHOLE) {
         typedef float V __attribute__((ext_vector_type(4), aligned(4)));
         s[i] = *reinterpret_cast<const V*>(state + r * p.dv + at[0]);
      } else {
#pragma unroll
         for(int e = 0; e < 4; e++) s[i][e] = state[r * p.dv + at[e]];
      }
      kk[i] = k[r];
      qq[i] = q[r];
   }
   float vv[4];
#pragma unroll
   for(int e = 0; e < 4; e++) vv[e] = (float)v[at[e]];
   // whether an earlier sequence has the same state
   bool mine = true;
   if(p.slots) {
      if(tid == 0) taken = 0;
      __syncthreads();
      bool found = false;
      for(int64_t i = tid; i < b; i += kStepLanes) found |= p.slots[i] == slot;
      if(found) taken = 1;
      __syncthreads();
      mine = !taken;
   }
   const float a = expf(p.log_decay[h]);
   float acc[4] = {};
#pragma unroll
   for(int i = 0; i < PASSES; i++) {
      const bool there = r0 + i * ROWS < p.dk;
#pragma unroll
      for(int e = 0; e < 4; e++) {
         s[i][e] = a * s[i][e] + (float)kk[i] * vv[e];
         acc[e] += there ? (float)qq[i] * s[i][e] : 0.0f;
      }
      if(mine && there) {
         float* const to = state + (r0 + i * ROWS) * p.dv;
         if constexpr(WHOLE) {
            typedef float V __attribute__((ext_vector_type(4), aligned(4)));
            if(j0 < p.dv) *reinterpret_cast<V*>(to + j0) = s[i];
         } else {
#pragma unroll
            for(int e = 0; e < 4; e++)
               if(j0 + e < p.dv) to[j0 + e] = s[i][e];
         }
      }
   }
   // the rows' sums: of a wavefront's lanes, then of the wavefronts in their order
#pragma unroll
   for(int e = 0; e < 4; e++)
#pragma unroll
      for(int by = LANES; by < 64; by *= 2) acc[e] += __shfl_xor(acc[e], by);
   if((tid & 63) < LANES)
#pragma unroll
      for(int e = 0; e < 4; e++) join[tid >> 6][c * 4 + e] = acc[e];
   __syncthreads();
   if(tid < LANES * 4 && first + tid < p.dv) {
      const float sum = ((join[0][tid] + join[1][tid]) + join[2][tid]) + join[3][tid];
      out[tid] = (T)(mine ? sum * p.scale : 0.0f);
   }
}

// ---- launches --------------------------------------------------------------------------------

template<class T, int DK, int DV, bool LOCAL, bool WHOLE, bool FINE>
hipError_t chunks_shape(DecayParams p, int roles, hipStream_t s)
{
   constexpr int bytes = Room<T, DK, DV, LOCAL, FINE>::BYTES;
   static_assert(bytes <= 160 * 1024, "fits the LDS");
   static std::atomic<uint64_t> mask{0};
   const hipError_t e = ensure_dynamic_lds(reinterpret_cast<const void*>(&decay_chunks<T, DK, DV, LOCAL, WHOLE, FINE>), bytes, mask);
   if(e != hipSuccess) return e;
   int most = 0;
   for(int r = 0; r < roles; r++) most = p.role[r].dv > most ? p.role[r].dv : most;
   p.slices = (most + DV - 1) / DV;
   p.items = p.pairs * (LOCAL ? p.parts : p.segments);         // the last part: where its sum is asked for
   const int64_t groups = (p.items + 7) / 8 * 8 * p.slices;
   if(!grid_ok(groups, kLanes)) return kTooLarge;
   decay_chunks<T, DK, DV, LOCAL, WHOLE, FINE><<<dim3((unsigned)groups, (unsigned)roles), kLanes, bytes, s>>>(p);
   return hipGetLastError();
}

template<class T, int DK, int DV, bool WHOLE, bool FINE>
hipError_t segments_launches(DecayParams p, int roles, hipStream_t s)
{
   // Segments so that each CU has a workgroup, where that pays, with a chunk's time in the last launch for a unit: a chunk in the
   // first launch half of it, the state of every part, which is written, read, written and read, 2.5 times its share of a
   // chunk's bytes in bf16, the launches 2; in the other types 5 and 3.5 (128 channels, out with its state, us unsplit / split.  bf16: 64
   // pairs of a sequence and a head 32 chunks 181 / 93, 8 chunks 48 / 42, 4 chunks 28 / 34; 85 pairs 32 chunks 181 / 117; 128 pairs 32 chunks
   // 188 / 169, 16 chunks 98 / 98, 8 chunks 48 / 62.  fp16: 64 pairs 32 chunks 154 / 105, 8 chunks 43 / 45; 128 pairs 32
   // chunks 159 / 194).
   // A segment of many chunks is two parts in the first launch, which has room for more workgroups on
   // a CU (65536 tokens x 16 heads: 197 us in one part, 152 in 3, 142 in 2).
   const int64_t chunks = (p.tokens + kChunk - 1) / kChunk;
   const int64_t groups = p.pairs * roles * ((p.role[0].dv + DV - 1) / DV);
   constexpr bool BF16 = std::is_same<T, bf16>::value;          // in halves of a chunk:
   constexpr int64_t STATES = (BF16 ? 5 : 10) * (4 * DK * DV) / (2 * kChunk * (DK + DV) * (int)sizeof(T)), LAUNCHES = BF16 ? 4 : 7;
   int64_t n = 256 / (groups > 0 ? groups : 1);
   if(n > p.splits) n = p.splits;
   if(n > chunks) n = chunks;
   if(n < 2 || 3 * ((chunks + n - 1) / n) + LAUNCHES + STATES >= 2 * chunks) n = 1;
   const int64_t parts = p.splits / n >= 2 && chunks / n >= 16 ? 2 : 1;
   const int64_t each = chunks > 0 ? (chunks + n * parts - 1) / (n * parts) : 1;       // chunks of a part
   p.part = each * kChunk;
   p.segment = p.part * parts;
   p.parts = chunks > 0 ? (chunks + each - 1) / each : 1;
   p.segments = (p.parts + parts - 1) / parts;
   // two parts of everything and three of the keys of 128 values leave neither registers nor LDS
   constexpr int ONE = Cores<T>::PARTS == 2 && FINE ? 64 : DV;
   if(p.segments == 1) return chunks_shape<T, DK, ONE, false, WHOLE, FINE>(p, roles, s);
   hipError_t e = chunks_shape<T, DK, DV, true, WHOLE, FINE>(p, roles, s);
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
   // the state behind the tokens is there, from the parts' sums
   for(int r = 0; r < roles; r++) p.role[r].new_state = nullptr;
   return chunks_shape<T, DK, DV, false, WHOLE, false>(p, roles, s);
}

// WHOLE: heads of whole groups of 8 channels.  Two parts of everything leave neither registers nor LDS for 128 values
// of other heads.
template<class T, int DK, int DV, bool FINE>
hipError_t chunks_fine(const DecayParams& p, int roles, hipStream_t s)
{
   const bool whole = p.role[0].dk % 8 == 0 && p.role[0].dv % 8 == 0;
   if(whole) return segments_launches<T, DK, DV, true, FINE>(p, roles, s);
   return segments_launches<T, DK, Cores<T>::PARTS == 2 ? 64 : DV, false, FINE>(p, roles, s);
}
template<class T, int DK, int DV>
hipError_t chunks_launches(const DecayParams& p, int roles, hipStream_t s)
{
   if constexpr(Cores<T>::FINE_PARTS > 1)
      for(int r = 0; r < roles; r++)
         if(p.role[r].new_state) return chunks_fine<T, DK, DV, true>(p, roles, s);
   return chunks_fine<T, DK, DV, false>(p, roles, s);
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

namespace {

template<class T, int LANES>
hipError_t step_shape(StepParams p, hipStream_t s)
{
   p.slices = (p.dv + LANES * 4 - 1) / (LANES * 4);
   const int64_t groups = p.batch * p.heads * p.slices;
   if(!grid_ok(groups, kStepLanes)) return kTooLarge;
   if(p.dv % 4 == 0) decay_step<T, LANES, true><<<(unsigned)groups, kStepLanes, 0, s>>>(p);
   else              decay_step<T, LANES, false><<<(unsigned)groups, kStepLanes, 0, s>>>(p);
   return hipGetLastError();
}

// Whole rows of the state a workgroup where there are states enough for all CUs, else 32 values.
template<class T>
hipError_t step_typed(const StepParams& p, hipStream_t s)
{
   if(p.dv <= 32 || p.batch * p.heads < 512) return step_shape<T, 8>(p, s);
   return p.dv <= 64 ? step_shape<T, 16>(p, s) : step_shape<T, 32>(p, s);
}

}  // namespace

hipError_t launch_decay_step(const StepParams& p, hipStream_t s)
{
   if(p.batch <= 0 || p.heads <= 0) return hipSuccess;
   switch(p.type) {
      case T_F32:  return step_typed<float>(p, s);
      case T_BF16: return step_typed<bf16>(p, s);
      default:     return step_typed<f16>(p, s);
   }
}

}  // namespace layer
}  // namespace fufft
