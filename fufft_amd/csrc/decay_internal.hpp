// Internal interface between the entry points of the decaying-attention calls
// (decay_capi.hip) and their kernels (decay.hip).
#pragma once

#include "layer_internal.hpp"

namespace fufft {
namespace layer {

constexpr int64_t kWidestHead = 128, kLongestText = (int64_t)1 << 30;

// in elements; the elements of a head are adjacent
struct Strides {
   int64_t batch, token, head;
};

// One use of the chunked sums: q, k and v stand for what takes their place in it.
struct DecayRole {
   const void*  q;
   const void*  k;
   const void*  v;
   void*        o;
   Strides      sq, sk, sv, so;
   const float* state;       // batch x heads x dk x dv, or dv x dk where turned; or NULL
   float*       new_state;   // the same, or NULL
   float*       work;        // parts x batch x heads x dk x dv
   int          dk, dv;
   int          turned;
   int          reverse;     // from the last token back
   int          late;        // the state given meets its first token undecayed, the one returned is decayed once more
   float        p_scale, kv_scale, out_scale;    // of scores, of what goes to the state, of results
};

struct DecayParams {
   DecayRole      role[3];
   const float*   log_decay;
   const int32_t* lens;      // or NULL
   int64_t        pairs;     // batch x heads
   int64_t        heads, tokens, splits;
   int64_t        segment, segments, part, parts, items, slices;     // set by the launch
   int            type;
};
hipError_t launch_decay(const DecayParams& p, int roles, hipStream_t s);

struct StepParams {
   const void*    q;
   const void*    k;
   const void*    v;
   void*          out;
   Strides        sq, sk, sv, so;
   const float*   log_decay;
   float*         state;     // slot_count x heads x dk x dv
   const int64_t* slots;     // or NULL
   int64_t        slot_count, batch, heads, slices;
   int            dk, dv, type;
   float          scale;
};
hipError_t launch_decay_step(const StepParams& p, hipStream_t s);

}  // namespace layer
}  // namespace fufft
