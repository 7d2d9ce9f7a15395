// Entry points of the decaying-attention calls: argument checks and dispatch.
// Declarations in include/fufft/fufft.h.
#include "decay_internal.hpp"
#include "mx4_arguments.hpp"

using namespace fufft::mx4;
using namespace fufft::layer;

namespace {

// One axis of an array: how many, how far apart (elements).
struct Axis {
   int64_t count, stride;
};
// A strided array: its axes from the widest stride to the narrowest, without those of one place; a
// row of `dim` adjacent elements at each place.
struct Array {
   const void* p;
   int64_t     element, dim;
   Axis        axis[3];
   int         axes;
   int64_t     places;
};

bool array_of(const void* p, int type, const fufft_strides* s, int64_t batch, int64_t tokens, int64_t heads, int64_t dim,
              Array* a)
{
   *a = Array{p, type_bytes(type), dim, {}, 0, batch * tokens * heads};
   if(!s) return a->places == 0;
   const Axis all[3] = {{batch, s->batch}, {tokens, s->token}, {heads, s->head}};
   for(const Axis& x : all) {
      if(!size_ok(x.stride) || !volume_ok(x.count, x.stride, 8)) return false;
      if(x.count == 1) continue;
      int at = a->axes++;
      while(at > 0 && a->axis[at - 1].stride < x.stride) {
         a->axis[at] = a->axis[at - 1];
         at--;
      }
      a->axis[at] = x;
   }
   return true;
}
// elements from the first to the last of the part of an array below its axis i
int64_t extent(const Array& a, int i)
{
   int64_t n = a.dim;
   for(int j = i; j < a.axes; j++) n += (a.axis[j].count - 1) * a.axis[j].stride;
   return n;
}
Span span_of(const Array& a) { return {a.p, a.places > 0 ? extent(a, 0) * a.element : 0}; }
// no element at two places
bool distinct(const Array& a)
{
   for(int i = 0; i < a.axes; i++)
      if(a.axis[i].stride < extent(a, i + 1)) return false;
   return true;
}
// Whether the parts below axis i of two arrays share nothing, the second one's `by` elements behind the first
// one's: far from each other, or, along an axis that both step through alike, each in the gaps of the other (parts
// of one row a token, whose heads may have other widths).  Parts longer than that step, which reach over several
// of the other's, are not taken.
bool parts_apart(const Array& a, const Array& b, int i, int64_t by)
{
   const int64_t wa = extent(a, i), wb = extent(b, i);
   if(by >= wa || by + wb <= 0) return true;
   if(i >= a.axes || i >= b.axes || a.axis[i].stride != b.axis[i].stride) return false;
   const int64_t s = a.axis[i].stride;
   const int64_t pa = extent(a, i + 1), pb = extent(b, i + 1);
   if(pa > s || pb > s) return false;
   // the second's first part in a step of the first: parts of at most a step meet that step's part and the next one's only
   const int64_t r = (by % s + s) % s;
   if(r < pa && !parts_apart(a, b, i + 1, r)) return false;
   return r + pb <= s || parts_apart(a, b, i + 1, r - s);
}
bool arrays_apart(const Array& a, const Array& b)
{
   if(disjoint(span_of(a), span_of(b))) return true;
   const int64_t bytes = static_cast<const char*>(b.p) - static_cast<const char*>(a.p);
   return a.element == b.element && bytes % a.element == 0 && parts_apart(a, b, 0, bytes / a.element);
}

Strides strides_of(const fufft_strides* s) { return s ? Strides{s->batch, s->token, s->head} : Strides{}; }

struct Sizes {
   int64_t batch, tokens, heads, dk, dv;
   bool    ok() const
   {
      return size_ok(batch) && size_ok(tokens) && size_ok(heads) && dk >= 1 && dv >= 1 && size_ok(dk) && size_ok(dv) &&
             volume_ok(batch, tokens, heads) && volume_ok(batch * heads, dk * 16, dv);
   }
   bool empty() const { return batch == 0 || heads == 0; }
   int64_t state_bytes(int64_t count = 1) const { return count * batch * heads * dk * dv * 4; }
};

// A small list of what a call reads and writes, and the checks of all of it.
struct Buffers {
   Array arrays[7];
   bool  written[7];
   int   count = 0;
   Span  flat[8];
   bool  flat_written[8];
   int   flats = 0;
   int   status = FUFFT_OK;

   void array(const void* p, int type, const fufft_strides* s, const Sizes& z, int64_t dim, bool out)
   {
      Array a;
      if(status != FUFFT_OK) return;
      if(!array_of(p, type, s, z.batch, z.tokens, z.heads, dim, &a) || (a.places > 0 && !p) || (out && !distinct(a))) {
         status = FUFFT_ERR_INVALID;
         return;
      }
      if(a.places == 0) return;
      if(!aligned(p, (uintptr_t)a.element)) {
         status = FUFFT_ERR_ALIGN;
         return;
      }
      arrays[count] = a;
      written[count++] = out;
   }
   // the number of the buffer among the flat ones
   int bytes(const void* p, int64_t n, uintptr_t align, bool out)
   {
      if(status != FUFFT_OK) return -1;
      const Span s{p, n};
      status = span_status(s, align);
      flat[flats] = s;
      flat_written[flats] = out;
      return flats++;
   }
   // Outputs share no byte with anything else, but for one pair of flat buffers of a size, by their numbers, that may start at one address.
   int check(int pair_a = -1, int pair_b = -1) const
   {
      if(status != FUFFT_OK) return status;
      for(int i = 0; i < count; i++) {
         for(int j = 0; j < i; j++)
            if((written[i] || written[j]) && !arrays_apart(arrays[i], arrays[j])) return FUFFT_ERR_INVALID;
         for(int j = 0; j < flats; j++)
            if((written[i] || flat_written[j]) && !disjoint(span_of(arrays[i]), flat[j])) return FUFFT_ERR_INVALID;
      }
      for(int i = 0; i < flats; i++)
         for(int j = 0; j < i; j++) {
            if(!flat_written[i] && !flat_written[j]) continue;
            const bool pair = i == pair_b && j == pair_a && flat[i].p == flat[j].p;
            if(!pair && !disjoint(flat[i], flat[j])) return FUFFT_ERR_INVALID;
         }
      return FUFFT_OK;
   }
};

// work and its number of splits, for `sets` states of each
bool splits_ok(const Sizes& z, int64_t splits, int64_t sets) { return size_ok(splits) && volume_ok(splits, z.state_bytes(sets)); }

}  // namespace

extern "C" {

int fufft_decay_attention(const void* q, const fufft_strides* q_strides, const void* k, const fufft_strides* k_strides,
                          const void* v, const fufft_strides* v_strides, int type, const float* log_decay, void* out,
                          const fufft_strides* out_strides, const float* state, float* new_state, const int32_t* lens,
                          float scale, int64_t batch, int64_t tokens, int64_t heads, int64_t dk, int64_t dv, float* work,
                          int64_t splits, void* stream)
{
   const Sizes z{batch, tokens, heads, dk, dv};
   if(!type_ok(type) || !z.ok() || !splits_ok(z, splits, 1)) return FUFFT_ERR_INVALID;
   if(z.empty()) return FUFFT_OK;
   Buffers all;
   all.array(q, type, q_strides, z, dk, false);
   all.array(k, type, k_strides, z, dk, false);
   all.array(v, type, v_strides, z, dv, false);
   all.array(out, type, out_strides, z, dv, true);
   all.bytes(log_decay, heads * 4, 4, false);
   const int before = all.bytes(state, state ? z.state_bytes() : 0, 4, false);
   const int behind = all.bytes(new_state, new_state ? z.state_bytes() : 0, 4, true);
   all.bytes(lens, lens ? batch * 4 : 0, 4, false);
   all.bytes(work, z.state_bytes(splits), 4, true);
   FUFFT_MX4_CHECK(all.check(before, behind));
   if(dk > kWidestHead || dv > kWidestHead || tokens > kLongestText) return FUFFT_ERR_UNSUPPORTED;
   DecayParams p{};
   p.role[0] = DecayRole{q, k, v, out, strides_of(q_strides), strides_of(k_strides), strides_of(v_strides), strides_of(out_strides),
                         state, new_state, work, (int)dk, (int)dv, 0, 0, 0, 1.0f, 1.0f, scale};
   p.log_decay = log_decay;
   p.lens = lens;
   p.pairs = batch * heads;
   p.heads = heads;
   p.tokens = tokens;
   p.splits = splits;
   p.type = type;
   return status_of(launch_decay(p, 1, static_cast<hipStream_t>(stream)));
}

int fufft_decay_attention_grad(const void* dout, const fufft_strides* dout_strides, const void* q,
                               const fufft_strides* q_strides, const void* k, const fufft_strides* k_strides, const void* v,
                               const fufft_strides* v_strides, int type, const float* log_decay, void* dq,
                               const fufft_strides* dq_strides, void* dk_out, const fufft_strides* dk_strides, void* dv_out,
                               const fufft_strides* dv_strides, const float* state, const float* dnew_state, float* dstate,
                               const int32_t* lens, float scale, int64_t batch, int64_t tokens, int64_t heads, int64_t dk,
                               int64_t dv, float* work, int64_t splits, void* stream)
{
   const Sizes z{batch, tokens, heads, dk, dv};
   if(!type_ok(type) || !z.ok() || !splits_ok(z, splits, 3)) return FUFFT_ERR_INVALID;
   if(z.empty()) return FUFFT_OK;
   Buffers all;
   all.array(dout, type, dout_strides, z, dv, false);
   all.array(q, type, q_strides, z, dk, false);
   all.array(k, type, k_strides, z, dk, false);
   all.array(v, type, v_strides, z, dv, false);
   all.array(dq, type, dq_strides, z, dk, true);
   all.array(dk_out, type, dk_strides, z, dk, true);
   all.array(dv_out, type, dv_strides, z, dv, true);
   all.bytes(log_decay, heads * 4, 4, false);
   all.bytes(state, state ? z.state_bytes() : 0, 4, false);
   all.bytes(dnew_state, dnew_state ? z.state_bytes() : 0, 4, false);
   all.bytes(dstate, dstate ? z.state_bytes() : 0, 4, true);
   all.bytes(lens, lens ? batch * 4 : 0, 4, false);
   all.bytes(work, z.state_bytes(splits * 3), 4, true);
   FUFFT_MX4_CHECK(all.check());
   if(dk > kWidestHead || dv > kWidestHead || tokens > kLongestText) return FUFFT_ERR_UNSUPPORTED;
   const Strides sd = strides_of(dout_strides), sq = strides_of(q_strides), sk = strides_of(k_strides), sv = strides_of(v_strides);
   const int64_t set = splits * batch * heads * dk * dv;
   DecayParams p{};
   // dq, from the first token on, meets the state turned; dk and dv, from the last one back, the gradient of the
   // state behind it, and dv's state ends as that of the state before it
   p.role[0] = DecayRole{dout, v, k, dq, sd, sv, sk, strides_of(dq_strides), state, nullptr, work,
                         (int)dv, (int)dk, 1, 0, 0, 1.0f, 1.0f, scale};
   p.role[1] = DecayRole{v, dout, q, dk_out, sv, sd, sq, strides_of(dk_strides), dnew_state, nullptr, work ? work + set : nullptr,
                         (int)dv, (int)dk, 1, 1, 1, scale, scale, 1.0f};
   p.role[2] = DecayRole{k, q, dout, dv_out, sk, sq, sd, strides_of(dv_strides), dnew_state, dstate, work ? work + 2 * set : nullptr,
                         (int)dk, (int)dv, 0, 1, 1, scale, scale, 1.0f};
   p.log_decay = log_decay;
   p.lens = lens;
   p.pairs = batch * heads;
   p.heads = heads;
   p.tokens = tokens;
   p.splits = splits;
   p.type = type;
   return status_of(launch_decay(p, 3, static_cast<hipStream_t>(stream)));
}

int fufft_decay_attention_step(const void* q, const fufft_strides* q_strides, const void* k, const fufft_strides* k_strides,
                               const void* v, const fufft_strides* v_strides, int type, const float* log_decay, void* out,
                               const fufft_strides* out_strides, float* state, int64_t slot_count, const int64_t* slots,
                               float scale, int64_t batch, int64_t heads, int64_t dk, int64_t dv, void* stream)
{
   const Sizes z{batch, 1, heads, dk, dv};
   if(!type_ok(type) || !z.ok() || !size_ok(slot_count) || !volume_ok(slot_count * heads, dk * 4, dv) ||
      !volume_ok(slot_count, heads))
      return FUFFT_ERR_INVALID;
   if(z.empty()) return FUFFT_OK;
   if(!slots && slot_count < batch) return FUFFT_ERR_INVALID;
   Buffers all;
   all.array(q, type, q_strides, z, dk, false);
   all.array(k, type, k_strides, z, dk, false);
   all.array(v, type, v_strides, z, dv, false);
   all.array(out, type, out_strides, z, dv, true);
   all.bytes(log_decay, heads * 4, 4, false);
   all.bytes(state, slot_count * heads * dk * dv * 4, 4, true);
   all.bytes(slots, slots ? batch * 8 : 0, 8, false);
   FUFFT_MX4_CHECK(all.check());
   if(dk > kWidestHead || dv > kWidestHead) return FUFFT_ERR_UNSUPPORTED;
   StepParams p{};
   p.q = q;
   p.k = k;
   p.v = v;
   p.out = out;
   p.sq = strides_of(q_strides);
   p.sk = strides_of(k_strides);
   p.sv = strides_of(v_strides);
   p.so = strides_of(out_strides);
   p.log_decay = log_decay;
   p.state = state;
   p.slots = slots;
   p.slot_count = slot_count;
   p.batch = batch;
   p.heads = heads;
   p.dk = (int)dk;
   p.dv = (int)dv;
   p.type = type;
   p.scale = scale;
   return status_of(launch_decay_step(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
