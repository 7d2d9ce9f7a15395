// Checks of arguments that the entry points on matrices share: types, sizes, alignment and
// the bytes that a call reads and writes.
#pragma once

#include "mx4_internal.hpp"
#include "../../include/fufft/fufft.h"

namespace fufft {
namespace mx4 {

inline bool type_ok(int type) { return type == FUFFT_F32 || type == FUFFT_BF16 || type == FUFFT_F16; }
inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// sizes of one argument: at most 2^40, so that no product of two below overflows
inline bool size_ok(int64_t n) { return n >= 0 && n <= ((int64_t)1 << 40); }
// a x b x c within 2^62
inline bool volume_ok(int64_t a, int64_t b, int64_t c = 1)
{
   const int64_t most = (int64_t)1 << 62;
   if(a == 0 || b == 0 || c == 0) return true;
   return a <= most / b && a * b <= most / c;
}

struct Span {
   const void* p;
   int64_t     bytes;
};
// present where it holds anything, and on its alignment
inline int span_status(const Span& a, uintptr_t align)
{
   if(a.bytes > 0 && !a.p) return FUFFT_ERR_INVALID;
   return a.bytes > 0 && !aligned(a.p, align) ? FUFFT_ERR_ALIGN : FUFFT_OK;
}
inline bool disjoint(const Span& a, const Span& b)
{
   if(!a.p || !b.p || a.bytes == 0 || b.bytes == 0) return true;
   const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
   return x + (uintptr_t)a.bytes <= y || y + (uintptr_t)b.bytes <= x;
}
template<int N>
inline bool apart(const Span& a, const Span (&others)[N])
{
   for(const Span& b : others)
      if(!disjoint(a, b)) return false;
   return true;
}

// bytes from the first to the last element of rows x k at leading dimension ld
inline Span matrix(const void* p, int type, int64_t ld, int64_t rows, int64_t k)
{
   return {p, rows == 0 || k == 0 ? 0 : ((rows - 1) * ld + k) * type_bytes(type)};
}
inline bool matrix_ok(int type, int64_t ld, int64_t rows, int64_t k)
{
   return type_ok(type) && size_ok(rows) && size_ok(k) && size_ok(ld) && (rows <= 1 || ld >= k) && volume_ok(rows, ld, 4);
}
// Two matrices of `rows` rows that share no byte: far from each other, or columns of one array, the rows
// of each in the gaps of the other's.
inline bool matrices_apart(const Span& a, int64_t pitch_a, int64_t width_a, const Span& b, int64_t pitch_b, int64_t width_b,
                    int64_t rows)
{
   if(disjoint(a, b)) return true;
   if(rows <= 1 || pitch_a != pitch_b) return false;
   const int64_t by = static_cast<const char*>(b.p) - static_cast<const char*>(a.p);
   const int64_t from = (by % pitch_a + pitch_a) % pitch_a;     // b's first byte in a row of a
   return from >= width_a && from + width_b <= pitch_a;
}
inline Span codes_of(const void* p, int64_t rows, int64_t k) { return {p, rows * (padded(k) / 2)}; }
inline Span scales_of(const void* p, int64_t rows, int64_t k) { return {p, rows * (padded(k) / 32)}; }

inline int status_of(hipError_t e)
{
   return e == hipSuccess ? FUFFT_OK : e == kTooLarge ? FUFFT_ERR_UNSUPPORTED : FUFFT_ERR_HIP;
}

#define FUFFT_MX4_CHECK(expr)                       \
   do {                                             \
      const int st_ = (expr);                       \
      if(st_ != FUFFT_OK) return st_;               \
   } while(0)

}  // namespace mx4
}  // namespace fufft
