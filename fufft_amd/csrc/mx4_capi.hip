// Entry points of the microscaled 4-bit calls: argument checks and dispatch.
// Declarations in include/fufft/fufft.h.
#include "mx4_internal.hpp"
#include "../../include/fufft/fufft.h"

namespace fufft {
namespace mx4 {

namespace {

bool type_ok(int type) { return type == FUFFT_F32 || type == FUFFT_BF16 || type == FUFFT_F16; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// sizes of one argument: at most 2^40, so that no product of two below overflows
bool size_ok(int64_t n) { return n >= 0 && n <= ((int64_t)1 << 40); }
// a x b x c within 2^62
bool volume_ok(int64_t a, int64_t b, int64_t c = 1)
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
int span_status(const Span& a, uintptr_t align)
{
   if(a.bytes > 0 && !a.p) return FUFFT_ERR_INVALID;
   return a.bytes > 0 && !aligned(a.p, align) ? FUFFT_ERR_ALIGN : FUFFT_OK;
}
bool disjoint(const Span& a, const Span& b)
{
   if(!a.p || !b.p || a.bytes == 0 || b.bytes == 0) return true;
   const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
   return x + (uintptr_t)a.bytes <= y || y + (uintptr_t)b.bytes <= x;
}
template<int N>
bool apart(const Span& a, const Span (&others)[N])
{
   for(const Span& b : others)
      if(!disjoint(a, b)) return false;
   return true;
}

// bytes from the first to the last element of rows x k at leading dimension ld
Span matrix(const void* p, int type, int64_t ld, int64_t rows, int64_t k)
{
   return {p, rows == 0 || k == 0 ? 0 : ((rows - 1) * ld + k) * type_bytes(type)};
}
bool matrix_ok(int type, int64_t ld, int64_t rows, int64_t k)
{
   return type_ok(type) && size_ok(rows) && size_ok(k) && size_ok(ld) && (rows <= 1 || ld >= k) && volume_ok(rows, ld, 4);
}
// Two matrices of `rows` rows that share no byte: far from each other, or columns of one array, the rows
// of each in the gaps of the other's.
bool matrices_apart(const Span& a, int64_t pitch_a, int64_t width_a, const Span& b, int64_t pitch_b, int64_t width_b,
                    int64_t rows)
{
   if(disjoint(a, b)) return true;
   if(rows <= 1 || pitch_a != pitch_b) return false;
   const int64_t by = static_cast<const char*>(b.p) - static_cast<const char*>(a.p);
   const int64_t from = (by % pitch_a + pitch_a) % pitch_a;     // b's first byte in a row of a
   return from >= width_a && from + width_b <= pitch_a;
}
Span codes_of(const void* p, int64_t rows, int64_t k) { return {p, rows * (padded(k) / 2)}; }
Span scales_of(const void* p, int64_t rows, int64_t k) { return {p, rows * (padded(k) / 32)}; }

int status_of(hipError_t e)
{
   return e == hipSuccess ? FUFFT_OK : e == kTooLarge ? FUFFT_ERR_UNSUPPORTED : FUFFT_ERR_HIP;
}

#define FUFFT_MX4_CHECK(expr)                       \
   do {                                             \
      const int st_ = (expr);                       \
      if(st_ != FUFFT_OK) return st_;               \
   } while(0)

}  // namespace

}  // namespace mx4
}  // namespace fufft

using namespace fufft::mx4;

extern "C" {

int64_t fufft_mx4_padded(int64_t k) { return size_ok(k) ? padded(k) : (int64_t)FUFFT_ERR_INVALID; }

int fufft_mx4_quantize(const void* x, int type, int64_t ld, int64_t rows, int64_t k, int rule, const uint8_t* rand,
                       void* codes, uint8_t* scales, void* codes_t, uint8_t* scales_t, void* stream)
{
   if(!matrix_ok(type, ld, rows, k) || !volume_ok(padded(rows), padded(k))) return FUFFT_ERR_INVALID;
   if(rule != FUFFT_MX4_FIT && rule != FUFFT_MX4_FLOOR) return FUFFT_ERR_INVALID;
   if(rows == 0 || k == 0) return FUFFT_OK;
   const bool along = codes || scales, across = codes_t || scales_t;
   if(!along && !across) return FUFFT_ERR_INVALID;
   const Span sx = matrix(x, type, ld, rows, k), sr{rand, rand ? rows * k : 0};
   const Span sc = codes_of(codes, along ? rows : 0, k), ss = scales_of(scales, along ? rows : 0, k);
   const Span tc = codes_of(codes_t, across ? k : 0, rows), ts = scales_of(scales_t, across ? k : 0, rows);
   FUFFT_MX4_CHECK(span_status(sx, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sc, 16));
   FUFFT_MX4_CHECK(span_status(ss, 4));
   FUFFT_MX4_CHECK(span_status(tc, 16));
   FUFFT_MX4_CHECK(span_status(ts, 4));
   if(!apart(sc, {sx, sr, ss, tc, ts}) || !apart(ss, {sx, sr, tc, ts}) || !apart(tc, {sx, sr, ts}) ||
      !apart(ts, {sx, sr}))
      return FUFFT_ERR_INVALID;
   QuantizeParams p{};
   p.x = x;
   p.rand = rand;
   p.codes = static_cast<uint8_t*>(codes);
   p.scales = scales;
   p.codes_t = static_cast<uint8_t*>(codes_t);
   p.scales_t = scales_t;
   p.slot_count = rows;
   p.ld = ld;
   p.rows = rows;
   p.k = k;
   p.type = type;
   p.fit = rule == FUFFT_MX4_FIT;
   return status_of(launch_quantize(p, static_cast<hipStream_t>(stream)));
}

int fufft_mx4_dequantize(const void* codes, const uint8_t* scales, void* out, int type, int64_t ld, int64_t rows,
                         int64_t k, void* stream)
{
   if(!matrix_ok(type, ld, rows, k)) return FUFFT_ERR_INVALID;
   if(rows == 0 || k == 0) return FUFFT_OK;
   const Span so = matrix(out, type, ld, rows, k), sc = codes_of(codes, rows, k), ss = scales_of(scales, rows, k);
   FUFFT_MX4_CHECK(span_status(so, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sc, 16));
   FUFFT_MX4_CHECK(span_status(ss, 4));
   if(!apart(so, {sc, ss})) return FUFFT_ERR_INVALID;
   DequantizeParams p{static_cast<const uint8_t*>(codes), scales, out, ld, rows, k, type};
   return status_of(launch_dequantize(p, static_cast<hipStream_t>(stream)));
}

int fufft_mx4_matmul(const void* a, const uint8_t* a_scales, const void* b, const uint8_t* b_scales,
                     const float* bias, void* out, int type, int64_t ld, int64_t m, int64_t n, int64_t k, void* stream)
{
   if(!matrix_ok(type, ld, m, n) || !size_ok(k) || !volume_ok(m, padded(k)) || !volume_ok(n, padded(k)))
      return FUFFT_ERR_INVALID;
   if(m == 0 || n == 0) return FUFFT_OK;
   const Span so = matrix(out, type, ld, m, n), sbias{bias, bias ? n * 4 : 0};
   const Span sa = codes_of(a, m, k), sas = scales_of(a_scales, m, k);
   const Span sb = codes_of(b, n, k), sbs = scales_of(b_scales, n, k);
   FUFFT_MX4_CHECK(span_status(so, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sa, 16));
   FUFFT_MX4_CHECK(span_status(sas, 4));
   FUFFT_MX4_CHECK(span_status(sb, 16));
   FUFFT_MX4_CHECK(span_status(sbs, 4));
   FUFFT_MX4_CHECK(span_status(sbias, 4));
   if(!apart(so, {sa, sas, sb, sbs, sbias})) return FUFFT_ERR_INVALID;
   MatmulParams p{};
   p.x = a;
   p.x_scales = a_scales;
   p.w = static_cast<const uint8_t*>(b);
   p.w_scales = b_scales;
   p.bias = bias;
   p.out = out;
   p.ld = ld;
   p.m = m;
   p.n = n;
   p.k = k;
   p.type = type;
   return status_of(launch_matmul(p, static_cast<hipStream_t>(stream)));
}

int fufft_mx4_linear(const void* x, int x_type, int64_t ldx, const void* w, const uint8_t* w_scales, const float* bias,
                     void* out, int type, int64_t ld, int64_t m, int64_t n, int64_t k, void* stream)
{
   if(!matrix_ok(type, ld, m, n) || !matrix_ok(x_type, ldx, m, k) || !volume_ok(n, padded(k))) return FUFFT_ERR_INVALID;
   if(m == 0 || n == 0) return FUFFT_OK;
   const Span so = matrix(out, type, ld, m, n), sbias{bias, bias ? n * 4 : 0}, sx = matrix(x, x_type, ldx, m, k);
   const Span sw = codes_of(w, n, k), sws = scales_of(w_scales, n, k);
   const int64_t xb = type_bytes(x_type), ob = type_bytes(type);
   FUFFT_MX4_CHECK(span_status(so, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sx, (uintptr_t)type_bytes(x_type)));
   FUFFT_MX4_CHECK(span_status(sw, 16));
   FUFFT_MX4_CHECK(span_status(sws, 4));
   FUFFT_MX4_CHECK(span_status(sbias, 4));
   if(!apart(so, {sw, sws, sbias}) || !matrices_apart(sx, ldx * xb, k * xb, so, ld * ob, n * ob, m))
      return FUFFT_ERR_INVALID;
   MatmulParams p{};
   p.x = x;
   p.w = static_cast<const uint8_t*>(w);
   p.w_scales = w_scales;
   p.bias = bias;
   p.out = out;
   p.ldx = ldx;
   p.ld = ld;
   p.m = m;
   p.n = n;
   p.k = k;
   p.x_type = x_type;
   p.type = type;
   return status_of(launch_linear(p, static_cast<hipStream_t>(stream)));
}

int fufft_mx4_cache_write(const void* x, int type, int64_t ld, const int64_t* slots, int64_t rows, int64_t channels,
                          void* codes, uint8_t* scales, int64_t slot_count, void* stream)
{
   if(!matrix_ok(type, ld, rows, channels) || !size_ok(slot_count) || !volume_ok(slot_count, padded(channels)) ||
      !volume_ok(rows, padded(channels)))
      return FUFFT_ERR_INVALID;
   if(rows == 0 || channels == 0 || slot_count == 0) return FUFFT_OK;
   const Span sx = matrix(x, type, ld, rows, channels), sl{slots, rows * 8};
   const Span sc = codes_of(codes, slot_count, channels), ss = scales_of(scales, slot_count, channels);
   FUFFT_MX4_CHECK(span_status(sx, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sl, 8));
   FUFFT_MX4_CHECK(span_status(sc, 16));
   FUFFT_MX4_CHECK(span_status(ss, 4));
   if(!apart(sc, {sx, sl, ss}) || !apart(ss, {sx, sl})) return FUFFT_ERR_INVALID;
   QuantizeParams p{};
   p.x = x;
   p.codes = static_cast<uint8_t*>(codes);
   p.scales = scales;
   p.slots = slots;
   p.slot_count = slot_count;
   p.ld = ld;
   p.rows = rows;
   p.k = channels;
   p.type = type;
   p.fit = 1;
   return status_of(launch_quantize(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"

namespace {

// the arguments that describe a cache, checked; FUFFT_OK with *c filled
int cache_params(const void* codes, const uint8_t* scales, int64_t pages, int64_t page, int64_t channels,
                 const int32_t* table, int64_t width, const int32_t* lens, int64_t batch, CacheParams* c)
{
   if(!size_ok(pages) || !size_ok(channels) || !size_ok(width) || !size_ok(batch)) return FUFFT_ERR_INVALID;
   if(page < 1 || page > 65536 || (page & (page - 1))) return FUFFT_ERR_INVALID;
   if(!volume_ok(pages, page, padded(channels)) || !volume_ok(batch, width, 4) || !volume_ok(width, page))
      return FUFFT_ERR_INVALID;
   FUFFT_MX4_CHECK(span_status(codes_of(codes, pages * page, channels), 16));
   FUFFT_MX4_CHECK(span_status(scales_of(scales, pages * page, channels), 4));
   FUFFT_MX4_CHECK(span_status({table, batch * width * 4}, 4));
   FUFFT_MX4_CHECK(span_status({lens, batch * 4}, 4));
   int log = 0;
   while(((int64_t)1 << log) < page) log++;
   *c = CacheParams{static_cast<const uint8_t*>(codes), scales, table, lens, pages, channels, width, batch, log};
   return FUFFT_OK;
}

}  // namespace

extern "C" {

int fufft_mx4_cache_read(const void* codes, const uint8_t* scales, int64_t pages, int64_t page, int64_t channels,
                         const int32_t* table, int64_t width, const int32_t* lens, int64_t batch, int64_t length,
                         void* out, int type, int order, void* stream)
{
   if(!type_ok(type) || !size_ok(length) || (order != FUFFT_MX4_TOKENS && order != FUFFT_MX4_CHANNELS))
      return FUFFT_ERR_INVALID;
   CacheParams c;
   FUFFT_MX4_CHECK(cache_params(codes, scales, pages, page, channels, table, width, lens, batch, &c));
   if(!volume_ok(batch, length, channels * 4)) return FUFFT_ERR_INVALID;
   const Span so{out, batch * length * channels * type_bytes(type)};
   FUFFT_MX4_CHECK(span_status(so, (uintptr_t)type_bytes(type)));
   const Span sc = codes_of(codes, pages * page, channels), ss = scales_of(scales, pages * page, channels);
   if(!apart(so, {sc, ss, Span{table, batch * width * 4}, Span{lens, batch * 4}})) return FUFFT_ERR_INVALID;
   return status_of(launch_cache_read(c, out, type, length, order == FUFFT_MX4_CHANNELS,
                                      static_cast<hipStream_t>(stream)));
}

int fufft_mx4_cache_conv(const void* codes, const uint8_t* scales, int64_t pages, int64_t page, int64_t channels,
                         const int32_t* table, int64_t width, const int32_t* lens, int64_t batch, const void* taps,
                         int tap_type, int64_t tap_count, void* out, int type, float* work, int64_t splits,
                         void* stream)
{
   if(!type_ok(type) || !type_ok(tap_type) || !size_ok(tap_count) || !size_ok(splits)) return FUFFT_ERR_INVALID;
   CacheParams c;
   FUFFT_MX4_CHECK(cache_params(codes, scales, pages, page, channels, table, width, lens, batch, &c));
   if(!volume_ok(tap_count, channels, 4) || !volume_ok(batch, channels, 4)) return FUFFT_ERR_INVALID;
   const int64_t count = batch * channels;
   if(count == 0) return FUFFT_OK;
   if(!volume_ok(splits, count * 4)) return FUFFT_ERR_INVALID;
   if(type != FUFFT_F32 && splits == 0) return FUFFT_ERR_INVALID;    // sums are fp32: a workspace of one split at least
   const Span so{out, count * type_bytes(type)}, st{taps, tap_count * channels * type_bytes(tap_type)};
   const Span sk{work, splits * count * 4};
   FUFFT_MX4_CHECK(span_status(so, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(st, (uintptr_t)type_bytes(tap_type)));
   FUFFT_MX4_CHECK(span_status(sk, 4));
   const Span sc = codes_of(codes, pages * page, channels), ss = scales_of(scales, pages * page, channels);
   const Span sp{table, batch * width * 4}, sl{lens, batch * 4};
   if(!apart(so, {sc, ss, sp, sl, st, sk}) || !apart(sk, {sc, ss, sp, sl, st})) return FUFFT_ERR_INVALID;
   return status_of(launch_cache_conv(c, taps, tap_type, tap_count, out, type, work, splits,
                                      static_cast<hipStream_t>(stream)));
}

}  // extern "C"
