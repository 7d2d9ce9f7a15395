// Entry points of the norm and 8-bit calls: argument checks and dispatch.
// Declarations in include/fufft/fufft.h.
#include "layer_internal.hpp"
#include "mx4_arguments.hpp"

using namespace fufft::mx4;
using namespace fufft::layer;

namespace {

Span bytes_of(const void* p, int64_t rows, int64_t k) { return {p, rows * padded(k)}; }
Span floats(const float* p, int64_t n) { return {p, n * 4}; }

// rows x k in elements of a type
struct Rows {
   const void* p;
   int         type;
   int64_t     ld;
};
Span span_of(const Rows& m, int64_t rows, int64_t k) { return m.p ? matrix(m.p, m.type, m.ld, rows, k) : Span{nullptr, 0}; }
// no byte shared: far from each other, or columns of one array
bool rows_apart(const Rows& a, const Rows& b, int64_t rows, int64_t k)
{
   if(!a.p || !b.p) return true;
   const int64_t ea = type_bytes(a.type), eb = type_bytes(b.type);
   return matrices_apart(span_of(a, rows, k), a.ld * ea, k * ea, span_of(b, rows, k), b.ld * eb, k * eb, rows);
}
// an output that may be an input, element for element, and otherwise shares no byte with it
bool same_or_apart(const Rows& out, const Rows& in, int64_t rows, int64_t k)
{
   if(out.p && out.p == in.p && out.type == in.type && (out.ld == in.ld || rows <= 1)) return true;
   return rows_apart(out, in, rows, k);
}
bool eps_ok(float eps) { return eps >= 0.0f && eps < __builtin_inff(); }

}  // namespace

extern "C" {

int64_t fufft_i8_padded(int64_t k) { return size_ok(k) ? padded(k) : (int64_t)FUFFT_ERR_INVALID; }

int fufft_i8_quantize(const void* x, int type, int64_t ld, int64_t rows, int64_t k, void* codes, float* scales,
                      void* stream)
{
   if(!matrix_ok(type, ld, rows, k) || !volume_ok(rows, padded(k))) return FUFFT_ERR_INVALID;
   if(rows == 0 || k == 0) return FUFFT_OK;
   const Span sx = matrix(x, type, ld, rows, k), sc = bytes_of(codes, rows, k), ss = floats(scales, rows);
   FUFFT_MX4_CHECK(span_status(sx, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sc, 16));
   FUFFT_MX4_CHECK(span_status(ss, 4));
   if(!apart(sc, {sx, ss}) || !apart(ss, {sx})) return FUFFT_ERR_INVALID;
   NormParams p{};
   p.x = x;
   p.codes = static_cast<int8_t*>(codes);
   p.scales = scales;
   p.ldx = ld;
   p.rows = rows;
   p.k = k;
   p.type = type;
   return status_of(launch_i8_quantize(p, static_cast<hipStream_t>(stream)));
}

int fufft_i8_dequantize(const void* codes, const float* scales, void* out, int type, int64_t ld, int64_t rows, int64_t k,
                        void* stream)
{
   if(!matrix_ok(type, ld, rows, k) || !volume_ok(rows, padded(k))) return FUFFT_ERR_INVALID;
   if(rows == 0 || k == 0) return FUFFT_OK;
   const Span so = matrix(out, type, ld, rows, k), sc = bytes_of(codes, rows, k), ss = floats(scales, rows);
   FUFFT_MX4_CHECK(span_status(so, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sc, 16));
   FUFFT_MX4_CHECK(span_status(ss, 4));
   if(!apart(so, {sc, ss})) return FUFFT_ERR_INVALID;
   return status_of(launch_i8_dequantize(static_cast<const int8_t*>(codes), scales, out, type, ld, rows, k,
                                         static_cast<hipStream_t>(stream)));
}

int fufft_i8_matmul(const void* a, const float* a_scales, const void* b, const float* b_scales, const float* bias,
                    void* out, int type, int64_t ld, int64_t m, int64_t n, int64_t k, void* stream)
{
   if(!matrix_ok(type, ld, m, n) || !size_ok(k) || !volume_ok(m, padded(k)) || !volume_ok(n, padded(k)))
      return FUFFT_ERR_INVALID;
   if(m == 0 || n == 0) return FUFFT_OK;
   const Span so = matrix(out, type, ld, m, n), sbias{bias, bias ? n * 4 : 0};
   const Span sa = bytes_of(a, m, k), sas = floats(a_scales, k ? m : 0);
   const Span sb = bytes_of(b, n, k), sbs = floats(b_scales, k ? n : 0);
   FUFFT_MX4_CHECK(span_status(so, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sa, 16));
   FUFFT_MX4_CHECK(span_status(sas, 4));
   FUFFT_MX4_CHECK(span_status(sb, 16));
   FUFFT_MX4_CHECK(span_status(sbs, 4));
   FUFFT_MX4_CHECK(span_status(sbias, 4));
   if(!apart(so, {sa, sas, sb, sbs, sbias})) return FUFFT_ERR_INVALID;
   if(k > kLongestI8) return FUFFT_ERR_UNSUPPORTED;
   const I8Params p{static_cast<const int8_t*>(a), static_cast<const int8_t*>(b), a_scales, b_scales, bias, out, ld, m, n,
                    k, type};
   return status_of(launch_i8_matmul(p, static_cast<hipStream_t>(stream)));
}

int fufft_rms_norm(const void* x, int type, int64_t ldx, const void* residual, int64_t ldr, void* total, int64_t ldt,
                   int sum_type, const float* weight, float eps, void* out, int64_t ldo, void* codes, float* scales,
                   int64_t rows, int64_t k, void* stream)
{
   if(!matrix_ok(type, ldx, rows, k) || !eps_ok(eps) || (sum_type != type && sum_type != FUFFT_F32))
      return FUFFT_ERR_INVALID;
   const bool eight = codes || scales;
   if((residual && !matrix_ok(sum_type, ldr, rows, k)) || (total && !matrix_ok(sum_type, ldt, rows, k)) ||
      (out && !matrix_ok(type, ldo, rows, k)) || (eight && !volume_ok(rows, padded(k))))
      return FUFFT_ERR_INVALID;
   if(rows == 0 || k == 0) return FUFFT_OK;
   if(!out && !eight) return FUFFT_ERR_INVALID;
   const Rows rx{x, type, ldx}, rr{residual, sum_type, ldr}, rt{total, sum_type, ldt}, ro{out, type, ldo};
   const Span sx = span_of(rx, rows, k), sr = span_of(rr, rows, k), st = span_of(rt, rows, k), so = span_of(ro, rows, k);
   const Span sw = floats(weight, weight ? k : 0);
   const Span sc = bytes_of(codes, eight ? rows : 0, k), ss = floats(scales, eight ? rows : 0);
   const uintptr_t element = (uintptr_t)type_bytes(type), stream_element = (uintptr_t)type_bytes(sum_type);
   if(!x) return FUFFT_ERR_INVALID;
   FUFFT_MX4_CHECK(span_status(sx, element));
   FUFFT_MX4_CHECK(span_status(sr, stream_element));
   FUFFT_MX4_CHECK(span_status(st, stream_element));
   FUFFT_MX4_CHECK(span_status(so, element));
   FUFFT_MX4_CHECK(span_status(sw, 4));
   FUFFT_MX4_CHECK(span_status(sc, 16));
   FUFFT_MX4_CHECK(span_status(ss, 4));
   if(!apart(sc, {sx, sr, st, so, sw, ss}) || !apart(ss, {sx, sr, st, so, sw}) || !apart(sw, {st, so}) ||
      !same_or_apart(rt, rr, rows, k) || !same_or_apart(rt, rx, rows, k) || !same_or_apart(ro, rx, rows, k) ||
      !rows_apart(ro, rr, rows, k) || !rows_apart(ro, rt, rows, k))
      return FUFFT_ERR_INVALID;
   const NormParams p{x,   residual, total, weight, out, static_cast<int8_t*>(codes), scales, ldx, ldr, ldt, ldo, rows, k,
                      eps, type,     sum_type};
   return status_of(launch_rms_norm(p, static_cast<hipStream_t>(stream)));
}

int fufft_rms_norm_grad(const void* dy, int type, int64_t ldy, const void* h, int64_t ldh, const void* dtotal, int64_t ldt,
                        int sum_type, const float* weight, float eps, void* dx, int dx_type, int64_t ldx, float* dweight,
                        float* work, int64_t splits, int64_t rows, int64_t k, void* stream)
{
   if(!matrix_ok(type, ldy, rows, k) || !eps_ok(eps) || (sum_type != type && sum_type != FUFFT_F32) ||
      (dx_type != type && dx_type != sum_type))
      return FUFFT_ERR_INVALID;
   if(!matrix_ok(sum_type, ldh, rows, k) || (dtotal && !matrix_ok(sum_type, ldt, rows, k)) ||
      !matrix_ok(dx_type, ldx, rows, k) || !size_ok(splits) || !volume_ok(splits, k, 4))
      return FUFFT_ERR_INVALID;
   if(k == 0) return FUFFT_OK;
   if(dweight && splits == 0) return FUFFT_ERR_INVALID;
   const Rows ry{dy, type, ldy}, rh{h, sum_type, ldh}, rt{dtotal, sum_type, ldt}, rx{dx, dx_type, ldx};
   const Span sy = span_of(ry, rows, k), sh = span_of(rh, rows, k), st = span_of(rt, rows, k), sx = span_of(rx, rows, k);
   const Span sw = floats(weight, weight ? k : 0), sd = floats(dweight, dweight ? k : 0);
   const Span sk = floats(work, dweight ? splits * k : 0);
   if(rows > 0 && (!dy || !h || !dx)) return FUFFT_ERR_INVALID;
   FUFFT_MX4_CHECK(span_status(sy, (uintptr_t)type_bytes(type)));
   FUFFT_MX4_CHECK(span_status(sh, (uintptr_t)type_bytes(sum_type)));
   FUFFT_MX4_CHECK(span_status(st, (uintptr_t)type_bytes(sum_type)));
   FUFFT_MX4_CHECK(span_status(sx, (uintptr_t)type_bytes(dx_type)));
   FUFFT_MX4_CHECK(span_status(sw, 4));
   FUFFT_MX4_CHECK(span_status(sd, 4));
   FUFFT_MX4_CHECK(span_status(sk, 4));
   if(!apart(sd, {sy, sh, st, sx, sw, sk}) || !apart(sk, {sy, sh, st, sx, sw}) || !apart(sx, {sw}) ||
      !rows_apart(rx, rh, rows, k) || !same_or_apart(rx, ry, rows, k) || !same_or_apart(rx, rt, rows, k))
      return FUFFT_ERR_INVALID;
   const NormGradParams p{dy,  h,    dtotal, weight,   dx,     dweight, work, ldy, ldh, ldt, ldx, rows, k, splits,
                          eps, type, sum_type, dx_type};
   return status_of(launch_rms_norm_grad(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
