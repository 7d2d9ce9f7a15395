// The short way from Python to the 4-bit, 8-bit, norm and decaying-attention calls: reads the tensors' properties, checks them
// and calls the C ABI, all in native code.  These calls are short (a few rows take
// the GPU 2 to 4 us), so what the host spends on a call is what a small one costs: 48 rows
// of 4096 made 4-bit, host time a call, 5.5 us through ctypes, 3.6 so, 3.2 of them the launch.
//
// Every function takes tensors, None where an argument is not given, then the
// stream's handle and the current GPU, and returns the C ABI's status, or None
// where an argument is not of the kind that the call takes: the caller then goes
// through the checks in Python, which say what is wrong.  No check is less here than there.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/fufft/fufft.h"

namespace {

struct Refused {};      // an argument that the checks in Python have to look at

const at::Tensor& tensor(PyObject* o, int64_t gpu)
{
   if(!THPVariable_CheckExact(o)) throw Refused();
   const at::Tensor& t = THPVariable_Unpack(o);
   if(!t.is_cuda() || t.get_device() != gpu) throw Refused();
   return t;
}

// a contiguous array of at least `bytes`
void* array(PyObject* o, at::ScalarType type, int64_t bytes, int64_t gpu)
{
   const at::Tensor& t = tensor(o, gpu);
   if(t.scalar_type() != type || !t.is_contiguous() || (int64_t)t.nbytes() < bytes) throw Refused();
   return t.data_ptr();
}

int element(const at::Tensor& t)
{
   switch(t.scalar_type()) {
      case at::kFloat:    return FUFFT_F32;
      case at::kBFloat16: return FUFFT_BF16;
      case at::kHalf:     return FUFFT_F16;
      default:            throw Refused();
   }
}

struct Matrix {
   void*   p;
   int     type;
   int64_t ld, rows, k;
};
Matrix matrix(PyObject* o, int64_t gpu)
{
   const at::Tensor& t = tensor(o, gpu);
   if(t.dim() != 2) throw Refused();
   Matrix m{nullptr, element(t), 0, t.size(0), t.size(1)};
   if(t.is_contiguous()) {
      m.ld = m.k;
   } else {
      if((m.k > 1 && t.stride(1) != 1) || (m.rows > 1 && t.stride(0) < m.k)) throw Refused();
      m.ld = m.rows > 1 ? t.stride(0) : m.k;
   }
   m.p = t.data_ptr();
   return m;
}

// `rows` rows of `width` bytes: a flat array, or one whose own rows have that length
void* rows_of(PyObject* o, int64_t rows, int64_t width, int64_t gpu)
{
   void* const p = array(o, at::kByte, rows * width, gpu);
   const at::Tensor& t = THPVariable_Unpack(o);
   if(t.dim() > 1 && rows * width > 0 && t.size(t.dim() - 1) != width) throw Refused();
   return p;
}

struct Blocks {
   void*    codes;
   uint8_t* scales;
};
Blocks blocks(PyObject* codes, PyObject* scales, int64_t rows, int64_t k, int64_t gpu)
{
   const int64_t groups = (k + 127) / 128;
   return {rows_of(codes, rows, groups * 64, gpu), static_cast<uint8_t*>(rows_of(scales, rows, groups * 4, gpu))};
}

// codes (pages, page, bytes of a row) and scales of the same pages
struct Cache {
   Blocks  b;
   int64_t pages, page;
};
Cache cache(PyObject* codes, PyObject* scales, int64_t channels, int64_t gpu)
{
   const at::Tensor &c = tensor(codes, gpu), &s = tensor(scales, gpu);
   const int64_t groups = (channels + 127) / 128;
   if(c.dim() != 3 || s.dim() != 3 || c.size(2) != groups * 64 || s.size(2) != groups * 4 || c.size(0) != s.size(0) ||
      c.size(1) != s.size(1))
      throw Refused();
   const int64_t page = c.size(1);
   if(page < 1 || page > 65536 || (page & (page - 1))) throw Refused();
   return {blocks(codes, scales, c.size(0) * page, channels, gpu), c.size(0), page};
}

struct Table {
   const int32_t *pages, *lens;
   int64_t        batch, width;
};
Table table(PyObject* pages, PyObject* lens, int64_t gpu)
{
   const at::Tensor &t = tensor(pages, gpu), &l = tensor(lens, gpu);
   if(t.dim() != 2 || l.dim() != 1 || t.size(0) != l.size(0)) throw Refused();
   const int64_t n = t.size(0), w = t.size(1);
   return {static_cast<const int32_t*>(array(pages, at::kInt, 4 * n * w, gpu)),
           static_cast<const int32_t*>(array(lens, at::kInt, 4 * n, gpu)), n, w};
}

int64_t integer(PyObject* o)
{
   const long long v = PyLong_AsLongLong(o);
   if(v == -1 && PyErr_Occurred()) throw Refused();
   return v;
}
void* handle(PyObject* o)
{
   void* const v = PyLong_AsVoidPtr(o);
   if(!v && PyErr_Occurred()) throw Refused();
   return v;
}

// the call without the interpreter's lock, its status as a Python number
template<class F>
PyObject* status_of(F call)
{
   int st;
   Py_BEGIN_ALLOW_THREADS
   st = call();
   Py_END_ALLOW_THREADS
   return PyLong_FromLong(st);
}

// `body` with `want` arguments; nothing it throws leaves
template<class F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F body)
{
   if(n != want) {
      PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
      return nullptr;
   }
   try {
      return body();
   } catch(...) {
      PyErr_Clear();
      Py_RETURN_NONE;
   }
}

PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 9, [&] {
      const int64_t gpu = integer(a[8]);
      void* const stream = handle(a[7]);
      const Matrix x = matrix(a[0], gpu);
      const bool along = a[1] != Py_None || a[2] != Py_None, across = a[3] != Py_None || a[4] != Py_None;
      if(!along && !across) throw Refused();
      const Blocks q = along ? blocks(a[1], a[2], x.rows, x.k, gpu) : Blocks{nullptr, nullptr};
      const Blocks t = across ? blocks(a[3], a[4], x.k, x.rows, gpu) : Blocks{nullptr, nullptr};
      const uint8_t* const rand =
         a[5] == Py_None ? nullptr : static_cast<const uint8_t*>(rows_of(a[5], x.rows, x.k, gpu));
      const int rule = (int)integer(a[6]);
      return status_of([&] {
         return fufft_mx4_quantize(x.p, x.type, x.ld, x.rows, x.k, rule, rand, q.codes, q.scales, t.codes, t.scales, stream);
      });
   });
}

PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 5, [&] {
      const int64_t gpu = integer(a[4]);
      void* const stream = handle(a[3]);
      const Matrix out = matrix(a[2], gpu);
      const Blocks q = blocks(a[0], a[1], out.rows, out.k, gpu);
      return status_of(
         [&] { return fufft_mx4_dequantize(q.codes, q.scales, out.p, out.type, out.ld, out.rows, out.k, stream); });
   });
}

const float* bias_of(PyObject* o, int64_t n, int64_t gpu)
{
   return o == Py_None ? nullptr : static_cast<const float*>(array(o, at::kFloat, 4 * n, gpu));
}

PyObject* matmul(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 9, [&] {
      const int64_t gpu = integer(a[8]), k = integer(a[5]);
      void* const stream = handle(a[7]);
      const Matrix out = matrix(a[4], gpu);
      if(k < 0) throw Refused();
      const Blocks x = blocks(a[0], a[1], out.rows, k, gpu), w = blocks(a[2], a[3], out.k, k, gpu);
      const float* const bias = bias_of(a[6], out.k, gpu);
      return status_of([&] {
         return fufft_mx4_matmul(x.codes, x.scales, w.codes, w.scales, bias, out.p, out.type, out.ld, out.rows, out.k, k,
                                 stream);
      });
   });
}

PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 7, [&] {
      const int64_t gpu = integer(a[6]);
      void* const stream = handle(a[5]);
      const Matrix x = matrix(a[0], gpu), out = matrix(a[3], gpu);
      if(x.rows != out.rows) throw Refused();
      const Blocks w = blocks(a[1], a[2], out.k, x.k, gpu);
      const float* const bias = bias_of(a[4], out.k, gpu);
      return status_of([&] {
         return fufft_mx4_linear(x.p, x.type, x.ld, w.codes, w.scales, bias, out.p, out.type, out.ld, out.rows, out.k, x.k,
                                 stream);
      });
   });
}

PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 6, [&] {
      const int64_t gpu = integer(a[5]);
      void* const stream = handle(a[4]);
      const Matrix x = matrix(a[0], gpu);
      const Cache c = cache(a[2], a[3], x.k, gpu);
      const int64_t* const slots = static_cast<const int64_t*>(array(a[1], at::kLong, 8 * x.rows, gpu));
      return status_of([&] {
         return fufft_mx4_cache_write(x.p, x.type, x.ld, slots, x.rows, x.k, c.b.codes, c.b.scales, c.pages * c.page,
                                      stream);
      });
   });
}

PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 8, [&] {
      const int64_t gpu = integer(a[7]);
      void* const stream = handle(a[6]);
      const int order = (int)integer(a[5]);
      const at::Tensor& out = tensor(a[4], gpu);
      if(out.dim() != 3 || !out.is_contiguous()) throw Refused();
      const int type = element(out);
      const int64_t channels = out.size(order == FUFFT_MX4_CHANNELS ? 1 : 2);
      const int64_t length = out.size(order == FUFFT_MX4_CHANNELS ? 2 : 1);
      const Cache c = cache(a[0], a[1], channels, gpu);
      const Table t = table(a[2], a[3], gpu);
      if(out.size(0) != t.batch) throw Refused();
      void* const to = out.data_ptr();
      return status_of([&] {
         return fufft_mx4_cache_read(c.b.codes, c.b.scales, c.pages, c.page, channels, t.pages, t.width, t.lens, t.batch,
                                     length, to, type, order, stream);
      });
   });
}

PyObject* cache_conv(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 9, [&] {
      const int64_t gpu = integer(a[8]);
      void* const stream = handle(a[7]);
      const Matrix taps = matrix(a[4], gpu), out = matrix(a[5], gpu);
      if(out.k != taps.k || (taps.rows > 1 && taps.ld != taps.k) || (out.rows > 1 && out.ld != out.k)) throw Refused();
      const Cache c = cache(a[0], a[1], taps.k, gpu);
      const Table t = table(a[2], a[3], gpu);
      if(t.batch != out.rows) throw Refused();
      const int64_t count = out.rows * out.k;
      int64_t splits = 0;
      float* work = nullptr;
      if(a[6] != Py_None && count > 0) {
         splits = tensor(a[6], gpu).numel() / count;
         if(splits > 0) work = static_cast<float*>(array(a[6], at::kFloat, 4 * splits * count, gpu));
      }
      if(out.type != FUFFT_F32 && splits == 0 && count > 0) throw Refused();
      return status_of([&] {
         return fufft_mx4_cache_conv(c.b.codes, c.b.scales, c.pages, c.page, taps.k, t.pages, t.width, t.lens, t.batch,
                                     taps.p, taps.type, taps.rows, out.p, out.type, work, splits, stream);
      });
   });
}

// ---- 8-bit rows and norms -----------------------------------------------------------------

struct Eight {
   void*  codes;
   float* scales;
};
// `rows` 8-bit rows of k values
Eight eight(PyObject* codes, PyObject* scales, int64_t rows, int64_t k, int64_t gpu)
{
   const int64_t width = (k + 127) / 128 * 128;
   void* const p = array(codes, at::kChar, rows * width, gpu);
   const at::Tensor& t = THPVariable_Unpack(codes);
   if(t.dim() > 1 && rows * width > 0 && t.size(t.dim() - 1) != width) throw Refused();
   return {p, static_cast<float*>(array(scales, at::kFloat, 4 * rows, gpu))};
}
float* floats_of(PyObject* o, int64_t n, int64_t gpu)
{
   return o == Py_None ? nullptr : static_cast<float*>(array(o, at::kFloat, 4 * n, gpu));
}
double number(PyObject* o)
{
   const double v = PyFloat_AsDouble(o);
   if(v == -1.0 && PyErr_Occurred()) throw Refused();
   return v;
}
// a matrix of rows x k, or nothing where None is given
Matrix like(PyObject* o, int64_t rows, int64_t k, int64_t gpu)
{
   if(o == Py_None) return Matrix{nullptr, -1, 0, rows, k};
   const Matrix m = matrix(o, gpu);
   if(m.rows != rows || m.k != k) throw Refused();
   return m;
}

PyObject* i8_quantize(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 5, [&] {
      const int64_t gpu = integer(a[4]);
      void* const stream = handle(a[3]);
      const Matrix x = matrix(a[0], gpu);
      const Eight q = eight(a[1], a[2], x.rows, x.k, gpu);
      return status_of([&] { return fufft_i8_quantize(x.p, x.type, x.ld, x.rows, x.k, q.codes, q.scales, stream); });
   });
}

PyObject* i8_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 5, [&] {
      const int64_t gpu = integer(a[4]);
      void* const stream = handle(a[3]);
      const Matrix out = matrix(a[2], gpu);
      const Eight q = eight(a[0], a[1], out.rows, out.k, gpu);
      return status_of([&] { return fufft_i8_dequantize(q.codes, q.scales, out.p, out.type, out.ld, out.rows, out.k, stream); });
   });
}

PyObject* i8_matmul(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 9, [&] {
      const int64_t gpu = integer(a[8]), k = integer(a[5]);
      void* const stream = handle(a[7]);
      const Matrix out = matrix(a[4], gpu);
      if(k < 0 || k > ((int64_t)1 << 40)) throw Refused();
      const Eight x = eight(a[0], a[1], out.rows, k, gpu), w = eight(a[2], a[3], out.k, k, gpu);
      const float* const bias = bias_of(a[6], out.k, gpu);
      return status_of([&] {
         return fufft_i8_matmul(x.codes, x.scales, w.codes, w.scales, bias, out.p, out.type, out.ld, out.rows, out.k, k, stream);
      });
   });
}

PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 10, [&] {
      const int64_t gpu = integer(a[9]);
      void* const stream = handle(a[8]);
      const float eps = (float)number(a[7]);
      const Matrix x = matrix(a[0], gpu);
      const Matrix out = like(a[2], x.rows, x.k, gpu), r = like(a[5], x.rows, x.k, gpu), t = like(a[6], x.rows, x.k, gpu);
      const int sum = r.p || a[5] != Py_None ? r.type : a[6] != Py_None ? t.type : x.type;
      if((a[2] != Py_None && out.type != x.type) || (sum != x.type && sum != FUFFT_F32) || (a[6] != Py_None && t.type != sum))
         throw Refused();
      const bool codes = a[3] != Py_None || a[4] != Py_None;
      if(!codes && a[2] == Py_None) throw Refused();
      const Eight q = codes ? eight(a[3], a[4], x.rows, x.k, gpu) : Eight{nullptr, nullptr};
      const float* const w = floats_of(a[1], x.k, gpu);
      return status_of([&] {
         return fufft_rms_norm(x.p, x.type, x.ld, r.p, r.ld, t.p, t.ld, sum, w, eps, out.p, out.ld, q.codes, q.scales, x.rows,
                               x.k, stream);
      });
   });
}

PyObject* rms_norm_grad(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 10, [&] {
      const int64_t gpu = integer(a[9]);
      void* const stream = handle(a[8]);
      const float eps = (float)number(a[7]);
      const Matrix dy = matrix(a[0], gpu);
      if(a[1] == Py_None || a[3] == Py_None) throw Refused();
      const Matrix h = like(a[1], dy.rows, dy.k, gpu), dx = like(a[3], dy.rows, dy.k, gpu), t = like(a[6], dy.rows, dy.k, gpu);
      if((h.type != dy.type && h.type != FUFFT_F32) || (dx.type != dy.type && dx.type != h.type) ||
         (a[6] != Py_None && t.type != h.type))
         throw Refused();
      const float* const w = floats_of(a[2], dy.k, gpu);
      float* const dw = floats_of(a[4], dy.k, gpu);
      int64_t splits = 0;
      float* work = nullptr;
      if(dw && a[5] != Py_None && dy.k > 0) {
         splits = tensor(a[5], gpu).numel() / dy.k;
         if(splits > 0) work = static_cast<float*>(array(a[5], at::kFloat, 4 * splits * dy.k, gpu));
      }
      if(a[4] != Py_None && splits == 0 && dy.k > 0) throw Refused();
      return status_of([&] {
         return fufft_rms_norm_grad(dy.p, dy.type, dy.ld, h.p, h.ld, t.p, t.ld, h.type, w, eps, dx.p, dx.type, dx.ld, dw, work,
                                    splits, dy.rows, dy.k, stream);
      });
   });
}

// ---- decaying attention ----------------------------------------------------------------------

// a tensor of (batch, tokens, heads, dim), or (batch, heads, dim) for one token
struct Heads {
   void*         p;
   int           type;
   fufft_strides s;
   int64_t       batch, tokens, heads, dim;
};
Heads heads_of(PyObject* o, int dims, int64_t gpu)
{
   const at::Tensor& t = tensor(o, gpu);
   if(t.dim() != dims) throw Refused();
   const bool many = dims == 4;
   Heads h{nullptr, element(t), {t.stride(0), many ? t.stride(1) : 0, t.stride(dims - 2)},
           t.size(0), many ? t.size(1) : 1, t.size(dims - 2), t.size(dims - 1)};
   if(h.dim > 1 && t.stride(dims - 1) != 1) throw Refused();
   h.p = t.data_ptr();
   return h;
}
void alike(const Heads& a, const Heads& b, bool dim)
{
   if(a.type != b.type || a.batch != b.batch || a.tokens != b.tokens || a.heads != b.heads || (dim && a.dim != b.dim))
      throw Refused();
}
float* states_of(PyObject* o, const Heads& q, int64_t dv, int64_t gpu)
{
   if(o == Py_None) return nullptr;
   float* const p = static_cast<float*>(array(o, at::kFloat, 4 * q.batch * q.heads * q.dim * dv, gpu));
   const at::Tensor& t = THPVariable_Unpack(o);
   if(t.dim() > 1 && (t.dim() != 4 || t.size(0) != q.batch || t.size(1) != q.heads || t.size(2) != q.dim || t.size(3) != dv))
      throw Refused();
   return p;
}
struct Work {
   float*  p;
   int64_t splits;
};
Work work_of(PyObject* o, int64_t each, int64_t gpu)
{
   if(o == Py_None || each == 0) return {nullptr, 0};
   const int64_t n = tensor(o, gpu).numel() / each;
   return {n == 0 ? nullptr : static_cast<float*>(array(o, at::kFloat, 4 * n * each, gpu)), n};
}
const int32_t* lens_of(PyObject* o, int64_t batch, int64_t gpu)
{
   return o == Py_None ? nullptr : static_cast<const int32_t*>(array(o, at::kInt, 4 * batch, gpu));
}

PyObject* decay_attention(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 12, [&] {
      const int64_t gpu = integer(a[11]);
      void* const stream = handle(a[10]);
      const float scale = (float)number(a[9]);
      const Heads q = heads_of(a[0], 4, gpu), k = heads_of(a[1], 4, gpu), v = heads_of(a[2], 4, gpu), out = heads_of(a[4], 4, gpu);
      alike(q, k, true);
      alike(q, v, false);
      alike(v, out, true);
      const float* const g = static_cast<const float*>(array(a[3], at::kFloat, 4 * q.heads, gpu));
      const float* const state = states_of(a[5], q, v.dim, gpu);
      float* const next = states_of(a[6], q, v.dim, gpu);
      const int32_t* const lens = lens_of(a[7], q.batch, gpu);
      const Work w = work_of(a[8], q.batch * q.heads * q.dim * v.dim, gpu);
      return status_of([&] {
         return fufft_decay_attention(q.p, &q.s, k.p, &k.s, v.p, &v.s, q.type, g, out.p, &out.s, state, next, lens, scale, q.batch,
                                      q.tokens, q.heads, q.dim, v.dim, w.p, w.splits, stream);
      });
   });
}

PyObject* decay_attention_grad(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 16, [&] {
      const int64_t gpu = integer(a[15]);
      void* const stream = handle(a[14]);
      const float scale = (float)number(a[13]);
      const Heads o = heads_of(a[0], 4, gpu), q = heads_of(a[1], 4, gpu), k = heads_of(a[2], 4, gpu), v = heads_of(a[3], 4, gpu);
      const Heads dq = heads_of(a[5], 4, gpu), dk = heads_of(a[6], 4, gpu), dv = heads_of(a[7], 4, gpu);
      alike(q, k, true);
      alike(q, v, false);
      alike(v, o, true);
      alike(q, dq, true);
      alike(q, dk, true);
      alike(v, dv, true);
      const float* const g = static_cast<const float*>(array(a[4], at::kFloat, 4 * q.heads, gpu));
      const float *const state = states_of(a[8], q, v.dim, gpu), *const dnew = states_of(a[9], q, v.dim, gpu);
      float* const dstate = states_of(a[10], q, v.dim, gpu);
      const int32_t* const lens = lens_of(a[11], q.batch, gpu);
      const Work w = work_of(a[12], 3 * q.batch * q.heads * q.dim * v.dim, gpu);
      return status_of([&] {
         return fufft_decay_attention_grad(o.p, &o.s, q.p, &q.s, k.p, &k.s, v.p, &v.s, q.type, g, dq.p, &dq.s, dk.p, &dk.s, dv.p,
                                           &dv.s, state, dnew, dstate, lens, scale, q.batch, q.tokens, q.heads, q.dim, v.dim, w.p,
                                           w.splits, stream);
      });
   });
}

PyObject* decay_attention_step(PyObject*, PyObject* const* a, Py_ssize_t n)
{
   return guarded(n, 10, [&] {
      const int64_t gpu = integer(a[9]);
      void* const stream = handle(a[8]);
      const float scale = (float)number(a[7]);
      const Heads q = heads_of(a[0], 3, gpu), k = heads_of(a[1], 3, gpu), v = heads_of(a[2], 3, gpu), out = heads_of(a[5], 3, gpu);
      alike(q, k, true);
      alike(q, v, false);
      alike(v, out, true);
      const float* const g = static_cast<const float*>(array(a[3], at::kFloat, 4 * q.heads, gpu));
      const at::Tensor& s = tensor(a[4], gpu);
      if(s.dim() != 4 || s.size(1) != q.heads || s.size(2) != q.dim || s.size(3) != v.dim) throw Refused();
      const int64_t count = s.size(0);
      if(a[6] == Py_None && count < q.batch) throw Refused();
      float* const state = static_cast<float*>(array(a[4], at::kFloat, 4 * count * q.heads * q.dim * v.dim, gpu));
      const int64_t* const slots = a[6] == Py_None ? nullptr : static_cast<const int64_t*>(array(a[6], at::kLong, 8 * q.batch, gpu));
      return status_of([&] {
         return fufft_decay_attention_step(q.p, &q.s, k.p, &k.s, v.p, &v.s, q.type, g, out.p, &out.s, state, count, slots, scale,
                                           q.batch, q.heads, q.dim, v.dim, stream);
      });
   });
}

#define FUFFT_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FUFFT_METHOD(quantize),    FUFFT_METHOD(dequantize), FUFFT_METHOD(matmul),
                         FUFFT_METHOD(linear),      FUFFT_METHOD(cache_write), FUFFT_METHOD(cache_read),
                         FUFFT_METHOD(cache_conv),
                         FUFFT_METHOD(i8_quantize), FUFFT_METHOD(i8_dequantize), FUFFT_METHOD(i8_matmul),
                         FUFFT_METHOD(rms_norm),    FUFFT_METHOD(rms_norm_grad), FUFFT_METHOD(decay_attention),
                         FUFFT_METHOD(decay_attention_grad), FUFFT_METHOD(decay_attention_step),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "The 4-bit, 8-bit, norm and decaying-attention calls, checked and made in native code.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void)
{
   PyObject* const m = PyModule_Create(&module);
   // what it was built for: tensors are read through inline code, and the calls through the header
   if(m && (PyModule_AddStringConstant(m, "TORCH", TORCH_VERSION) || PyModule_AddIntConstant(m, "ABI", FUFFT_ABI_VERSION))) {
      Py_DECREF(m);
      return nullptr;
   }
   return m;
}
