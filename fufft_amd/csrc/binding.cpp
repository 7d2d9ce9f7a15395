// The short way from Python to the 4-bit calls: reads the tensors' properties, checks them
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

#define FUFFT_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FUFFT_METHOD(quantize),    FUFFT_METHOD(dequantize), FUFFT_METHOD(matmul),
                         FUFFT_METHOD(linear),      FUFFT_METHOD(cache_write), FUFFT_METHOD(cache_read),
                         FUFFT_METHOD(cache_conv), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "The 4-bit calls, checked and made in native code.", -1, methods,
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
