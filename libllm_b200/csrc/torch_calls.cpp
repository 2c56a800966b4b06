// The quick way from torch tensors to the kernels of a step's output end (ops.py): a call's tensors are looked at, its result is allocated and its
// kernel launched without a Python-level step for each.  Interpreted, these steps take three times as long as the launch and more than a small
// kernel itself (8 rows x 2,048 brought into four bits: 6.6 us a call for a kernel of 1.4; one row of 128,256 logits: 10.3 for 2.3).
//
// Every function answers None when anything about a call is not plainly right, and ops.py then goes through its own checks, which say what it
// is; a tensor when the kernel was launched; and a status when the kernel's library refused.  No C++ exception leaves a function.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "fp4.h"
#include "logits.h"

namespace {

int (*g_quantize)(const Fp4QuantizeCall *) = nullptr;
int (*g_dequantize)(const Fp4DequantizeCall *) = nullptr;
int (*g_gemm)(const Fp4GemmCall *) = nullptr;
int (*g_adjust)(const AdjustLogitsCall *) = nullptr;

struct Wrong {};
void need(bool ok) {
  if (!ok) throw Wrong();
}

// bind(name, address): where a kernel family's function lies.
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  const char *name = n == 2 ? PyUnicode_AsUTF8(args[0]) : nullptr;
  void *p = name ? PyLong_AsVoidPtr(args[1]) : nullptr;
  if (!p || PyErr_Occurred()) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_TypeError, "bind(name, address)");
  const std::string f = name;
  if (f == "llm_fp4_quantize") g_quantize = (int (*)(const Fp4QuantizeCall *))p;
  else if (f == "llm_fp4_dequantize") g_dequantize = (int (*)(const Fp4DequantizeCall *))p;
  else if (f == "llm_fp4_gemm") g_gemm = (int (*)(const Fp4GemmCall *))p;
  else if (f == "llm_adjust_logits") g_adjust = (int (*)(const AdjustLogitsCall *))p;
  else return PyErr_Format(PyExc_ValueError, "no function '%s'", name);
  Py_RETURN_NONE;
}

const at::Tensor &tensor(PyObject *o) {
  need(THPVariable_CheckExact(o));
  return THPVariable_Unpack(o);
}
const at::Tensor *tensor_or_none(PyObject *o) { return o == Py_None ? nullptr : &tensor(o); }
long long number(PyObject *o) {
  need(PyLong_CheckExact(o));
  const long long v = PyLong_AsLongLong(o);
  need(!(v == -1 && PyErr_Occurred()));
  return v;
}
// The current device's stream, if the tensor lies there and is an ordinary one.
struct Place {
  int device;
  void *stream;
  explicit Place(const at::Tensor &t) {
    device = on_gpu(t) ? t.get_device() : -1;
    need(device >= 0 && device == c10::cuda::current_device());
    stream = (void *)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  }
  static bool on_gpu(const at::Tensor &t) { return t.is_cuda() && t.layout() == at::kStrided && t.has_storage(); }
  void same(const at::Tensor &t) const { need(on_gpu(t) && t.get_device() == device); }
};
int code(at::ScalarType t) {
  need(t == at::kFloat || t == at::kBFloat16);
  return t == at::kFloat ? 0 : 1;
}
PyObject *answer(int status, at::Tensor &&t) { return status ? PyLong_FromLong(status) : THPVariable_Wrap(std::move(t)); }

// A matrix in four bits as ops.Fp4Matrix lays it out.
struct Layout {
  long long scales, row_scale, bytes;
  Layout(long long rows, long long cols, long long format) {
    need(rows >= 0 && rows < (1ll << 40) && cols > 0 && cols <= (1ll << 28) && (format == 0 || format == 1));
    scales = (rows * ((cols + 31) / 32 * 16) + 511) / 512 * 512;
    row_scale = scales + (rows + 127) / 128 * ((cols + 255) / 256) * (format == 0 ? 2048 : 1024);
    bytes = row_scale + 4 * rows;
  }
};

template <typename Body>
PyObject *guarded(Body body) {
  try {
    return body();
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// fp4_quantize(x, format) -> the bytes of the matrix
PyObject *fp4_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    need(n == 2 && g_quantize);
    const at::Tensor &x = tensor(args[0]);
    need(x.dim() == 2 && (x.stride(1) == 1 || x.size(1) == 1));
    Fp4QuantizeCall c = {};
    c.dtype = code(x.scalar_type());
    c.rows = x.size(0);
    c.cols = x.size(1);
    c.format = number(args[1]);
    const Layout l(c.rows, c.cols, c.format);
    const Place place(x);
    at::Tensor data = at::empty({l.bytes}, x.options().dtype(at::kByte));
    unsigned char *p = (unsigned char *)data.data_ptr();
    c.x = x.data_ptr();
    c.ldx = x.stride(0);
    c.codes = p;
    c.scales = p + l.scales;
    c.row_scale = (float *)(p + l.row_scale);
    c.stream = place.stream;
    return answer(g_quantize(&c), std::move(data));
  });
}

// fp4_dequantize(data, rows, cols, format, is bfloat16) -> values
PyObject *fp4_dequantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    need(n == 5 && g_dequantize);
    const at::Tensor &data = tensor(args[0]);
    Fp4DequantizeCall c = {};
    c.rows = number(args[1]);
    c.cols = c.ldo = number(args[2]);
    c.format = number(args[3]);
    c.dtype = number(args[4]);
    need(c.dtype == 0 || c.dtype == 1);
    const Layout l(c.rows, c.cols, c.format);
    need(data.scalar_type() == at::kByte && data.is_contiguous() && data.numel() == l.bytes);
    const Place place(data);
    at::Tensor out = at::empty({c.rows, c.cols}, data.options().dtype(c.dtype ? at::kBFloat16 : at::kFloat));
    const unsigned char *p = (const unsigned char *)data.data_ptr();
    c.codes = p;
    c.scales = p + l.scales;
    c.row_scale = (const float *)(p + l.row_scale);
    c.out = out.data_ptr();
    c.stream = place.stream;
    return answer(g_dequantize(&c), std::move(out));
  });
}

// fp4_gemm(x data, w data, M, N, K, format, is bfloat16, status word) -> out
PyObject *fp4_gemm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    need(n == 8 && g_gemm);
    const at::Tensor &x = tensor(args[0]), &w = tensor(args[1]);
    Fp4GemmCall c = {};
    c.M = number(args[2]);
    c.N = c.ldo = number(args[3]);
    c.K = number(args[4]);
    c.format = number(args[5]);
    c.out_dtype = number(args[6]);
    c.status = (int *)number(args[7]);
    need((c.out_dtype == 0 || c.out_dtype == 1) && c.M < (1 << 30) && c.N < (1 << 30) && c.status);
    const Layout lx(c.M, c.K, c.format), lw(c.N, c.K, c.format);
    need(x.scalar_type() == at::kByte && x.is_contiguous() && x.numel() == lx.bytes);
    need(w.scalar_type() == at::kByte && w.is_contiguous() && w.numel() == lw.bytes);
    const Place place(w);
    place.same(x);
    at::Tensor out = at::empty({c.M, c.N}, w.options().dtype(c.out_dtype ? at::kBFloat16 : at::kFloat));
    const unsigned char *px = (const unsigned char *)x.data_ptr(), *pw = (const unsigned char *)w.data_ptr();
    c.x_codes = px;
    c.x_scales = px + lx.scales;
    c.x_row = (const float *)(px + lx.row_scale);
    c.w_codes = pw;
    c.w_scales = pw + lw.scales;
    c.w_row = (const float *)(pw + lw.row_scale);
    c.out = out.data_ptr();
    c.stream = place.stream;
    return answer(g_gemm(&c), std::move(out));
  });
}

bool per_row(const at::Tensor &t, at::ScalarType type, long long rows) {
  return t.scalar_type() == type && t.dim() == 1 && t.size(0) == rows && (rows <= 1 || t.stride(0) == 1);
}
// A number for all rows, or a tensor with one per row.
void penalty(PyObject *o, long long rows, const Place &place, bool positive, const float **p, double *all) {
  if (PyFloat_CheckExact(o)) {
    *all = PyFloat_AS_DOUBLE(o);
    need(std::isfinite((float)*all) && (!positive || (float)*all > 0));
    return;
  }
  const at::Tensor &t = tensor(o);
  need(per_row(t, at::kFloat, rows));
  place.same(t);
  *p = (const float *)t.data_ptr();
}

// adjust_logits(logits, out, history, slots, lengths, repetition, presence, frequency, bias, allowed) -> out; tensors that are not given None
PyObject *adjust_logits(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    need(n == 10 && g_adjust);
    const at::Tensor &x = tensor(args[0]);
    need(x.dim() == 2 && x.scalar_type() == at::kFloat && (x.stride(1) == 1 || x.size(1) == 1));
    AdjustLogitsCall c = {};
    c.B = x.size(0);
    c.V = x.size(1);
    need(c.B <= 65535 && c.V <= (1ll << 30));
    c.ld = x.stride(0);
    const Place place(x);
    c.stream = place.stream;
    const at::Tensor *given = tensor_or_none(args[1]);
    if (given) {
      need(given->dim() == 2 && given->scalar_type() == at::kFloat && given->size(0) == c.B && given->size(1) == c.V);
      need((given->stride(1) == 1 || c.V <= 1) && (given->stride(0) >= c.V || c.B <= 1));
      place.same(*given);
      c.ldo = given->stride(0);
    }
    if (const at::Tensor *h = tensor_or_none(args[2])) {
      need(h->dim() == 2 && h->scalar_type() == at::kInt && (h->stride(1) == 1 || h->size(1) <= 1) && h->numel() > 0);
      place.same(*h);
      const at::Tensor &lengths = tensor(args[4]);
      need(per_row(lengths, at::kInt, c.B));
      place.same(lengths);
      c.history = (const int *)h->data_ptr();
      c.ldh = h->stride(0);
      c.places = h->size(0);
      c.longest = h->size(1);
      c.lengths = (const int *)lengths.data_ptr();
      if (const at::Tensor *slots = tensor_or_none(args[3])) {
        need(per_row(*slots, at::kInt, c.B));
        place.same(*slots);
        c.slots = (const int *)slots->data_ptr();
      } else {
        need(c.B <= c.places);
      }
    } else {
      need(args[3] == Py_None && args[4] == Py_None);
    }
    penalty(args[5], c.B, place, true, &c.repetition, &c.repetition_all);
    penalty(args[6], c.B, place, false, &c.presence, &c.presence_all);
    penalty(args[7], c.B, place, false, &c.frequency, &c.frequency_all);
    if (const at::Tensor *b = tensor_or_none(args[8])) {
      const int64_t d = b->dim();
      need(b->scalar_type() == at::kFloat && (d == 1 || (d == 2 && b->size(0) == c.B)) && b->size(d - 1) == c.V && (b->stride(d - 1) == 1 || c.V <= 1));
      place.same(*b);
      c.bias = (const float *)b->data_ptr();
      c.ld_bias = d == 2 ? b->stride(0) : 0;
    }
    if (const at::Tensor *m = tensor_or_none(args[9])) {
      const int64_t d = m->dim(), words = (c.V + 31) / 32;
      need(m->scalar_type() == at::kInt && (d == 1 || (d == 2 && m->size(0) == c.B)) && m->size(d - 1) == words && (m->stride(d - 1) == 1 || words <= 1));
      place.same(*m);
      c.allowed = (const unsigned *)m->data_ptr();
      c.ld_allowed = d == 2 ? m->stride(0) : 0;
    }
    at::Tensor out = given ? *given : at::empty({c.B, c.V}, x.options());
    if (!given) c.ldo = c.V;
    c.logits = (const float *)x.data_ptr();
    c.out = (float *)out.data_ptr();
    const int status = g_adjust(&c);
    if (status || !given) return answer(status, std::move(out));
    Py_INCREF(args[1]);
    return args[1];
  });
}

PyMethodDef METHODS[] = {{"bind", (PyCFunction)(void *)bind, METH_FASTCALL, nullptr},
                         {"fp4_quantize", (PyCFunction)(void *)fp4_quantize, METH_FASTCALL, nullptr},
                         {"fp4_dequantize", (PyCFunction)(void *)fp4_dequantize, METH_FASTCALL, nullptr},
                         {"fp4_gemm", (PyCFunction)(void *)fp4_gemm, METH_FASTCALL, nullptr},
                         {"adjust_logits", (PyCFunction)(void *)adjust_logits, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "llm_torch_calls", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_llm_torch_calls() { return PyModule_Create(&MODULE); }
