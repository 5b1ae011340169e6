// The operators over torch tensors (ops.py) without an interpreter between the tensors and the C ABI: shapes, types and places are read and
// checked here, results are made here, and the entry points of libfr_b200.so are called with torch's current stream.  A call costs 3.5 to
// 5 us of the host this way, of which the memory of the result is 1.3 and the launch most of the rest; through ctypes it took 10 to 28.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>

#include <string>
#include <vector>

#include "../../include/fr_b200.h"

namespace {

decltype(&fr_b200_linear) p_linear;
decltype(&fr_b200_linear_workspace) p_linear_workspace;
decltype(&fr_b200_conv_seq) p_conv_seq;
decltype(&fr_b200_conv_step) p_conv_step;
decltype(&fr_b200_ssm_seq) p_ssm_seq;
decltype(&fr_b200_ssm_step) p_ssm_step;
decltype(&fr_b200_ssm_seq_workspace) p_ssm_workspace;
decltype(&fr_b200_slots_copy) p_slots_copy;

struct Bad {};   // a Python error is set
[[noreturn]] void bad(const char *fmt, ...) {
  va_list v;
  va_start(v, fmt);
  PyErr_FormatV(PyExc_ValueError, fmt, v);
  va_end(v);
  throw Bad{};
}
const at::Tensor *tensor(PyObject *o, const char *what) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) bad("%s is not a tensor", what);
  const at::Tensor &t = THPVariable_Unpack(o);
  if (t.requires_grad() && c10::GradMode::is_enabled()) bad("%s requires a gradient, and none flows through this operator: call it under torch.no_grad()", what);
  return &t;
}
const at::Tensor &needed(PyObject *o, const char *what) {
  const at::Tensor *t = tensor(o, what);
  if (!t) bad("%s is missing", what);
  return *t;
}
int element_of(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return FR_B200_T_F16;
    case at::kFloat: return FR_B200_T_F32;
    case at::kBFloat16: return FR_B200_T_BF16;
    default: return -1;
  }
}
int element_of(const at::Tensor &x) {
  if (!x.is_cuda()) bad("x is not on a GPU: there is no CPU path");
  const int e = element_of(x.scalar_type());
  if (e < 0) bad("x has a type other than float16, bfloat16 and float32");
  return e;
}

// a [rows, width] tensor with adjacent elements
struct Rows {
  void *p = nullptr;
  int64_t ld = 0;
};
Rows rows_of(const at::Tensor &t, const char *what, int64_t width, const at::Tensor *like) {
  if (t.dim() != 2) bad("%s has %lld dimensions instead of 2", what, (long long)t.dim());
  const auto size = t.sizes(), stride = t.strides();
  if (width >= 0 && size[1] != width) bad("%s is %lld wide instead of %lld", what, (long long)size[1], (long long)width);
  if (like && (t.scalar_type() != like->scalar_type() || t.device() != like->device() || size[0] != like->sizes()[0]))
    bad("%s differs from x in type, device or rows", what);
  if (size[1] > 1 && stride[1] != 1) bad("the elements of a row of %s are not adjacent", what);
  return {t.data_ptr(), size[0] > 1 ? stride[0] : size[1]};
}
Rows rows_of(const at::Tensor *t, const char *what, int64_t width, const at::Tensor *like) { return t ? rows_of(*t, what, width, like) : Rows{}; }
// an fp32 parameter of [a] or [a, b], or none
const float *param(PyObject *o, const char *what, int64_t a, int64_t b, const at::Tensor &like) {
  const at::Tensor *t = tensor(o, what);
  if (!t) return nullptr;
  const auto size = t->sizes();
  const bool shape = b < 0 ? size.size() == 1 && size[0] == a : size.size() == 2 && size[0] == a && size[1] == b;
  if (!shape || t->scalar_type() != at::kFloat || t->device() != like.device() || !t->is_contiguous())
    bad("%s is not a contiguous fp32 tensor of its shape on the device of x", what);
  return static_cast<const float *>(t->data_ptr());
}
// a pool [slots, ...] of whole slots of `inner` elements
struct Pool {
  void *p = nullptr;
  int64_t stride = 0;
  int slots = 0;
};
int64_t slot_elements(const at::Tensor &t, const char *what) {
  int64_t want = 1;
  for (int64_t i = t.dim() - 1; i >= 1; --i) {
    if (t.sizes()[i] > 1 && t.strides()[i] != want) bad("a slot of %s is not contiguous", what);
    want *= t.sizes()[i];
  }
  return want;
}
Pool pool_of(PyObject *o, at::ScalarType type, int64_t a, int64_t b, const at::Tensor &like) {
  const at::Tensor *t = tensor(o, "state");
  if (!t) return {};
  if (t->dim() != 3 || t->scalar_type() != type || t->device() != like.device() || t->sizes()[1] != a || t->sizes()[2] != b)
    bad("state is not a [slots, %lld, %lld] tensor of its type on the device of x", (long long)a, (long long)b);
  const int64_t each = slot_elements(*t, "state"), slots = t->sizes()[0];
  if (slots > INT32_MAX) bad("too many slots");
  return {t->data_ptr(), slots > 1 ? t->strides()[0] : each, (int)slots};
}
at::Tensor result(PyObject *o, const at::Tensor &x, int64_t rows, int64_t width, at::ScalarType type) {
  const at::Tensor *t = tensor(o, "out");
  if (!t) return at::empty({rows, width}, x.options().dtype(type));
  if (t->dim() != 2 || t->scalar_type() != type || t->device() != x.device() || t->sizes()[0] != rows || t->sizes()[1] != width)
    bad("out is not a [%lld, %lld] tensor of its type on the device of x", (long long)rows, (long long)width);
  return *t;
}

// host integers: a list, a buffer of int32 (numpy), another sequence of integers, a CPU tensor; one number stands for all where that is
// allowed.  n < 0: as many as there are.
struct Ints {
  std::vector<int32_t> own;
  Py_buffer view{};
  const int32_t *p = nullptr;
  int64_t n = 0;
  ~Ints() { if (view.obj) PyBuffer_Release(&view); }
  void take(PyObject *o, int64_t want, const char *what, bool one_for_all) {
    if (o == Py_None) return;
    if (one_for_all && PyLong_Check(o)) {
      own.assign(want > 0 ? want : 1, number(o, what));
      p = own.data();
      n = want;
      return;
    }
    if (THPVariable_Check(o)) {
      const at::Tensor &t = THPVariable_Unpack(o);
      if (t.is_cuda()) bad("%s is on the GPU: the call holds it by value, from the host", what);
      if (t.dim() != 1 || !at::isIntegralType(t.scalar_type(), false)) bad("%s is not a list of integers", what);
      const at::Tensor w = t.to(at::kLong).contiguous();
      for (int64_t i = 0; i < w.sizes()[0]; ++i) own.push_back(checked(w.data_ptr<int64_t>()[i], what));
      p = own.data();
      n = (int64_t)own.size();
    } else if (PyObject_CheckBuffer(o) && PyObject_GetBuffer(o, &view, PyBUF_FORMAT | PyBUF_C_CONTIGUOUS) == 0 && view.ndim == 1 && view.itemsize == 4 &&
               view.format && view.format[1] == 0 && (view.format[0] == 'i' || view.format[0] == 'l')) {
      p = static_cast<const int32_t *>(view.buf);
      n = view.shape[0];
    } else {
      PyErr_Clear();
      PyObject *s = PySequence_Fast(o, "");
      if (!s) bad("%s is not a list of integers", what);
      const int64_t len = PySequence_Fast_GET_SIZE(s);
      try {
        for (int64_t i = 0; i < len; ++i) {
          PyObject *index = PyNumber_Index(PySequence_Fast_GET_ITEM(s, i));
          if (!index) bad("%s is not a list of integers", what);
          try { own.push_back(number(index, what)); } catch (...) { Py_DECREF(index); throw; }
          Py_DECREF(index);
        }
      } catch (...) { Py_DECREF(s); throw; }
      Py_DECREF(s);
      own.reserve(1);
      p = own.data();
      n = len;
    }
    if (want >= 0 && n != want) bad("%s has %lld entries instead of %lld", what, (long long)n, (long long)want);
  }
  static int32_t checked(int64_t v, const char *what) {
    if (v < INT32_MIN || v > INT32_MAX) bad("%s has an entry that is no 32-bit integer", what);
    return (int32_t)v;
  }
  static int32_t number(PyObject *o, const char *what) {
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &over);
    if (over) bad("%s has an entry that is no 32-bit integer", what);
    if (v == -1 && PyErr_Occurred()) throw Bad{};
    return checked(v, what);
  }
};

void arguments(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) bad("%lld arguments instead of %lld", (long long)got, (long long)want);
}
int fit(int64_t v, const char *what) {
  if (v > INT32_MAX) bad("%s is too long", what);
  return (int)v;
}
struct Place {
  int device;
  void *stream;
  explicit Place(const at::Tensor &x) : device(x.get_device()), stream(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)x.get_device()).stream()) {}
};
// Scratch of a call.  It goes back to the allocator behind the call: what gets it next on this stream comes after.
at::Tensor work_area(size_t bytes, const at::Tensor &x) { return bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : at::Tensor(); }
// a tensor, or the negative status
PyObject *answer(int rc, const at::Tensor &t) { return rc < 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(t); }

template <typename F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (const Bad &) {
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// x, w, bias, activation, residual, out, out dtype
PyObject *py_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    arguments(n, 7);
    const at::Tensor &x = needed(a[0], "x"), &w = needed(a[1], "w");
    const int dt = element_of(x);
    const Rows xr = rows_of(x, "x", -1, nullptr);
    const int64_t rows = x.sizes()[0], k = x.sizes()[1];
    if (w.scalar_type() != x.scalar_type() || w.device() != x.device()) bad("w differs from x in type or device");
    const Rows wr = rows_of(w, "w", k, nullptr);
    const int64_t channels = w.sizes()[0];
    at::ScalarType type = x.scalar_type();
    if (a[6] != Py_None) {
      if (!THPDtype_Check(a[6])) bad("out_dtype is not a dtype");
      type = reinterpret_cast<THPDtype *>(a[6])->scalar_type;
    } else if (const at::Tensor *o = tensor(a[5], "out")) type = o->scalar_type();
    const int out_dt = element_of(type);
    if (out_dt < 0) bad("the result is of the type of x, or float32");
    const at::Tensor out = result(a[5], x, rows, channels, type);
    const Rows orow = rows_of(out, "out", -1, nullptr);
    const at::Tensor *res = tensor(a[4], "the residual");
    if (res && (res->scalar_type() != type || res->device() != x.device() || res->dim() != 2 || res->sizes()[0] != rows))
      bad("the residual differs from the result in type, device or rows");
    const Rows rr = rows_of(res, "the residual", channels, nullptr);
    const float *bias = param(a[2], "bias", channels, -1, x);
    const Place at(x);
    const int ki = fit(k, "x"), ni = fit(channels, "w");
    const size_t need = p_linear_workspace(xr.p, xr.ld, wr.p, wr.ld, rows, ki, ni);
    const at::Tensor work = work_area(need, x);
    return answer(p_linear(xr.p, xr.ld, wr.p, wr.ld, dt, rows, ki, ni, bias, (int)PyLong_AsLong(a[3]), rr.p, rr.ld, orow.p, orow.ld, out_dt,
                           need ? work.data_ptr() : nullptr, need, at.device, at.stream), out);
  });
}

// x, w, bias, activation, state, from, to, out, starts, whether sequences
PyObject *py_conv(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    arguments(n, 10);
    const at::Tensor &x = needed(a[0], "x"), &w = needed(a[1], "w");
    const int dt = element_of(x);
    const Rows xr = rows_of(x, "x", -1, nullptr);
    const int64_t rows = x.sizes()[0], d = x.sizes()[1];
    if (w.dim() != 2) bad("w has %lld dimensions instead of 2", (long long)w.dim());
    const int64_t taps = w.sizes()[1];
    const float *wp = param(a[1], "w", d, taps, x), *bias = param(a[2], "bias", d, -1, x);
    const at::Tensor out = result(a[7], x, rows, d, x.scalar_type());
    const Rows orow = rows_of(out, "out", -1, nullptr);
    const Pool pool = pool_of(a[4], x.scalar_type(), taps - 1, d, x);
    const bool seq = a[9] == Py_True;
    Ints starts, from, to;
    int64_t streams = rows;
    if (seq) {
      starts.take(a[8], -1, "starts", false);
      if (starts.p && starts.n < 1) bad("starts has the first row of every sequence and the end of the last");
      streams = a[8] == Py_None ? 1 : starts.n - 1;
    }
    from.take(a[5], streams, "from_slots", true);
    to.take(a[6], streams, "to_slots", true);
    const int act = (int)PyLong_AsLong(a[3]);
    const Place at(x);
    const int rc = seq ? p_conv_seq(xr.p, xr.ld, dt, rows, fit(d, "x"), wp, fit(taps, "w"), bias, act, starts.p, fit(streams, "starts"), pool.p, pool.stride,
                                    pool.slots, from.p, to.p, orow.p, orow.ld, at.device, at.stream)
                       : p_conv_step(xr.p, xr.ld, dt, fit(rows, "x"), fit(d, "x"), wp, fit(taps, "w"), bias, act, pool.p, pool.stride, pool.slots, from.p, to.p,
                                     orow.p, orow.ld, at.device, at.stream);
    return answer(rc, out);
  });
}

// x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, from, to, out, starts, whether sequences
PyObject *py_ssm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    arguments(n, 15);
    const at::Tensor &x = needed(a[0], "x"), &A = needed(a[2], "A"), &B = needed(a[3], "B"), &C = needed(a[4], "C");
    const int dt = element_of(x);
    const Rows xr = rows_of(x, "x", -1, nullptr);
    const int64_t rows = x.sizes()[0], d = x.sizes()[1];
    if (A.dim() != 2) bad("A has %lld dimensions instead of 2", (long long)A.dim());
    const int64_t states = A.sizes()[1];
    const float *Ap = param(a[2], "A", d, states, x), *skip = param(a[5], "D", d, -1, x), *bias = param(a[7], "dt_bias", d, -1, x);
    const Rows tr = rows_of(needed(a[1], "dt"), "dt", d, &x), br = rows_of(B, "B", -1, &x), cr = rows_of(C, "C", B.sizes()[1], &x);
    if (states < 1 || B.sizes()[1] % states) bad("B is not [rows, groups * N]");
    const int64_t groups = B.sizes()[1] / states;
    const Rows zr = rows_of(tensor(a[6], "z"), "z", d, &x);
    const at::Tensor out = result(a[12], x, rows, d, x.scalar_type());
    const Rows orow = rows_of(out, "out", -1, nullptr);
    const Pool pool = pool_of(a[9], at::kFloat, d, states, x);
    const bool seq = a[14] == Py_True;
    Ints starts, from, to;
    int64_t streams = rows;
    if (seq) {
      starts.take(a[13], -1, "starts", false);
      if (starts.p && starts.n < 1) bad("starts has the first row of every sequence and the end of the last");
      streams = a[13] == Py_None ? 1 : starts.n - 1;
    }
    from.take(a[10], streams, "from_slots", true);
    to.take(a[11], streams, "to_slots", true);
    const int softplus = PyObject_IsTrue(a[8]);
    if (softplus < 0) throw Bad{};
    const int di = fit(d, "x"), ni = fit(states, "A"), gi = fit(groups, "B");
    const Place at(x);
    if (!seq)
      return answer(p_ssm_step(xr.p, xr.ld, tr.p, tr.ld, Ap, br.p, br.ld, cr.p, cr.ld, skip, zr.p, zr.ld, bias, softplus, dt, fit(rows, "x"), di, ni, gi,
                               static_cast<float *>(pool.p), pool.stride, pool.slots, from.p, to.p, orow.p, orow.ld, at.device, at.stream), out);
    const size_t need = p_ssm_workspace(rows, fit(streams, "starts"), di, ni);
    const at::Tensor work = work_area(need, x);
    return answer(p_ssm_seq(xr.p, xr.ld, tr.p, tr.ld, Ap, br.p, br.ld, cr.p, cr.ld, skip, zr.p, zr.ld, bias, softplus, dt, rows, di, ni, gi, starts.p,
                            (int)streams, static_cast<float *>(pool.p), pool.stride, pool.slots, from.p, to.p, orow.p, orow.ld,
                            need ? work.data_ptr() : nullptr, need, at.device, at.stream), out);
  });
}

// pool, src, dst
PyObject *py_copy_slots(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    arguments(n, 3);
    const at::Tensor &pool = needed(a[0], "pool");
    if (!pool.is_cuda() || pool.dim() < 1) bad("pool is not a GPU tensor of slots");
    const int64_t es = pool.element_size(), each = slot_elements(pool, "the pool") * es, slots = pool.sizes()[0];
    Ints src, dst;
    src.take(a[1], -1, "src", false);
    dst.take(a[2], src.n, "dst", false);
    if (a[1] == Py_None || a[2] == Py_None) bad("src and dst are two lists of as many slots");
    const Place at(pool);
    const int rc = p_slots_copy(pool.data_ptr(), each, (slots > 1 ? pool.strides()[0] * es : each), fit(slots, "the pool"), fit(src.n, "src"), src.p, dst.p,
                                at.device, at.stream);
    if (rc < 0) return PyLong_FromLong(rc);
    Py_INCREF(a[0]);
    return a[0];
  });
}

// the path of libfr_b200.so
PyObject *py_bind(PyObject *, PyObject *path) {
  const char *s = PyUnicode_AsUTF8(path);
  if (!s) return nullptr;
  void *h = dlopen(s, RTLD_NOW | RTLD_LOCAL);
  if (!h) { PyErr_SetString(PyExc_RuntimeError, dlerror()); return nullptr; }
  bool ok = true;
  auto get = [&](auto &f, const char *name) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(h, name)); ok = ok && f; };
  get(p_linear, "fr_b200_linear");
  get(p_linear_workspace, "fr_b200_linear_workspace");
  get(p_conv_seq, "fr_b200_conv_seq");
  get(p_conv_step, "fr_b200_conv_step");
  get(p_ssm_seq, "fr_b200_ssm_seq");
  get(p_ssm_step, "fr_b200_ssm_step");
  get(p_ssm_workspace, "fr_b200_ssm_seq_workspace");
  get(p_slots_copy, "fr_b200_slots_copy");
  if (!ok) { PyErr_SetString(PyExc_RuntimeError, "libfr_b200.so lacks an operator"); return nullptr; }
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"bind", py_bind, METH_O, nullptr}, {"linear", FAST(py_linear), nullptr}, {"conv", FAST(py_conv), nullptr},
                         {"ssm", FAST(py_ssm), nullptr}, {"copy_slots", FAST(py_copy_slots), nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fr_b200_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fr_b200_torch() { return PyModule_Create(&module); }
