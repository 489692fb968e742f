// The host path of ops.py: looks at the tensors of a call, allocates what it returns and calls the C ABI.
//
// A one-token op runs for 4 us on the device, and checking its ten tensors in Python, converting 27 arguments in ctypes
// and launching took 14; here it takes 9, of which the launch is 3.  Only Python's C API is used (tensors are looked at through
// their own methods), so that this file depends on no version of torch, and the entry points come from the library that
// _lib.py has loaded.
//
// A function returns its outputs; None when the arguments do not fit (ops.py finds out what is wrong and says so); an
// error code of the C ABI; or NotImplemented when another device than the tensors' is current.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <cstdint>

namespace {

typedef int (*StepFn)(const void*, int, const void*, int, const void*, int, const void*, int, const void*, int, const float*,
                      const float*, float*, int, const int32_t*, int, void*, int, int, int, int, int, float, int, int, void*);
typedef size_t (*WorkspaceFn)(int, int, int, int, int, int, int);
typedef int (*PrefillFn)(const void*, int, const void*, int, const void*, int, const void*, int, const void*, int, const float*,
                         const float*, float*, int, const int32_t*, const int32_t*, int, int, void*, int, int, int, int, int,
                         float, int, int, void*, size_t, void*);
typedef int (*SampleFn)(const void*, int64_t, int, int, int, const float*, const int32_t*, const float*, const float*,
                        const uint32_t*, float, const float*, int32_t*, int32_t*, float*, void*);
StepFn step_fn;
WorkspaceFn workspace_fn;
PrefillFn prefill_fn;
SampleFn sample_fn;

enum Type { kF16, kBF16, kF32, kI32, kU8, kTypes };  // the first three as dfssm_dtype
PyObject *types[kTypes], *tensor_type, *empty_like, *stream_of, *current_device;
PyObject *s_dtype, *s_shape, *s_get_device, *s_is_contiguous, *s_data_ptr, *s_stride, *s_new_empty, *kw_dtype;

// A reference that is given up at the end of its scope.
struct Ref {
  PyObject* o;
  explicit Ref(PyObject* p = nullptr) : o(p) {}
  ~Ref() { Py_XDECREF(o); }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
  PyObject* release() {
    PyObject* p = o;
    o = nullptr;
    return p;
  }
};

PyObject* method(PyObject* self, PyObject* name) { return PyObject_VectorcallMethod(name, &self, 1, nullptr); }

struct Tensor {
  PyObject* obj;
  char* ptr;
  int type;
  long device;
  int dims;
  long long n[4];
  bool contiguous;
  bool is(int t, long d, int nd) const { return type == t && device == d && dims == nd; }
  bool vector(int t, long d, long long len) const { return is(t, d, 1) && n[0] == len && contiguous; }
};

// In the functions below 1 is success, 0 an argument that does not fit, -1 a Python exception.
enum { kOk = 1, kNo = 0, kRaised = -1 };

int read(PyObject* o, Tensor& t) {
  if (!PyObject_TypeCheck(o, reinterpret_cast<PyTypeObject*>(tensor_type))) return kNo;
  t.obj = o;
  Ref dtype(PyObject_GetAttr(o, s_dtype)), shape(PyObject_GetAttr(o, s_shape));
  if (!dtype.o || !shape.o) return kRaised;
  t.type = -1;
  for (int i = 0; i < kTypes; ++i)
    if (dtype.o == types[i]) t.type = i;
  if (!PyTuple_Check(shape.o) || PyTuple_GET_SIZE(shape.o) > 4) return kNo;
  t.dims = (int)PyTuple_GET_SIZE(shape.o);
  for (int i = 0; i < t.dims; ++i) {
    t.n[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape.o, i));
    if (t.n[i] == -1 && PyErr_Occurred()) return kRaised;
    if (t.n[i] > INT32_MAX && !(t.type == kU8 && t.dims == 1)) return kNo;
  }
  Ref device(method(o, s_get_device));
  if (!device.o) return kRaised;
  t.device = PyLong_AsLong(device.o);
  if (t.device == -1 && PyErr_Occurred()) return kRaised;
  if (t.device < 0) return kNo;
  Ref contiguous(method(o, s_is_contiguous)), ptr(method(o, s_data_ptr));
  if (!contiguous.o || !ptr.o) return kRaised;
  t.contiguous = contiguous.o == Py_True;
  t.ptr = static_cast<char*>(PyLong_AsVoidPtr(ptr.o));
  return !t.ptr && PyErr_Occurred() ? kRaised : kOk;
}

// The stride of rows that are each contiguous, [rows][heads][width] or [rows][width]
int row_stride(const Tensor& t, long long& ld) {
  const long long width = t.dims == 3 ? t.n[1] * t.n[2] : t.n[1];
  ld = width;
  if (!t.contiguous) {
    Ref s(method(t.obj, s_stride));
    if (!s.o) return kRaised;
    long long st[3] = {};
    for (int i = 0; i < t.dims; ++i) {
      st[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(s.o, i));
      if (st[i] == -1 && PyErr_Occurred()) return kRaised;
    }
    if (st[t.dims - 1] != 1 && t.n[t.dims - 1] != 1) return kNo;
    if (t.dims == 3 && st[1] != t.n[2] && t.n[1] != 1) return kNo;
    if (t.n[0] > 1) ld = st[0];
  }
  return ld >= width && ld <= INT32_MAX ? kOk : kNo;
}

int on_current_device(long device, void*& stream, bool& elsewhere) {
  Ref now(PyObject_CallNoArgs(current_device));
  if (!now.o) return kRaised;
  const long d = PyLong_AsLong(now.o);
  if (d == -1 && PyErr_Occurred()) return kRaised;
  elsewhere = d != device;
  if (elsewhere) return kOk;
  Ref index(PyLong_FromLong(device)), s(index.o ? PyObject_CallOneArg(stream_of, index.o) : nullptr);
  if (!s.o) return kRaised;
  stream = PyLong_AsVoidPtr(s.o);
  return !stream && PyErr_Occurred() ? kRaised : kOk;
}

// empty_like(t, dtype=...) / t.new_empty(size, dtype=...)
PyObject* like(PyObject* t, PyObject* dtype) {
  PyObject* a[2] = {t, dtype};
  return PyObject_Vectorcall(empty_like, a, 1, dtype ? kw_dtype : nullptr);
}
PyObject* new_empty(PyObject* t, PyObject* size, PyObject* dtype) {
  PyObject* a[3] = {t, size, dtype};
  return PyObject_VectorcallMethod(s_new_empty, a, 2, dtype ? kw_dtype : nullptr);
}
int pointer(PyObject* t, void*& p) {
  Ref ptr(method(t, s_data_ptr));
  if (!ptr.o) return kRaised;
  p = PyLong_AsVoidPtr(ptr.o);
  return !p && PyErr_Occurred() ? kRaised : kOk;
}

struct Delta {
  Tensor q, k, v, a, b, A_log, dt_bias, state, slots;
  long long lq, lk, lv, la, lb, lo;
  const int32_t* slot;
  Ref out;
  void *o, *stream;
  float scale;
  int qk_norm;
  bool elsewhere;
  int n() const { return (int)q.n[0]; }
};

// x: q, k, v, a, b, A_log, dt_bias, state
int delta(PyObject* const* x, PyObject* slots, long long n_seq, PyObject* scale, PyObject* qk_norm, PyObject* out, Delta& d) {
  Tensor* const t[8] = {&d.q, &d.k, &d.v, &d.a, &d.b, &d.A_log, &d.dt_bias, &d.state};
  for (int i = 0; i < 8; ++i)
    if (const int rc = read(x[i], *t[i]); rc != kOk) return rc;
  const Tensor &q = d.q, &k = d.k, &v = d.v, &a = d.a, &b = d.b, &s = d.state;
  const int type = q.type;
  const long dev = q.device;
  if ((type != kF16 && type != kBF16) || q.dims != 3 || !k.is(type, dev, 3) || !v.is(type, dev, 3) || !a.is(type, dev, 2) ||
      !b.is(type, dev, 2) || !s.is(kF32, dev, 4) || !s.contiguous)
    return kNo;
  const long long n = q.n[0], hk = q.n[1], dk = q.n[2], hv = v.n[1], dv = v.n[2];
  if (k.n[0] != n || k.n[1] != hk || k.n[2] != dk || v.n[0] != n || a.n[0] != n || a.n[1] != hv || b.n[0] != n || b.n[1] != hv ||
      s.n[1] != hv || s.n[2] != dv || s.n[3] != dk || !d.A_log.vector(kF32, dev, hv) || !d.dt_bias.vector(kF32, dev, hv))
    return kNo;
  d.slot = nullptr;
  if (slots != Py_None) {
    if (const int rc = read(slots, d.slots); rc != kOk) return rc;
    if (!d.slots.vector(kI32, dev, n_seq)) return kNo;
    d.slot = reinterpret_cast<const int32_t*>(d.slots.ptr);
  }
  const Tensor* const rows[5] = {&q, &k, &v, &a, &b};
  long long* const ld[5] = {&d.lq, &d.lk, &d.lv, &d.la, &d.lb};
  for (int i = 0; i < 5; ++i)
    if (const int rc = row_stride(*rows[i], *ld[i]); rc != kOk) return rc;
  double f = std::pow((double)dk, -0.5);
  if (scale != Py_None) {
    f = PyFloat_AsDouble(scale);
    if (f == -1.0 && PyErr_Occurred()) return kRaised;
  }
  d.scale = (float)f;
  d.qk_norm = PyObject_IsTrue(qk_norm);
  if (d.qk_norm < 0) return kRaised;
  if (const int rc = on_current_device(dev, d.stream, d.elsewhere); rc != kOk) return rc;
  if (d.elsewhere) return kOk;
  if (out != Py_None) {
    Tensor o;
    if (const int rc = read(out, o); rc != kOk) return rc;
    if (!o.is(type, dev, 3) || o.n[0] != n || o.n[1] != hv || o.n[2] != dv) return kNo;
    if (const int rc = row_stride(o, d.lo); rc != kOk) return rc;
    d.o = o.ptr;
    Py_INCREF(out);
    d.out.o = out;
    return kOk;
  }
  if (v.contiguous) {
    d.out.o = like(v.obj, nullptr);
  } else {
    Ref shape(PyObject_GetAttr(v.obj, s_shape));
    d.out.o = shape.o ? new_empty(v.obj, shape.o, nullptr) : nullptr;
  }
  d.lo = hv * dv;
  return d.out.o ? pointer(d.out.o, d.o) : kRaised;
}

PyObject* answer(int state) {  // of what did not come to a call
  if (state == kRaised) return nullptr;
  Py_RETURN_NONE;
}
PyObject* answer(int rc, Ref& out) { return rc ? PyLong_FromLong(rc) : out.release(); }

// q, k, v, a, b, A_log, dt_bias, state, slots, scale, qk_norm, out
PyObject* gated_delta_step(PyObject*, PyObject* const* x, Py_ssize_t count) {
  if (count != 12) return PyErr_Format(PyExc_TypeError, "12 arguments");
  Delta d;
  Tensor q;
  int rc = read(x[0], q);
  if (rc != kOk || q.dims != 3) return answer(rc == kOk ? kNo : rc);
  rc = delta(x, x[8], q.n[0], x[9], x[10], x[11], d);
  if (rc != kOk) return answer(rc);
  if (d.elsewhere) Py_RETURN_NOTIMPLEMENTED;
  Py_BEGIN_ALLOW_THREADS
  rc = step_fn(d.q.ptr, (int)d.lq, d.k.ptr, (int)d.lk, d.v.ptr, (int)d.lv, d.a.ptr, (int)d.la, d.b.ptr, (int)d.lb,
               reinterpret_cast<const float*>(d.A_log.ptr), reinterpret_cast<const float*>(d.dt_bias.ptr),
               reinterpret_cast<float*>(d.state.ptr), (int)d.state.n[0], d.slot, d.n(), d.o, (int)d.lo, (int)d.q.n[1],
               (int)d.v.n[1], (int)d.q.n[2], (int)d.v.n[2], d.scale, d.qk_norm, d.q.type, d.stream);
  Py_END_ALLOW_THREADS
  return answer(rc, d.out);
}

// q, k, v, a, b, A_log, dt_bias, state, cu_seqlens, slots, scale, qk_norm, out, workspace
PyObject* gated_delta_prefill(PyObject*, PyObject* const* x, Py_ssize_t count) {
  if (count != 14) return PyErr_Format(PyExc_TypeError, "14 arguments");
  Delta d;
  Tensor cu;
  int rc = read(x[8], cu);
  if (rc != kOk) return answer(rc);
  if (cu.dims != 1 || cu.n[0] < 1) return answer(kNo);
  const int n_seq = (int)(cu.n[0] - 1);
  rc = delta(x, x[9], n_seq, x[10], x[11], x[12], d);
  if (rc != kOk) return answer(rc);
  if (!cu.vector(kI32, d.q.device, cu.n[0])) return answer(kNo);
  if (d.elsewhere) Py_RETURN_NOTIMPLEMENTED;
  const int hk = (int)d.q.n[1], hv = (int)d.v.n[1], dk = (int)d.q.n[2], dv = (int)d.v.n[2];
  const size_t need = workspace_fn(d.n(), n_seq, hk, hv, dk, dv, d.q.type);
  size_t bytes = 0;
  void* workspace = nullptr;
  Ref own;
  if (x[13] != Py_None) {
    Tensor w;
    rc = read(x[13], w);
    if (rc != kOk) return answer(rc);
    if (w.type != kU8 || w.device != d.q.device || !w.contiguous) return answer(kNo);
    bytes = 1;
    for (int i = 0; i < w.dims; ++i) bytes *= (size_t)w.n[i];
    if (bytes < need) return answer(kNo);
    workspace = w.ptr;
  } else if (need) {
    Ref size(PyLong_FromSize_t(need));
    own.o = size.o ? new_empty(d.v.obj, size.o, types[kU8]) : nullptr;
    if (!own.o || pointer(own.o, workspace) != kOk) return nullptr;
    bytes = need;
  }
  Py_BEGIN_ALLOW_THREADS
  rc = prefill_fn(d.q.ptr, (int)d.lq, d.k.ptr, (int)d.lk, d.v.ptr, (int)d.lv, d.a.ptr, (int)d.la, d.b.ptr, (int)d.lb,
                  reinterpret_cast<const float*>(d.A_log.ptr), reinterpret_cast<const float*>(d.dt_bias.ptr),
                  reinterpret_cast<float*>(d.state.ptr), (int)d.state.n[0], d.slot, reinterpret_cast<const int32_t*>(cu.ptr),
                  n_seq, d.n(), d.o, (int)d.lo, hk, hv, dk, dv, d.scale, d.qk_norm, d.q.type, workspace, bytes, d.stream);
  Py_END_ALLOW_THREADS
  return answer(rc, d.out);
}

// logits, uniform, temperature, top_k, top_p, min_p, seen_bits (each None or a tensor), rep_penalty, out
PyObject* sample_filtered(PyObject*, PyObject* const* x, Py_ssize_t count) {
  if (count != 9) return PyErr_Format(PyExc_TypeError, "9 arguments");
  Tensor l, u, seen;
  int rc = read(x[0], l);
  if (rc == kOk) rc = read(x[1], u);
  if (rc != kOk) return answer(rc);
  if (l.type > kF32 || l.type < 0 || l.dims != 2 || l.n[1] < 1) return answer(kNo);
  const long dev = l.device;
  const long long B = l.n[0], V = l.n[1];
  long long ld = V;
  if (!l.contiguous) {
    Ref s(method(l.obj, s_stride));
    if (!s.o) return nullptr;
    const long long st0 = PyLong_AsLongLong(PyTuple_GET_ITEM(s.o, 0)), st1 = PyLong_AsLongLong(PyTuple_GET_ITEM(s.o, 1));
    if (PyErr_Occurred()) return nullptr;
    if (V > 1 && st1 != 1) return answer(kNo);
    if (B > 1) ld = st0;
    if (ld < V) return answer(kNo);
  }
  if (!u.vector(kF32, dev, B)) return answer(kNo);
  const void* setting[4] = {};
  for (int i = 0; i < 4; ++i) {
    if (x[2 + i] == Py_None) continue;
    Tensor t;
    rc = read(x[2 + i], t);
    if (rc != kOk) return answer(rc);
    if (!t.vector(i == 1 ? kI32 : kF32, dev, B)) return answer(kNo);
    setting[i] = t.ptr;
  }
  const uint32_t* bits = nullptr;
  if (x[6] != Py_None) {
    rc = read(x[6], seen);
    if (rc != kOk) return answer(rc);
    if (!seen.is(kI32, dev, 2) || !seen.contiguous || seen.n[0] != B || seen.n[1] != (V + 31) / 32) return answer(kNo);
    bits = reinterpret_cast<const uint32_t*>(seen.ptr);
  }
  const double rep = PyFloat_AsDouble(x[7]);
  if (rep == -1.0 && PyErr_Occurred()) return nullptr;
  void *stream, *p[3];
  bool elsewhere;
  if (on_current_device(dev, stream, elsewhere) != kOk) return nullptr;
  if (elsewhere) Py_RETURN_NOTIMPLEMENTED;
  Ref out;
  if (x[8] != Py_None) {
    if (!PyTuple_Check(x[8]) || PyTuple_GET_SIZE(x[8]) != 3) return answer(kNo);
    for (int i = 0; i < 3; ++i) {
      Tensor t;
      rc = read(PyTuple_GET_ITEM(x[8], i), t);
      if (rc != kOk) return answer(rc);
      if (!t.vector(i < 2 ? kI32 : kF32, dev, B)) return answer(kNo);
      p[i] = t.ptr;
    }
    Py_INCREF(x[8]);
    out.o = x[8];
  } else {
    out.o = PyTuple_New(3);
    if (!out.o) return nullptr;
    for (int i = 0; i < 3; ++i) {
      PyObject* t = like(u.obj, i < 2 ? types[kI32] : nullptr);
      if (!t) return nullptr;
      PyTuple_SET_ITEM(out.o, i, t);
      if (pointer(t, p[i]) != kOk) return nullptr;
    }
  }
  Py_BEGIN_ALLOW_THREADS
  rc = sample_fn(l.ptr, ld, l.type, (int)B, (int)V, static_cast<const float*>(setting[0]), static_cast<const int32_t*>(setting[1]),
                 static_cast<const float*>(setting[2]), static_cast<const float*>(setting[3]), bits, (float)rep,
                 reinterpret_cast<const float*>(u.ptr), static_cast<int32_t*>(p[0]), static_cast<int32_t*>(p[1]),
                 static_cast<float*>(p[2]), stream);
  Py_END_ALLOW_THREADS
  return answer(rc, out);
}

// Addresses of the four C entry points; the type Tensor, the five dtypes, and the functions empty_like, (device) ->
// current stream's handle and () -> current device.
PyObject* bind(PyObject*, PyObject* const* x, Py_ssize_t count) {
  if (count != 13) return PyErr_Format(PyExc_TypeError, "13 arguments");
  void* fn[4];
  for (int i = 0; i < 4; ++i) {
    fn[i] = PyLong_AsVoidPtr(x[i]);
    if (!fn[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "no address");
  }
  if (!PyType_Check(x[4])) return PyErr_Format(PyExc_TypeError, "a type");
  step_fn = reinterpret_cast<StepFn>(fn[0]);
  workspace_fn = reinterpret_cast<WorkspaceFn>(fn[1]);
  prefill_fn = reinterpret_cast<PrefillFn>(fn[2]);
  sample_fn = reinterpret_cast<SampleFn>(fn[3]);
  PyObject** const to[9] = {&tensor_type, &types[0], &types[1], &types[2], &types[3], &types[4], &empty_like, &stream_of, &current_device};
  for (int i = 0; i < 9; ++i) {
    Py_INCREF(x[4 + i]);
    PyObject* old = *to[i];
    *to[i] = x[4 + i];
    Py_XDECREF(old);
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {"gated_delta_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gated_delta_step)), METH_FASTCALL, nullptr},
    {"gated_delta_prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gated_delta_prefill)), METH_FASTCALL, nullptr},
    {"sample_filtered", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sample_filtered)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "dfssm_pycalls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dfssm_pycalls() {
  struct Name {
    PyObject** to;
    const char* text;
  } const names[] = {{&s_dtype, "dtype"},           {&s_shape, "shape"},       {&s_get_device, "get_device"},
                     {&s_is_contiguous, "is_contiguous"}, {&s_data_ptr, "data_ptr"}, {&s_stride, "stride"},
                     {&s_new_empty, "new_empty"}};
  for (const Name& n : names)
    if (!(*n.to = PyUnicode_InternFromString(n.text))) return nullptr;
  kw_dtype = PyTuple_Pack(1, s_dtype);
  return kw_dtype ? PyModule_Create(&module) : nullptr;
}
