// CPython extension spoc_amd._host: the launch calls of spoc_amd/sarek.py, and the operators of spoc_amd/hip.py on microscaled rows and on
// a paged cache, with their argument lists turned into the C ones here.  A launch takes the HIP runtime 2.8 us; building the same structures with ctypes took 2.3 us more for
// one kernel and 5.3 us for a pipeline of two.  The entry points are those of the library the ctypes front end has loaded
// (bind() gets their addresses), so there is one library per process whichever build it is, and their statuses come back
// to the caller, who turns them into exceptions as for every other entry point.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <tuple>
#include <type_traits>
#include <utility>
#include <vector>

#include "sarek_hip.h"

namespace {

decltype(&sarek_hip_execute_run_vectors) g_run_vectors;
decltype(&sarek_hip_execute_run_source) g_run_source;
decltype(&sarek_hip_execute_run_pipeline) g_run_pipeline;
decltype(&sarek_hip_last_run_path) g_last_run_path;
decltype(&sarek_hip_fold_partials_f64) g_fold_partials;

PyObject *s_h, *s_value;   // "_h", "value"

bool bound() {
  if (g_run_vectors) return true;
  PyErr_SetString(PyExc_RuntimeError, "spoc_amd._host: bind() has not been called");
  return false;
}

// What a ctypes integer field takes: an integer (or what __index__ makes one), cut to the field's width.
bool as_bits(PyObject *o, unsigned long long *out) {
  if (PyFloat_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "int expected instead of float instance");
    return false;
  }
  *out = PyLong_AsUnsignedLongLongMask(o);
  return !(*out == static_cast<unsigned long long>(-1) && PyErr_Occurred());
}
bool as_int(PyObject *o, int *out) {
  unsigned long long v;
  if (!as_bits(o, &v)) return false;
  *out = static_cast<int>(v);
  return true;
}

// Sequences are read as tuples: a conversion below may run the caller's code (__index__), which may change a list.

// block or grid: up to three integers, missing ones zero
bool as_dims(PyObject *o, int out[3]) {
  PyObject *seq = PySequence_Tuple(o);
  if (!seq) return false;
  const Py_ssize_t n = PyTuple_GET_SIZE(seq);
  bool ok = n <= 3;
  if (!ok) PyErr_SetString(PyExc_IndexError, "invalid index");
  for (Py_ssize_t i = 0; i < 3 && ok; ++i) {
    out[i] = 0;
    if (i < n) ok = as_int(PyTuple_GET_ITEM(seq, i), out + i);
  }
  Py_DECREF(seq);
  return ok;
}

// A vector's handle: its _h is a ctypes pointer, or None once it is destroyed (the library reports that one)
bool as_handle(PyObject *vector, sarek_hip_vector *out) {
  PyObject *h = PyObject_GetAttr(vector, s_h);
  if (!h) return false;
  bool ok = true;
  *out = nullptr;
  if (h != Py_None) {
    PyObject *value = PyObject_GetAttr(h, s_value);
    ok = value != nullptr;
    if (ok && value != Py_None) {
      *out = static_cast<sarek_hip_vector>(PyLong_AsVoidPtr(value));
      ok = !PyErr_Occurred();
    }
    Py_XDECREF(value);
  }
  Py_DECREF(h);
  return ok;
}

// [(kind, value), ...] as Execute.Vec, .Int, ... make them
bool as_args(PyObject *o, std::vector<sarek_hip_varg> &out) {
  PyObject *seq = PySequence_Tuple(o);
  if (!seq) return false;
  const Py_ssize_t n = PyTuple_GET_SIZE(seq);
  out.resize(static_cast<size_t>(n));
  bool ok = true;
  for (Py_ssize_t i = 0; i < n && ok; ++i) {
    PyObject *item = PySequence_Tuple(PyTuple_GET_ITEM(seq, i));
    if (!item) {
      ok = false;
      break;
    }
    if (PyTuple_GET_SIZE(item) != 2) {
      PyErr_SetString(PyExc_ValueError, "an argument is a pair of kind and value");
      Py_DECREF(item);
      ok = false;
      break;
    }
    PyObject *kind = PyTuple_GET_ITEM(item, 0), *value = PyTuple_GET_ITEM(item, 1);
    sarek_hip_varg &a = out[static_cast<size_t>(i)];
    std::memset(&a, 0, sizeof(a));
    const char *k = PyUnicode_Check(kind) ? PyUnicode_AsUTF8(kind) : "";
    unsigned long long bits = 0;
    if (!k) {
      ok = false;
    } else if (!std::strcmp(k, "vec")) {
      a.kind = SAREK_HIP_VARG_VEC;
      ok = as_handle(value, &a.vec);
    } else if (!std::strcmp(k, "i32")) {
      a.kind = SAREK_HIP_VARG_INT32;
      ok = as_bits(value, &bits);
      a.i32 = static_cast<int32_t>(bits);
    } else if (!std::strcmp(k, "i64")) {
      a.kind = SAREK_HIP_VARG_INT64;
      ok = as_bits(value, &bits);
      a.i64 = static_cast<int64_t>(bits);
    } else if (!std::strcmp(k, "f32")) {
      a.kind = SAREK_HIP_VARG_FLOAT32;
      const double v = PyFloat_AsDouble(value);
      ok = !(v == -1.0 && PyErr_Occurred());
      a.f32 = static_cast<float>(v);
    } else if (!std::strcmp(k, "f64")) {
      a.kind = SAREK_HIP_VARG_FLOAT64;
      a.f64 = PyFloat_AsDouble(value);
      ok = !(a.f64 == -1.0 && PyErr_Occurred());
    } else {
      PyErr_Format(PyExc_ValueError, "unknown vector_arg %R", kind);
      ok = false;
    }
    Py_DECREF(item);
  }
  Py_DECREF(seq);
  return ok;
}

// The status where a call failed, otherwise what `done` makes
template <typename Call, typename Done>
PyObject *finish(Call call, Done done) {
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = call();
  Py_END_ALLOW_THREADS
  return status != SAREK_HIP_OK ? PyLong_FromLong(status) : done();
}
PyObject *path() { return PyUnicode_FromString(g_last_run_path()); }

bool arity(Py_ssize_t given, Py_ssize_t wanted, const char *what) {
  if (given == wanted) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", what, wanted, given);
  return false;
}

// run_vectors(ir, args, block, grid, shared_mem) -> path | status
PyObject *run_vectors(PyObject *, PyObject *const *a, Py_ssize_t n) {
  std::vector<sarek_hip_varg> args;
  int block[3], grid[3], shared;
  if (!bound() || !arity(n, 5, "run_vectors")) return nullptr;
  const char *ir = PyUnicode_AsUTF8(a[0]);
  if (!ir || !as_args(a[1], args) || !as_dims(a[2], block) || !as_dims(a[3], grid) || !as_int(a[4], &shared)) return nullptr;
  return finish([&] { return g_run_vectors(ir, block, grid, shared, args.data(), static_cast<int>(args.size())); }, path);
}

// run_source(source, lang, kernel_name, block, grid, shared_mem, inject_lengths, args) -> path | status
PyObject *run_source(PyObject *, PyObject *const *a, Py_ssize_t n) {
  std::vector<sarek_hip_varg> args;
  int lang, block[3], grid[3], shared, inject;
  if (!bound() || !arity(n, 8, "run_source")) return nullptr;
  const char *source = PyUnicode_AsUTF8(a[0]), *name = source ? PyUnicode_AsUTF8(a[2]) : nullptr;
  if (!name || !as_int(a[1], &lang) || !as_dims(a[3], block) || !as_dims(a[4], grid) || !as_int(a[5], &shared) ||
      !as_int(a[6], &inject) || !as_args(a[7], args))
    return nullptr;
  return finish(
      [&] {
        return g_run_source(source, lang, name, block, grid, shared, inject, args.data(), static_cast<int>(args.size()));
      },
      path);
}

// run_pipeline([(ir, args, block, grid[, shared_mem]), ...]) -> (path, launches) | status
PyObject *run_pipeline(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!bound() || !arity(n, 1, "run_pipeline")) return nullptr;
  PyObject *seq = PySequence_Tuple(a[0]);
  if (!seq) return nullptr;
  const size_t count = static_cast<size_t>(PyTuple_GET_SIZE(seq));
  std::vector<sarek_hip_pipeline_stage> stages(count);
  std::vector<std::vector<sarek_hip_varg>> args(count);
  // The stages as tuples of their own: they keep the IR texts, which the library reads while other threads run and may
  // change a stage that is a list.
  std::vector<PyObject *> held;
  bool ok = true;
  for (size_t i = 0; i < count && ok; ++i) {
    PyObject *stage = PySequence_Tuple(PyTuple_GET_ITEM(seq, static_cast<Py_ssize_t>(i)));
    if (!stage) {
      ok = false;
      break;
    }
    held.push_back(stage);
    const Py_ssize_t parts = PyTuple_GET_SIZE(stage);
    if (parts < 4) {
      PyErr_Format(PyExc_ValueError, "not enough values to unpack (expected 4, got %zd)", parts);
      ok = false;
      break;
    }
    sarek_hip_pipeline_stage &s = stages[i];
    s.ir_text = PyUnicode_AsUTF8(PyTuple_GET_ITEM(stage, 0));
    s.shared_mem_bytes = 0;
    ok = s.ir_text && as_args(PyTuple_GET_ITEM(stage, 1), args[i]) && as_dims(PyTuple_GET_ITEM(stage, 2), s.block) &&
         as_dims(PyTuple_GET_ITEM(stage, 3), s.grid) && (parts == 4 || as_int(PyTuple_GET_ITEM(stage, 4), &s.shared_mem_bytes));
    s.args = args[i].data();
    s.n_args = static_cast<int>(args[i].size());
  }
  PyObject *result = nullptr;
  int launches = 0;
  if (ok)
    result = finish([&] { return g_run_pipeline(stages.data(), static_cast<int>(count), &launches); },
                    [&] { return Py_BuildValue("(si)", g_last_run_path(), launches); });
  for (PyObject *o : held) Py_DECREF(o);
  Py_DECREF(seq);
  return result;
}

// fold_partials(partials, count, sum, stream) -> status; the pointers and the stream as integers
PyObject *fold_partials(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!bound() || !arity(n, 4, "fold_partials")) return nullptr;
  void *partials = PyLong_AsVoidPtr(a[0]), *sum = PyLong_AsVoidPtr(a[2]), *stream = PyLong_AsVoidPtr(a[3]);
  const long long count = PyLong_AsLongLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_fold_partials(static_cast<const float *>(partials), count, static_cast<double *>(sum), stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

// The operators on microscaled rows, called with their C arguments: pointers and the stream as integers or None, numbers.  (ctypes takes
// 1.7 us for the 9 arguments of mx_quantize, this 0.3.)
decltype(&sarek_hip_mx_quantize) g_mx_quantize;
decltype(&sarek_hip_mx_dequantize) g_mx_dequantize;
decltype(&sarek_hip_rms_norm_mx) g_rms_norm_mx;
decltype(&sarek_hip_rms_norm_backward) g_rms_norm_backward;
decltype(&sarek_hip_gemm_mx) g_gemm_mx;
// and those on a paged cache
decltype(&sarek_hip_rotary) g_rotary;
decltype(&sarek_hip_kv_append) g_kv_append;
decltype(&sarek_hip_attention_paged) g_attention_paged;
decltype(&sarek_hip_attention_shared) g_attention_shared;

template <typename T>
T as_c(PyObject *o) {
  if constexpr (std::is_pointer_v<T>) {
    return o == Py_None ? nullptr : static_cast<T>(PyLong_AsVoidPtr(o));
  } else if constexpr (std::is_floating_point_v<T>) {
    return static_cast<T>(PyFloat_AsDouble(o));
  } else {
    const long long v = PyLong_AsLongLong(o);
    if (v != static_cast<long long>(static_cast<T>(v))) PyErr_SetString(PyExc_OverflowError, "an integer argument does not fit its type");
    return static_cast<T>(v);
  }
}
template <typename... Args, size_t... Is>
PyObject *call_with(int (*f)(Args...), PyObject *const *a, std::index_sequence<Is...>) {
  const std::tuple<Args...> args{as_c<Args>(a[Is])...};
  if (PyErr_Occurred()) return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = std::apply(f, args);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}
template <typename... Args>
PyObject *call(int (*f)(Args...), PyObject *const *a, Py_ssize_t n, const char *what) {
  if (!f) {
    PyErr_SetString(PyExc_RuntimeError, "spoc_amd._host: bind_mx() and bind_attention() have not been called");
    return nullptr;
  }
  if (!arity(n, sizeof...(Args), what)) return nullptr;
  return call_with(f, a, std::index_sequence_for<Args...>{});
}
PyObject *mx_quantize(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_mx_quantize, a, n, "mx_quantize"); }
PyObject *mx_dequantize(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_mx_dequantize, a, n, "mx_dequantize"); }
PyObject *rms_norm_mx(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_rms_norm_mx, a, n, "rms_norm_mx"); }
PyObject *rms_norm_backward(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_rms_norm_backward, a, n, "rms_norm_backward"); }
PyObject *gemm_mx(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_gemm_mx, a, n, "gemm_mx"); }
PyObject *rotary(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_rotary, a, n, "rotary"); }
PyObject *kv_append(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_kv_append, a, n, "kv_append"); }
PyObject *attention_paged(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_attention_paged, a, n, "attention_paged"); }
PyObject *attention_shared(PyObject *, PyObject *const *a, Py_ssize_t n) { return call(g_attention_shared, a, n, "attention_shared"); }

// The operators on a paged cache with their tensors as they are.  The ordinary call is looked through and made here: the checks of
// hip.py take 4 to 8 us of the interpreter, reading what they need of the tensors 0.25 us each.  Whatever is not as it has to be, and a call that
// fails, gives None, and hip.py, which then goes through it with the same checks, says what it was.
PyObject *g_tensor, *g_types[3], *g_int32, *g_int64, *g_get_device, *g_raw_stream;   // SAREK_HIP_TYPE_* order
PyObject *s_shape, *s_stride, *s_dtype, *s_data_ptr, *s_get_device, *s_new_empty;
decltype(&sarek_hip_attention_workspace_bytes) g_workspace_bytes;

struct Held {      // a new reference, or none
  PyObject *o;
  explicit Held(PyObject *p) : o(p) {}
  ~Held() { Py_XDECREF(o); }
  Held(const Held &) = delete;
  Held &operator=(const Held &) = delete;
};
struct TensorOf {
  PyObject *dtype;             // (the type objects live as long as torch does)
  long long shape[3], stride[3];
  void *data;
};
bool as_longs(PyObject *tuple, int n, long long *out) {
  if (!tuple || !PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) != n) return false;
  for (int i = 0; i < n; ++i) out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
  return !PyErr_Occurred();
}
// A plain tensor of `dims` dimensions on that device, its last dimension adjacent
bool read(PyObject *t, int dims, long device, TensorOf *out) {
  if (reinterpret_cast<PyObject *>(Py_TYPE(t)) != g_tensor) return false;
  const Held where(PyObject_CallMethodNoArgs(t, s_get_device));
  if (!where.o || PyLong_AsLong(where.o) != device) return false;
  const Held shape(PyObject_GetAttr(t, s_shape)), stride(PyObject_CallMethodNoArgs(t, s_stride)), dtype(PyObject_GetAttr(t, s_dtype)),
      data(PyObject_CallMethodNoArgs(t, s_data_ptr));
  if (!dtype.o || !data.o || !as_longs(shape.o, dims, out->shape) || !as_longs(stride.o, dims, out->stride)) return false;
  out->dtype = dtype.o;
  out->data = PyLong_AsVoidPtr(data.o);
  return !PyErr_Occurred() && (out->stride[dims - 1] == 1 || out->shape[dims - 1] == 1);
}
bool same_shape(const TensorOf &a, const TensorOf &b) { return a.shape[0] == b.shape[0] && a.shape[1] == b.shape[1] && a.shape[2] == b.shape[2]; }
// [tokens, heads, head dim] that go with a cache
bool read_heads(PyObject *t, long device, PyObject *dtype, long long tokens, long long heads, long long d, TensorOf *out) {
  return read(t, 3, device, out) && out->dtype == dtype && (tokens < 0 || out->shape[0] == tokens) && (heads < 0 || out->shape[1] == heads) && out->shape[2] == d;
}
// The device and its stream; false where an error is set
bool here(long *device, void **stream) {
  const Held index(PyObject_CallNoArgs(g_get_device));
  if (!index.o) return false;
  const Held raw(PyObject_CallOneArg(g_raw_stream, index.o));
  if (!raw.o) return false;
  *device = PyLong_AsLong(index.o);
  *stream = PyLong_AsVoidPtr(raw.o);
  return !PyErr_Occurred();
}
PyObject *long_way() {
  PyErr_Clear();
  Py_RETURN_NONE;
}
PyObject *new_like(PyObject *t) {
  const Held shape(PyObject_GetAttr(t, s_shape));
  return shape.o ? PyObject_CallMethodOneArg(t, s_new_empty, shape.o) : nullptr;
}
template <class Call> bool succeeds(Call call) {
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = call();
  Py_END_ALLOW_THREADS
  return status == SAREK_HIP_OK;
}
// What a Rotary and a KvCache hold for this: (address, values turned, device) and (address, heads, head dim, device, type)
struct PlanOf {
  const sarek_hip_rotary_plan *at;
  long long dim, device;
};
bool read_plan(PyObject *o, PlanOf *out) {
  long long v[3];
  if (!as_longs(o, 3, v)) return false;
  *out = {reinterpret_cast<const sarek_hip_rotary_plan *>(static_cast<uintptr_t>(v[0])), v[1], v[2]};
  return true;
}
struct CacheOf {
  const sarek_hip_kv_cache *at;
  long long heads, d, device;
  PyObject *dtype;
};
bool read_cache(PyObject *o, CacheOf *out) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 5) return false;
  long long v[4];
  for (int i = 0; i < 4; ++i) v[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
  *out = {reinterpret_cast<const sarek_hip_kv_cache *>(static_cast<uintptr_t>(v[0])), v[1], v[2], v[3], PyTuple_GET_ITEM(o, 4)};
  return !PyErr_Occurred();
}
struct SequencesOf {
  const int *pages, *lengths, *starts;
  long long pages_stride;
  int max_pages, batch;
};
bool read_sequences(PyObject *pages, PyObject *lengths, PyObject *starts, long device, long long tokens, SequencesOf *out) {
  TensorOf p, l, s;
  if (!read(lengths, 1, device, &l) || l.dtype != g_int32 || !read(pages, 2, device, &p) || p.dtype != g_int32 || p.shape[0] != l.shape[0] ||
      l.shape[0] > INT32_MAX || p.shape[1] > INT32_MAX)
    return false;
  s.data = nullptr;
  if (starts == Py_None) {
    if (l.shape[0] != tokens) return false;
  } else if (!read(starts, 1, device, &s) || s.dtype != g_int32 || s.shape[0] != l.shape[0] + 1) {
    return false;
  }
  *out = {static_cast<const int *>(p.data), static_cast<const int *>(l.data), static_cast<const int *>(s.data),
          l.shape[0] > 1 ? p.stride[0] : p.shape[1], static_cast<int>(p.shape[1]), static_cast<int>(l.shape[0])};
  return true;
}

// rotary_tensors(x, positions, plan, out or None, inverse) -> out | None
PyObject *rotary_tensors(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!g_rotary || !g_tensor || !arity(n, 5, "rotary_tensors")) return long_way();
  long device;
  void *stream;
  TensorOf x, at, to;
  PlanOf plan;
  if (!here(&device, &stream) || !read(a[0], 3, device, &x) || !read(a[1], 1, device, &at) || !read_plan(a[2], &plan)) return long_way();
  int type = 0;
  while (type < 3 && x.dtype != g_types[type]) ++type;
  if (type == 3 || (at.dtype != g_int64 && at.dtype != g_int32) || at.shape[0] != x.shape[0] || plan.device != device || plan.dim > x.shape[2] ||
      x.shape[1] > 65535 || x.shape[2] > 65536)
    return long_way();
  const Held out(a[3] == Py_None ? new_like(a[0]) : Py_NewRef(a[3]));
  if (!out.o || !read(out.o, 3, device, &to) || to.dtype != x.dtype || !same_shape(to, x)) return long_way();
  const int inverse = a[4] == Py_True;
  if (!succeeds([&] {
        return g_rotary(plan.at, x.data, x.stride[0], x.stride[1], type, at.data, at.dtype == g_int64 ? 8 : 4, inverse, to.data, to.stride[0], to.stride[1],
                        x.shape[0], static_cast<int>(x.shape[1]), static_cast<int>(x.shape[2]), stream);
      }))
    return long_way();
  return Py_NewRef(out.o);
}

// kv_append_tensors(k, v, cache, pages, lengths, starts or None, plan or None, q or None, q_out or None, first) -> q_out | False without a q | None
PyObject *kv_append_tensors(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!g_kv_append || !g_tensor || !arity(n, 10, "kv_append_tensors")) return long_way();
  long device;
  void *stream;
  TensorOf k, v, q, to;
  CacheOf cache;
  PlanOf plan = {nullptr, 0, 0};
  SequencesOf s;
  if (!here(&device, &stream) || !read_cache(a[2], &cache) || cache.device != device || !read_heads(a[0], device, cache.dtype, -1, cache.heads, cache.d, &k) ||
      !read_heads(a[1], device, cache.dtype, k.shape[0], cache.heads, cache.d, &v) || !read_sequences(a[3], a[4], a[5], device, k.shape[0], &s))
    return long_way();
  if (a[6] != Py_None && (!read_plan(a[6], &plan) || plan.device != device || plan.dim > cache.d)) return long_way();
  const long long first = PyLong_AsLongLong(a[9]);
  if (PyErr_Occurred()) return long_way();
  const bool with_q = a[7] != Py_None;
  const Held out(!with_q ? Py_NewRef(Py_False) : a[8] == Py_None ? new_like(a[7]) : Py_NewRef(a[8]));
  q.data = to.data = nullptr, q.stride[0] = q.stride[1] = q.shape[1] = to.stride[0] = to.stride[1] = 0;
  if (!out.o || (with_q && (!read_heads(a[7], device, cache.dtype, k.shape[0], -1, cache.d, &q) || q.shape[1] > 65535 || q.shape[1] < 1 ||
                            !read_heads(out.o, device, cache.dtype, k.shape[0], q.shape[1], cache.d, &to))))
    return long_way();
  if (!succeeds([&] {
        return g_kv_append(cache.at, k.data, k.stride[0], k.stride[1], v.data, v.stride[0], v.stride[1], q.data, q.stride[0], q.stride[1], to.data, to.stride[0],
                           to.stride[1], static_cast<int>(q.shape[1]), plan.at, s.pages, s.pages_stride, s.max_pages, s.lengths, s.starts, s.batch, k.shape[0],
                           first, stream);
      }))
    return long_way();
  return Py_NewRef(out.o);
}

// attention_tensors(q, cache, prefix_pages or None, prefix_length, pages, lengths, starts or None, causal, scale or None, out or None, lse or None) -> out | None
PyObject *attention_tensors(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!g_attention_shared || !g_tensor || !arity(n, 11, "attention_tensors")) return long_way();
  long device;
  void *stream;
  TensorOf q, to, lse, prefix;
  CacheOf cache;
  SequencesOf s;
  if (!here(&device, &stream) || !read_cache(a[1], &cache) || cache.device != device || !read_heads(a[0], device, cache.dtype, -1, -1, cache.d, &q) ||
      q.shape[1] < 1 || q.shape[1] > 65535 || q.shape[1] % cache.heads != 0 || !read_sequences(a[4], a[5], a[6], device, q.shape[0], &s))
    return long_way();
  prefix.data = lse.data = nullptr;
  long long prefix_length = 0;
  if (a[2] != Py_None) {
    prefix_length = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred() || !read(a[2], 1, device, &prefix) || prefix.dtype != g_int32 || prefix_length < 0 || prefix_length > prefix.shape[0] * cache.at->page_size)
      return long_way();
  }
  if (a[10] != Py_None && (!read(a[10], 2, device, &lse) || lse.dtype != g_types[SAREK_HIP_TYPE_F32] || lse.shape[0] != q.shape[0] || lse.shape[1] != q.shape[1] ||
                           (lse.shape[0] > 1 && lse.stride[0] != lse.shape[1])))
    return long_way();
  const int causal = PyObject_IsTrue(a[7]);
  const double scale = a[8] == Py_None ? 1.0 / std::sqrt(static_cast<double>(cache.d)) : PyFloat_AsDouble(a[8]);
  if (PyErr_Occurred()) return long_way();
  const Held out(a[9] == Py_None ? new_like(a[0]) : Py_NewRef(a[9]));
  if (!out.o || !read_heads(out.o, device, cache.dtype, q.shape[0], q.shape[1], cache.d, &to)) return long_way();
  const int heads = static_cast<int>(q.shape[1]);
  const int64_t held = g_workspace_bytes(cache.at, heads, s.batch, q.shape[0], s.max_pages, prefix_length);
  TensorOf space;
  space.data = nullptr;
  const Held values(held > 0 ? Py_BuildValue("(L)", static_cast<long long>(held + 1) / 2) : nullptr);      // of q's type, of 2 bytes
  const Held workspace(held > 0 ? PyObject_CallMethodOneArg(a[0], s_new_empty, values.o) : nullptr);
  if (held > 0 && (!workspace.o || !read(workspace.o, 1, device, &space))) return long_way();
  if (!succeeds([&] {
        return g_attention_shared(cache.at, q.data, q.stride[0], q.stride[1], heads, to.data, to.stride[0], to.stride[1], static_cast<float *>(lse.data),
                                  prefix_length > 0 ? static_cast<const int *>(prefix.data) : nullptr, prefix_length, s.pages, s.pages_stride, s.max_pages, s.lengths,
                                  s.starts, s.batch, q.shape[0], causal, static_cast<float>(scale), space.data, held, stream);
      }))
    return long_way();
  return Py_NewRef(out.o);
}

// bind_torch(Tensor, float32, bfloat16, float16, int32, int64, _cuda_getDevice, _cuda_getCurrentRawStream, address of attention_workspace_bytes)
PyObject *bind_torch(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!arity(n, 9, "bind_torch")) return nullptr;
  void *const bytes = PyLong_AsVoidPtr(a[8]);
  if (PyErr_Occurred()) return nullptr;
  PyObject **const to[8] = {&g_tensor, &g_types[0], &g_types[1], &g_types[2], &g_int32, &g_int64, &g_get_device, &g_raw_stream};
  for (int i = 0; i < 8; ++i) Py_XSETREF(*to[i], Py_NewRef(a[i]));
  g_workspace_bytes = reinterpret_cast<decltype(g_workspace_bytes)>(bytes);
  Py_RETURN_NONE;
}

// bind(addresses of the first five entry points above, in the order of their declaration)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!arity(n, 5, "bind")) return nullptr;
  void *p[5];
  for (int i = 0; i < 5; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_run_source = reinterpret_cast<decltype(g_run_source)>(p[1]);
  g_run_pipeline = reinterpret_cast<decltype(g_run_pipeline)>(p[2]);
  g_last_run_path = reinterpret_cast<decltype(g_last_run_path)>(p[3]);
  g_fold_partials = reinterpret_cast<decltype(g_fold_partials)>(p[4]);
  g_run_vectors = reinterpret_cast<decltype(g_run_vectors)>(p[0]);
  Py_RETURN_NONE;
}

// bind_mx(addresses of the five on microscaled rows)
PyObject *bind_mx(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!arity(n, 5, "bind_mx")) return nullptr;
  void *p[5];
  for (int i = 0; i < 5; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_mx_dequantize = reinterpret_cast<decltype(g_mx_dequantize)>(p[1]);
  g_rms_norm_mx = reinterpret_cast<decltype(g_rms_norm_mx)>(p[2]);
  g_rms_norm_backward = reinterpret_cast<decltype(g_rms_norm_backward)>(p[3]);
  g_gemm_mx = reinterpret_cast<decltype(g_gemm_mx)>(p[4]);
  g_mx_quantize = reinterpret_cast<decltype(g_mx_quantize)>(p[0]);
  Py_RETURN_NONE;
}

// bind_attention(addresses of the four on a paged cache)
PyObject *bind_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (!arity(n, 4, "bind_attention")) return nullptr;
  void *p[4];
  for (int i = 0; i < 4; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_rotary = reinterpret_cast<decltype(g_rotary)>(p[0]);
  g_kv_append = reinterpret_cast<decltype(g_kv_append)>(p[1]);
  g_attention_paged = reinterpret_cast<decltype(g_attention_paged)>(p[2]);
  g_attention_shared = reinterpret_cast<decltype(g_attention_shared)>(p[3]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(bind), METH_FASTCALL, "Addresses of the library's entry points."},
    {"bind_mx", reinterpret_cast<PyCFunction>(bind_mx), METH_FASTCALL, "The same for the operators on microscaled rows."},
    {"run_vectors", reinterpret_cast<PyCFunction>(run_vectors), METH_FASTCALL, "sarek_hip_execute_run_vectors"},
    {"run_source", reinterpret_cast<PyCFunction>(run_source), METH_FASTCALL, "sarek_hip_execute_run_source"},
    {"run_pipeline", reinterpret_cast<PyCFunction>(run_pipeline), METH_FASTCALL, "sarek_hip_execute_run_pipeline"},
    {"fold_partials", reinterpret_cast<PyCFunction>(fold_partials), METH_FASTCALL, "sarek_hip_fold_partials_f64"},
    {"mx_quantize", reinterpret_cast<PyCFunction>(mx_quantize), METH_FASTCALL, "sarek_hip_mx_quantize"},
    {"mx_dequantize", reinterpret_cast<PyCFunction>(mx_dequantize), METH_FASTCALL, "sarek_hip_mx_dequantize"},
    {"rms_norm_mx", reinterpret_cast<PyCFunction>(rms_norm_mx), METH_FASTCALL, "sarek_hip_rms_norm_mx"},
    {"rms_norm_backward", reinterpret_cast<PyCFunction>(rms_norm_backward), METH_FASTCALL, "sarek_hip_rms_norm_backward"},
    {"gemm_mx", reinterpret_cast<PyCFunction>(gemm_mx), METH_FASTCALL, "sarek_hip_gemm_mx"},
    {"bind_attention", reinterpret_cast<PyCFunction>(bind_attention), METH_FASTCALL, "The same for the operators on a paged cache."},
    {"rotary", reinterpret_cast<PyCFunction>(rotary), METH_FASTCALL, "sarek_hip_rotary"},
    {"kv_append", reinterpret_cast<PyCFunction>(kv_append), METH_FASTCALL, "sarek_hip_kv_append"},
    {"attention_paged", reinterpret_cast<PyCFunction>(attention_paged), METH_FASTCALL, "sarek_hip_attention_paged"},
    {"attention_shared", reinterpret_cast<PyCFunction>(attention_shared), METH_FASTCALL, "sarek_hip_attention_shared"},
    {"bind_torch", reinterpret_cast<PyCFunction>(bind_torch), METH_FASTCALL, "What the next three need of torch."},
    {"rotary_tensors", reinterpret_cast<PyCFunction>(rotary_tensors), METH_FASTCALL, "sarek_hip_rotary of tensors, None where it is not the ordinary call"},
    {"kv_append_tensors", reinterpret_cast<PyCFunction>(kv_append_tensors), METH_FASTCALL, "sarek_hip_kv_append, likewise"},
    {"attention_tensors", reinterpret_cast<PyCFunction>(attention_tensors), METH_FASTCALL, "sarek_hip_attention_paged and _shared, likewise"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Argument lists of launches, built natively.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
  s_h = PyUnicode_InternFromString("_h");
  s_value = PyUnicode_InternFromString("value");
  PyObject **const names[] = {&s_shape, &s_stride, &s_dtype, &s_data_ptr, &s_get_device, &s_new_empty};
  const char *const texts[] = {"shape", "stride", "dtype", "data_ptr", "get_device", "new_empty"};
  for (int i = 0; i < 6; ++i)
    if (!(*names[i] = PyUnicode_InternFromString(texts[i]))) return nullptr;
  return s_h && s_value ? PyModule_Create(&module) : nullptr;
}
