// Python's way to the operators: checks the tensors, allocates what is not given (on the launching
// stream) and calls the C entry points of libhgemm_b200.so, whose addresses operators.py hands over. In C++
// because a small call is bound by the host: with the same checks in Python the norms of 48 tokens
// took 13 us a call, of which the launch is 3.5.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <optional>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "hgemm_b200.h"

namespace {

decltype(&hgemm_lora) g_lora;
decltype(&hgemm_lora_workspace_bytes) g_lora_bytes;
decltype(&hgemm_qk_norm_rope) g_norm;
decltype(&hgemm_attn_prompt) g_attn;
decltype(&hgemm_attn_prompt_workspace_bytes) g_attn_bytes;
PyObject *g_error;  // HgemmError

struct Refused {};  // a Python error is set
template <class... A>
[[noreturn]] void refuse(PyObject *type, const char *format, A... args) {
  PyErr_Format(type, format, args...);
  throw Refused();
}

const at::Tensor &tensor(const char *name, PyObject *o) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
void type_is(const char *name, const at::Tensor &t, at::ScalarType type) {
  if (t.scalar_type() != type)
    refuse(PyExc_TypeError, "%s must be %s, got %s", name, c10::toString(type), c10::toString(t.scalar_type()));
}
void dims_are(const char *name, const at::Tensor &t, int64_t dims) {
  if (t.dim() != dims)
    refuse(PyExc_ValueError, "%s must have %lld dimensions, got %lld", name, static_cast<long long>(dims),
           static_cast<long long>(t.dim()));
}
int as_int(int64_t n) {
  if (n > INT_MAX) refuse(PyExc_ValueError, "a size of %lld is too large", static_cast<long long>(n));
  return static_cast<int>(n);
}
c10::Device cuda(const at::Tensor &t) {
  if (!t.is_cuda()) refuse(PyExc_ValueError, "the operators take CUDA tensors");
  return t.device();
}
void on(const char *name, const at::Tensor &t, c10::Device dev) {
  if (t.device() != dev) refuse(PyExc_ValueError, "%s must be on cuda:%d", name, static_cast<int>(dev.index()));
}

// A contiguous operand of the given shape.
template <class T>
T *dense(const char *name, PyObject *o, at::ScalarType type, at::IntArrayRef shape, c10::Device dev) {
  const at::Tensor &t = tensor(name, o);
  type_is(name, t, type);
  dims_are(name, t, static_cast<int64_t>(shape.size()));
  for (size_t i = 0; i < shape.size(); ++i)
    if (t.size(i) != shape[i])
      refuse(PyExc_ValueError, "dimension %d of %s must be %lld, got %lld", static_cast<int>(i), name,
             static_cast<long long>(shape[i]), static_cast<long long>(t.size(i)));
  on(name, t, dev);
  if (!t.is_contiguous()) refuse(PyExc_ValueError, "%s must be contiguous", name);
  return static_cast<T *>(t.data_ptr());
}

// tokens x heads x head_dim with the heads of a token adjacent: its address, and the token stride.
hgemm_half_t *heads(const char *name, const at::Tensor &t, c10::Device dev, long long *stride) {
  type_is(name, t, at::kHalf);
  dims_are(name, t, 3);
  on(name, t, dev);
  const int64_t n = t.size(0), h = t.size(1), d = t.size(2);
  if (n && h && ((d > 1 && t.stride(2) != 1) || (h > 1 && t.stride(1) != d)))
    refuse(PyExc_ValueError, "the heads of a token must be adjacent in %s", name);
  *stride = n > 1 ? t.stride(0) : std::max<long long>(t.stride(0), h * d);
  return static_cast<hgemm_half_t *>(t.data_ptr());
}
bool same_shape(const at::Tensor &a, const at::Tensor &b) { return a.sizes() == b.sizes(); }

// The launching stream: None for the device's current one, an address or a torch stream. While it lives
// the device is current, and so is the stream: memory of this call comes from its pool and is free for later work on
// it.
struct Launch {
  std::optional<c10::cuda::CUDAGuard> device;
  std::optional<c10::cuda::CUDAStreamGuard> guard;
  hgemm_stream_t stream;
  Launch(c10::Device dev, PyObject *o) {
    if (o == Py_None) {
      device.emplace(dev);
      stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
      return;
    }
    PyObject *address = PyLong_Check(o) ? Py_NewRef(o) : PyObject_GetAttrString(o, "cuda_stream");
    if (!address) throw Refused();
    stream = static_cast<cudaStream_t>(PyLong_AsVoidPtr(address));
    Py_DECREF(address);
    if (PyErr_Occurred()) throw Refused();
    guard.emplace(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(stream), dev.index()));
  }
};

at::Tensor fresh(at::IntArrayRef shape, c10::Device dev) {
  return at::Tensor(at::detail::empty_cuda(shape, at::kHalf, dev, std::nullopt));
}

// The caller's workspace or one of this call, which `keep` holds until the launch is made.
template <class Args>
void scratch(Args &args, size_t need, PyObject *workspace, c10::Device dev, at::Tensor &keep) {
  args.workspace = nullptr;
  args.workspace_bytes = 0;
  if (workspace == Py_None) {
    if (need == 0) return;
    keep = fresh({static_cast<int64_t>((need + 1) / 2)}, dev);
  } else {
    keep = tensor("workspace", workspace);
    on("workspace", keep, dev);
    if (!keep.is_contiguous()) refuse(PyExc_ValueError, "workspace must be contiguous");
  }
  args.workspace = keep.data_ptr();
  args.workspace_bytes = keep.nbytes();
}

template <class Entry, class Args>
void call(const char *name, Entry entry, const Args &args, hgemm_stream_t stream) {
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = entry(&args, stream);
  Py_END_ALLOW_THREADS
  if (status == HGEMM_OK) return;
  if (PyObject *e = PyObject_CallFunction(g_error, "is", status, name)) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw Refused();
}

// A tensor of the caller's that was written: what autograd has saved of it is no longer that, and it says so.
void written(PyObject *o) {
  if (o == Py_None) return;
  const at::Tensor &t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

template <class F>
PyObject *guarded(Py_ssize_t got, Py_ssize_t want, F &&f) {
  HANDLE_TH_ERRORS
  if (got != want || !g_error) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments, or bind() was not called");
    return nullptr;
  }
  try {
    return f();
  } catch (const Refused &) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// X, W, down, up, scale, seg_start, seg_adapter, Y, workspace, stream
PyObject *lora(PyObject *, PyObject *const *p, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject * {
    const at::Tensor &X = tensor("X", p[0]), &W = tensor("W", p[1]), &down = tensor("down", p[2]),
                     &ids = tensor("seg_adapter", p[6]);
    const c10::Device dev = cuda(X);
    dims_are("X", X, 2);
    dims_are("W", W, 2);
    dims_are("down", down, 3);
    dims_are("seg_adapter", ids, 1);
    const int64_t T = X.size(0), K = X.size(1), N = W.size(1), A = down.size(0), r = down.size(2),
                  S = ids.size(0);
    hgemm_lora_t a;
    a.tokens = as_int(T);
    a.N = as_int(N);
    a.K = as_int(K);
    a.rank = as_int(r);
    a.adapters = as_int(A);
    a.segments = as_int(S);
    a.X = dense<hgemm_half_t>("X", p[0], at::kHalf, {T, K}, dev);
    a.W = dense<hgemm_half_t>("W", p[1], at::kHalf, {K, N}, dev);
    a.down = dense<hgemm_half_t>("down", p[2], at::kHalf, {A, K, r}, dev);
    a.up = dense<hgemm_half_t>("up", p[3], at::kHalf, {A, r, N}, dev);
    a.scale = dense<float>("scale", p[4], at::kFloat, {A}, dev);
    a.seg_start = dense<int>("seg_start", p[5], at::kInt, {S + 1}, dev);
    a.seg_adapter = dense<int>("seg_adapter", p[6], at::kInt, {S}, dev);
    if (p[7] != Py_None) a.Y = dense<hgemm_half_t>("Y", p[7], at::kHalf, {T, N}, dev);
    const Launch launch(dev, p[9]);
    at::Tensor Y, keep;
    if (p[7] == Py_None) {
      Y = fresh({T, N}, dev);
      a.Y = static_cast<hgemm_half_t *>(Y.data_ptr());
    }
    scratch(a, g_lora_bytes(a.tokens, a.N, a.K, a.rank, a.adapters, a.segments), p[8], dev, keep);
    call("hgemm_lora", g_lora, a, launch.stream);
    written(p[7]);
    return p[7] == Py_None ? THPVariable_Wrap(Y) : Py_NewRef(p[7]);
  });
}

// q, k, q_weight, k_weight, positions, inv_freq, eps, axis_of, interleaved, q_out, k_out, stream
PyObject *qk_norm_rope(PyObject *, PyObject *const *p, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject * {
    const at::Tensor &q = tensor("q", p[0]), &k = tensor("k", p[1]), &pos = tensor("positions", p[4]),
                     &inv = tensor("inv_freq", p[5]);
    const c10::Device dev = cuda(q);
    hgemm_qk_norm_rope_t a;
    a.q = heads("q", q, dev, &a.q_stride);
    a.k = heads("k", k, dev, &a.k_stride);
    const int64_t T = q.size(0), hq = q.size(1), hk = k.size(1), d = q.size(2);
    if (k.size(0) != T || k.size(2) != d) refuse(PyExc_ValueError, "tokens or head_dim of q and k differ");
    dims_are("inv_freq", inv, 1);
    const int64_t half = inv.size(0), axes = pos.dim() == 2 ? pos.size(0) : 1;
    a.tokens = as_int(T);
    a.heads_q = as_int(hq);
    a.heads_kv = as_int(hk);
    a.head_dim = as_int(d);
    a.rot_dim = as_int(2 * half);
    a.axes = as_int(axes);
    a.q_weight = dense<hgemm_half_t>("q_weight", p[2], at::kHalf, {d}, dev);
    a.k_weight = dense<hgemm_half_t>("k_weight", p[3], at::kHalf, {d}, dev);
    a.positions = pos.dim() == 2 ? dense<int>("positions", p[4], at::kInt, {axes, T}, dev)
                                 : dense<int>("positions", p[4], at::kInt, {T}, dev);
    a.inv_freq = dense<float>("inv_freq", p[5], at::kFloat, {half}, dev);
    a.axis_of = p[7] == Py_None ? nullptr : dense<unsigned char>("axis_of", p[7], at::kByte, {half}, dev);
    a.eps = static_cast<float>(PyFloat_AsDouble(p[6]));
    a.interleaved = PyObject_IsTrue(p[8]);
    if (PyErr_Occurred()) throw Refused();
    auto given = [&](const char *name, PyObject *o, const at::Tensor &in, long long *stride) {
      const at::Tensor &t = tensor(name, o);
      hgemm_half_t *at = heads(name, t, dev, stride);
      if (!same_shape(t, in)) refuse(PyExc_ValueError, "%s has another shape than its input", name);
      return at;
    };
    if (p[9] != Py_None) a.q_out = given("q_out", p[9], q, &a.q_out_stride);
    if (p[10] != Py_None) a.k_out = given("k_out", p[10], k, &a.k_out_stride);
    const Launch launch(dev, p[11]);
    at::Tensor q_out, k_out;
    if (p[9] == Py_None) {
      q_out = fresh(q.sizes(), dev);
      a.q_out = static_cast<hgemm_half_t *>(q_out.data_ptr());
      a.q_out_stride = hq * d;
    }
    if (p[10] == Py_None) {
      k_out = fresh(k.sizes(), dev);
      a.k_out = static_cast<hgemm_half_t *>(k_out.data_ptr());
      a.k_out_stride = hk * d;
    }
    call("hgemm_qk_norm_rope", g_norm, a, launch.stream);
    written(p[9]);
    written(p[10]);
    PyObject *y0 = p[9] == Py_None ? THPVariable_Wrap(q_out) : Py_NewRef(p[9]);
    PyObject *y1 = p[10] == Py_None ? THPVariable_Wrap(k_out) : Py_NewRef(p[10]);
    PyObject *both = y0 && y1 ? PyTuple_Pack(2, y0, y1) : nullptr;
    Py_XDECREF(y0);
    Py_XDECREF(y1);
    return both;
  });
}

// q, k, v, cu_q, cu_k, scale, causal, out, lse, workspace, stream
PyObject *attn_prompt(PyObject *, PyObject *const *p, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject * {
    const at::Tensor &q = tensor("q", p[0]), &k = tensor("k", p[1]), &v = tensor("v", p[2]),
                     &cu = tensor("cu_q", p[3]);
    const c10::Device dev = cuda(q);
    hgemm_attn_prompt_t a;
    a.q = heads("q", q, dev, &a.q_stride);
    a.k = heads("k", k, dev, &a.k_stride);
    a.v = heads("v", v, dev, &a.v_stride);
    const int64_t Tq = q.size(0), hq = q.size(1), d = q.size(2);
    if (!same_shape(k, v) || k.size(2) != d)
      refuse(PyExc_ValueError, "shapes of k and v, or head_dim of q and k, differ");
    dims_are("cu_q", cu, 1);
    const int64_t starts = cu.size(0);
    a.total_q = as_int(Tq);
    a.total_k = as_int(k.size(0));
    a.batch = as_int(starts - 1);
    a.heads_q = as_int(hq);
    a.heads_kv = as_int(k.size(1));
    a.head_dim = as_int(d);
    a.cu_q = dense<int>("cu_q", p[3], at::kInt, {starts}, dev);
    a.cu_k = p[4] == Py_None ? nullptr : dense<int>("cu_k", p[4], at::kInt, {starts}, dev);
    a.scale = static_cast<float>(p[5] == Py_None ? 1.0 / std::sqrt(static_cast<double>(d)) : PyFloat_AsDouble(p[5]));
    a.causal = PyObject_IsTrue(p[6]);
    if (PyErr_Occurred()) throw Refused();
    a.lse = p[8] == Py_None ? nullptr : dense<float>("lse", p[8], at::kFloat, {Tq, hq}, dev);
    if (p[7] != Py_None) {
      const at::Tensor &out = tensor("out", p[7]);
      a.out = heads("out", out, dev, &a.out_stride);
      if (!same_shape(out, q)) refuse(PyExc_ValueError, "out has another shape than q");
    }
    const Launch launch(dev, p[10]);
    at::Tensor out, keep;
    if (p[7] == Py_None) {
      out = fresh(q.sizes(), dev);
      a.out = static_cast<hgemm_half_t *>(out.data_ptr());
      a.out_stride = hq * d;
    }
    scratch(a, g_attn_bytes(a.total_q, a.total_k, a.batch, a.heads_q, a.heads_kv, a.head_dim), p[9], dev, keep);
    call("hgemm_attn_prompt", g_attn, a, launch.stream);
    written(p[7]);
    written(p[8]);
    return p[7] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(p[7]);
  });
}

// Addresses of the five entry points, in the order of the variables above, and the exception class.
PyObject *bind(PyObject *, PyObject *args) {
  Py_ssize_t f[5];
  PyObject *error;
  if (!PyArg_ParseTuple(args, "nnnnnO", &f[0], &f[1], &f[2], &f[3], &f[4], &error)) return nullptr;
  g_lora = reinterpret_cast<decltype(g_lora)>(f[0]);
  g_lora_bytes = reinterpret_cast<decltype(g_lora_bytes)>(f[1]);
  g_norm = reinterpret_cast<decltype(g_norm)>(f[2]);
  g_attn = reinterpret_cast<decltype(g_attn)>(f[3]);
  g_attn_bytes = reinterpret_cast<decltype(g_attn_bytes)>(f[4]);
  Py_XSETREF(g_error, Py_NewRef(error));
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"lora", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(lora)), METH_FASTCALL, nullptr},
    {"qk_norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qk_norm_rope)), METH_FASTCALL,
     nullptr},
    {"attn_prompt", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attn_prompt)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operators", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__operators() {
  PyObject *m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", OPERATORS_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
