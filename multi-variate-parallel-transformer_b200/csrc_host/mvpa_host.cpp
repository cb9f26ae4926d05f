// Host path of the torch operators: what Python did around the C ABI (include/mvpa.h) - checks, outputs, scratch, views and,
// for a block, the projections - as single calls.  A small operator call needs 10 us of the device; the same work took
// 25 us in Python, a training step of a block 1.1 ms where the device needs 0.6.
//
// Every function here works on ordinary CUDA tensors that nothing watches (no mode, transform or tracer) and answers None
// for anything else, which the callers then take through their Python path; results and errors are the same either way.
#include <Python.h>
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/autocast_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/PyInterpreter.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "mvpa.h"

namespace {

using at::Tensor;

struct Api {
  decltype(&mvpa_fwd_workspace_bytes) fwd_bytes;
  decltype(&mvpa_bwd_workspace_bytes) bwd_bytes;
  decltype(&mvpa_fwd) fwd;
  decltype(&mvpa_bwd) bwd;
  decltype(&mvpa_rmsnorm) rmsnorm;
  decltype(&mvpa_rmsnorm_bwd) rmsnorm_bwd;
  decltype(&mvpa_rmsnorm_bwd_workspace_bytes) rmsnorm_bwd_bytes;
  decltype(&mvpa_silu_mul) silu_mul;
  decltype(&mvpa_silu_mul_bwd) silu_mul_bwd;
  decltype(&mvpa_workspace_status) fwd_status;
  decltype(&mvpa_bwd_status) bwd_status;
  decltype(&mvpa_last_error_string) last_error;
  decltype(&mvpa_quantize_fp8) quantize_fp8;
  decltype(&mvpa_rmsnorm_fp8) rmsnorm_fp8;
  decltype(&mvpa_silu_mul_fp8) silu_mul_fp8;
  decltype(&mvpa_matmul_fp8) matmul_fp8;
  decltype(&mvpa_gated_linear) gated_linear;
  decltype(&mvpa_gated_linear_bwd) gated_linear_bwd;
  decltype(&mvpa_gated_linear_saved_bytes) gated_saved_bytes;
  decltype(&mvpa_gated_linear_bwd_workspace_bytes) gated_bwd_bytes;
  decltype(&mvpa_quantize_int4) quantize_int4;
  decltype(&mvpa_dequantize_int4) dequantize_int4;
  decltype(&mvpa_matmul_int4) matmul_int4;
  decltype(&mvpa_matmul_int4_workspace_bytes) int4_workspace_bytes;
} api;

PyObject* device_mode = nullptr;  // torch.utils._device.DeviceContext

void check(int status, const char* what) {
  if (status != 0)
    throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(status) + "): " + api.last_error());
}

// Nothing follows the current call operation by operation.  (Forward-mode levels and compilers are looked at in Python.)
bool watched() {
  using c10::DispatchKey;
  static constexpr c10::DispatchKeySet keys({DispatchKey::FuncTorchDynamicLayerFrontMode, DispatchKey::FuncTorchDynamicLayerBackMode,
                                             DispatchKey::FuncTorchVmapMode, DispatchKey::FuncTorchBatched, DispatchKey::Python,
                                             DispatchKey::Functionalize, DispatchKey::Tracer, DispatchKey::PreDispatch});
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || !(c10::impl::tls_local_dispatch_key_set().included_ & keys).empty() ||
         torch::jit::tracer::isTracing();
}
// (A default device is a function mode as well; it only fills in where new tensors live.)
bool function_modes() {
  for (int64_t i = 0, n = at::impl::PythonTorchFunctionTLS::stack_len(); i < n; ++i) {
    const int device = PyObject_IsInstance(at::impl::PythonTorchFunctionTLS::get_stack_at(i)->ptr(getPyInterpreter()), device_mode);
    if (device < 0) throw python_error();
    if (device == 0) return true;
  }
  return false;
}

bool ordinary(const Tensor& t) {  // a strided CUDA tensor with storage and no wrapper or lazy bit
  using c10::DispatchKey;
  static constexpr c10::DispatchKeySet allowed =
      c10::DispatchKeySet(DispatchKey::CUDA) | c10::DispatchKeySet({DispatchKey::ADInplaceOrView, DispatchKey::AutogradCUDA, DispatchKey::AutocastCUDA});
  return t.defined() && t.is_cuda() && t.has_storage() && (t.key_set() | allowed) == allowed;
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return MVPA_BF16;
    case at::kFloat: return MVPA_F32;
    case at::kHalf: return MVPA_F16;
    default: return -1;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// (B, heads, N, D) as the kernels read it in place: contiguous last dimension, 16-byte aligned base and strides
bool rows_fit(const Tensor& t) {
  if (t.dim() != 4 || t.stride(3) != 1) return false;
  const int64_t es = t.element_size();
  return ((t.stride(0) | t.stride(1) | t.stride(2)) * es & 15) == 0 && aligned16(t.const_data_ptr());
}

mvpa_tensor view4(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }
// `heads` heads of D columns starting at column `col` of a (B * N, ld) matrix
mvpa_tensor columns(const Tensor& m, int64_t col, int64_t N, int64_t D) {
  const int64_t ld = m.stride(0);
  return {static_cast<char*>(m.data_ptr()) + col * m.element_size(), N * ld, D, ld};
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

struct Ops {  // q, u, vt, z, k, r_time, r_chan, v
  Tensor t[8];
  bool take(PyObject* const* a, int64_t steps = 0) {  // `steps` time steps of queries, 0 for all
    for (int i = 0; i < 8; ++i) {
      if (!THPVariable_CheckExact(a[i])) return false;
      t[i] = THPVariable_Unpack(a[i]);
      if (!ordinary(t[i]) || t[i].device() != t[0].device() || t[i].scalar_type() != t[0].scalar_type() || t[i].numel() == 0) return false;
    }
    if (dtype_code(t[0]) < 0 || !rows_fit(t[0]) || !rows_fit(t[4]) || !rows_fit(t[7]) || t[5].dim() < 2 || t[6].dim() < 2) return false;
    for (int i : {1, 2, 3, 5, 6})
      if (!t[i].is_contiguous()) return false;
    const int64_t Hkv = t[4].size(1), N = t[4].size(2), D = t[4].size(3), T = t[5].size(-2), C = t[6].size(-2);
    return t[4].sizes() == t[7].sizes() && t[0].size(0) == t[4].size(0) && t[0].size(3) == D && T * C == N &&
           t[0].size(2) == (steps ? steps : T) * C && t[1].numel() == Hkv * D && t[2].numel() == Hkv * D && t[3].numel() == Hkv * D &&
           t[5].numel() == Hkv * T * D && t[6].numel() == Hkv * C * D;
  }
  mvpa_problem problem(double scale, int64_t window, int64_t t0, int64_t tn) const {
    mvpa_problem p = {};
    p.B = (int32_t)t[0].size(0); p.H = (int32_t)t[0].size(1); p.Hkv = (int32_t)t[4].size(1); p.D = (int32_t)t[0].size(3);
    p.T = (int32_t)t[5].size(-2); p.C = (int32_t)t[6].size(-2);
    p.window = (int32_t)window; p.dtype = dtype_code(t[0]); p.sm_scale = (float)scale;
    p.q_time_begin = (int32_t)t0; p.q_time_count = (int32_t)tn;
    return p;
  }
};

Tensor scratch(size_t bytes, const Tensor& like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte).requires_grad(false)); }

void launch_fwd(const mvpa_problem& p, const mvpa_tensor& q, const mvpa_tensor& k, const mvpa_tensor& v, const void* u, const void* vt,
                const void* z, const Tensor& rt, const Tensor& rc, const mvpa_tensor& o, float* lse, bool status) {
  const size_t bytes = api.fwd_bytes(&p);
  const Tensor ws = bytes ? scratch(bytes, rt) : Tensor();
  check(api.fwd(&p, &q, &k, &v, u, vt, z, rt.const_data_ptr(), rc.const_data_ptr(), &o, lse, bytes ? ws.data_ptr() : nullptr, bytes,
                stream_of(rt)), "mvpa_fwd");
  if (status && bytes) check(api.fwd_status(ws.data_ptr(), bytes, stream_of(rt)), "mvpa_fwd kernels");  // synchronises the stream
}

// Gradients of u, vt, z, r_time, r_chan one after the other, flat, in the operands' type (they leave the library as fp32; one
// buffer means one cast, and every piece is a whole number of rows of D >= 16 elements, hence 16-byte aligned).
Tensor launch_bwd(const mvpa_problem& p, const mvpa_tensor& q, const mvpa_tensor& k, const mvpa_tensor& v, const void* u, const void* vt,
                  const void* z, const Tensor& rt, const Tensor& rc, const mvpa_tensor& o, const Tensor& lse, const mvpa_tensor& d_o,
                  const mvpa_tensor& dq, const mvpa_tensor& dk, const mvpa_tensor& dv, bool status) {
  const int64_t nb = (int64_t)p.Hkv * p.D, nt = rt.numel(), nc = rc.numel();
  const Tensor small = at::empty({3 * nb + nt + nc}, rt.options().dtype(at::kFloat).requires_grad(false));
  float* f = small.data_ptr<float>();
  const size_t bytes = api.bwd_bytes(&p);
  const Tensor ws = scratch(bytes < 16 ? 16 : bytes, rt);
  check(api.bwd(&p, &q, &k, &v, u, vt, z, rt.const_data_ptr(), rc.const_data_ptr(), &o, lse.const_data_ptr<float>(), &d_o, &dq, &dk, &dv,
                f, f + nb, f + 2 * nb, f + 3 * nb, f + 3 * nb + nt, ws.data_ptr(), bytes, stream_of(rt)), "mvpa_bwd");
  if (status) check(api.bwd_status(&p, ws.data_ptr(), bytes, stream_of(rt)), "mvpa_bwd kernels");
  return small.to(rt.scalar_type());
}

bool numbers(PyObject* scale, PyObject* window, double* s, int64_t* w) {
  if (!PyFloat_Check(scale) || !PyLong_CheckExact(window)) return false;
  *s = PyFloat_AS_DOUBLE(scale);
  int overflow = 0;
  *w = PyLong_AsLongLongAndOverflow(window, &overflow);
  return !overflow && *w >= INT32_MIN && *w <= INT32_MAX;
}

PyObject* wrap(std::vector<Tensor>&& ts) {  // undefined tensors become None
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  if (!out) throw python_error();
  for (size_t i = 0; i < ts.size(); ++i) {
    PyObject* o;
    if (ts[i].defined()) o = THPVariable_Wrap(std::move(ts[i]));
    else { o = Py_None; Py_INCREF(o); }
    PyTuple_SET_ITEM(out, (Py_ssize_t)i, o);
  }
  return out;
}

bool arguments(Py_ssize_t given, Py_ssize_t wanted) {
  if (given == wanted) return true;
  PyErr_SetString(PyExc_TypeError, "mvpa_host: wrong number of arguments");
  return false;
}

// attend(q, u, vt, z, k, r_time, r_chan, v, sm_scale, window, status): the whole of an operator call that no gradient flows through,
// shapes as `flash_mvpa` wants them.  -> o or None
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 11)) return nullptr;
  const bool status = a[10] == Py_True;
  Ops x;
  double scale;
  int64_t window;
  if (!numbers(a[8], a[9], &scale, &window) || function_modes() || watched() || !x.take(a)) Py_RETURN_NONE;
  const Tensor &q = x.t[0], &k = x.t[4], &rt = x.t[5], &rc = x.t[6];
  const int64_t D = q.size(3);
  if (c10::GradMode::is_enabled())
    for (const Tensor& t : x.t)
      if (t.requires_grad()) Py_RETURN_NONE;
  if (q.size(1) % k.size(1) != 0 || (D != 16 && D != 32 && D != 64 && D != 128) || rt.dim() != 4 || rc.dim() != 4)
    Py_RETURN_NONE;
  Tensor o;
  {
    pybind11::gil_scoped_release nogil;
    c10::cuda::CUDAGuard guard(q.device());
    c10::NoGradGuard no_grad;
    o = at::empty_like(q);
    launch_fwd(x.problem(scale, window, 0, 0), view4(q), view4(k), view4(x.t[7]), x.t[1].const_data_ptr(), x.t[2].const_data_ptr(),
               x.t[3].const_data_ptr(), rt, rc, view4(o), nullptr, status);
  }
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

// forward(q, u, vt, z, k, r_time, r_chan, v, sm_scale, window, t0, tn, status) -> (o, lse) or None
PyObject* forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 13)) return nullptr;
  const bool status = a[12] == Py_True;
  Ops x;
  double scale;
  int64_t window;
  if (!numbers(a[8], a[9], &scale, &window) || !PyLong_CheckExact(a[10]) || !PyLong_CheckExact(a[11]) || function_modes() ||
      watched())
    Py_RETURN_NONE;
  const int64_t t0 = PyLong_AsLongLong(a[10]), tn = PyLong_AsLongLong(a[11]);
  if (PyErr_Occurred()) return nullptr;
  if (!x.take(a, tn)) Py_RETURN_NONE;
  const Tensor& q = x.t[0];
  Tensor o, lse;
  {
    pybind11::gil_scoped_release nogil;
    c10::cuda::CUDAGuard guard(q.device());
    c10::NoGradGuard no_grad;
    o = at::empty_like(q);
    lse = at::empty({q.size(0) * q.size(1), q.size(2)}, q.options().dtype(at::kFloat).requires_grad(false));
    launch_fwd(x.problem(scale, window, t0, tn), view4(q), view4(x.t[4]), view4(x.t[7]), x.t[1].const_data_ptr(),
               x.t[2].const_data_ptr(), x.t[3].const_data_ptr(), x.t[5], x.t[6], view4(o), lse.data_ptr<float>(), status);
  }
  return wrap({std::move(o), std::move(lse)});
  END_HANDLE_TH_ERRORS
}

// backward(do, q, u, vt, z, k, r_time, r_chan, v, o, lse, sm_scale, window, status) -> the eight gradients or None
PyObject* backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 14)) return nullptr;
  const bool status = a[13] == Py_True;
  Ops x;
  double scale;
  int64_t window;
  for (int i : {0, 9, 10})
    if (!THPVariable_CheckExact(a[i])) Py_RETURN_NONE;
  if (!numbers(a[11], a[12], &scale, &window) || function_modes() || watched() || !x.take(a + 1)) Py_RETURN_NONE;
  Tensor d_o = THPVariable_Unpack(a[0]);
  const Tensor o = THPVariable_Unpack(a[9]), lse = THPVariable_Unpack(a[10]);
  const Tensor &q = x.t[0], &k = x.t[4], &v = x.t[7];
  for (const Tensor& t : {d_o, o})
    if (!ordinary(t) || t.device() != q.device() || t.scalar_type() != q.scalar_type() || t.sizes() != q.sizes()) Py_RETURN_NONE;
  if (!ordinary(lse) || lse.scalar_type() != at::kFloat || lse.device() != q.device() || !lse.is_contiguous() ||
      lse.numel() != q.size(0) * q.size(1) * q.size(2) || !rows_fit(o))
    Py_RETURN_NONE;
  std::vector<Tensor> g(8);
  {
    pybind11::gil_scoped_release nogil;
    c10::cuda::CUDAGuard guard(q.device());
    c10::NoGradGuard no_grad;
    if (!rows_fit(d_o)) d_o = d_o.contiguous();
    g[0] = at::empty_like(q);
    g[4] = at::empty_like(k);
    g[7] = at::empty_like(v);
    const Tensor small = launch_bwd(x.problem(scale, window, 0, 0), view4(q), view4(k), view4(v), x.t[1].const_data_ptr(),
                                    x.t[2].const_data_ptr(), x.t[3].const_data_ptr(), x.t[5], x.t[6], view4(o), lse, view4(d_o),
                                    view4(g[0]), view4(g[4]), view4(g[7]), status);
    int64_t at = 0;
    for (int i : {1, 2, 3, 5, 6}) {
      g[i] = small.narrow(0, at, x.t[i].numel()).view(x.t[i].sizes());
      at += x.t[i].numel();
    }
  }
  return wrap(std::move(g));
  END_HANDLE_TH_ERRORS
}

// plain(*tensors): 1 if the kernels can take these contiguous tensors and nothing watches the call, 0 if not, -1 if Python has to look
PyObject* plain(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  long answer = 1;
  if (n == 0 || function_modes()) return PyLong_FromLong(-1);
  for (Py_ssize_t i = 0; i < n && answer == 1; ++i)
    if (!THPVariable_CheckExact(a[i])) answer = 0;
  if (answer == 1 && watched()) answer = 0;
  if (answer == 1) {
    const Tensor& t0 = THPVariable_Unpack(a[0]);
    for (Py_ssize_t i = 0; i < n && answer == 1; ++i) {
      const Tensor& t = THPVariable_Unpack(a[i]);
      if (!ordinary(t) || (t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kFloat) || t.scalar_type() != t0.scalar_type() ||
               t.device() != t0.device() || !t.is_contiguous() || t.numel() == 0 || !aligned16(t.const_data_ptr()))
        answer = 0;
    }
  }
  return PyLong_FromLong(answer);
  END_HANDLE_TH_ERRORS
}

struct Dims {
  int64_t B, T, C, E, H, Hkv, D, I, N, KV, rows;
  mvpa_problem problem(int dtype, double scale, int window) const {
    mvpa_problem p = {};
    p.B = (int32_t)B; p.H = (int32_t)H; p.Hkv = (int32_t)Hkv; p.T = (int32_t)T; p.C = (int32_t)C; p.D = (int32_t)D;
    p.window = window; p.dtype = dtype; p.sm_scale = (float)scale;
    return p;
  }
};

// What the kernels read of a block through pointers: one type and device, contiguous, 16-byte aligned, of the given sizes.
bool fits(const Tensor& t, const Tensor& like, at::ScalarType type, at::IntArrayRef sizes) {
  return ordinary(t) && t.scalar_type() == type && t.device() == like.device() && t.is_contiguous() && t.sizes() == sizes &&
         aligned16(t.const_data_ptr());
}

// The sizes of a block's call; false where an input (x, pos, chan, ln_w, wq, wkv, wpos, wchan, bias, wc, wg, wu, wd) is not of them.
bool block_dims(const Tensor* in, PyObject* const* heads, Dims& d) {
  const Tensor &x = in[0], &bias = in[8], &wg = in[10];
  d.H = PyLong_AsLongLong(heads[0]); d.Hkv = PyLong_AsLongLong(heads[1]); d.D = PyLong_AsLongLong(heads[2]);
  if (PyErr_Occurred()) throw python_error();
  if (!ordinary(x) || x.dim() != 4 || x.numel() == 0 || dtype_code(x) < 0 || !ordinary(wg) || wg.dim() != 2 || !ordinary(bias) ||
      d.H <= 0 || d.Hkv <= 0 || d.D <= 0)
    return false;
  d.B = x.size(0); d.T = x.size(1); d.C = x.size(2); d.E = x.size(3); d.I = wg.size(0);
  d.N = d.T * d.C; d.KV = d.Hkv * d.D; d.rows = d.B * d.N;
  const int64_t Q = d.H * d.D;
  const std::vector<int64_t> sizes[13] = {x.sizes().vec(), {1, d.T, d.E}, {1, d.C, d.E}, {d.E}, {Q, d.E}, {2 * d.KV, d.E}, {d.KV, d.E},
                                          {d.KV, d.E}, bias.sizes().vec(), {d.E, Q}, {d.I, d.E}, {d.I, d.E}, {d.E, d.I}};
  for (int i = 0; i < 13; ++i)
    if (!fits(in[i], x, x.scalar_type(), sizes[i])) return false;
  return bias.numel() == 3 * d.KV && d.I > 0 && d.I * x.element_size() % 16 == 0;
}

// What the body of a block's call runs under.  No autocast: a backward may run inside a region that the forward was outside of, and
// the kernels read every product as the type that the forward had.
struct Body {
  pybind11::gil_scoped_release nogil;
  c10::cuda::CUDAGuard guard;
  c10::NoGradGuard no_grad;
  c10::impl::ExcludeDispatchKeyGuard no_autocast{c10::autocast_dispatch_keyset};
  explicit Body(const Tensor& t) : guard(t.device()) {}
};

// The kernels' status word, looked at after a call (which synchronises the stream) where calls are checked; else no tensor.
Tensor status_word(bool status, const Tensor& like) {
  return status ? at::zeros({64}, like.options().dtype(at::kInt).requires_grad(false)) : Tensor();
}
int32_t* word_of(const Tensor& word) { return word.defined() ? word.data_ptr<int32_t>() : nullptr; }
void look_at(const Tensor& word, const Tensor& like, const char* what) {
  if (word.defined()) check(api.fwd_status(word.data_ptr(), 256, stream_of(like)), what);
}

const char* part(const Tensor& t, int64_t elements) { return static_cast<const char*>(t.const_data_ptr()) + elements * t.element_size(); }

// block_forward(x, pos, chan, ln_w, wq, wkv, wpos, wchan, bias, wc, wg, wu, wd, eps, window, H, Hkv, D, status, gated)
//   -> (h, xn, q, kv, g, up, rt, rc, o, lse, act): `block_grad.BlockFunction.forward`, or None.  `gated` (bf16): the gate as one kernel,
//   which keeps what the backward wants in one tensor of bytes, in g's place; up is None.
PyObject* block_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 20)) return nullptr;
  const bool status = a[18] == Py_True, gated = a[19] == Py_True;
  Tensor in[13];
  for (int i = 0; i < 13; ++i) {
    if (!THPVariable_CheckExact(a[i])) Py_RETURN_NONE;
    in[i] = THPVariable_Unpack(a[i]);
  }
  Dims d;
  if (watched() || !block_dims(in, a + 15, d) || (gated && (in[0].scalar_type() != at::kBFloat16 || d.E % 8 != 0 || d.I % 8 != 0))) Py_RETURN_NONE;
  const Tensor &x = in[0], &pos = in[1], &chan = in[2], &ln_w = in[3], &wq = in[4], &wkv = in[5], &wpos = in[6], &wchan = in[7],
               &bias = in[8], &wc = in[9], &wg = in[10], &wu = in[11], &wd = in[12];
  const double eps = PyFloat_AsDouble(a[13]);
  const int64_t window = PyLong_AsLongLong(a[14]);
  if (PyErr_Occurred()) return nullptr;
  Tensor h, xn, q, kv, g, up, rt, rc, o, lse, act;
  {
    const Body body(x);
    const int dt = dtype_code(x);
    const Tensor x2 = x.view({d.rows, d.E});
    xn = at::empty_like(x2);
    check(api.rmsnorm(x2.const_data_ptr(), nullptr, ln_w.const_data_ptr(), nullptr, xn.data_ptr(), d.rows, (int32_t)d.E, (float)eps, dt,
                      stream_of(x)), "mvpa_rmsnorm");
    q = at::mm(xn, wq.t());
    kv = at::mm(xn, wkv.t());
    if (!gated) {
      g = at::mm(xn, wg.t());
      up = at::mm(xn, wu.t());
    }
    const auto keys = [&](const Tensor& embeds, const Tensor& w) {  // (Hkv, rows, D)
      return at::mm(embeds.select(0, 0), w.t()).view({-1, d.Hkv, d.D}).transpose(0, 1).contiguous();
    };
    rt = keys(pos, wpos);
    rc = keys(chan, wchan);
    o = at::empty_like(q);
    lse = at::empty({d.B * d.H, d.N}, x.options().dtype(at::kFloat).requires_grad(false));
    launch_fwd(d.problem(dt, 1.0 / std::sqrt((double)d.D), (int)window), columns(q, 0, d.N, d.D), columns(kv, 0, d.N, d.D),
               columns(kv, d.KV, d.N, d.D), part(bias, 0), part(bias, d.KV), part(bias, 2 * d.KV), rt, rc, columns(o, 0, d.N, d.D),
               lse.data_ptr<float>(), status);
    act = at::empty({d.rows, d.I}, xn.options());
    if (gated) {
      g = scratch(api.gated_saved_bytes(d.rows, (int32_t)d.I), x);
      const Tensor word = status_word(status, x);
      check(api.gated_linear(xn.const_data_ptr(), d.E, wg.const_data_ptr(), wu.const_data_ptr(), act.data_ptr(), d.I, g.data_ptr(), d.rows,
                             (int32_t)d.E, (int32_t)d.I, word_of(word), stream_of(x)), "mvpa_gated_linear");
      look_at(word, x, "mvpa_gated_linear kernel");
    } else {
      check(api.silu_mul(g.const_data_ptr(), up.const_data_ptr(), g.stride(0), act.data_ptr(), act.stride(0), d.rows, (int32_t)g.size(1), dt,
                         stream_of(x)), "mvpa_silu_mul");
    }
    h = at::empty_like(x);  // (not a view of a matrix: the caller may change it in place)
    Tensor h2 = h.view({d.rows, d.E});
    at::addmm_out(h2, x2, act, wd.t());
    h2.addmm_(o, wc.t());
  }
  return wrap({h, xn, q, kv, g, up, rt, rc, o, lse, act});
  END_HANDLE_TH_ERRORS
}

// block_backward(dh, x, pos, chan, ln_w, wq, wkv, wpos, wchan, bias, wc, wg, wu, wd, xn, q, kv, g, up, rt, rc, o, lse, act, need, eps,
//   window, H, Hkv, D, status, gated) -> the thirteen gradients (None where the bit of `need` is clear), or None
PyObject* block_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 32)) return nullptr;
  const bool status = a[30] == Py_True, gated = a[31] == Py_True;
  Tensor in[24];
  for (int i = 0; i < 24; ++i) {
    if (gated && i == 18) continue;  // (no `up`)
    if (!THPVariable_CheckExact(a[i])) Py_RETURN_NONE;
    in[i] = THPVariable_Unpack(a[i]);
  }
  Dims d;
  if (watched() || !block_dims(in + 1, a + 27, d) || !ordinary(in[0]) || in[0].device() != in[1].device() ||
      in[0].scalar_type() != in[1].scalar_type() || in[0].sizes() != in[1].sizes())
    Py_RETURN_NONE;
  // (a saved-tensor hook may have brought anything back)
  const std::vector<int64_t> saved[10] = {{d.rows, d.E}, {d.rows, d.H * d.D}, {d.rows, 2 * d.KV}, {d.rows, d.I}, {d.rows, d.I},
                                          {d.Hkv, d.T, d.D}, {d.Hkv, d.C, d.D}, {d.rows, d.H * d.D}, {d.B * d.H, d.N}, {d.rows, d.I}};
  for (int i = 0; i < 10; ++i) {
    if (gated && (i == 3 || i == 4)) continue;
    if (!fits(in[14 + i], in[1], i == 8 ? at::kFloat : in[1].scalar_type(), saved[i])) Py_RETURN_NONE;
  }
  if (gated && (in[1].scalar_type() != at::kBFloat16 || !fits(in[17], in[1], at::kByte, {(int64_t)api.gated_saved_bytes(d.rows, (int32_t)d.I)})))
    Py_RETURN_NONE;
  const Tensor &x = in[1], &pos = in[2], &chan = in[3], &ln_w = in[4], &wq = in[5], &wkv = in[6], &wpos = in[7], &wchan = in[8],
               &bias = in[9], &wc = in[10], &wg = in[11], &wu = in[12], &wd = in[13], &xn = in[14], &q = in[15], &kv = in[16],
               &g = in[17], &up = in[18], &rt = in[19], &rc = in[20], &o = in[21], &lse = in[22], &act = in[23];
  const int64_t need = PyLong_AsLongLong(a[24]), window = PyLong_AsLongLong(a[26]);
  const double eps = PyFloat_AsDouble(a[25]);
  if (PyErr_Occurred()) return nullptr;
  std::vector<Tensor> grad(13);
  {
    const Body body(x);
    const int dt = dtype_code(x);
    const auto needs = [&](int i) { return (need >> i & 1) != 0; };
    const auto weight = [&](int i, const Tensor& dy, const Tensor& y) {  // d W = d^T input
      if (needs(i)) grad[i] = at::mm(dy.t(), y);
    };
    const Tensor dh = in[0].contiguous(), dh2 = dh.view({d.rows, d.E});
    weight(9, dh2, o);
    weight(12, dh2, act);
    const Tensor dact = at::mm(dh2, wd);
    const Tensor dg = at::empty({d.rows, d.I}, xn.options().requires_grad(false)), dup = at::empty_like(dg);
    Tensor dxn;  // of the normalised input
    if (gated) {
      if (needs(0) || needs(3)) dxn = at::empty_like(xn);
      Tensor dwg, dwu;
      if (needs(10) || needs(11)) {
        dwg = at::empty_like(wg);
        dwu = at::empty_like(wu);
      }
      const auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
      const Tensor word = status_word(status, x);
      const size_t bytes = api.gated_bwd_bytes(d.rows, (int32_t)d.E, (int32_t)d.I);
      const Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte).requires_grad(false)) : Tensor();
      check(api.gated_linear_bwd(dact.const_data_ptr(), d.I, g.const_data_ptr(), xn.const_data_ptr(), d.E, wg.const_data_ptr(), wu.const_data_ptr(),
                                 dg.data_ptr(), dup.data_ptr(), ptr(dxn), ptr(dwg), ptr(dwu), d.rows, (int32_t)d.E, (int32_t)d.I, ptr(ws),
                                 bytes, word_of(word), stream_of(x)), "mvpa_gated_linear_bwd");
      look_at(word, x, "mvpa_gated_linear_bwd kernel");
      if (needs(10)) grad[10] = dwg;
      if (needs(11)) grad[11] = dwu;
    } else {
      check(api.silu_mul_bwd(g.const_data_ptr(), up.const_data_ptr(), g.stride(0), dact.const_data_ptr(), dact.stride(0), dg.data_ptr(),
                             dup.data_ptr(), g.size(1), d.rows, (int32_t)g.size(1), dt, stream_of(x)), "mvpa_silu_mul_bwd");
    }
    const Tensor d_o = at::mm(dh2, wc), dq = at::empty_like(q), dkv = at::empty_like(kv);
    const auto q4 = [&](const Tensor& t) { return columns(t, 0, d.N, d.D); };
    const auto v4 = [&](const Tensor& t) { return columns(t, d.KV, d.N, d.D); };
    const Tensor small = launch_bwd(d.problem(dt, 1.0 / std::sqrt((double)d.D), (int)window), q4(q), q4(kv), v4(kv), part(bias, 0),
                                    part(bias, d.KV), part(bias, 2 * d.KV), rt, rc, q4(o), lse, q4(d_o), q4(dq), q4(dkv), v4(dkv), status);
    if (needs(8)) grad[8] = small.narrow(0, 0, 3 * d.KV).view(bias.sizes());
    const auto keys = [&](int64_t at, int64_t rows, const Tensor& e, int i_e, const Tensor& w, int i_w) {
      const Tensor dk = small.narrow(0, at, rows * d.KV).view({d.Hkv, rows, d.D}).transpose(0, 1).reshape({rows, d.KV});
      weight(i_w, dk, e.select(0, 0));
      if (needs(i_e)) grad[i_e] = at::mm(dk, w).view(e.sizes());
    };
    keys(3 * d.KV, d.T, pos, 1, wpos, 6);
    keys(3 * d.KV + d.T * d.KV, d.C, chan, 2, wchan, 7);
    weight(4, dq, xn);
    weight(5, dkv, xn);
    if (!gated) {
      weight(10, dg, xn);
      weight(11, dup, xn);
    }
    if (needs(0) || needs(3)) {
      if (gated) dxn.addmm_(dq, wq);
      else dxn = at::mm(dq, wq);
      dxn.addmm_(dkv, wkv);
      if (!gated) {
        dxn.addmm_(dg, wg);
        dxn.addmm_(dup, wu);
      }
      grad[0] = at::empty(x.sizes(), x.options().requires_grad(false));
      grad[3] = at::empty_like(ln_w);
      const size_t bytes = api.rmsnorm_bwd_bytes(d.rows, (int32_t)d.E);
      const Tensor ws = scratch(bytes, x);
      check(api.rmsnorm_bwd(x.const_data_ptr(), ln_w.const_data_ptr(), dxn.const_data_ptr(), dh2.const_data_ptr(), grad[0].data_ptr(),
                            grad[3].data_ptr(), d.rows, (int32_t)d.E, (float)eps, dt, ws.data_ptr(), bytes, stream_of(x)), "mvpa_rmsnorm_bwd");
    }
  }
  return wrap(std::move(grad));
  END_HANDLE_TH_ERRORS
}

// branches(x, w_in, w_out, bias, r_time, r_chan, window, B, T, C, H, Hkv, D, status[, gated]): MLP(x) + Attn(x) of the fused inference block
//   (`MVPFormerBlock.fused_branches`), or None.  `gated` (bf16): the gate's projections and the gate as one kernel.
PyObject* branches(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14 && !arguments(n, 15)) return nullptr;
  const bool status = a[13] == Py_True, gated = n > 14 && a[14] == Py_True;
  Tensor in[6];
  for (int i = 0; i < 6; ++i) {
    if (!THPVariable_CheckExact(a[i])) Py_RETURN_NONE;
    in[i] = THPVariable_Unpack(a[i]);
    if (!ordinary(in[i]) || !in[i].is_contiguous() || in[i].device() != in[0].device() || in[i].scalar_type() != in[0].scalar_type() ||
        in[i].numel() == 0 || !aligned16(in[i].const_data_ptr()))
      Py_RETURN_NONE;
  }
  const Tensor &x = in[0], &w_in = in[1], &w_out = in[2], &bias = in[3], &rt = in[4], &rc = in[5];
  int64_t v[7];
  for (int i = 0; i < 7; ++i) v[i] = PyLong_AsLongLong(a[6 + i]);
  if (PyErr_Occurred()) return nullptr;
  Dims d;
  d.B = v[1]; d.T = v[2]; d.C = v[3]; d.H = v[4]; d.Hkv = v[5]; d.D = v[6];
  d.N = d.T * d.C; d.KV = d.Hkv * d.D; d.rows = d.B * d.N; d.E = d.H * d.D;
  const int dt = dtype_code(x);
  const int64_t I = x.dim() == 2 && w_in.dim() == 2 ? (w_in.size(0) - d.E - 2 * d.KV) / 2 : 0, es = x.element_size();
  if (I <= 0 || w_in.size(0) != d.E + 2 * (d.KV + I) || w_out.dim() != 2 || w_out.size(1) != d.E + I || d.KV <= 0 || d.rows <= 0 ||
      (dt != MVPA_BF16 && dt != MVPA_F32) || x.size(0) != d.rows || x.size(1) != d.E || I * es % 16 != 0 || bias.numel() != 3 * d.KV ||
      d.D * es % 16 != 0 || rt.numel() != d.T * d.KV || rc.numel() != d.C * d.KV || rt.size(-2) != d.T || rc.size(-2) != d.C ||
      function_modes() || watched())
    Py_RETURN_NONE;
  Tensor out;
  {
    pybind11::gil_scoped_release nogil;
    c10::cuda::CUDAGuard guard(x.device());
    c10::NoGradGuard no_grad;
    const int64_t g0 = d.E + 2 * d.KV;
    const bool one = gated && dt == MVPA_BF16 && d.E % 8 == 0 && I % 8 == 0 && !at::autocast::is_autocast_enabled(at::kCUDA);
    const Tensor big = at::linear(x, one ? w_in.narrow(0, 0, g0) : w_in);  // (rows, E + 2 KV (+ 2 I))
    if (big.scalar_type() == x.scalar_type()) {  // (autocast may have formed it in another type: Python's path follows that)
      const Tensor cat = at::empty({d.rows, d.E + I}, x.options().requires_grad(false));
      launch_fwd(d.problem(dt, 1.0 / std::sqrt((double)d.D), (int)v[0]), columns(big, 0, d.N, d.D), columns(big, d.E, d.N, d.D),
                 columns(big, d.E + d.KV, d.N, d.D), part(bias, 0), part(bias, d.KV), part(bias, 2 * d.KV), rt, rc,
                 columns(cat, 0, d.N, d.D), nullptr, status);
      if (one) {
        const Tensor word = status_word(status, x);
        check(api.gated_linear(x.const_data_ptr(), d.E, part(w_in, g0 * d.E), part(w_in, (g0 + I) * d.E), const_cast<char*>(part(cat, d.E)),
                               cat.stride(0), nullptr, d.rows, (int32_t)d.E, (int32_t)I, word_of(word), stream_of(x)), "mvpa_gated_linear");
        look_at(word, x, "mvpa_gated_linear kernel");
      } else {
        check(api.silu_mul(part(big, g0), part(big, g0 + I), big.stride(0), const_cast<char*>(part(cat, d.E)), cat.stride(0), d.rows, (int32_t)I,
                           dt, stream_of(x)), "mvpa_silu_mul");
      }
      out = at::linear(cat, w_out);
    }
  }
  if (!out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- the block in 8 bits (`mvpa_ops.quantize_fp8` and its neighbours): ordinary calls; anything else is answered None, and the Python
// ---- path serves or refuses it ----

constexpr int64_t kFp8Block = 128;
int64_t blocks_of(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

// Tensors on one device that nothing watches and no gradient has to flow through.
bool fp8_inputs(std::initializer_list<const Tensor*> ts) {
  const Tensor& t0 = **ts.begin();
  const bool grad = c10::GradMode::is_enabled();
  for (const Tensor* t : ts)
    if (t->defined() && (!ordinary(*t) || t->device() != t0.device() || (grad && t->requires_grad()))) return false;
  return !function_modes() && !watched();
}
// A matrix with at least one element, unit inner stride and rows that do not overlap; -> its leading dimension, or 0.
int64_t matrix_ld(const Tensor& t) {
  if (t.dim() != 2 || t.numel() == 0 || (t.stride(1) != 1 && t.size(1) > 1)) return 0;
  if (t.size(0) < 2) return (t.size(1) + 15) / 16 * 16;
  return t.stride(0) < t.size(1) ? 0 : t.stride(0);
}
bool bf16_or_fp32(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

// A new tensor beside `like`.  (The operators' calls are a few microseconds long, and the dispatcher's way to the same two
// functions is a third of one for each tensor.)
Tensor fresh(at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_strided_cuda(sizes, strides, type, like.device()));
}

// What an operator writes: the caller's pair, or a new one.
struct Pair {
  Tensor q, scales;
  int64_t ld = 0, ld_s = 0;
  // Whether the caller's tensors (undefined: none) are a pair of these sizes.
  bool fits(int64_t rows, int64_t width, int64_t tall) {
    if (!q.defined() || !scales.defined()) return q.defined() == scales.defined();
    ld = matrix_ld(q);
    ld_s = matrix_ld(scales);
    return q.scalar_type() == at::kFloat8_e4m3fn && scales.scalar_type() == at::kFloat8_e8m0fnu && ld != 0 && ld_s != 0 &&
           q.sizes() == at::IntArrayRef({rows, width}) && scales.sizes() == at::IntArrayRef({(rows + tall - 1) / tall, blocks_of(width)});
  }
  void make(int64_t rows, int64_t width, int64_t tall, const Tensor& like) {
    if (q.defined()) return;
    ld = (width + 15) / 16 * 16;
    ld_s = blocks_of(width);
    q = fresh({rows, width}, {ld, 1}, at::kFloat8_e4m3fn, like);
    scales = fresh({(rows + tall - 1) / tall, ld_s}, {ld_s, 1}, at::kFloat8_e8m0fnu, like);
  }
};

bool take(PyObject* a, Tensor& t) {  // (None leaves the tensor undefined)
  if (a == Py_None) return true;
  if (!THPVariable_CheckExact(a)) return false;
  t = THPVariable_Unpack(a);
  return true;
}

// quantize_fp8(x, block_rows, q or None, scales or None) -> (q, scales) or None
PyObject* quantize_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 4)) return nullptr;
  Tensor x;
  Pair out;
  if (a[0] == Py_None || !take(a[0], x) || !PyLong_CheckExact(a[1]) || !take(a[2], out.q) || !take(a[3], out.scales)) Py_RETURN_NONE;
  const int64_t tall = PyLong_AsLongLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  if ((tall != 1 && tall != kFp8Block) || !fp8_inputs({&x, &out.q, &out.scales}) || !bf16_or_fp32(x)) Py_RETURN_NONE;
  const int64_t ld = matrix_ld(x);
  if (ld == 0 || x.size(1) > INT32_MAX || !out.fits(x.size(0), x.size(1), tall)) Py_RETURN_NONE;
  std::optional<Body> body(std::in_place, x);
  out.make(x.size(0), x.size(1), tall, x);
  check(api.quantize_fp8(x.const_data_ptr(), ld, out.q.data_ptr(), out.ld, out.scales.data_ptr(), out.ld_s, x.size(0),
                         (int32_t)x.size(1), (int32_t)tall, dtype_code(x), stream_of(x)), "mvpa_quantize_fp8");
  body.reset();  // (the interpreter is wanted again)
  return wrap({std::move(out.q), std::move(out.scales)});
  END_HANDLE_TH_ERRORS
}

// rmsnorm_fp8(x, weight, eps, add or None, sum_out or None, q or None, scales or None) -> (q, scales) or None
PyObject* rmsnorm_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 7)) return nullptr;
  Tensor x, w, add, sum;
  Pair out;
  if (a[0] == Py_None || a[1] == Py_None || !take(a[0], x) || !take(a[1], w) || !PyFloat_Check(a[2]) || !take(a[3], add) || !take(a[4], sum) ||
      !take(a[5], out.q) || !take(a[6], out.scales))
    Py_RETURN_NONE;
  if (!fp8_inputs({&x, &w, &add, &sum, &out.q, &out.scales}) || !bf16_or_fp32(x) || x.dim() < 1 || x.numel() == 0) Py_RETURN_NONE;
  const int64_t E = x.size(-1);
  for (const Tensor* t : {&x, &w, &add, &sum})
    if (t->defined() && (!t->is_contiguous() || t->scalar_type() != x.scalar_type())) Py_RETURN_NONE;
  for (const Tensor* t : {&add, &sum})
    if (t->defined() && (t->numel() != x.numel() || t->dim() < 1 || t->size(-1) != E)) Py_RETURN_NONE;
  if (w.dim() != 1 || w.size(0) != E || E > 4096 || !out.fits(x.numel() / E, E, 1)) Py_RETURN_NONE;
  std::optional<Body> body(std::in_place, x);
  out.make(x.numel() / E, E, 1, x);
  check(api.rmsnorm_fp8(x.const_data_ptr(), add.defined() ? add.const_data_ptr() : nullptr, w.const_data_ptr(),
                        sum.defined() ? sum.data_ptr() : nullptr, out.q.data_ptr(), out.ld, out.scales.data_ptr(), out.ld_s,
                        x.numel() / E, (int32_t)E, (float)PyFloat_AS_DOUBLE(a[2]), dtype_code(x), stream_of(x)), "mvpa_rmsnorm_fp8");
  body.reset();  // (the interpreter is wanted again)
  return wrap({std::move(out.q), std::move(out.scales)});
  END_HANDLE_TH_ERRORS
}

// silu_mul_fp8(gate, up, q or None, scales or None) -> (q, scales) or None
PyObject* silu_mul_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 4)) return nullptr;
  Tensor g, u;
  Pair out;
  if (a[0] == Py_None || a[1] == Py_None || !take(a[0], g) || !take(a[1], u) || !take(a[2], out.q) || !take(a[3], out.scales) ||
      !fp8_inputs({&g, &u, &out.q, &out.scales}) || !bf16_or_fp32(g))
    Py_RETURN_NONE;
  const int64_t ld = matrix_ld(g);
  if (ld == 0 || matrix_ld(u) != ld || u.sizes() != g.sizes() || u.scalar_type() != g.scalar_type() || g.size(1) > INT32_MAX || !out.fits(g.size(0), g.size(1), 1))
    Py_RETURN_NONE;
  std::optional<Body> body(std::in_place, g);
  out.make(g.size(0), g.size(1), 1, g);
  check(api.silu_mul_fp8(g.const_data_ptr(), u.const_data_ptr(), ld, out.q.data_ptr(), out.ld, out.scales.data_ptr(), out.ld_s,
                         g.size(0), (int32_t)g.size(1), dtype_code(g), stream_of(g)), "mvpa_silu_mul_fp8");
  body.reset();  // (the interpreter is wanted again)
  return wrap({std::move(out.q), std::move(out.scales)});
  END_HANDLE_TH_ERRORS
}

// matmul_fp8(a, a_scales, b, b_scales, out or None, out is fp32, status) -> out or None
PyObject* matmul_fp8(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 7)) return nullptr;
  const bool status = p[6] == Py_True;
  Tensor a, sa, b, sb, out;
  if (p[0] == Py_None || p[1] == Py_None || p[2] == Py_None || p[3] == Py_None || !take(p[0], a) || !take(p[1], sa) || !take(p[2], b) ||
      !take(p[3], sb) || !take(p[4], out) || !fp8_inputs({&a, &sa, &b, &sb, &out}))
    Py_RETURN_NONE;
  const int64_t ld_a = matrix_ld(a), ld_b = matrix_ld(b);
  const bool exponents = sa.scalar_type() == at::kFloat8_e8m0fnu;
  if (ld_a == 0 || ld_b == 0 || a.scalar_type() != at::kFloat8_e4m3fn || b.scalar_type() != at::kFloat8_e4m3fn ||
      sa.scalar_type() != sb.scalar_type() || (!exponents && sa.scalar_type() != at::kFloat))
    Py_RETURN_NONE;
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0), KB = blocks_of(K);
  if (b.size(1) != K || sa.sizes() != at::IntArrayRef({M, KB}) || sb.sizes() != at::IntArrayRef({blocks_of(N), KB}) || N > INT32_MAX ||
      K > INT32_MAX || (out.defined() && (out.sizes() != at::IntArrayRef({M, N}) || !bf16_or_fp32(out) || matrix_ld(out) == 0)))
    Py_RETURN_NONE;
  {
    const Body body(a);
    if (!out.defined()) out = fresh({M, N}, {N, 1}, p[5] == Py_True ? at::kFloat : at::kBFloat16, a);
    const Tensor word = status ? at::zeros({64}, a.options().dtype(at::kInt).requires_grad(false)) : Tensor();
    int32_t* w = status ? word.data_ptr<int32_t>() : nullptr;
    check(api.matmul_fp8(a.const_data_ptr(), ld_a, sa.const_data_ptr(), sa.stride(0), sa.stride(1), b.const_data_ptr(), ld_b,
                         sb.const_data_ptr(), sb.stride(0), sb.stride(1), exponents ? MVPA_E8M0 : MVPA_F32, out.data_ptr(), matrix_ld(out),
                         M, (int32_t)N, (int32_t)K, dtype_code(out), w, stream_of(a)), "mvpa_matmul_fp8");
    if (status) check(api.fwd_status(w, 256, stream_of(a)), "mvpa_matmul_fp8 kernel");  // synchronises the stream
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// branches_fp8(q, scales, w_in q, w_in scales, w_out q, w_out scales, bias, r_time, r_chan, window, B, T, C, H, Hkv, D, status): the fused
//   inference block with its projections in 8 bits (`MVPFormerBlock.fused_branches_fp8`), in the type of `bias`; or None
PyObject* branches_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 17)) return nullptr;
  const bool status = a[16] == Py_True;
  Tensor in[9];
  for (int i = 0; i < 9; ++i)
    if (a[i] == Py_None || !take(a[i], in[i])) Py_RETURN_NONE;
  const Tensor &xq = in[0], &xs = in[1], &iq = in[2], &is = in[3], &oq = in[4], &os = in[5], &bias = in[6], &rt = in[7], &rc = in[8];
  if (!fp8_inputs({&xq, &xs, &iq, &is, &oq, &os, &bias, &rt, &rc})) Py_RETURN_NONE;
  int64_t v[7];
  for (int i = 0; i < 7; ++i) v[i] = PyLong_AsLongLong(a[9 + i]);
  if (PyErr_Occurred()) return nullptr;
  Dims d;
  d.B = v[1]; d.T = v[2]; d.C = v[3]; d.H = v[4]; d.Hkv = v[5]; d.D = v[6];
  d.N = d.T * d.C; d.KV = d.Hkv * d.D; d.rows = d.B * d.N; d.E = d.H * d.D;
  const int64_t ld_x = matrix_ld(xq), ld_i = matrix_ld(iq), ld_o = matrix_ld(oq);
  const int64_t I = iq.dim() == 2 ? (iq.size(0) - d.E - 2 * d.KV) / 2 : 0, es = bias.element_size(), K = d.E + I, kb = blocks_of(K);
  const auto pair_of = [](const Tensor& q, const Tensor& s, int64_t rows, int64_t width, int64_t tall) {
    return q.scalar_type() == at::kFloat8_e4m3fn && s.scalar_type() == at::kFloat8_e8m0fnu && q.sizes() == at::IntArrayRef({rows, width}) &&
           s.sizes() == at::IntArrayRef({(rows + tall - 1) / tall, blocks_of(width)});
  };
  if (I <= 0 || d.KV <= 0 || d.rows <= 0 || ld_x == 0 || ld_i == 0 || ld_o == 0 || d.E % kFp8Block != 0 || !bf16_or_fp32(bias) ||
      d.E + 2 * (d.KV + I) > INT32_MAX || !pair_of(xq, xs, d.rows, d.E, 1) || !pair_of(iq, is, d.E + 2 * (d.KV + I), d.E, kFp8Block) ||
      !pair_of(oq, os, d.E, K, kFp8Block) || bias.numel() != 3 * d.KV || d.D * es % 16 != 0 || rt.numel() != d.T * d.KV ||
      rc.numel() != d.C * d.KV || rt.dim() < 2 || rc.dim() < 2 || rt.size(-2) != d.T || rc.size(-2) != d.C)
    Py_RETURN_NONE;
  // (the attention reads q, k and v in place: the product's rows have to start on 16-byte boundaries)
  if ((d.E + 2 * (d.KV + I)) * es % 16 != 0) Py_RETURN_NONE;
  for (const Tensor* t : {&bias, &rt, &rc})
    if (!t->is_contiguous() || t->scalar_type() != bias.scalar_type() || !aligned16(t->const_data_ptr())) Py_RETURN_NONE;
  Tensor out;
  {
    const Body body(xq);
    const Tensor word = status ? at::zeros({64}, bias.options().dtype(at::kInt).requires_grad(false)) : Tensor();
    int32_t* w = status ? word.data_ptr<int32_t>() : nullptr;
    const int dt = dtype_code(bias);
    const auto product = [&](const Tensor& a, int64_t ld_a, const Tensor& sa, const Tensor& b, int64_t ld_b, const Tensor& sb) {
      Tensor o = fresh({a.size(0), b.size(0)}, {b.size(0), 1}, bias.scalar_type(), bias);
      check(api.matmul_fp8(a.const_data_ptr(), ld_a, sa.const_data_ptr(), sa.stride(0), sa.stride(1), b.const_data_ptr(), ld_b,
                           sb.const_data_ptr(), sb.stride(0), sb.stride(1), MVPA_E8M0, o.data_ptr(), o.size(1), a.size(0), (int32_t)b.size(0),
                           (int32_t)a.size(1), dt, w, stream_of(a)), "mvpa_matmul_fp8");
      return o;
    };
    const Tensor big = product(xq, ld_x, xs, iq, ld_i, is);  // (rows, E + 2 KV + 2 I)
    const Tensor att = fresh({d.rows, d.E}, {d.E, 1}, bias.scalar_type(), bias);
    launch_fwd(d.problem(dt, 1.0 / std::sqrt((double)d.D), (int)v[0]), columns(big, 0, d.N, d.D), columns(big, d.E, d.N, d.D),
               columns(big, d.E + d.KV, d.N, d.D), part(bias, 0), part(bias, d.KV), part(bias, 2 * d.KV), rt, rc, columns(att, 0, d.N, d.D),
               nullptr, status);
    const int64_t ld = (K + 15) / 16 * 16, g0 = d.E + 2 * d.KV;
    const Tensor q = fresh({d.rows, K}, {ld, 1}, at::kFloat8_e4m3fn, bias), scales = fresh({d.rows, kb}, {kb, 1}, at::kFloat8_e8m0fnu, bias);
    uint8_t *qp = static_cast<uint8_t*>(q.data_ptr()), *sp = static_cast<uint8_t*>(scales.data_ptr());
    check(api.quantize_fp8(att.const_data_ptr(), d.E, qp, ld, sp, kb, d.rows, (int32_t)d.E, 1, dt, stream_of(xq)), "mvpa_quantize_fp8");
    check(api.silu_mul_fp8(part(big, g0), part(big, g0 + I), big.stride(0), qp + d.E, ld, sp + d.E / kFp8Block, kb, d.rows, (int32_t)I, dt,
                           stream_of(xq)), "mvpa_silu_mul_fp8");
    out = product(q, ld, scales, oq, ld_o, os);
    if (status) check(api.fwd_status(w, 256, stream_of(xq)), "mvpa_matmul_fp8 kernel");  // synchronises the stream
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- the gated projection (`mvpa_ops.gated_linear`) ----

// x (..., E), w_gate and w_up (I, E) as the kernels read them: bf16, contiguous, 16-byte aligned, E and I multiples of 8, not empty.
struct Gated {
  Tensor x, wg, wu;
  int64_t rows, E, I;
  bool take(PyObject* const* a) {
    for (int i = 0; i < 3; ++i)
      if (!THPVariable_CheckExact(a[i])) return false;
    x = THPVariable_Unpack(a[0]);
    wg = THPVariable_Unpack(a[1]);
    wu = THPVariable_Unpack(a[2]);
    if (!ordinary(x) || x.scalar_type() != at::kBFloat16 || x.dim() < 2 || x.numel() == 0 || !ordinary(wg) || wg.dim() != 2 || function_modes() ||
        watched())
      return false;
    E = x.size(-1);
    I = wg.size(0);
    rows = x.numel() / E;
    constexpr int64_t kMost = INT32_MAX - 1024;
    return E % 8 == 0 && I % 8 == 0 && I > 0 && E <= kMost && I <= kMost && rows <= kMost && fits(x, x, at::kBFloat16, x.sizes()) &&
           fits(wg, x, at::kBFloat16, {I, E}) && fits(wu, x, at::kBFloat16, {I, E});
  }
  Tensor like_x(int64_t width) const {  // (..., width)
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = width;
    return at::empty(sizes, x.options().requires_grad(false));
  }
  Tensor forward(Tensor* saved, bool status) const {
    Tensor h = like_x(I);
    if (saved) *saved = scratch(api.gated_saved_bytes(rows, (int32_t)I), x);
    const Tensor w = status_word(status, x);
    check(api.gated_linear(x.const_data_ptr(), E, wg.const_data_ptr(), wu.const_data_ptr(), h.data_ptr(), I, saved ? saved->data_ptr() : nullptr,
                           rows, (int32_t)E, (int32_t)I, word_of(w), stream_of(x)), "mvpa_gated_linear");
    look_at(w, x, "mvpa_gated_linear kernel");
    return h;
  }
};

// gated_linear(x, w_gate, w_up, status): a call that no gradient flows through -> h or None
PyObject* gated_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 4)) return nullptr;
  Gated g;
  if (!g.take(a) || at::autocast::is_autocast_enabled(at::kCUDA) ||
      (c10::GradMode::is_enabled() && (g.x.requires_grad() || g.wg.requires_grad() || g.wu.requires_grad())))
    Py_RETURN_NONE;
  Tensor h;
  {
    const Body body(g.x);
    h = g.forward(nullptr, a[3] == Py_True);
  }
  return THPVariable_Wrap(std::move(h));
  END_HANDLE_TH_ERRORS
}

// gated_forward(x, w_gate, w_up, save, status) -> (h, saved or None) or None
PyObject* gated_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 5)) return nullptr;
  Gated g;
  if (!g.take(a)) Py_RETURN_NONE;
  Tensor h, saved;
  {
    const Body body(g.x);
    h = g.forward(a[3] == Py_True ? &saved : nullptr, a[4] == Py_True);
  }
  return wrap({std::move(h), std::move(saved)});
  END_HANDLE_TH_ERRORS
}

// gated_backward(dh, x, w_gate, w_up, saved, need, status) -> the three gradients (None where the bit of `need` is clear), or None
PyObject* gated_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 7)) return nullptr;
  Gated g;
  if (!THPVariable_CheckExact(a[0]) || !THPVariable_CheckExact(a[4]) || !g.take(a + 1)) Py_RETURN_NONE;
  const Tensor &dh = THPVariable_Unpack(a[0]), &saved = THPVariable_Unpack(a[4]);
  std::vector<int64_t> sizes = g.x.sizes().vec();
  sizes.back() = g.I;
  if (!ordinary(dh) || dh.scalar_type() != at::kBFloat16 || dh.device() != g.x.device() || dh.sizes() != at::IntArrayRef(sizes) ||
      !fits(saved, g.x, at::kByte, {(int64_t)api.gated_saved_bytes(g.rows, (int32_t)g.I)}))
    Py_RETURN_NONE;
  const int64_t need = PyLong_AsLongLong(a[5]);
  if (PyErr_Occurred()) return nullptr;
  std::vector<Tensor> grad(3);
  {
    const Body body(g.x);
    const Tensor d = dh.is_contiguous() && aligned16(dh.const_data_ptr()) ? dh : dh.clone(at::MemoryFormat::Contiguous);
    const Tensor dg = at::empty({2, g.rows, g.I}, g.x.options().requires_grad(false)), w = status_word(a[6] == Py_True, g.x);
    if (need & 1) grad[0] = g.like_x(g.E);
    Tensor dwg, dwu;
    if (need & 6) {
      dwg = at::empty_like(g.wg);
      dwu = at::empty_like(g.wu);
    }
    const auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    const size_t bytes = api.gated_bwd_bytes(g.rows, (int32_t)g.E, (int32_t)g.I);
    const Tensor ws = bytes ? at::empty({(int64_t)bytes}, g.x.options().dtype(at::kByte).requires_grad(false)) : Tensor();
    check(api.gated_linear_bwd(d.const_data_ptr(), g.I, saved.const_data_ptr(), g.x.const_data_ptr(), g.E, g.wg.const_data_ptr(),
                               g.wu.const_data_ptr(), dg.data_ptr(), const_cast<char*>(part(dg, g.rows * g.I)), ptr(grad[0]), ptr(dwg), ptr(dwu),
                               g.rows, (int32_t)g.E, (int32_t)g.I, ptr(ws), bytes, word_of(w), stream_of(g.x)),
          "mvpa_gated_linear_bwd");
    look_at(w, g.x, "mvpa_gated_linear_bwd kernel");
    if (need & 2) grad[1] = std::move(dwg);
    if (need & 4) grad[2] = std::move(dwu);
  }
  return wrap(std::move(grad));
  END_HANDLE_TH_ERRORS
}

// ---- weights in 4 bits (`mvpa_ops.quantize_int4` and its neighbours): as for 8 bits ----

// (q, scales, zeros or None) of N rows of K values.
struct Int4 {
  Tensor q, scales, zeros;
  mvpa_int4 c = {};
  bool take(PyObject* const* a) { return a[0] != Py_None && a[1] != Py_None && take_(a[0], q) && take_(a[1], scales) && take_(a[2], zeros); }
  bool fits(int64_t N, int64_t K, int64_t group) {
    const int64_t groups = (K + group - 1) / group;
    if (q.scalar_type() != at::kByte || !bf16_or_fp32(scales) || q.sizes() != at::IntArrayRef({N, (K + 1) / 2}) ||
        scales.sizes() != at::IntArrayRef({N, groups}))
      return false;
    c.ld_q = matrix_ld(q);
    c.ld_s = matrix_ld(scales);
    if (zeros.defined()) {
      if (zeros.scalar_type() != at::kByte || zeros.sizes() != at::IntArrayRef({N, groups})) return false;
      c.ld_z = matrix_ld(zeros);
      if (c.ld_z == 0) return false;
    }
    c.q = q.const_data_ptr();
    c.scales = scales.const_data_ptr();
    c.zeros = zeros.defined() ? zeros.const_data_ptr() : nullptr;
    return c.ld_q != 0 && c.ld_s != 0;
  }

 private:
  static bool take_(PyObject* a, Tensor& t) {  // (None leaves the tensor undefined)
    if (a == Py_None) return true;
    if (!THPVariable_CheckExact(a)) return false;
    t = THPVariable_Unpack(a);
    return true;
  }
};
bool group_of(PyObject* a, int64_t* group) {
  if (!PyLong_CheckExact(a)) return false;
  int overflow = 0;
  *group = PyLong_AsLongLongAndOverflow(a, &overflow);
  return *group == 32 || *group == 64 || *group == 128;
}

// quantize_int4(w, group, zeros) -> (q, scales[, zeros]) or None
PyObject* quantize_int4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 3)) return nullptr;
  Tensor w;
  int64_t group;
  if (a[0] == Py_None || !take(a[0], w) || !group_of(a[1], &group) || (a[2] != Py_True && a[2] != Py_False) || !fp8_inputs({&w}) ||
      !bf16_or_fp32(w))
    Py_RETURN_NONE;
  const int64_t ld = matrix_ld(w);
  if (ld == 0 || w.size(1) > INT32_MAX - 1024) Py_RETURN_NONE;
  const int64_t N = w.size(0), K = w.size(1), groups = (K + group - 1) / group, half = (K + 1) / 2, ld_q = (half + 15) / 16 * 16;
  Tensor q, scales, zeros;
  {
    const Body body(w);
    q = fresh({N, half}, {ld_q, 1}, at::kByte, w);
    scales = fresh({N, groups}, {groups, 1}, w.scalar_type(), w);
    if (a[2] == Py_True) zeros = fresh({N, groups}, {groups, 1}, at::kByte, w);
    const mvpa_int4 to = {q.data_ptr(), scales.data_ptr(), zeros.defined() ? zeros.data_ptr() : nullptr, ld_q, groups, groups};
    check(api.quantize_int4(w.const_data_ptr(), ld, &to, N, (int32_t)K, (int32_t)group, dtype_code(w), stream_of(w)), "mvpa_quantize_int4");
  }
  if (zeros.defined()) return wrap({std::move(q), std::move(scales), std::move(zeros)});
  return wrap({std::move(q), std::move(scales)});
  END_HANDLE_TH_ERRORS
}

// dequantize_int4(q, scales, zeros or None, width, group, out is fp32) -> the values or None
PyObject* dequantize_int4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 6)) return nullptr;
  Int4 w;
  int64_t group;
  if (!w.take(a) || !PyLong_CheckExact(a[3]) || !group_of(a[4], &group) || !fp8_inputs({&w.q, &w.scales, &w.zeros})) Py_RETURN_NONE;
  int overflow = 0;
  const int64_t K = PyLong_AsLongLongAndOverflow(a[3], &overflow);
  if (overflow || K <= 0 || K > INT32_MAX - 1024 || w.q.dim() != 2 || !w.fits(w.q.size(0), K, group)) Py_RETURN_NONE;
  Tensor out;
  {
    const Body body(w.q);
    out = fresh({w.q.size(0), K}, {K, 1}, a[5] == Py_True ? at::kFloat : at::kBFloat16, w.q);
    check(api.dequantize_int4(&w.c, dtype_code(w.scales), out.data_ptr(), K, w.q.size(0), (int32_t)K, (int32_t)group, dtype_code(out),
                              stream_of(w.q)), "mvpa_dequantize_int4");
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// matmul_int4(x, q, scales, zeros or None, and the same three of the second weight of a gate, or None three times, group, out or None,
//   status) -> out or None
PyObject* matmul_int4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 10)) return nullptr;
  const bool status = a[9] == Py_True, two = a[4] != Py_None;
  Tensor x, out;
  Int4 w, up;
  int64_t group;
  if (a[0] == Py_None || !take(a[0], x) || !w.take(a + 1) || (two && !up.take(a + 4)) || !group_of(a[7], &group) || !take(a[8], out) ||
      !fp8_inputs({&x, &w.q, &w.scales, &w.zeros, &up.q, &up.scales, &up.zeros, &out}) || !bf16_or_fp32(x) || x.dim() < 1 || x.numel() == 0 ||
      w.q.dim() != 2 || w.q.numel() == 0)
    Py_RETURN_NONE;
  const int64_t K = x.size(-1), M = x.numel() / K, N = w.q.size(0);
  int64_t ld = K;
  if (x.dim() == 2) ld = matrix_ld(x);
  else if (!x.is_contiguous()) ld = 0;
  if (ld == 0 || K > INT32_MAX - 1024 || !w.fits(N, K, group) || (two && (!up.fits(N, K, group) || up.scales.scalar_type() != w.scales.scalar_type())))
    Py_RETURN_NONE;
  if (out.defined() && (out.sizes() != at::IntArrayRef({M, N}) || out.scalar_type() != x.scalar_type() || matrix_ld(out) == 0)) Py_RETURN_NONE;
  {
    const Body body(x);
    const int dt = dtype_code(x);
    int64_t ld_out = N;
    if (out.defined()) {
      ld_out = matrix_ld(out);
    } else if (x.dim() == 2) {
      out = fresh({M, N}, {N, 1}, x.scalar_type(), x);
    } else {
      std::vector<int64_t> sizes = x.sizes().vec();
      sizes.back() = N;
      out = at::empty(sizes, x.options().requires_grad(false));
    }
    const size_t bytes = api.int4_workspace_bytes(x.const_data_ptr(), ld, M, (int32_t)K, dt);
    const Tensor ws = bytes ? fresh({(int64_t)bytes}, {1}, at::kByte, x) : Tensor();
    const Tensor word = status ? at::zeros({64}, x.options().dtype(at::kInt).requires_grad(false)) : Tensor();
    check(api.matmul_int4(x.const_data_ptr(), ld, &w.c, two ? &up.c : nullptr, dtype_code(w.scales), out.data_ptr(), ld_out, M, (int32_t)N,
                          (int32_t)K, (int32_t)group, dt, bytes ? ws.data_ptr() : nullptr, bytes, status ? word.data_ptr<int32_t>() : nullptr,
                          stream_of(x)), "mvpa_matmul_int4");
    if (status) check(api.fwd_status(word.data_ptr<int32_t>(), 256, stream_of(x)), "mvpa_matmul_int4 kernel");  // synchronises the stream
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// branches_int4(x, then (q, scales, zeros or None) of q k v, gate, up and the output, bias, r_time, r_chan, window, B, T, C, H, Hkv, D, group,
//   status): the fused inference block with its weights in 4 bits (`MVPFormerBlock.fused_branches_int4`), or None
PyObject* branches_int4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments(n, 25)) return nullptr;
  const bool status = a[24] == Py_True;
  Tensor x, bias, rt, rc;
  Int4 w[4];  // q k v, gate, up, out
  int64_t group, v[7];
  if (a[0] == Py_None || a[13] == Py_None || a[14] == Py_None || a[15] == Py_None || !take(a[0], x) || !take(a[13], bias) || !take(a[14], rt) ||
      !take(a[15], rc) || !group_of(a[23], &group))
    Py_RETURN_NONE;
  for (int i = 0; i < 4; ++i)
    if (!w[i].take(a + 1 + 3 * i) || !fp8_inputs({&x, &w[i].q, &w[i].scales, &w[i].zeros})) Py_RETURN_NONE;
  if (!fp8_inputs({&x, &bias, &rt, &rc}) || !bf16_or_fp32(x) || x.dim() != 2 || x.numel() == 0 || !x.is_contiguous()) Py_RETURN_NONE;
  for (int i = 0; i < 7; ++i) v[i] = PyLong_AsLongLong(a[16 + i]);
  if (PyErr_Occurred()) return nullptr;
  Dims d;
  d.B = v[1]; d.T = v[2]; d.C = v[3]; d.H = v[4]; d.Hkv = v[5]; d.D = v[6];
  d.N = d.T * d.C; d.KV = d.Hkv * d.D; d.rows = d.B * d.N; d.E = d.H * d.D;
  const int64_t I = w[1].q.dim() == 2 ? w[1].q.size(0) : 0, es = x.element_size(), K = d.E + I, Q = d.E + 2 * d.KV;
  if (I <= 0 || d.KV <= 0 || d.rows <= 0 || x.size(0) != d.rows || x.size(1) != d.E || K > INT32_MAX - 1024 || !w[0].fits(Q, d.E, group) ||
      !w[1].fits(I, d.E, group) || !w[2].fits(I, d.E, group) || !w[3].fits(d.E, K, group) || bias.numel() != 3 * d.KV || d.D * es % 16 != 0 ||
      Q * es % 16 != 0 || rt.numel() != d.T * d.KV || rc.numel() != d.C * d.KV || rt.dim() < 2 || rc.dim() < 2 ||
      rt.size(-2) != d.T || rc.size(-2) != d.C || w[2].scales.scalar_type() != w[1].scales.scalar_type())
    Py_RETURN_NONE;
  for (const Tensor* t : {&bias, &rt, &rc})
    if (!t->is_contiguous() || t->scalar_type() != x.scalar_type() || !aligned16(t->const_data_ptr())) Py_RETURN_NONE;
  Tensor out;
  {
    const Body body(x);
    const int dt = dtype_code(x);
    const Tensor word = status_word(status, x);
    const auto product = [&](const Tensor& a, const Int4& w, const Int4* up, void* to, int64_t ld) {
      const int64_t K = a.size(1);
      const size_t bytes = api.int4_workspace_bytes(a.const_data_ptr(), a.stride(0), d.rows, (int32_t)K, dt);
      const Tensor ws = bytes ? fresh({(int64_t)bytes}, {1}, at::kByte, x) : Tensor();
      check(api.matmul_int4(a.const_data_ptr(), a.stride(0), &w.c, up ? &up->c : nullptr, dtype_code(w.scales), to, ld, d.rows,
                            (int32_t)w.q.size(0), (int32_t)K, (int32_t)group, dt, bytes ? ws.data_ptr() : nullptr, bytes, word_of(word),
                            stream_of(x)), "mvpa_matmul_int4");
    };
    const int64_t ld = (K + 7) / 8 * 8;  // (the attention writes 16-byte aligned rows)
    const Tensor big = fresh({d.rows, Q}, {Q, 1}, x.scalar_type(), x), cat = fresh({d.rows, K}, {ld, 1}, x.scalar_type(), x);
    product(x, w[0], nullptr, big.data_ptr(), Q);
    launch_fwd(d.problem(dt, 1.0 / std::sqrt((double)d.D), (int)v[0]), columns(big, 0, d.N, d.D), columns(big, d.E, d.N, d.D),
               columns(big, d.E + d.KV, d.N, d.D), part(bias, 0), part(bias, d.KV), part(bias, 2 * d.KV), rt, rc, columns(cat, 0, d.N, d.D),
               nullptr, status);
    product(x, w[1], &w[2], const_cast<char*>(part(cat, d.E)), ld);
    out = fresh({d.rows, d.E}, {d.E, 1}, x.scalar_type(), x);
    product(cat, w[3], nullptr, out.data_ptr(), d.E);
    look_at(word, x, "mvpa_matmul_int4 kernel");
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// init(path of libmvpa_b200.so, which is already loaded; the class of the mode that a default device is)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 2)) return nullptr;
  const char* p = PyUnicode_AsUTF8(a[0]);
  if (!p) return nullptr;
  Py_INCREF(a[1]);
  device_mode = a[1];
  void* so = dlopen(p, RTLD_NOW);
  if (!so) { PyErr_SetString(PyExc_ImportError, dlerror()); return nullptr; }
  const char* missing = nullptr;
  const auto get = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(so, name));
    if (!f) missing = name;
  };
  get(api.fwd_bytes, "mvpa_fwd_workspace_bytes"); get(api.bwd_bytes, "mvpa_bwd_workspace_bytes");
  get(api.fwd, "mvpa_fwd"); get(api.bwd, "mvpa_bwd");
  get(api.rmsnorm, "mvpa_rmsnorm"); get(api.rmsnorm_bwd, "mvpa_rmsnorm_bwd");
  get(api.rmsnorm_bwd_bytes, "mvpa_rmsnorm_bwd_workspace_bytes");
  get(api.silu_mul, "mvpa_silu_mul"); get(api.silu_mul_bwd, "mvpa_silu_mul_bwd");
  get(api.fwd_status, "mvpa_workspace_status"); get(api.bwd_status, "mvpa_bwd_status");
  get(api.last_error, "mvpa_last_error_string");
  get(api.quantize_fp8, "mvpa_quantize_fp8"); get(api.rmsnorm_fp8, "mvpa_rmsnorm_fp8");
  get(api.silu_mul_fp8, "mvpa_silu_mul_fp8"); get(api.matmul_fp8, "mvpa_matmul_fp8");
  get(api.gated_linear, "mvpa_gated_linear"); get(api.gated_linear_bwd, "mvpa_gated_linear_bwd");
  get(api.gated_saved_bytes, "mvpa_gated_linear_saved_bytes"); get(api.gated_bwd_bytes, "mvpa_gated_linear_bwd_workspace_bytes");
  get(api.quantize_int4, "mvpa_quantize_int4"); get(api.dequantize_int4, "mvpa_dequantize_int4");
  get(api.matmul_int4, "mvpa_matmul_int4"); get(api.int4_workspace_bytes, "mvpa_matmul_int4_workspace_bytes");
  if (missing) { PyErr_Format(PyExc_ImportError, "%s has no %s", p, missing); return nullptr; }
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(init), FAST(attend), FAST(forward), FAST(backward), FAST(plain), FAST(block_forward),
                         FAST(block_backward), FAST(branches), FAST(quantize_fp8), FAST(rmsnorm_fp8), FAST(silu_mul_fp8),
                         FAST(matmul_fp8), FAST(branches_fp8), FAST(gated_linear), FAST(gated_forward), FAST(gated_backward),
                         FAST(quantize_int4), FAST(dequantize_int4), FAST(matmul_int4), FAST(branches_int4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "mvpa_host_b200", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_mvpa_host_b200() { return PyModule_Create(&module_def); }
