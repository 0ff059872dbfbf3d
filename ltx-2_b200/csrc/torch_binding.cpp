// Tensor-level calls of the residual-path and training operators (include/ltxfp8.h): argument
// checks, output and workspace allocation from torch's caching allocator, the launch on the
// current stream of the tensors' device.
//
// These operators are called per token step and per layer, where the host's time for a call
// matters: building four output tensors, the checks and a 16-argument ctypes call from Python
// take 17-28 us, most of it more than the kernel; here a call takes 5-13 us.  The functions
// take positional arguments only; the Python wrappers in ltx_kernels/blockwise/ops.py name
// and document them.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <string>

#include "ltxfp8.h"

namespace {

using at::Tensor;

PyObject* g_check = nullptr;  // ltx_kernels._lib.check: raises for a non-zero return code

// The caller's Python error for a failed C-ABI call.
struct AbiError {
  int code;
};

void abi(int rc) {
  if (rc != LTXFP8_OK) throw AbiError{rc};
}

// A Python tensor argument, or None where `optional`.
Tensor tensor_arg(const char* name, const char* what, PyObject* o, bool optional = false) {
  if (optional && o == Py_None) return Tensor();
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, ": ", what, " must be a tensor");
  return THPVariable_Unpack(o);
}

// CUDA tensors, all on one device.
c10::Device one_device(const char* name, std::initializer_list<const Tensor*> ts) {
  c10::optional<c10::Device> dev;
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), name, ": ltx-2_b200 kernels need CUDA (sm_100) tensors, got ", t->device());
    if (!dev)
      dev = t->device();
    else
      TORCH_CHECK(*dev == t->device(), name, ": all tensors must be on one device, got ", *dev, " and ", t->device());
  }
  return *dev;
}

bool misaligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0; }

// bf16 [..., K] as [M, K] with 16-byte aligned rows (a copy only where it has none).
struct Rows {
  Tensor t;  // keeps the copy, if one was made
  int64_t M = 0, K = 0, ld = 0;
  const void* ptr() const { return t.const_data_ptr(); }
};

Rows bf16_rows(const char* name, const char* what, const Tensor& x) {
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, name, ": ", what, ": expected bf16, got ", x.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, name, ": ", what, ": expected a [..., K] tensor, got shape ", x.sizes());
  Rows r;
  r.K = x.size(-1);
  r.t = x.dim() == 2 ? x : x.reshape({-1, r.K});
  r.M = r.t.size(0);
  r.ld = r.K;
  if (r.M > 0) {
    const bool strided = r.M > 1;
    if (r.t.stride(1) != 1 || misaligned(r.t) || (strided && (r.t.stride(0) % 8 != 0 || r.t.stride(0) < r.K)))
      r.t = r.t.clone(at::MemoryFormat::Contiguous);
    if (strided) r.ld = r.t.stride(0);
  }
  return r;
}

// Leading dimension of activation scales holding (m, kb) at [kb * ld + m]: the (M, KB)
// MN-major view the quantisers return, or a contiguous (KB, M) tensor.
int64_t scale_ld(const Tensor& s, int64_t M, int64_t KB) {
  TORCH_CHECK(s.scalar_type() == at::kFloat, "activation scales must be float32, got ", s.scalar_type());
  if (s.dim() == 2) {
    if (s.size(0) == M && s.size(1) == KB && (s.stride(0) == 1 || M == 1) && (KB == 1 || s.stride(1) >= M))
      return KB > 1 ? s.stride(1) : std::max<int64_t>(M, 1);
    if (s.size(0) == KB && s.size(1) == M && (s.stride(1) == 1 || M == 1) && (KB == 1 || s.stride(0) >= M))
      return KB > 1 ? s.stride(0) : std::max<int64_t>(M, 1);
  }
  TORCH_CHECK(false, "activation scales of shape ", s.sizes(), " strides ", s.strides(), " are not an MN-major (", M,
              ", ", KB, ") view or a contiguous (", KB, ", ", M, ") tensor");
}

// e4m3 codes [..., K] as a contiguous aligned [M, K] matrix with their scales.
struct Codes {
  Tensor q;
  const float* s = nullptr;
  int64_t M = 0, K = 0, ld = 1;
};

Codes code_rows(const char* name, const char* what, const Tensor& q, const Tensor& s) {
  TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn, name, ": ", what, ": codes must be float8_e4m3fn, got ",
              q.scalar_type());
  TORCH_CHECK(q.dim() >= 1 && q.size(-1) > 0 && q.size(-1) % 128 == 0, name, ": ", what,
              ": expected [..., K] codes with K a positive multiple of 128, got ", q.sizes());
  Codes c;
  c.K = q.size(-1);
  c.q = (q.dim() == 2 ? q : q.reshape({-1, c.K})).contiguous();
  if (misaligned(c.q)) c.q = c.q.clone();
  c.M = c.q.size(0);
  if (c.M > 0) {
    c.ld = scale_ld(s, c.M, c.K / 128);
    c.s = s.const_data_ptr<float>();
  }
  return c;
}

Tensor new_tensor(c10::Device dev, at::IntArrayRef sizes, at::ScalarType t) {
  return at::detail::empty_cuda(sizes, t, dev, c10::nullopt);
}

int64_t align4(int64_t n) { return (n + 3) / 4 * 4; }

// (M, KB) fp32 scales with strides (1, align4(M)), as blockwise::quantize returns.
Tensor new_scales(c10::Device dev, int64_t M, int64_t KB) {
  return at::detail::empty_strided_cuda({M, KB}, {1, align4(M)}, at::kFloat, dev);
}

Tensor new_workspace(c10::Device dev, size_t bytes) {
  return bytes ? new_tensor(dev, {static_cast<int64_t>(bytes)}, at::kByte) : Tensor();
}

void* data(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const void* cdata(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

PyObject* wrap_all(std::initializer_list<const Tensor*> ts) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor* t : ts) {
    PyObject* o = wrap(*t);
    if (!o) {
      Py_DECREF(out);
      throw python_error();
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

int activation_arg(const char* name, PyObject* o, bool allow_none) {
  if (o == Py_None && allow_none) return LTXFP8_ACT_NONE;
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "gelu_tanh") == 0) return LTXFP8_ACT_GELU_TANH;
    if (PyUnicode_CompareWithASCIIString(o, "silu") == 0) return LTXFP8_ACT_SILU;
  }
  PyObject* r = PyObject_Repr(o);
  const std::string got = r ? PyUnicode_AsUTF8(r) : "?";
  Py_XDECREF(r);
  TORCH_CHECK(false, name, ": activation must be ", allow_none ? "None, " : "", "'gelu_tanh' or 'silu', got ", got);
}

bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

double double_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

// The gain of a norm: contiguous, aligned fp32 or bf16 [H].
Tensor gain_arg(const char* name, const Tensor& w, int64_t H, int* dtype) {
  *dtype = LTXFP8_DTYPE_F32;
  if (!w.defined()) return w;
  const bool f32 = w.scalar_type() == at::kFloat;
  TORCH_CHECK((f32 || w.scalar_type() == at::kBFloat16) && w.dim() == 1 && w.size(0) == H, name,
              ": weight must be fp32 or bf16 [", H, "], got ", w.scalar_type(), " ", w.sizes());
  *dtype = f32 ? LTXFP8_DTYPE_F32 : LTXFP8_DTYPE_BF16;
  Tensor c = w.contiguous();
  return misaligned(c) ? c.clone() : c;
}

// (x, weight, residual, eps, quantize)
PyObject* rms_norm_quantize(PyObject* const* a) {
  const char* name = "rms_norm_quantize";
  const Tensor x = tensor_arg(name, "x", a[0]), weight = tensor_arg(name, "weight", a[1], true),
               residual = tensor_arg(name, "residual", a[2], true);
  const double eps = double_arg(a[3]);
  const bool quantize = bool_arg(a[4]);
  const c10::Device dev = one_device(name, {&x, &weight, &residual});
  const Rows xr = bf16_rows(name, "x", x);
  const int64_t M = xr.M, H = xr.K;
  Rows rr;
  Tensor h = xr.t, q, s, y;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  if (residual.defined()) {
    TORCH_CHECK(residual.sizes() == x.sizes(), name, ": residual must have x's shape ", x.sizes(), ", got ",
                residual.sizes());
    rr = bf16_rows(name, "residual", residual);
    h = new_tensor(dev, {M, H}, at::kBFloat16);
  }
  int wdt;
  const Tensor w = gain_arg(name, weight, H, &wdt);
  if (quantize) {
    q = new_tensor(dev, {M, H}, at::kFloat8_e4m3fn);
    s = new_scales(dev, M, H / 128);
  } else {
    y = new_tensor(dev, {M, H}, at::kBFloat16);
  }
  const Tensor rstd = new_tensor(dev, {M}, at::kFloat);
  abi(ltxfp8_rms_norm_quantize(xr.ptr(), xr.ld, cdata(rr.t), rr.ld, M, H, cdata(w), wdt, static_cast<float>(eps),
                               rr.t.defined() ? data(h) : nullptr, data(q), static_cast<float*>(data(s)), align4(M),
                               data(y), static_cast<float*>(data(rstd)), stream_of(dev)));
  return quantize ? wrap_all({&q, &s, &h, &rstd}) : wrap_all({&y, &h, &rstd});
}

// (dy, h, rstd, weight, dh)
PyObject* rms_norm_backward(PyObject* const* a) {
  const char* name = "rms_norm_backward";
  const Tensor dy = tensor_arg(name, "dy", a[0]), h = tensor_arg(name, "h", a[1]), rstd = tensor_arg(name, "rstd", a[2]),
               weight = tensor_arg(name, "weight", a[3], true), dh = tensor_arg(name, "dh", a[4], true);
  const c10::Device dev = one_device(name, {&dy, &h, &rstd, &weight, &dh});
  const Rows yr = bf16_rows(name, "dy", dy), hr = bf16_rows(name, "h", h);
  const int64_t M = yr.M, H = yr.K;
  TORCH_CHECK(hr.M == M && hr.K == H, name, ": h has ", hr.t.sizes(), " values, dy ", yr.t.sizes());
  TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.numel() == M, name, ": rstd must be fp32 [", M, "]");
  const Tensor rs = rstd.contiguous();
  Rows dr;
  if (dh.defined()) {
    dr = bf16_rows(name, "dh", dh);
    TORCH_CHECK(dr.M == M && dr.K == H, name, ": dh has ", dr.t.sizes(), " values, dy ", yr.t.sizes());
  }
  int wdt;
  const Tensor w = gain_arg(name, weight, H, &wdt);
  const c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor dx = new_tensor(dev, {M, H}, at::kBFloat16), dw, ws;
  size_t bytes = 0;
  if (w.defined()) {
    abi(ltxfp8_rms_norm_backward_workspace_bytes(M, H, &bytes));
    dw = new_tensor(dev, {H}, weight.scalar_type());
    ws = new_workspace(dev, bytes);
  }
  abi(ltxfp8_rms_norm_backward(yr.ptr(), yr.ld, hr.ptr(), hr.ld, static_cast<const float*>(cdata(rs)), cdata(w), wdt,
                               cdata(dr.t), dr.ld, M, H, data(dx), data(dw), data(ws), bytes, stream_of(dev)));
  if (dy.dim() != 2) dx = dx.view(dy.sizes());
  return wrap_all({&dx, &dw});
}

// (a_q, sfa, w_q, sfb, bias, residual, activation, out, split_k)
PyObject* gemm_residual(PyObject* const* a) {
  const char* name = "gemm_residual";
  const Tensor aq = tensor_arg(name, "a_q", a[0]), sfa = tensor_arg(name, "sfa", a[1]),
               wq = tensor_arg(name, "w_q", a[2]), sfb = tensor_arg(name, "sfb", a[3]),
               bias = tensor_arg(name, "bias", a[4], true), residual = tensor_arg(name, "residual", a[5], true);
  const Tensor given = tensor_arg(name, "out", a[7], true);
  const c10::Device dev = one_device(name, {&aq, &sfa, &wq, &sfb, &bias, &residual, &given});
  const int act = activation_arg(name, a[6], true);
  const bool split_k = bool_arg(a[8]);
  TORCH_CHECK(aq.dim() == 2 && wq.dim() == 2, name, " expects 2-D operands");
  const int64_t M = aq.size(0), K = aq.size(1), N = wq.size(0);
  TORCH_CHECK(wq.size(1) == K, name, ": K mismatch (", K, " vs ", wq.size(1), ")");
  TORCH_CHECK(aq.scalar_type() == at::kFloat8_e4m3fn && wq.scalar_type() == at::kFloat8_e4m3fn, name,
              ": operands must be float8_e4m3fn");
  TORCH_CHECK(aq.is_contiguous() && wq.is_contiguous(), name, ": operands must be contiguous (K-major)");
  const int64_t KB = K / 128;
  TORCH_CHECK(sfb.scalar_type() == at::kFloat && sfb.dim() == 2 && sfb.size(0) == N / 128 && sfb.size(1) == KB &&
                  sfb.is_contiguous(),
              name, ": weight scales must be contiguous fp32 [", N / 128, ", ", KB, "]");
  Tensor b = bias;
  if (b.defined()) {
    TORCH_CHECK(b.scalar_type() == at::kFloat && b.numel() == N, name, ": bias must be fp32 [", N, "]");
    b = b.contiguous();
    if (misaligned(b)) b = b.clone();
  }
  TORCH_CHECK(!residual.defined() || (residual.scalar_type() == at::kBFloat16 && residual.dim() == 2 &&
                                      residual.size(0) == M && residual.size(1) == N),
              name, ": residual must be bf16 [", M, ", ", N, "]");
  TORCH_CHECK(!given.defined() || (given.scalar_type() == at::kBFloat16 && given.dim() == 2 && given.size(0) == M &&
                                   given.size(1) == N && given.is_contiguous()),
              name, ": out must be a contiguous bf16 [", M, ", ", N, "] tensor");
  const c10::cuda::OptionalCUDAGuard guard(dev);
  Tensor out = given.defined() ? given : new_tensor(dev, {M, N}, at::kBFloat16);
  if (M > 0) {
    Rows rr;
    if (residual.defined()) rr = bf16_rows(name, "residual", residual);
    const int64_t ld = scale_ld(sfa, M, KB);
    size_t bytes = 0;
    if (split_k) abi(ltxfp8_gemm_workspace_bytes(M, N, K, &bytes));
    const Tensor ws = new_workspace(dev, bytes);
    abi(ltxfp8_gemm_residual(cdata(aq), static_cast<const float*>(cdata(sfa)), ld, cdata(wq),
                             static_cast<const float*>(cdata(sfb)), static_cast<const float*>(cdata(b)), cdata(rr.t),
                             rr.ld, data(out), M, N, K, act, data(ws), bytes, stream_of(dev)));
  }
  if (given.defined()) {
    Py_INCREF(a[7]);
    return a[7];
  }
  return wrap(out);
}

// (z, activation, save)
PyObject* act_quantize_save(PyObject* const* a) {
  const char* name = "act_quantize_save";
  const Tensor z = tensor_arg(name, "z", a[0]);
  const c10::Device dev = one_device(name, {&z});
  const int act = activation_arg(name, a[1], false);
  const bool save = bool_arg(a[2]);
  const Rows zr = bf16_rows(name, "z", z);
  const int64_t M = zr.M, N = zr.K;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const Tensor yq = new_tensor(dev, {M, N}, at::kFloat8_e4m3fn), ys = new_scales(dev, M, N / 128);
  Tensor zq, zs;
  if (save) {
    zq = new_tensor(dev, {M, N}, at::kFloat8_e4m3fn);
    zs = new_scales(dev, M, N / 128);
  }
  abi(ltxfp8_act_quantize_save(zr.ptr(), zr.ld, M, N, act, data(yq), static_cast<float*>(data(ys)), align4(M), data(zq),
                               static_cast<float*>(data(zs)), align4(M), stream_of(dev)));
  return wrap_all({&yq, &ys, &zq, &zs});
}

// (dy, z_q, z_scales, activation, quantize, dbias)
PyObject* act_backward(PyObject* const* a) {
  const char* name = "act_backward";
  const Tensor dy = tensor_arg(name, "dy", a[0]), zq = tensor_arg(name, "z_q", a[1]),
               zs = tensor_arg(name, "z_scales", a[2]);
  const c10::Device dev = one_device(name, {&dy, &zq, &zs});
  const int act = activation_arg(name, a[3], false);
  const bool quantize = bool_arg(a[4]), dbias = bool_arg(a[5]);
  const Rows yr = bf16_rows(name, "dy", dy);
  const Codes zc = code_rows(name, "z", zq, zs);
  const int64_t M = yr.M, N = yr.K;
  TORCH_CHECK(zc.M == M && zc.K == N, name, ": the checkpoint has ", zc.q.sizes(), " values, dy ", yr.t.sizes());
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const Tensor dz = new_tensor(dev, {M, N}, at::kBFloat16);
  Tensor dq, ds, db, ws;
  size_t bytes = 0;
  if (quantize) {
    dq = new_tensor(dev, {M, N}, at::kFloat8_e4m3fn);
    ds = new_scales(dev, M, N / 128);
  }
  if (dbias) {
    abi(ltxfp8_act_backward_workspace_bytes(M, N, &bytes));
    db = new_tensor(dev, {N}, at::kFloat);
    ws = new_workspace(dev, bytes);
  }
  abi(ltxfp8_act_backward(yr.ptr(), yr.ld, cdata(zc.q), zc.s, zc.ld, M, N, act, data(dz), data(dq),
                          static_cast<float*>(data(ds)), align4(M), static_cast<float*>(data(db)), data(ws), bytes,
                          stream_of(dev)));
  return wrap_all({&dz, &dq, &ds, &db});
}

PyObject* wgrad_call(const char* name, c10::Device dev, const Tensor& g, const void* x, int64_t x_rows, int64_t K,
                     int64_t x_ld, const float* xs, int64_t xs_ld, double alpha, bool transposed) {
  const Rows gr = bf16_rows(name, "g", g);
  TORCH_CHECK(x_rows == gr.M, name, ": g has ", gr.M, " rows, x ", x_rows);
  const int64_t M = gr.M, N = gr.K;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  size_t bytes = 0;
  abi(ltxfp8_wgrad_workspace_bytes(M, N, K, &bytes));
  const Tensor out = transposed ? new_tensor(dev, {K, N}, at::kBFloat16) : new_tensor(dev, {N, K}, at::kBFloat16);
  const Tensor ws = new_workspace(dev, bytes);
  abi(ltxfp8_wgrad(gr.ptr(), gr.ld, x, x_ld, xs, xs_ld, static_cast<float>(alpha), data(out), transposed ? 1 : 0, M, N, K,
                   data(ws), bytes, stream_of(dev)));
  return wrap(out);
}

// (g, x_q, x_scales, alpha, transposed)
PyObject* wgrad_1x128(PyObject* const* a) {
  const char* name = "wgrad_1x128";
  const Tensor g = tensor_arg(name, "g", a[0]), xq = tensor_arg(name, "x_q", a[1]),
               xs = tensor_arg(name, "x_scales", a[2]);
  const c10::Device dev = one_device(name, {&g, &xq, &xs});
  const Codes xc = code_rows(name, "x", xq, xs);
  return wgrad_call(name, dev, g, cdata(xc.q), xc.M, xc.K, xc.K, xc.s, xc.ld, double_arg(a[3]), bool_arg(a[4]));
}

// (g, x, alpha, transposed)
PyObject* wgrad_bf16(PyObject* const* a) {
  const char* name = "wgrad_bf16";
  const Tensor g = tensor_arg(name, "g", a[0]), x = tensor_arg(name, "x", a[1]);
  const c10::Device dev = one_device(name, {&g, &x});
  const Rows xr = bf16_rows(name, "x", x);
  return wgrad_call(name, dev, g, xr.ptr(), xr.M, xr.K, xr.ld, nullptr, 0, double_arg(a[2]), bool_arg(a[3]));
}

// (name, leaves): refuse a capture in which autograd would reach a leaf's gradient node that was
// made on the default stream and is still alive.
PyObject* check_capture(PyObject* const* a) {
  const char* name = PyUnicode_AsUTF8(a[0]);
  if (!name) throw python_error();
  TORCH_CHECK_TYPE(PyList_Check(a[1]), name, ": expected a list of tensors");
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[1]); ++i) {
    const Tensor t = tensor_arg(name, "a leaf", PyList_GET_ITEM(a[1], i));
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node || !t.is_cuda()) continue;
    const auto s = node->stream();
    TORCH_CHECK(!s || c10::cuda::CUDAStream(*s) != c10::cuda::getDefaultCUDAStream(t.device().index()), name,
                ": a leaf's gradient node from an earlier eager result on the default stream is still alive; release "
                "that result (or compute it on a side stream) before capturing");
  }
  Py_RETURN_NONE;
}

// (check): the Python function that raises for a C-ABI return code.
PyObject* set_check(PyObject* const* a) {
  Py_INCREF(a[0]);
  Py_XDECREF(g_check);
  g_check = a[0];
  Py_RETURN_NONE;
}

// One Python entry: the argument count, C++ exceptions as Python errors.
template <PyObject* (*kFn)(PyObject* const*), Py_ssize_t kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == kArgs, "expected ", kArgs, " positional arguments, got ", nargs);
  try {
    return kFn(args);
  } catch (const AbiError& e) {
    PyObject* r = g_check ? PyObject_CallFunction(g_check, "i", e.code) : nullptr;
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "ltxfp8 error %d: %s", e.code, ltxfp8_last_error());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define LTXFP8_ENTRY(fn, n) \
  {#fn, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<fn, n>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {
    LTXFP8_ENTRY(rms_norm_quantize, 5), LTXFP8_ENTRY(rms_norm_backward, 5), LTXFP8_ENTRY(gemm_residual, 9),
    LTXFP8_ENTRY(act_quantize_save, 3), LTXFP8_ENTRY(act_backward, 6),      LTXFP8_ENTRY(wgrad_1x128, 5),
    LTXFP8_ENTRY(wgrad_bf16, 4),        LTXFP8_ENTRY(check_capture, 2),
    LTXFP8_ENTRY(set_check, 1),         {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ltxfp8_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ltxfp8_torch(void) {
  PyObject* m = PyModule_Create(&kModule);
  // The torch it was compiled against, compared with the running one by the loader.
  if (m && PyModule_AddStringConstant(m, "torch_version", LTXFP8_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
