// _fmlp_fast: the per-call fast path of flashmlp_fwd / flashmlp_bwd (flashmlp_amd/flashmlp.py), and of the gated
// block's operators, the experts' and the orthogonalised updates (gated.py, block.py, clip.py, experts.py, muon.py;
// below).
//
// A CPython module (METH_FASTCALL) over the C ABI of libflashmlp.so for the common case:
// inputs on one GPU, a shape with kernels of its own (views that they do not read in place are copied
// to dense tensors first). It allocates the
// outputs and the workspace with ATen on the inputs' device, launches on torch's current HIP
// stream of that device and returns the C ABI status with the outputs; for any other input it
// returns None and the Python wrapper takes its general path (which also raises the reference's
// errors). Same entry points, same results as the ctypes calls of the general path; only the
// host work per call is smaller (no ctypes argument conversion, allocations from C++).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/Exception.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <memory>
#include <vector>

#include "flashmlp.h"

namespace {

int io_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return FMLP_DTYPE_F16;
    case at::kBFloat16: return FMLP_DTYPE_BF16;
    case at::kFloat: return FMLP_DTYPE_F32;
    default: return -1;
  }
}

bool dense16(const at::Tensor& t) {
  return t.dim() == 3 && t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

// x and dout: dense 16-byte aligned rows, heads any multiple of 16 bytes apart (0: one matrix
// expanded to every head)
bool rows16(const at::Tensor& t) {
  return t.dim() == 3 && t.stride(2) == 1 && t.stride(1) == t.size(2) &&
         (t.stride(0) * (int64_t)t.element_size()) % 16 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

// the tensors of a call that those kernels take, as they are or (bit i of *copy) as a dense copy: one GPU,
// one dtype, strided; sets the io dtype code
bool eligible(PyObject* const* args, int n, const at::Tensor** ts, int* code, unsigned* copy) {
  for (int i = 0; i < n; ++i) {
    if (!THPVariable_Check(args[i])) return false;
    ts[i] = &THPVariable_Unpack(args[i]);
  }
  const at::Tensor& x = *ts[0];
  if (!x.is_cuda()) return false;
  const int c = io_code(x);
  if (c < 0) return false;
  *copy = 0;
  for (int i = 0; i < n; ++i) {
    const at::Tensor& t = *ts[i];
    if (t.scalar_type() != x.scalar_type() || t.device() != x.device() || t.layout() != at::kStrided || t.dim() != 3 ||
        t.is_neg())  // (a lazily negated view: its memory holds the other sign)
      return false;
    if (!dense16(t) && !((i == 0 || i == 3) && rows16(t))) *copy |= 1u << i;
  }
  *code = c;
  return true;
}

// A call's inputs as the kernels take them: the caller's tensors, or dense copies held here.
struct Inputs {
  const void* p[4];
  int64_t st[4][3];
  at::Tensor held[4];
};

at::Tensor bytes_on(const at::Tensor& like, size_t n) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

// Elements up to which a call's copies are one launch (fmlp_copy_dense); above, ATen copies each view by
// itself, which streams rows of large ones faster (bf16 padded rows, this launch / ATen: 2^20 elements 4.4 /
// 6.2 us, 2^21 4.8 / 6.1, 2^22 7.1 / 6.1, 2^24 19.3 / 13.1).
constexpr int64_t kFusedElems = (int64_t)1 << 21;

// status of the copies (FMLP_OK); throws c10::OutOfMemoryError when they do not fit
int take_inputs(const at::Tensor* const* ts, int n, unsigned copy, hipStream_t stream, Inputs* in) {
  int64_t total = 0;
  for (int i = 0; i < n; ++i) {
    const at::Tensor& t = *ts[i];
    if (copy >> i & 1u) total += t.numel();
    in->p[i] = t.data_ptr();
    for (int k = 0; k < 3; ++k) in->st[i][k] = t.stride(k);
  }
  if (copy == 0) return FMLP_OK;
  const bool fused = total <= kFusedElems;
  const int64_t es = ts[0]->element_size();
  if (fused) in->held[0] = bytes_on(*ts[0], (size_t)(total * es + 4 * 256));
  char* next = fused ? (char*)in->held[0].data_ptr() : nullptr;
  const void* src[4];
  void* dst[4];
  int64_t sizes[12], strides[12];
  int m = 0;
  for (int i = 0; i < n; ++i) {
    if (!(copy >> i & 1u)) continue;
    const at::Tensor& t = *ts[i];
    if (fused) {
      src[m] = t.data_ptr();
      dst[m] = next;
      for (int k = 0; k < 3; ++k) {
        sizes[3 * m + k] = t.size(k);
        strides[3 * m + k] = t.stride(k);
      }
      ++m;
      in->p[i] = next;
      next += (t.numel() * es + 255) / 256 * 256;
    } else {
      in->held[i] = t.is_contiguous() ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
      in->p[i] = in->held[i].data_ptr();
    }
    in->st[i][0] = t.size(1) * t.size(2);
    in->st[i][1] = t.size(2);
    in->st[i][2] = 1;
  }
  return m ? fmlp_copy_dense(m, src, dst, sizes, strides, (int)es, stream) : FMLP_OK;
}

// a dense output of t's shape
at::Tensor empty_dense(const at::Tensor& t) {
  return t.is_contiguous() ? at::empty_like(t) : at::empty(t.sizes(), t.options());
}

PyObject* wrap_or_none(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

// fwd(x, w1, w2, act) -> (status, o) or None
PyObject* fast_fwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 4) {
    PyErr_SetString(PyExc_TypeError, "fwd(x, w1, w2, act)");
    return nullptr;
  }
  const at::Tensor* ts[3];
  int code = 0;
  unsigned copy = 0;
  if (!eligible(args, 3, ts, &code, &copy)) Py_RETURN_NONE;
  const at::Tensor &x = *ts[0], &w1 = *ts[1];
  const int act = (int)PyLong_AsLong(args[3]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  const int64_t H = x.size(0), B = x.size(1), D = x.size(2), E = w1.size(2);
  if (!fmlp_shape_dense(D, E, code)) Py_RETURN_NONE;
  c10::DeviceGuard guard(x.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
  Inputs in;
  try {
    const int st = take_inputs(ts, 3, copy, stream, &in);
    if (st != FMLP_OK) return Py_BuildValue("(iO)", st, Py_None);
  } catch (const c10::OutOfMemoryError&) {
    if (copy == 0) throw;
    Py_RETURN_NONE;
  }
  at::Tensor o = empty_dense(x);
  size_t n = fmlp_fwd_workspace_bytes(H, B, D, E, code);
  at::Tensor ws;
  if (n) {
    try {
      ws = bytes_on(x, n);
    } catch (const c10::OutOfMemoryError&) {  // the kernels then run every tile whole
      n = 0;
    }
  }
  const int st = fmlp_fwd_strided_ws(in.p[0], in.p[1], in.p[2], o.data_ptr(), H, B, D, E, in.st[0], in.st[1], in.st[2],
                                     code, act, n ? ws.data_ptr() : nullptr, n, stream);
  return Py_BuildValue("(iN)", st, THPVariable_Wrap(o));
  END_HANDLE_TH_ERRORS
}

// bwd(x, w1, w2, do, act, flags) -> (status, dx, dw1, dw2) or None; flags: the backward's flag
// bits (FMLP_DW_HILO, FMLP_BWD_RECOMPUTE, FMLP_BWD_NO_DX, FMLP_BWD_NO_DW), the io dtype is added
PyObject* fast_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 6) {
    PyErr_SetString(PyExc_TypeError, "bwd(x, w1, w2, do, act, flags)");
    return nullptr;
  }
  const at::Tensor* ts[4];
  int code = 0;
  unsigned copy = 0;
  if (!eligible(args, 4, ts, &code, &copy)) Py_RETURN_NONE;
  const at::Tensor &x = *ts[0], &w1 = *ts[1], &w2 = *ts[2];
  const int act = (int)PyLong_AsLong(args[4]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  int flags = (int)PyLong_AsLong(args[5]);
  if (flags == -1 && PyErr_Occurred()) return nullptr;
  const int64_t H = x.size(0), B = x.size(1), D = x.size(2), E = w1.size(2);
  if (!fmlp_shape_dense(D, E, code)) Py_RETURN_NONE;
  flags |= code;
  const bool need_dx = (flags & FMLP_BWD_NO_DX) == 0, need_dw = (flags & FMLP_BWD_NO_DW) == 0;
  c10::DeviceGuard guard(x.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
  Inputs in;
  try {
    const int st = take_inputs(ts, 4, copy, stream, &in);
    if (st != FMLP_OK) return Py_BuildValue("(iOOO)", st, Py_None, Py_None, Py_None);
  } catch (const c10::OutOfMemoryError&) {
    if (copy == 0) throw;
    Py_RETURN_NONE;
  }
  at::Tensor dx, dw1, dw2, ws;
  if (need_dx) dx = empty_dense(x);
  if (need_dw) {
    dw1 = empty_dense(w1);
    dw2 = empty_dense(w2);
  }
  // the workspace this call's plan needs (one plan lookup, for its own activation)
  auto ws_need = [&](int f) -> size_t {
    int64_t info[9];
    if (fmlp_bwd_plan(H, B, D, E, f, act, info, 9) == FMLP_OK) return (size_t)info[8];
    return fmlp_bwd_workspace_bytes(H, B, D, E, f);
  };
  size_t n = ws_need(flags);
  if (n) {
    try {
      ws = bytes_on(x, n);
    } catch (const c10::OutOfMemoryError&) {
      // the stored-dZ form's workspace does not fit: the recompute form needs at most the fp32
      // dW partials (as the general path does)
      const bool any_ws = !fmlp_shape_tuned(D, E, code);  // such calls accept any workspace
      if ((flags & FMLP_BWD_RECOMPUTE) && !any_ws) throw;
      flags |= FMLP_BWD_RECOMPUTE;
      n = ws_need(flags);
      try {
        if (n) ws = bytes_on(x, n);
      } catch (const c10::OutOfMemoryError&) {
        if (!any_ws) throw;
        n = 0;
      }
    }
  }
  const int st = fmlp_bwd_strided(in.p[0], in.p[1], in.p[2], in.p[3], need_dx ? dx.data_ptr() : nullptr,
                                  need_dw ? dw1.data_ptr() : nullptr, need_dw ? dw2.data_ptr() : nullptr, H, B, D, E,
                                  in.st[0], in.st[1], in.st[2], in.st[3], flags, act, n ? ws.data_ptr() : nullptr, n,
                                  stream);
  return Py_BuildValue("(iNNN)", st, wrap_or_none(dx), wrap_or_none(dw1), wrap_or_none(dw2));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------
// The gated block's operators. Calls that need no copies and no error message run here, with their
// autograd nodes in C++; for any other call these return None and the Python module takes its general path.
// ---------------------------------------------------------------------------------------------
[[noreturn]] void raise_status(int st, const char* what) {
  TORCH_CHECK(false, "flashmlp ", what, " failed: ", fmlp_status_string(st), ": ", fmlp_last_error());
  __builtin_unreachable();
}
void check_status(int st, const char* what) {
  if (st != FMLP_OK) raise_status(st, what);
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A second derivative would need these backward passes to be differentiable. Under create_graph=True the gradients of
// `run`, made from the tensors `of`, are returned with a node that raises once it is differentiated (flashmlp_amd/gated.py's
// first_derivatives_only).
template <typename F>
variable_list once(const variable_list& of, F run) {
  const bool graph = at::GradMode::is_enabled();
  variable_list g;
  {
    at::AutoGradMode off(false);
    g = run();
  }
  if (!graph || !torch::autograd::any_variable_requires_grad(of)) return g;
  const auto node = std::make_shared<torch::autograd::Error>("FlashMLP's gradients cannot be differentiated again",
                                                             torch::autograd::collect_next_edges(of));
  for (const at::Tensor& t : g)
    if (t.defined()) torch::autograd::set_history(t, node);
  return g;
}
// the incoming gradients and the saved tensors of a node
variable_list joined(const variable_list& a, const variable_list& b) {
  variable_list r(a);
  r.insert(r.end(), b.begin(), b.end());
  return r;
}

// x (0), weights (1 .. 3) and dout (4) as the kernels read them in place
bool gated_ok(const at::Tensor* const* ts, int n, int* code) {
  const at::Tensor& x = *ts[0];
  if (!x.is_cuda()) return false;
  *code = io_code(x);
  if (*code < 0) return false;
  for (int i = 0; i < n; ++i) {
    const at::Tensor& t = *ts[i];
    if (t.scalar_type() != x.scalar_type() || t.device() != x.device() || t.layout() != at::kStrided || t.dim() != 3 ||
        t.is_neg())
      return false;
    if (!dense16(t) && !((i == 0 || i == 4) && rows16(t))) return false;
  }
  const at::Tensor &wg = *ts[1], &wu = *ts[2], &w2 = *ts[3];
  const int64_t H = x.size(0), D = x.size(2), E = wg.size(2);
  if (wg.size(0) != H || wg.size(1) != D || wu.sizes() != wg.sizes() || w2.size(0) != H || w2.size(1) != E || w2.size(2) != D)
    return false;
  return n < 5 || ts[4]->sizes() == x.sizes();
}

// the call's workspace of n bytes; where it does not fit, the least that the call runs with (n is then that)
at::Tensor gated_ws(const at::Tensor& x, size_t& n, int64_t H, int64_t D, int64_t E, int code) {
  if (n == 0) return at::Tensor();
  try {
    return bytes_on(x, n);
  } catch (const c10::OutOfMemoryError&) {
    const size_t least = fmlp_gated_min_workspace_bytes(H, D, E, code);
    if (least >= n) throw;
    n = least;
  }
  return n ? bytes_on(x, n) : at::Tensor();
}

// (x may be one matrix for every head: its head stride is 0; out_f32: unrounded)
at::Tensor gated_fwd_run(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& w2, int code,
                         int act, bool out_f32 = false) {
  const int64_t H = x.size(0), B = x.size(1), D = x.size(2), E = wg.size(2);
  c10::DeviceGuard guard(x.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
  at::Tensor o = out_f32 ? at::empty(x.sizes(), x.options().dtype(at::kFloat)) : empty_dense(x);
  if (out_f32) code |= FMLP_OUT_F32;
  size_t n = fmlp_gated_fwd_workspace_bytes(H, B, D, E, code);
  const at::Tensor ws = gated_ws(x, n, H, D, E, code);
  check_status(fmlp_gated_fwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), w2.data_ptr(), o.data_ptr(), H, B, D, E,
                              x.stride(0), code, act, n ? ws.data_ptr() : nullptr, n, stream),
               "gated forward");
  return o;
}

// (dx, dwg, dwu, dw2); those that are not wanted undefined
std::vector<at::Tensor> gated_bwd_run(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& w2,
                                      const at::Tensor& dout, int code, int act, bool need_dx, bool need_dw,
                                      bool out_f32 = false, float dw_scale = 1.f) {
  std::vector<at::Tensor> g(4);
  if (!need_dx && !need_dw) return g;
  const int64_t H = x.size(0), B = x.size(1), D = x.size(2), E = wg.size(2);
  c10::DeviceGuard guard(x.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
  if (need_dx) g[0] = out_f32 ? at::empty(x.sizes(), x.options().dtype(at::kFloat)) : empty_dense(x);
  if (need_dw) {
    g[1] = at::empty_like(wg);
    g[2] = at::empty_like(wu);
    g[3] = at::empty_like(w2);
  }
  const int flags = code | (need_dx ? 0 : FMLP_BWD_NO_DX) | (need_dw ? 0 : FMLP_BWD_NO_DW) | (out_f32 ? FMLP_OUT_F32 : 0);
  size_t n = fmlp_gated_bwd_workspace_bytes(H, B, D, E, flags);
  const at::Tensor ws = gated_ws(x, n, H, D, E, flags);
  auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  check_status(fmlp_gated_bwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), w2.data_ptr(), dout.data_ptr(), ptr(g[0]),
                              ptr(g[1]), ptr(g[2]), ptr(g[3]), H, B, D, E, x.stride(0), dout.stride(0), flags, act, dw_scale,
                              n ? ws.data_ptr() : nullptr, n, stream),
               "gated backward");
  return g;
}

// A node's saved tensors may have been through hooks, which keep values, sizes and type but no layout: they are laid out
// for the kernels again, and checked again.
void laid_out(at::Tensor& t, bool fits) {
  if (fits && !t.is_neg()) return;
  t = t.resolve_neg().contiguous();
  if ((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) != 0) t = t.clone(at::MemoryFormat::Contiguous);
}
// x (H, B, D), the weights and dout (H, B, D) of a backward pass
void gated_laid_out(at::Tensor& x, variable_list& s, at::Tensor& dout, int code) {
  laid_out(x, rows16(x));
  for (int i = 1; i < 4; ++i) laid_out(s[i], dense16(s[i]));
  laid_out(dout, rows16(dout));
  const at::Tensor* ts[5] = {&x, &s[1], &s[2], &s[3], &dout};
  int now = 0;
  TORCH_CHECK(gated_ok(ts, 5, &now) && now == code, "a saved tensor of the gated MLP came back with another size, type or device");
}

struct GatedFn : torch::autograd::Function<GatedFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu,
                            const at::Tensor& w2, int64_t code, int64_t act) {
    ctx->save_for_backward({x, wg, wu, w2});
    ctx->saved_data["code"] = code;
    ctx->saved_data["act"] = act;
    return gated_fwd_run(x, wg, wu, w2, (int)code, (int)act);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    return once(joined(grads, s), [&] { return first(ctx, s, grads); });
  }
  static variable_list first(AutogradContext* ctx, const variable_list& s, const variable_list& grads) {
    const int code = (int)ctx->saved_data["code"].toInt(), act = (int)ctx->saved_data["act"].toInt();
    at::Tensor dout = grads[0], x = s[0];
    if (!dout.defined()) return variable_list(6);
    variable_list w = s;
    gated_laid_out(x, w, dout, code);
    const bool dw = ctx->needs_input_grad(1) || ctx->needs_input_grad(2) || ctx->needs_input_grad(3);
    auto g = gated_bwd_run(x, w[1], w[2], w[3], dout, code, act, ctx->needs_input_grad(0), dw);
    variable_list r(6);
    for (int i = 0; i < 4; ++i)
      if (ctx->needs_input_grad(i)) r[i] = g[i];
    return r;
  }
};

at::Tensor head_sum(const at::Tensor& t, float scale, const at::Tensor& like) {
  c10::DeviceGuard guard(t.device());
  at::Tensor out = at::empty({t.size(1), t.size(2)}, like.options());
  check_status(fmlp_head_sum(t.data_ptr<float>(), out.data_ptr(), t.size(0), out.numel(), scale, io_code(like),
                             c10::hip::getCurrentHIPStream(t.device().index()).stream()),
               "head sum");
  return out;
}
at::Tensor every_head(const at::Tensor& t, int64_t H) { return t.unsqueeze(0).expand({H, t.size(0), t.size(1)}); }

// One input (B, D) through every head, the mean over heads (gated.py's _SharedGatedFunction)
struct SharedGatedFn : torch::autograd::Function<SharedGatedFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu,
                            const at::Tensor& w2, int64_t code, int64_t act) {
    ctx->save_for_backward({x, wg, wu, w2});
    ctx->saved_data["code"] = code;
    ctx->saved_data["act"] = act;
    const int64_t H = wg.size(0);
    return head_sum(gated_fwd_run(every_head(x, H), wg, wu, w2, (int)code, (int)act, true), 1.f / (float)H, x);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    return once(joined(grads, s), [&] { return first(ctx, s, grads); });
  }
  static variable_list first(AutogradContext* ctx, const variable_list& s, const variable_list& grads) {
    const int code = (int)ctx->saved_data["code"].toInt(), act = (int)ctx->saved_data["act"].toInt();
    variable_list r(6);
    if (!grads[0].defined()) return r;
    const int64_t H = s[1].size(0);
    at::Tensor d2 = grads[0], x2 = s[0];
    laid_out(d2, rows16(every_head(d2, H)));
    laid_out(x2, rows16(every_head(x2, H)));
    at::Tensor dout = every_head(d2, H), x = every_head(x2, H);
    variable_list w = s;
    gated_laid_out(x, w, dout, code);
    const bool dw = ctx->needs_input_grad(1) || ctx->needs_input_grad(2) || ctx->needs_input_grad(3);
    const float scale = 1.f / (float)H;
    auto g = gated_bwd_run(x, w[1], w[2], w[3], dout, code, act, ctx->needs_input_grad(0), dw, true, scale);
    if (ctx->needs_input_grad(0)) r[0] = head_sum(g[0], scale, s[0]);
    for (int i = 1; i < 4; ++i)
      if (ctx->needs_input_grad(i)) r[i] = g[i];
    return r;
  }
};

// Under torch.jit.trace a call that launches by itself would leave its allocations in the graph, never filled: the Python
// modules call what the graph can hold.
bool traced() { return at::tracer::impl::is_dispatch_enabled(); }

bool unpack(PyObject* const* args, int n, const at::Tensor** ts) {
  if (traced()) return false;
  for (int i = 0; i < n; ++i) {
    if (!THPVariable_Check(args[i])) return false;
    ts[i] = &THPVariable_Unpack(args[i]);
  }
  return true;
}

// gated_fwd(x, wg, wu, w2, act) -> o, or None
PyObject* fast_gated_fwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* ts[4];
  int code = 0;
  if (nargs != 5 || !unpack(args, 4, ts) || !gated_ok(ts, 4, &code)) Py_RETURN_NONE;
  const int act = (int)PyLong_AsLong(args[4]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  return THPVariable_Wrap(gated_fwd_run(*ts[0], *ts[1], *ts[2], *ts[3], code, act));
  END_HANDLE_TH_ERRORS
}

// gated(x, wg, wu, w2, act) -> o with its autograd node, or None
PyObject* fast_gated(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* ts[4];
  int code = 0;
  if (nargs != 5 || !unpack(args, 4, ts) || !gated_ok(ts, 4, &code)) Py_RETURN_NONE;
  const int act = (int)PyLong_AsLong(args[4]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  return THPVariable_Wrap(GatedFn::apply(*ts[0], *ts[1], *ts[2], *ts[3], (int64_t)code, (int64_t)act));
  END_HANDLE_TH_ERRORS
}

// gated_shared(x (B, D), wg, wu, w2, act) -> the mean over heads with its autograd node, or None
PyObject* fast_gated_shared(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* ts[4];
  int code = 0;
  if (nargs != 5 || !unpack(args, 4, ts) || ts[0]->dim() != 2 || ts[1]->dim() != 3 || !ts[0]->is_cuda()) Py_RETURN_NONE;
  const at::Tensor x3 = every_head(ts[0]->detach(), ts[1]->size(0));
  const at::Tensor* t3[4] = {&x3, ts[1], ts[2], ts[3]};
  if (!gated_ok(t3, 4, &code)) Py_RETURN_NONE;
  const int act = (int)PyLong_AsLong(args[4]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  return THPVariable_Wrap(SharedGatedFn::apply(*ts[0], *ts[1], *ts[2], *ts[3], (int64_t)code, (int64_t)act));
  END_HANDLE_TH_ERRORS
}

// gated_bwd(x, wg, wu, w2, do, act, need_dx, need_dw) -> (dx, dwg, dwu, dw2), or None
PyObject* fast_gated_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* ts[5];
  int code = 0;
  if (nargs != 8 || !unpack(args, 5, ts) || !gated_ok(ts, 5, &code)) Py_RETURN_NONE;
  const int act = (int)PyLong_AsLong(args[5]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  auto g = gated_bwd_run(*ts[0], *ts[1], *ts[2], *ts[3], *ts[4], code, act, PyObject_IsTrue(args[6]) == 1,
                         PyObject_IsTrue(args[7]) == 1);
  return Py_BuildValue("(NNNN)", wrap_or_none(g[0]), wrap_or_none(g[1]), wrap_or_none(g[2]), wrap_or_none(g[3]));
  END_HANDLE_TH_ERRORS
}

// ---- join ----
struct JoinCfg {
  double scale, eps;
  bool post;
  int64_t heads;  // without o: heads of y, 0 for rows
  at::ScalarType dtype;
};

// (what has no memory of its own, a wrapper around other tensors, would pass for an input that is not there)
const void* cptr(const at::Tensor& t) {
  const void* p = t.defined() ? t.data_ptr() : nullptr;
  TORCH_CHECK_TYPE(p != nullptr || !t.defined() || t.numel() == 0,
                   "a tensor without memory of its own cannot be read by the kernels");
  return p;
}
void* mptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void head_strides(const at::Tensor& t, int64_t* sh, int64_t* sr) {
  *sh = t.dim() == 3 ? t.stride(0) : 0;
  *sr = t.stride(t.dim() - 2);
}
int code_of(at::ScalarType t) { return t == at::kHalf ? FMLP_DTYPE_F16 : t == at::kBFloat16 ? FMLP_DTYPE_BF16 : FMLP_DTYPE_F32; }

fmlp_join join_call(const at::Tensor& r, const at::Tensor& o, const at::Tensor& w_post, const at::Tensor& gate,
                    const at::Tensor& w_pre, const JoinCfg& c) {
  fmlp_join j{};
  j.o = cptr(o);
  j.w_post = cptr(w_post);
  j.gate = cptr(gate);
  j.w_pre = cptr(w_pre);
  j.B = r.size(0);
  j.H = o.defined() ? (o.dim() == 3 ? o.size(0) : 1) : std::max<int64_t>(c.heads, 1);
  j.D = r.size(1) / j.H;
  j.groups = gate.defined() && gate.dim() == 2 ? gate.size(0) : 1;
  j.r_stride = r.stride(0);
  if (o.defined()) head_strides(o, &j.o_head_stride, &j.o_row_stride);
  j.scale = (float)c.scale;
  j.eps = (float)c.eps;
  j.post = c.post ? 1 : 0;
  j.dtype = code_of(c.dtype);
  j.r_dtype = code_of(r.scalar_type());
  return j;
}

bool cols1(const at::Tensor& t) { return t.stride(t.dim() - 1) == 1 && !t.is_neg(); }

// the call needs no copies, and no error: (r (B, C), o (H, B, D) or (B, C) or none, vectors of C)
bool join_ok(const at::Tensor& r, const at::Tensor& o, const at::Tensor& w_post, const at::Tensor& gate,
             const at::Tensor& w_pre, const JoinCfg& c) {
  if (!r.is_cuda() || r.layout() != at::kStrided || r.dim() != 2 || r.size(1) < 1 || !cols1(r)) return false;
  if (c.dtype != at::kHalf && c.dtype != at::kBFloat16 && c.dtype != at::kFloat) return false;
  if (r.scalar_type() != c.dtype && r.scalar_type() != at::kFloat) return false;
  const int64_t B = r.size(0), C = r.size(1);
  for (const at::Tensor* t : {&r, &o, &w_post, &gate, &w_pre})
    if (t->defined() && t->numel() > 0 && t->data_ptr() == nullptr) return false;  // (the general path refuses it)
  for (const at::Tensor* t : {&o, &w_post, &gate, &w_pre})
    if (t->defined() && (t->scalar_type() != c.dtype || t->device() != r.device() || t->layout() != at::kStrided || t->is_neg()))
      return false;
  if (o.defined()) {
    if (o.dim() != 2 && o.dim() != 3) return false;
    if (o.size(o.dim() - 2) != B || !cols1(o) || (o.dim() == 3 ? o.size(0) * o.size(2) : o.size(1)) != C) return false;
  } else if (w_post.defined() || gate.defined() || c.heads < 0 || (c.heads > 0 && C % c.heads != 0)) {
    return false;
  }
  if (w_post.defined() && !c.post) return false;
  for (const at::Tensor* t : {&w_post, &w_pre})
    if (t->defined() && (t->dim() != 1 || t->size(0) != C || !t->is_contiguous())) return false;
  if (gate.defined()) {
    if ((gate.dim() != 1 && gate.dim() != 2) || gate.size(gate.dim() - 1) != C || !gate.is_contiguous()) return false;
    if (gate.dim() == 2 && (gate.size(0) < 1 || B % gate.size(0) != 0)) return false;
  }
  return true;
}

// (r', y, rs); r' undefined without o, rs (2, B) undefined unless saved
std::tuple<at::Tensor, at::Tensor, at::Tensor> join_fwd_run(const at::Tensor& r, const at::Tensor& o, const at::Tensor& w_post,
                                                            const at::Tensor& gate, const at::Tensor& w_pre,
                                                            const JoinCfg& c, bool save) {
  c10::DeviceGuard guard(r.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(r.device().index()).stream();
  fmlp_join j = join_call(r, o, w_post, gate, w_pre, c);
  at::Tensor r2, y, rs;
  const auto opt = r.options().dtype(c.dtype);
  if (o.defined()) r2 = r.is_contiguous() ? at::empty_like(r) : at::empty(r.sizes(), r.options());
  if (o.defined() ? o.dim() == 3 : c.heads > 0) y = at::empty({j.H, j.B, j.D}, opt);
  else y = at::empty({j.B, j.D}, opt);
  if (save) rs = at::empty({2, j.B}, r.options().dtype(at::kFloat));
  j.r = cptr(r);
  j.r_out = mptr(r2);
  j.y = mptr(y);
  head_strides(y, &j.y_head_stride, &j.y_row_stride);
  if (save) {
    j.rs_o = rs.data_ptr<float>();
    j.rs_r = j.rs_o + j.B;
  }
  check_status(fmlp_join_fwd(&j, stream), "join forward");
  return {r2, y, rs};
}

at::Tensor cols(const at::Tensor& t) { return !t.defined() || cols1(t) ? t : t.resolve_neg().contiguous(); }

// A 16-bit stream's backward makes the unrounded r' again from r; else r' itself is what is saved.
bool from_r(const at::Tensor& r, const at::Tensor& o) { return o.defined() && r.scalar_type() != at::kFloat; }

// (dr, do, dw_post, dgate, dw_pre); those that are not wanted undefined. r2: r' or, where from_r, r
std::vector<at::Tensor> join_bwd_run(const at::Tensor& r2, const at::Tensor& o, const at::Tensor& rs, at::Tensor dr2,
                                     at::Tensor dy, const at::Tensor& w_post, const at::Tensor& gate,
                                     const at::Tensor& w_pre, const JoinCfg& c, const bool* need) {
  c10::DeviceGuard guard(r2.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(r2.device().index()).stream();
  fmlp_join j = join_call(r2, o, w_post, gate, w_pre, c);
  std::vector<at::Tensor> g(5);
  dr2 = cols(dr2);
  dy = cols(dy);
  if (need[0]) g[0] = at::empty(r2.sizes(), r2.options());
  if (need[1] && o.defined()) g[1] = at::empty(o.sizes(), o.options());
  if (need[2] && w_post.defined()) g[2] = at::empty_like(w_post);
  if (need[3] && gate.defined()) g[3] = at::empty_like(gate);
  if (need[4] && w_pre.defined()) g[4] = dy.defined() ? at::empty_like(w_pre) : at::zeros_like(w_pre);
  if (from_r(r2, o)) j.r = cptr(r2);
  else j.r_out = const_cast<void*>(cptr(r2));
  j.rs_o = rs.data_ptr<float>();
  j.rs_r = j.rs_o + j.B;
  j.dr_out = cptr(dr2);
  j.dy = cptr(dy);
  if (!dy.defined()) j.w_pre = nullptr;
  j.dr = mptr(g[0]);
  j.d_o = mptr(g[1]);
  j.dw_post = mptr(g[2]);
  j.dgate = mptr(g[3]);
  j.dw_pre = dy.defined() ? mptr(g[4]) : nullptr;
  if (dr2.defined()) j.dr_out_stride = dr2.stride(0);
  if (dy.defined()) head_strides(dy, &j.y_head_stride, &j.y_row_stride);
  if (g[1].defined()) head_strides(g[1], &j.d_o_head_stride, &j.d_o_row_stride);
  at::Tensor ws;
  const size_t n = fmlp_join_bwd_workspace_bytes(&j);
  if (n) ws = bytes_on(r2, n);
  check_status(fmlp_join_bwd(&j, n ? ws.data_ptr() : nullptr, n, stream), "join backward");
  return g;
}

struct JoinFn : torch::autograd::Function<JoinFn> {
  using Opt = std::optional<at::Tensor>;
  // with o: (r', y); without: (y)
  static variable_list forward(AutogradContext* ctx, const at::Tensor& r, const Opt& o_, const Opt& w_post_,
                               const Opt& gate_, const Opt& w_pre_, const JoinCfg& c) {
    const at::Tensor o = o_.value_or(at::Tensor()), w_post = w_post_.value_or(at::Tensor()),
                     gate = gate_.value_or(at::Tensor()), w_pre = w_pre_.value_or(at::Tensor());
    auto [r2, y, rs] = join_fwd_run(r, o, w_post, gate, w_pre, c, true);
    ctx->save_for_backward({r2.defined() && !from_r(r, o) ? r2 : r, o, rs, w_post, gate, w_pre});
    ctx->saved_data["scale"] = c.scale;
    ctx->saved_data["eps"] = c.eps;
    ctx->saved_data["post"] = c.post;
    ctx->saved_data["heads"] = c.heads;
    ctx->saved_data["dtype"] = (int64_t)c.dtype;
    ctx->set_materialize_grads(false);
    if (!r2.defined()) return {y};
    return {r2, y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    return once(joined(grads, s), [&] { return first(ctx, s, grads); });
  }
  static variable_list first(AutogradContext* ctx, const variable_list& s, const variable_list& grads) {
    const bool with_o = s[1].defined();
    const JoinCfg c{ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["post"].toBool(),
                    ctx->saved_data["heads"].toInt(), (at::ScalarType)ctx->saved_data["dtype"].toInt()};
    const at::Tensor dr2 = with_o ? grads[0] : at::Tensor(), dy = with_o ? grads[1] : grads[0];
    variable_list r(6);
    if (!dr2.defined() && !dy.defined()) return r;
    // the node has an edge for each tensor that is there
    const bool there[5] = {true, with_o, s[3].defined(), s[4].defined(), s[5].defined()};
    bool need[5];
    for (int i = 0, edge = 0; i < 5; ++i) need[i] = there[i] && ctx->needs_input_grad(edge++);
    variable_list t = s;
    t[0] = cols(t[0]);
    t[1] = cols(t[1]);
    for (int i = 2; i < 6; ++i)
      if (t[i].defined()) t[i] = t[i].resolve_neg().contiguous();
    const at::Tensor& rs = t[2];
    TORCH_CHECK(join_ok(t[0], t[1], t[3], t[4], t[5], c) && rs.scalar_type() == at::kFloat && rs.device() == t[0].device() &&
                    rs.dim() == 2 && rs.size(0) == 2 && rs.size(1) == t[0].size(0) &&
                    (!dr2.defined() || dr2.sizes() == t[0].sizes()) && (!dy.defined() || dy.numel() == t[0].numel()),
                "a saved tensor of the join came back with another size, type or device");
    auto g = join_bwd_run(t[0], t[1], rs, dr2, dy, t[3], t[4], t[5], c, need);
    for (int i = 0; i < 5; ++i) r[i] = g[i];
    return r;
  }
};

at::Tensor or_none(PyObject* o, bool* ok) {
  if (o == Py_None) return at::Tensor();
  if (!THPVariable_Check(o)) {
    *ok = false;
    return at::Tensor();
  }
  return THPVariable_Unpack(o);
}

// join(r, o, w_post, gate, w_pre, scale, post, eps, heads, dtype_of) -> (r', y), or None. o None: block_norm, with
// heads (0: rows) and the dtype of `dtype_of` (0 fp16, 1 bf16, 2 fp32)
PyObject* fast_join(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 10 || traced()) Py_RETURN_NONE;
  at::Tensor t[5];
  bool ok = true;
  for (int i = 0; i < 5; ++i) t[i] = or_none(args[i], &ok);
  if (!ok || !t[0].defined()) Py_RETURN_NONE;
  for (int i : {5, 7})  // scale and eps are numbers: a tensor's value would be taken, and its gradient lost
    if (!PyFloat_Check(args[i]) && !PyLong_Check(args[i])) Py_RETURN_NONE;
  JoinCfg c{PyFloat_AsDouble(args[5]), PyFloat_AsDouble(args[7]), PyObject_IsTrue(args[6]) == 1, PyLong_AsLong(args[8]),
            at::kFloat};
  const long code = PyLong_AsLong(args[9]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  c.dtype = t[1].defined() ? t[1].scalar_type() : code == 0 ? at::kHalf : code == 1 ? at::kBFloat16 : at::kFloat;
  if (!(c.eps >= 0) || !join_ok(t[0], t[1], t[2], t[3], t[4], c)) Py_RETURN_NONE;
  // a tensor with a tangent goes to the node too, which refuses forward mode
  bool grad = false;
  for (auto& v : t) grad = grad || (v.defined() && ((at::GradMode::is_enabled() && v.requires_grad()) || v._fw_grad(0).defined()));
  at::Tensor r2, y;
  if (grad) {
    const auto opt = [&](int i) { return t[i].defined() ? JoinFn::Opt(t[i]) : JoinFn::Opt(); };
    variable_list out = JoinFn::apply(t[0], opt(1), opt(2), opt(3), opt(4), c);
    if (out.size() == 2) r2 = out[0];
    y = out.back();
  } else {
    std::tie(r2, y, std::ignore) = join_fwd_run(t[0], t[1], t[2], t[3], t[4], c, false);
  }
  return Py_BuildValue("(NN)", wrap_or_none(r2), wrap_or_none(y));
  END_HANDLE_TH_ERRORS
}

// ---- clipping ----
// clip(grads, outs, max_norm) -> norm, or None; lists of tensors, outs None for the norm alone
PyObject* fast_clip(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 3 || traced() || !PyList_Check(args[0]) || (args[1] != Py_None && !PyList_Check(args[1]))) Py_RETURN_NONE;
  const bool clip = args[1] != Py_None;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  if (n == 0 || n > (1 << 24) || (clip && PyList_GET_SIZE(args[1]) != n)) Py_RETURN_NONE;
  const double max_norm = PyFloat_AsDouble(args[2]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!(max_norm >= 0)) Py_RETURN_NONE;
  std::vector<const void*> g((size_t)n);
  std::vector<void*> o((size_t)(clip ? n : 0));
  std::vector<int64_t> numel((size_t)n);
  std::vector<int> gt((size_t)n), ot(o.size());
  const at::Tensor* first = nullptr;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *a = PyList_GET_ITEM(args[0], i), *b = clip ? PyList_GET_ITEM(args[1], i) : nullptr;
    if (!THPVariable_Check(a) || (b && !THPVariable_Check(b))) Py_RETURN_NONE;
    const at::Tensor& t = THPVariable_Unpack(a);
    if (i == 0) {
      if (!t.is_cuda()) Py_RETURN_NONE;
      first = &t;
    }
    const auto fits = [&](const at::Tensor& v, int* code) {
      *code = io_code(v);
      return *code >= 0 && v.layout() == at::kStrided && v.device() == first->device() && v.is_contiguous() && !v.is_neg();
    };
    if (!fits(t, &gt[i])) Py_RETURN_NONE;
    g[i] = t.data_ptr();
    numel[i] = t.numel();
    if (b) {
      const at::Tensor& v = THPVariable_Unpack(b);
      if (!fits(v, &ot[i]) || v.sizes() != t.sizes()) Py_RETURN_NONE;
      o[i] = v.data_ptr();
    }
  }
  c10::DeviceGuard guard(first->device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream(first->device().index()).stream();
  at::Tensor norm = at::empty({}, first->options().dtype(at::kFloat));
  const size_t bytes = fmlp_clip_workspace_bytes((int)n, numel.data());
  at::Tensor ws = bytes_on(*first, bytes);
  const int st = clip ? fmlp_clip_grads((int)n, g.data(), o.data(), numel.data(), gt.data(), ot.data(), (float)max_norm,
                                        norm.data_ptr<float>(), ws.data_ptr(), bytes, stream)
                      : fmlp_grad_norm((int)n, g.data(), numel.data(), gt.data(), norm.data_ptr<float>(), ws.data_ptr(),
                                       bytes, stream);
  check_status(st, clip ? "gradient clipping" : "gradient norm");
  if (clip)  // as any in-place operation, so that autograd notices a saved tensor that has changed
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor& v = THPVariable_Unpack(PyList_GET_ITEM(args[1], i));
      if (!v.is_inference()) v.unsafeGetTensorImpl()->bump_version();
    }
  return THPVariable_Wrap(norm);
  END_HANDLE_TH_ERRORS
}

// ---- experts ----
// a strided tensor on a GPU with memory of its own
bool on_gpu(const at::Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && (t.numel() == 0 || t.data_ptr() != nullptr);
}
// a dense tensor of `type` on the device of `like`
bool dense_beside(const at::Tensor& t, const at::Tensor& like, at::ScalarType type) {
  return on_gpu(t) && t.device() == like.device() && t.scalar_type() == type && t.is_contiguous();
}
at::Tensor dense(const at::Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }
bool wants_node(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)  // (a tensor with a tangent goes to the node too, which refuses forward mode)
    if (t->defined() && ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}
hipStream_t stream_on(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool route_ok(const at::Tensor& l, int64_t k) {
  return on_gpu(l) && io_code(l) >= 0 && l.dim() == 2 && k >= 1 && k <= l.size(1) && cols1(l);
}
std::pair<at::Tensor, at::Tensor> route_run(const at::Tensor& l, int64_t k, bool normalize) {
  c10::DeviceGuard guard(l.device());
  const int64_t T = l.size(0);
  at::Tensor w = at::empty({T, k}, l.options().dtype(at::kFloat)), e = at::empty({T, k}, l.options().dtype(at::kInt));
  check_status(fmlp_route_fwd(l.data_ptr(), w.data_ptr<float>(), e.data_ptr<int>(), T, l.size(1), l.stride(0), k, normalize,
                              io_code(l), stream_on(l)),
               "route forward");
  return {w, e};
}

struct RouteFn : torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& l, int64_t k, bool normalize) {
    auto [w, e] = route_run(l, k, normalize);
    ctx->save_for_backward({normalize ? at::Tensor() : l, w, e});
    ctx->saved_data["normalize"] = normalize;
    ctx->saved_data["N"] = l.size(1);
    ctx->saved_data["dtype"] = (int64_t)l.scalar_type();
    ctx->mark_non_differentiable({e});
    return {w, e};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    return once(joined({grads[0]}, s), [&] { return first(ctx, s, grads); });
  }
  static variable_list first(AutogradContext* ctx, const variable_list& s, const variable_list& grads) {
    variable_list r(3);
    if (!grads[0].defined()) return r;
    const bool normalize = ctx->saved_data["normalize"].toBool();
    const int64_t N = ctx->saved_data["N"].toInt();
    const auto dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
    const at::Tensor w = dense(s[1]), e = dense(s[2]), dw = dense(grads[0]), l = s[0].defined() ? cols(s[0]) : s[0];
    TORCH_CHECK(w.dim() == 2 && dense_beside(w, w, at::kFloat) && dense_beside(e, w, at::kInt) && dense_beside(dw, w, at::kFloat) &&
                    e.sizes() == w.sizes() && dw.sizes() == w.sizes() &&
                    (normalize || (route_ok(l, w.size(1)) && l.device() == w.device() && l.scalar_type() == dtype &&
                                   l.size(0) == w.size(0) && l.size(1) == N)),
                "a saved tensor of the routing came back with another size, type or device");
    c10::DeviceGuard guard(w.device());
    r[0] = at::empty({w.size(0), N}, w.options().dtype(dtype));
    check_status(fmlp_route_bwd(normalize ? nullptr : l.data_ptr(), w.data_ptr<float>(), e.data_ptr<int>(), dw.data_ptr<float>(),
                                r[0].data_ptr(), w.size(0), N, normalize ? 0 : l.stride(0), w.size(1), normalize, code_of(dtype),
                                stream_on(w)),
                 "route backward");
    return r;
  }
};

// whole numbers as Python has them
bool whole(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o) || PyBool_Check(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// expert_route(logits, k, normalize) -> (weights, experts), or None
PyObject* fast_route(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* l;
  int64_t k;
  if (nargs != 3 || !unpack(args, 1, &l) || !whole(args[1], &k) || !route_ok(*l, k)) Py_RETURN_NONE;
  const bool normalize = PyObject_IsTrue(args[2]) == 1;
  at::Tensor w, e;
  if (wants_node({l})) {
    variable_list out = RouteFn::apply(*l, k, normalize);
    w = out[0];
    e = out[1];
  } else {
    std::tie(w, e) = route_run(*l, k, normalize);
  }
  return Py_BuildValue("(NN)", THPVariable_Wrap(w), THPVariable_Wrap(e));
  END_HANDLE_TH_ERRORS
}

// expert_plan(experts, num_experts, capacity) -> (slots, counts), or None
PyObject* fast_plan(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* ex;
  int64_t N, capacity;
  if (nargs != 3 || !unpack(args, 1, &ex) || !whole(args[1], &N) || !whole(args[2], &capacity) || N < 1 || capacity < 0) Py_RETURN_NONE;
  const at::Tensor& e = *ex;
  const bool wide = e.scalar_type() == at::kLong;
  if (!on_gpu(e) || (!wide && e.scalar_type() != at::kInt) || e.dim() != 2 || e.size(1) < 1 || !e.is_contiguous()) Py_RETURN_NONE;
  c10::DeviceGuard guard(e.device());
  const int64_t T = e.size(0), k = e.size(1);
  const auto opt = e.options().dtype(at::kInt);
  at::Tensor slots = at::empty({T, k}, opt), counts = at::empty({N}, opt), ws;
  const size_t n = fmlp_expert_plan_workspace_bytes(T, k, N);
  if (n) ws = bytes_on(e, n);
  check_status(fmlp_expert_plan(e.data_ptr(), wide ? 8 : 4, slots.data_ptr<int>(), counts.data_ptr<int>(), T, k, N, capacity,
                                n ? ws.data_ptr() : nullptr, n, stream_on(e)),
               "expert plan");
  return Py_BuildValue("(NN)", THPVariable_Wrap(slots), THPVariable_Wrap(counts));
  END_HANDLE_TH_ERRORS
}

// slots (T, k), counts (N) of a plan for T tokens, or for any number where T < 0
bool plan_ok(const at::Tensor& slots, const at::Tensor& counts, const at::Tensor& like, int64_t T, int64_t N, int64_t capacity) {
  return N >= 1 && capacity >= 0 && dense_beside(slots, like, at::kInt) && slots.dim() == 2 && slots.size(1) >= 1 &&
         (T < 0 || slots.size(0) == T) && dense_beside(counts, like, at::kInt) && counts.dim() == 1 && counts.size(0) == N;
}
const float* weights_ptr(const at::Tensor& w) { return w.defined() ? w.data_ptr<float>() : nullptr; }

// (rows, dweights); those that are not wanted undefined
std::pair<at::Tensor, at::Tensor> scatter_run(const at::Tensor& x, const at::Tensor& w, const at::Tensor& slots, const at::Tensor& counts,
                                              int64_t N, int64_t capacity, const at::Tensor& rows_in, bool want_rows, bool want_dw) {
  c10::DeviceGuard guard(x.device());
  at::Tensor rows, dw;
  if (want_rows) rows = at::empty({N, capacity, x.size(1)}, x.options());
  if (want_dw) dw = at::empty(slots.sizes(), x.options().dtype(at::kFloat));
  if (!want_rows && !want_dw) return {rows, dw};
  check_status(fmlp_expert_scatter(x.data_ptr(), x.stride(0), weights_ptr(w), slots.data_ptr<int>(), counts.data_ptr<int>(),
                                   want_dw ? rows_in.data_ptr() : nullptr, mptr(rows), want_dw ? dw.data_ptr<float>() : nullptr,
                                   slots.size(0), slots.size(1), N, capacity, x.size(1), io_code(x), stream_on(x)),
               "expert scatter");
  return {rows, dw};
}
at::Tensor gather_run(const at::Tensor& rows, const at::Tensor& w, const at::Tensor& slots) {
  c10::DeviceGuard guard(rows.device());
  at::Tensor o = at::empty({slots.size(0), rows.size(2)}, rows.options());
  check_status(fmlp_expert_gather(rows.data_ptr(), weights_ptr(w), slots.data_ptr<int>(), o.data_ptr(), slots.size(0), slots.size(1),
                                  rows.size(0), rows.size(1), rows.size(2), io_code(rows), stream_on(rows)),
               "expert gather");
  return o;
}

struct DispatchFn : torch::autograd::Function<DispatchFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& slots, const at::Tensor& counts, int64_t N,
                            int64_t capacity) {
    ctx->save_for_backward({slots});
    ctx->saved_data["T"] = x.size(0);
    return scatter_run(x, at::Tensor(), slots, counts, N, capacity, at::Tensor(), true, false).first;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    return once(joined(grads, s), [&] { return first(ctx, s, grads); });
  }
  static variable_list first(AutogradContext* ctx, const variable_list& s, const variable_list& grads) {
    variable_list r(5);
    if (!grads[0].defined()) return r;
    const at::Tensor drows = dense(grads[0]), slots = dense(s[0]);
    TORCH_CHECK(dense_beside(slots, drows, at::kInt) && slots.dim() == 2 && slots.size(0) == ctx->saved_data["T"].toInt(),
                "a saved tensor of the dispatch came back with another size, type or device");
    r[0] = gather_run(drows, at::Tensor(), slots);
    return r;
  }
};

bool rows_ok(const at::Tensor& rows) {
  return on_gpu(rows) && io_code(rows) >= 0 && rows.dim() == 3 && rows.size(2) >= 1 && rows.is_contiguous();
}

// Saves the rows for the weights' gradient alone.
struct CombineFn : torch::autograd::Function<CombineFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows, const std::optional<at::Tensor>& w_, const at::Tensor& slots,
                            const at::Tensor& counts) {
    const at::Tensor w = w_.value_or(at::Tensor());
    ctx->save_for_backward({w.defined() && w.requires_grad() ? rows : at::Tensor(), w, slots, counts});
    ctx->saved_data["rows"] = rows.sizes();
    ctx->saved_data["dtype"] = (int64_t)rows.scalar_type();
    return gather_run(rows, w, slots);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    return once(joined(grads, s), [&] { return first(ctx, s, grads); });
  }
  static variable_list first(AutogradContext* ctx, const variable_list& s, const variable_list& grads) {
    variable_list r(4);
    if (!grads[0].defined()) return r;
    const auto shape = ctx->saved_data["rows"].toIntVector();
    const auto dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
    const at::Tensor dout = cols(grads[0]), rows = dense(s[0]), w = dense(s[1]), slots = dense(s[2]), counts = dense(s[3]);
    TORCH_CHECK(dout.dim() == 2 && dout.size(1) == shape[2] && dout.scalar_type() == dtype &&
                    plan_ok(slots, counts, dout, dout.size(0), shape[0], shape[1]) &&
                    (!rows.defined() || (dense_beside(rows, dout, dtype) && rows.sizes() == shape)) &&
                    (!w.defined() || (dense_beside(w, dout, at::kFloat) && w.sizes() == slots.sizes())),
                "a saved tensor of the combination came back with another size, type or device");
    // (the node has an edge for each tensor that is there: rows, then the weights)
    auto g = scatter_run(dout, w, slots, counts, shape[0], shape[1], rows, ctx->needs_input_grad(0),
                         rows.defined() && ctx->needs_input_grad(1));
    r[0] = g.first;
    r[1] = g.second;
    return r;
  }
};

// expert_dispatch(x, slots, counts, num_experts, capacity) -> rows, or None
PyObject* fast_dispatch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* t[3];
  int64_t N, capacity;
  if (nargs != 5 || !unpack(args, 3, t) || !whole(args[3], &N) || !whole(args[4], &capacity)) Py_RETURN_NONE;
  const at::Tensor& x = *t[0];
  if (!on_gpu(x) || io_code(x) < 0 || x.dim() != 2 || x.size(1) < 1 || !cols1(x) || !plan_ok(*t[1], *t[2], x, x.size(0), N, capacity))
    Py_RETURN_NONE;
  if (wants_node({&x})) return THPVariable_Wrap(DispatchFn::apply(x, *t[1], *t[2], N, capacity));
  return THPVariable_Wrap(scatter_run(x, at::Tensor(), *t[1], *t[2], N, capacity, at::Tensor(), true, false).first);
  END_HANDLE_TH_ERRORS
}

// expert_combine(rows, weights, slots, counts, num_experts, capacity) -> o, or None
PyObject* fast_combine(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int64_t N, capacity;
  if (nargs != 6 || traced() || !whole(args[4], &N) || !whole(args[5], &capacity)) Py_RETURN_NONE;
  bool ok = true;
  at::Tensor t[4];
  for (int i = 0; i < 4; ++i) t[i] = or_none(args[i], &ok);
  const at::Tensor &rows = t[0], &w = t[1], &slots = t[2], &counts = t[3];
  if (!ok || !rows.defined() || !slots.defined() || !counts.defined()) Py_RETURN_NONE;
  if (!rows_ok(rows) || rows.size(0) != N || rows.size(1) != capacity || !plan_ok(slots, counts, rows, -1, N, capacity)) Py_RETURN_NONE;
  if (w.defined() && (!dense_beside(w, rows, at::kFloat) || w.sizes() != slots.sizes())) Py_RETURN_NONE;
  if (wants_node({&rows, &w}))
    return THPVariable_Wrap(CombineFn::apply(rows, w.defined() ? std::optional<at::Tensor>(w) : std::optional<at::Tensor>(), slots, counts));
  return THPVariable_Wrap(gather_run(rows, w, slots));
  END_HANDLE_TH_ERRORS
}

// ---- orthogonalised updates ----
// a, b, c of every step, from one triple of numbers
bool triple(PyObject* o, int64_t steps, std::vector<float>* abc) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 3 || steps < 1 || steps > 10) return false;
  float v[3];
  for (int i = 0; i < 3; ++i) {
    PyObject* x = PyTuple_GET_ITEM(o, i);
    if (!PyFloat_Check(x)) return false;
    v[i] = (float)PyFloat_AS_DOUBLE(x);
  }
  for (int64_t i = 0; i < steps; ++i) abc->insert(abc->end(), v, v + 3);
  return true;
}
bool number(PyObject* o, double* v) {
  if (!PyFloat_Check(o) && !(PyLong_Check(o) && !PyBool_Check(o))) return false;
  *v = PyFloat_AsDouble(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}
// a dense stack of matrices of a type that the kernels take (one with a tangent goes to Python, which refuses forward mode)
bool stack_ok(const at::Tensor& t) {
  return on_gpu(t) && io_code(t) >= 0 && t.dim() >= 2 && t.is_contiguous() && !t._fw_grad(0).defined();
}
int64_t heads_of(const at::Tensor& t) {
  int64_t h = 1;
  for (int64_t i = 0; i + 2 < t.dim(); ++i) h *= t.size(i);
  return h;
}
void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// orthogonalize(x, out, steps, coefficients, eps) -> the result, or None; out None: a new tensor
PyObject* fast_ortho(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* px;
  int64_t steps;
  double eps;
  bool ok = true;
  std::vector<float> abc;
  if (nargs != 5 || !unpack(args, 1, &px) || !whole(args[2], &steps) || !triple(args[3], steps, &abc) || !number(args[4], &eps))
    Py_RETURN_NONE;
  const at::Tensor& x = *px;
  at::Tensor out = or_none(args[1], &ok);
  if (!ok || !stack_ok(x)) Py_RETURN_NONE;
  if (out.defined() && (!stack_ok(out) || out.device() != x.device() || out.scalar_type() != x.scalar_type() || out.sizes() != x.sizes()))
    Py_RETURN_NONE;
  c10::DeviceGuard guard(x.device());
  const bool mine = !out.defined();
  if (mine) out = at::empty(x.sizes(), x.options());
  const int64_t H = heads_of(x), R = x.size(-2), C = x.size(-1);
  const size_t n = fmlp_orthogonalize_workspace_bytes_for(H, R, C, io_code(x), (int)steps, abc.data());
  at::Tensor ws;
  if (n) ws = bytes_on(x, n);
  check_status(fmlp_orthogonalize(x.data_ptr(), out.data_ptr(), H, R, C, io_code(x), (int)steps, abc.data(), (float)eps,
                                  n ? ws.data_ptr() : nullptr, n, stream_on(x)),
               "orthogonalisation");
  if (!mine) changed(out);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// muon_step(params, grads, momenta, lr, momentum, nesterov, weight_decay, scale, steps, coefficients, eps) -> True, or None;
// lists, scale None: sqrt(max(1, R / C))
PyObject* fast_muon(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 11 || traced()) Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i)
    if (!PyList_Check(args[i])) Py_RETURN_NONE;
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  double lr, momentum, decay, scale = 0, eps;
  int64_t steps;
  std::vector<float> abc;
  if (n == 0 || n > (1 << 24) || PyList_GET_SIZE(args[1]) != n || PyList_GET_SIZE(args[2]) != n || !number(args[3], &lr) ||
      !number(args[4], &momentum) || !number(args[6], &decay) || (args[7] != Py_None && !number(args[7], &scale)) ||
      !whole(args[8], &steps) || !triple(args[9], steps, &abc) || !number(args[10], &eps))
    Py_RETURN_NONE;
  if (!(lr >= 0) || !(decay >= 0) || !(momentum >= 0 && momentum <= 1)) Py_RETURN_NONE;
  std::vector<fmlp_muon_tensor> t((size_t)n);
  const at::Tensor* first = nullptr;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* v[3];
    for (int k = 0; k < 3; ++k) {
      PyObject* o = PyList_GET_ITEM(args[k], i);
      if (!THPVariable_Check(o)) Py_RETURN_NONE;
      v[k] = &THPVariable_Unpack(o);
      if (first == nullptr) first = v[k];
      if (!stack_ok(*v[k]) || v[k]->device() != first->device() || v[k]->sizes() != v[0]->sizes()) Py_RETURN_NONE;
    }
    const int64_t R = v[0]->size(-2), C = v[0]->size(-1);
    const double s = args[7] != Py_None ? scale : std::sqrt(std::max(1.0, C ? (double)R / (double)C : 1.0));
    t[(size_t)i] = fmlp_muon_tensor{v[0]->data_ptr(), v[1]->data_ptr(), v[2]->data_ptr(), heads_of(*v[0]), R, C,
                                    io_code(*v[0]), io_code(*v[1]), io_code(*v[2]), (float)s};
  }
  c10::DeviceGuard guard(first->device());
  const size_t bytes = fmlp_muon_workspace_bytes_for((int)n, t.data(), (int)steps, abc.data());
  at::Tensor ws;
  if (bytes) ws = bytes_on(*first, bytes);
  check_status(fmlp_muon_step((int)n, t.data(), lr, momentum, PyObject_IsTrue(args[5]) == 1, decay, (int)steps, abc.data(), (float)eps,
                              bytes ? ws.data_ptr() : nullptr, bytes, stream_on(*first)),
               "muon step");
  for (Py_ssize_t i = 0; i < n; ++i)
    for (int k : {0, 2}) changed(THPVariable_Unpack(PyList_GET_ITEM(args[k], i)));
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"fwd", (PyCFunction)(void (*)(void))fast_fwd, METH_FASTCALL, "fwd(x, w1, w2, act) -> (status, o) or None"},
    {"bwd", (PyCFunction)(void (*)(void))fast_bwd, METH_FASTCALL,
     "bwd(x, w1, w2, do, act, flags) -> (status, dx, dw1, dw2) or None"},
    {"gated_fwd", (PyCFunction)(void (*)(void))fast_gated_fwd, METH_FASTCALL, "gated_fwd(x, wg, wu, w2, act) -> o or None"},
    {"gated", (PyCFunction)(void (*)(void))fast_gated, METH_FASTCALL, "gated(x, wg, wu, w2, act) -> o or None"},
    {"gated_shared", (PyCFunction)(void (*)(void))fast_gated_shared, METH_FASTCALL,
     "gated_shared(x, wg, wu, w2, act) -> the mean over heads or None"},
    {"gated_bwd", (PyCFunction)(void (*)(void))fast_gated_bwd, METH_FASTCALL,
     "gated_bwd(x, wg, wu, w2, do, act, need_dx, need_dw) -> (dx, dwg, dwu, dw2) or None"},
    {"join", (PyCFunction)(void (*)(void))fast_join, METH_FASTCALL,
     "join(r, o, w_post, gate, w_pre, scale, post, eps, heads, dtype) -> (r', y) or None"},
    {"clip", (PyCFunction)(void (*)(void))fast_clip, METH_FASTCALL, "clip(grads, outs, max_norm) -> norm or None"},
    {"expert_route", (PyCFunction)(void (*)(void))fast_route, METH_FASTCALL,
     "expert_route(logits, k, normalize) -> (weights, experts) or None"},
    {"expert_plan", (PyCFunction)(void (*)(void))fast_plan, METH_FASTCALL,
     "expert_plan(experts, num_experts, capacity) -> (slots, counts) or None"},
    {"expert_dispatch", (PyCFunction)(void (*)(void))fast_dispatch, METH_FASTCALL,
     "expert_dispatch(x, slots, counts, num_experts, capacity) -> rows or None"},
    {"expert_combine", (PyCFunction)(void (*)(void))fast_combine, METH_FASTCALL,
     "expert_combine(rows, weights, slots, counts, num_experts, capacity) -> o or None"},
    {"orthogonalize", (PyCFunction)(void (*)(void))fast_ortho, METH_FASTCALL,
     "orthogonalize(x, out, steps, coefficients, eps) -> the result or None"},
    {"muon_step", (PyCFunction)(void (*)(void))fast_muon, METH_FASTCALL,
     "muon_step(params, grads, momenta, lr, momentum, nesterov, weight_decay, scale, steps, coefficients, eps) -> True or None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fmlp_fast", "fast path of the Python wrappers", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__fmlp_fast() { return PyModule_Create(&kModule); }
