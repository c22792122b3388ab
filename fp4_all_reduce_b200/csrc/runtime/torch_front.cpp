// Native front end of the torch ops: argument checks, output allocation and the launch of one call in one C++ function,
// for the Python wrappers (`ops/codec.py`, `ops/gemm.py`, `parallel/context.py`) and for `torch.ops.fp4ar.*`.
//
// Why it exists: with the checks in Python and the C interface reached through ctypes a call cost 13 - 28 us of host time
// (encode 15.6, add_rmsnorm through its custom op 18.2, decode_sum of eight sources 23.7, reduce_reencode 24.6 - 31, a
// fused block 17.4, a GEMM 14.9), which is what every call of fewer than about 2000 rows then takes, several times the
// device time of its kernel.  What is left here is the allocation of the outputs and the launch itself.
//
// Loaded as the extension module `_fp4ar_front` (see `_native.front()`).  The C interface is bound at run time from the
// library that `_native.cuda()` loaded, so there is one copy of its state whatever FP4AR_LIBRARY names.
#include <Python.h>
#include <dlfcn.h>
#include <string>
#include <vector>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/library.h>
#include "../include/fp4ar.h"
#include "../include/fp4ar_gemm.h"
#include "../include/fp4ar_layer.h"

namespace {

using at::Tensor;

constexpr int64_t kHidden = FP4AR_HIDDEN, kQRow = FP4AR_QROW_BYTES, kMxRow = FP4AR_MXROW_BYTES, kRec = FP4AR_REC_STRIDE;
constexpr int64_t kValues = kHidden / 2;

// ---- the C interface ----
struct Api {
  decltype(&fp4ar_launch) launch;
  decltype(&fp4ar_last_cuda_error) last_error;
  decltype(&fp4ar_encode) encode;
  decltype(&fp4ar_encode_static) encode_static;
  decltype(&fp4ar_decode_sum) decode_sum;
  decltype(&fp4ar_reduce_reencode) reduce_reencode;
  decltype(&fp4ar_add_rmsnorm) add_rmsnorm;
  decltype(&fp4ar_gemm_nvfp4) gemm;
  decltype(&fp4ar_gated_linear) gated_linear;
  decltype(&fp4ar_gated_backward) gated_backward;
  decltype(&fp4ar_adapters_workspace) adapters_workspace;
  decltype(&fp4ar_linear_adapters) linear_adapters;
};
Api api{};
PyObject* check_rc = nullptr;      // _native.check(rc, what): raises the Python error of a return code

template <class F>
bool bind(void* lib, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(lib, name));
  return f != nullptr;
}

// ---- checks, with the messages users of the Python wrappers know ----
std::string dtype_name(at::ScalarType t) { return std::string("torch.") + torch::getTHPDtype(t)->name; }
std::string shape_text(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); i++) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}
[[noreturn]] void bad_layout(const Tensor& t, at::ScalarType dtype, int64_t cols, const char* name) {
  if (t.scalar_type() != dtype) TORCH_CHECK_VALUE(false, name, " must be ", dtype_name(dtype), ", got ", dtype_name(t.scalar_type()));
  if (cols >= 0 && (t.dim() != 2 || t.size(1) != cols))
    TORCH_CHECK_VALUE(false, name, " must have shape [rows, ", cols, "], got ", shape_text(t));
  if (!t.is_contiguous()) TORCH_CHECK_VALUE(false, name, " must be contiguous");
  TORCH_CHECK_VALUE(false, name, " must be a CUDA tensor");
}
inline bool layout_ok(const Tensor& t, at::ScalarType dtype, int64_t cols) {
  return t.scalar_type() == dtype && (cols < 0 || (t.dim() == 2 && t.size(1) == cols)) && t.is_contiguous();
}
inline void require(const Tensor& t, at::ScalarType dtype, int64_t cols, const char* name) {
  if (!layout_ok(t, dtype, cols) || !t.is_cuda()) bad_layout(t, dtype, cols, name);
}
// The kernels trust their pointers: every tensor of a call lives on the device that it is launched on.
inline void require_on(const Tensor& t, c10::Device dev, const char* name) {
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", the call runs on ", dev);
}

inline Tensor new_empty(at::IntArrayRef size, at::ScalarType dtype, c10::Device dev) {
  return Tensor(at::detail::empty_cuda(size, dtype, dev, std::nullopt));
}
inline fp4ar_stream stream_of(c10::Device dev) { return (fp4ar_stream)c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

void raise_rc(int rc, const char* what) {
  static const char* names[] = {"ok", "bad argument", "unsupported combination", "CUDA error", "context poisoned"};
  std::string msg = std::string(what) + " failed: " + (rc >= 0 && rc <= 4 ? std::string(names[rc]) : std::to_string(rc));
  if (rc == FP4AR_ERR_CUDA) msg += std::string(": ") + api.last_error();
  throw std::runtime_error(msg);
}
inline void ok(int rc, const char* what) {
  if (rc != FP4AR_OK) raise_rc(rc, what);
}

// Kernels write behind autograd's back: who has saved a tensor for a backward pass learns of it by the version.  (A tensor made under
// inference mode has none and cannot have been saved.)
inline void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---- one function per op: used by the Python entry points (GIL released) and by torch.ops ----
std::tuple<Tensor, Tensor> op_encode(const Tensor& x) {
  require(x, at::kBFloat16, kHidden, "x");
  const c10::Device dev = x.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t rows = x.size(0);
  Tensor q = new_empty({rows, kQRow}, at::kByte, dev), rs = new_empty({rows}, at::kFloat, dev);
  char* qp = (char*)q.mutable_data_ptr();
  ok(api.encode(x.data_ptr(), (int)rows, qp, kQRow, qp + kValues, kQRow, (float*)rs.mutable_data_ptr(), stream_of(dev)), "fp4ar_encode");
  return {std::move(q), std::move(rs)};
}

Tensor op_encode_static(const Tensor& x, double gs) {
  require(x, at::kBFloat16, kHidden, "x");
  const c10::Device dev = x.device();
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t rows = x.size(0);
  Tensor q = new_empty({rows, kQRow}, at::kByte, dev);
  ok(api.encode_static(x.data_ptr(), (int)rows, (float)gs, q.mutable_data_ptr(), stream_of(dev)), "fp4ar_encode_static");
  return q;
}

// Sources of a decode-sum; row_scales[i] undefined: the static scale gs[i].
struct Sources {
  int n = 0;
  int64_t pitch = 0, rows = 0;
  const void* src[FP4AR_MAX_RANKS];
  const float* rs[FP4AR_MAX_RANKS];
  float gs[FP4AR_MAX_RANKS] = {};
};
Sources sources(const std::vector<Tensor>& q, const std::vector<Tensor>& row_scales, const std::vector<double>& gs, bool have_gs) {
  Sources s;
  TORCH_CHECK_VALUE(!q.empty() && q.size() <= FP4AR_MAX_RANKS, "1..8 sources");
  s.n = (int)q.size();
  s.pitch = q[0].dim() == 2 ? q[0].size(1) : -1;
  if (s.pitch < 0) bad_layout(q[0], at::kByte, kQRow, "source");
  for (const Tensor& t : q) {
    require(t, at::kByte, s.pitch, "source");
    require_on(t, q[0].device(), "source");
    TORCH_CHECK_VALUE(t.sizes() == q[0].sizes(), "sources must have one shape");
  }
  TORCH_CHECK_VALUE(s.pitch == kQRow || s.pitch == kRec, "source rows must be 3456 B (NVFP4 rows) or 3584 B (receive records)");
  TORCH_CHECK_INDEX(row_scales.empty() || row_scales.size() >= q.size(), "list index out of range");
  s.rows = q[0].size(0);
  for (int i = 0; i < s.n; i++) {
    s.src[i] = q[i].data_ptr();
    s.rs[i] = nullptr;
    if (!row_scales.empty() && row_scales[i].defined()) {
      require(row_scales[i], at::kFloat, -1, "row_scales");
      require_on(row_scales[i], q[0].device(), "row_scales");
      TORCH_CHECK_VALUE(row_scales[i].numel() >= s.rows, "row_scales must have ", s.rows, " elements, got ", row_scales[i].numel());
      s.rs[i] = (const float*)row_scales[i].data_ptr();
    } else {
      TORCH_CHECK_VALUE(have_gs, "a source without row scales needs a static scale");
      s.gs[i] = (float)gs[i];
    }
  }
  return s;
}

Tensor op_decode_sum(const std::vector<Tensor>& q, const std::vector<Tensor>& row_scales, const std::vector<double>& gs, bool have_gs) {
  const Sources s = sources(q, row_scales, gs, have_gs);
  const c10::Device dev = q[0].device();
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = new_empty({s.rows, kHidden}, at::kBFloat16, dev);
  ok(api.decode_sum(s.n, s.src, s.pitch, s.rs, s.gs, (int)s.rows, out.mutable_data_ptr(), stream_of(dev)), "fp4ar_decode_sum");
  return out;
}

std::tuple<Tensor, Tensor> op_reduce_reencode(const std::vector<Tensor>& q, const std::vector<Tensor>& row_scales,
                                              const std::vector<double>& gs, bool have_gs) {
  const Sources s = sources(q, row_scales, gs, have_gs);
  const c10::Device dev = q[0].device();
  const c10::cuda::CUDAGuard guard(dev);
  Tensor rec = new_empty({s.rows, kRec}, at::kByte, dev);      // the kernel writes whole records, their zero tail included
  Tensor out = new_empty({s.rows, kHidden}, at::kBFloat16, dev);
  ok(api.reduce_reencode(s.n, s.src, s.pitch, s.rs, s.gs, (int)s.rows, rec.mutable_data_ptr(), out.mutable_data_ptr(), stream_of(dev)),
     "fp4ar_reduce_reencode");
  return {std::move(rec), std::move(out)};
}

// `out` undefined: allocated; given: any contiguous memory of the device that holds the rows.  `inplace`: the updated
// residual replaces `residual`.
std::tuple<Tensor, Tensor> op_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps, double weight_bias,
                                   int64_t epilogue, double qscale, bool inplace, Tensor out) {
  require(x, at::kBFloat16, kHidden, "x");
  require(residual, at::kBFloat16, kHidden, "residual");
  TORCH_CHECK_VALUE(weight.scalar_type() == at::kBFloat16 && weight.numel() == kHidden && weight.is_cuda() && weight.is_contiguous(),
                    "weight must be a contiguous CUDA BF16 tensor of 6144 elements");
  const int64_t rows = x.size(0);
  TORCH_CHECK_VALUE(residual.size(0) >= rows, "residual must have ", rows, " rows, got ", residual.size(0));
  TORCH_CHECK_VALUE(epilogue >= FP4AR_EPI_NORM_BF16 && epilogue <= FP4AR_EPI_NORM_MXFP8, "epilogue must be 1 (BF16), 2 (NVFP4) or 3 (MXFP8)");
  const c10::Device dev = x.device();
  require_on(residual, dev, "residual");
  require_on(weight, dev, "weight");
  const bool bf16 = epilogue == FP4AR_EPI_NORM_BF16;
  const int64_t cols = bf16 ? kHidden : epilogue == FP4AR_EPI_NORM_NVFP4 ? kQRow : kMxRow;
  if (out.defined()) {
    const int64_t bytes = rows * cols * (bf16 ? 2 : 1);
    TORCH_CHECK_VALUE(out.device() == dev && out.is_contiguous() && (int64_t)out.nbytes() >= bytes,
                      "out must be contiguous, on ", dev, " and hold ", bytes, " bytes");
  }
  const c10::cuda::CUDAGuard guard(dev);
  const bool given = out.defined();
  Tensor res_out = inplace ? residual : new_empty(residual.sizes(), at::kBFloat16, dev);
  if (!given) out = new_empty({rows, cols}, bf16 ? at::kBFloat16 : at::kByte, dev);
  void* op = out.mutable_data_ptr();
  ok(api.add_rmsnorm(x.data_ptr(), residual.data_ptr(), res_out.mutable_data_ptr(), weight.data_ptr(), (float)eps, (float)weight_bias,
                     (int)epilogue, (float)qscale, bf16 ? op : nullptr, bf16 ? nullptr : op, (int)rows, stream_of(dev)),
     "fp4ar_add_rmsnorm");
  if (given) written(out);
  if (inplace) written(res_out);
  return {std::move(out), std::move(res_out)};
}

std::tuple<Tensor, Tensor> op_gemm(const Tensor& x, const Tensor& wt, double gs, bool want_acc, Tensor q) {
  TORCH_CHECK_VALUE(x.is_cuda() && wt.is_cuda() && x.scalar_type() == at::kBFloat16 && wt.scalar_type() == at::kBFloat16,
                    "x and wt must be CUDA BF16 tensors");
  TORCH_CHECK_VALUE(x.dim() == 2 && wt.dim() == 2 && x.size(1) == wt.size(1) && x.is_contiguous() && wt.is_contiguous(),
                    "x [M, K] and wt [N, K] must be contiguous with equal K");
  const int64_t M = x.size(0), K = x.size(1), Nn = wt.size(0);
  TORCH_CHECK_VALUE(K % 64 == 0 && Nn % 256 == 0, "K must be a multiple of 64 and N a multiple of 256");
  const c10::Device dev = x.device();
  require_on(wt, dev, "wt");
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t qb = Nn / 2 + Nn / 16;
  const bool given = q.defined();
  if (!given) {
    q = new_empty({M, qb}, at::kByte, dev);
  } else {
    TORCH_CHECK_VALUE(layout_ok(q, at::kByte, qb) && q.size(0) == M && q.device() == dev,
                      "out must be a contiguous uint8 [M, N/2 + N/16] tensor on the device of x");
  }
  Tensor acc;
  if (want_acc) acc = new_empty({M, Nn}, at::kFloat, dev);
  ok(api.gemm(nullptr, 0, x.data_ptr(), wt.data_ptr(), (int)M, (int)Nn, (int)K, (float)gs, q.mutable_data_ptr(),
              want_acc ? (float*)acc.mutable_data_ptr() : nullptr, stream_of(dev)), "fp4ar_gemm_nvfp4");
  if (given) written(q);
  return {std::move(q), std::move(acc)};
}

// ---- gated projections, adapters ----
// A contiguous tensor of this shape that the tensor maps can describe.
void require_matrix(const Tensor& t, at::ScalarType dtype, at::IntArrayRef shape, c10::Device dev, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == dtype, name, " must be ", dtype_name(dtype), ", got ", dtype_name(t.scalar_type()));
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", shape_text(t));
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  require_on(t, dev, name);
  TORCH_CHECK_VALUE((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 || t.numel() == 0, name, " must start on a 16-byte boundary");
}
void require_apart(const Tensor& out, const Tensor& in, const char* name) {
  const char *a = (const char*)out.data_ptr(), *b = (const char*)in.data_ptr();
  TORCH_CHECK_VALUE(out.numel() == 0 || in.numel() == 0 || a + out.nbytes() <= b || b + in.nbytes() <= a, "out must not overlap ", name);
}
// Rows and columns as the C interface takes them: 32-bit, with room for a tile.
void require_size(int64_t n, const char* name) { TORCH_CHECK_VALUE(n <= 0x7fff0000, name, " is too large: ", n); }

bool recording(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Values with a gradient of their own are not written over: it would go on to whoever made them.
void require_no_history(const Tensor& out) { TORCH_CHECK_VALUE(!recording({&out}), "out must not require a gradient"); }
// A tangent that a kernel does not see would be lost: torch takes a result without one as constant.
void require_no_tangent(std::initializer_list<const Tensor*> ts, const char* op) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error(std::string(op) + " has no forward-mode derivative");
}

struct GatedShape {
  int64_t M, K, F;
  GatedShape(const Tensor& x, const Tensor& wt, int64_t act) {
    TORCH_CHECK_VALUE(x.dim() == 2, "x must have shape [rows, K], got ", shape_text(x));
    TORCH_CHECK_VALUE(wt.dim() == 2 && wt.size(1) == x.size(1), "wt must have shape [2 F, ", x.size(1), "], got ", shape_text(wt));
    M = x.size(0); K = x.size(1); F = wt.size(0) / 2;
    TORCH_CHECK_VALUE(K >= 8 && K % 8 == 0, "K must be a positive multiple of 8, got ", K);
    TORCH_CHECK_VALUE(F >= 8 && wt.size(0) % 16 == 0, "wt must have 2 F rows, F a positive multiple of 8, got ", wt.size(0), " rows");
    TORCH_CHECK_VALUE(act >= FP4AR_ACT_SILU && act <= FP4AR_ACT_GELU_TANH, "activation must be 0 (silu), 1 (gelu) or 2 (gelu_tanh)");
    require_size(M, "rows"); require_size(K, "K"); require_size(2 * F, "2 F");
    require_matrix(x, at::kBFloat16, {M, K}, x.device(), "x");
    require_matrix(wt, at::kBFloat16, {2 * F, K}, x.device(), "wt");
  }
};

std::tuple<Tensor, Tensor> op_gated_linear(const Tensor& x, const Tensor& wt, int64_t act, bool want_pre, Tensor out) {
  require_no_tangent({&x, &wt, &out}, "gated_linear");
  require_no_history(out);
  const GatedShape s(x, wt, act);
  const c10::Device dev = x.device();
  if (out.defined()) {
    require_matrix(out, at::kBFloat16, {s.M, s.F}, dev, "out");
    require_apart(out, x, "x");
    require_apart(out, wt, "wt");
  }
  const c10::cuda::CUDAGuard guard(dev);
  const bool given = out.defined();
  if (!given) out = new_empty({s.M, s.F}, at::kBFloat16, dev);
  Tensor pre;
  if (want_pre) pre = new_empty({s.M, 2 * s.F}, at::kFloat, dev);
  ok(api.gated_linear(x.data_ptr(), wt.data_ptr(), (int)s.M, (int)s.F, (int)s.K, (int)act, out.mutable_data_ptr(),
                      want_pre ? pre.mutable_data_ptr() : nullptr, stream_of(dev)), "fp4ar_gated_linear");
  if (given) written(out);
  return {std::move(out), std::move(pre)};
}

std::tuple<Tensor, Tensor> op_gated_backward(const Tensor& dh_, const Tensor& pre, const Tensor& x, const Tensor& wt, int64_t act, bool need_dx,
                                             bool need_dw) {
  require_no_tangent({&dh_, &pre, &x, &wt}, "gated_linear");
  const GatedShape s(x, wt, act);
  const c10::Device dev = x.device();
  TORCH_CHECK_VALUE(dh_.dim() == 2 && dh_.size(0) == s.M && dh_.size(1) == s.F, "dh must have shape [", s.M, ", ", s.F, "], got ", shape_text(dh_));
  require_on(dh_, dev, "dh");
  const c10::cuda::CUDAGuard guard(dev);
  // a gradient comes as autograd made it: any strides, any place in its storage
  Tensor dh = dh_.contiguous();
  if (reinterpret_cast<uintptr_t>(dh.data_ptr()) & 15) dh = dh.clone();
  require_matrix(dh, at::kBFloat16, {s.M, s.F}, dev, "dh");
  require_matrix(pre, at::kFloat, {s.M, 2 * s.F}, dev, "pre");
  Tensor dx, dw;
  if (!need_dx && !need_dw) return {dx, dw};
  if (need_dx) dx = new_empty({s.M, s.K}, at::kBFloat16, dev);
  if (need_dw) dw = new_empty({2 * s.F, s.K}, at::kBFloat16, dev);
  Tensor dpre = new_empty({s.M, 2 * s.F}, at::kBFloat16, dev);
  ok(api.gated_backward(dh.data_ptr(), pre.data_ptr(), x.data_ptr(), wt.data_ptr(), (int)s.M, (int)s.F, (int)s.K, (int)act,
                        dpre.mutable_data_ptr(), need_dx ? dx.mutable_data_ptr() : nullptr, need_dw ? dw.mutable_data_ptr() : nullptr,
                        stream_of(dev)), "fp4ar_gated_backward");
  return {std::move(dx), std::move(dw)};
}

// Records h for autograd: 12 us of host time for both passes beside the autograd engine's own (as a Python function 30).
struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& wt, int64_t act) {
    auto r = op_gated_linear(x, wt, act, true, Tensor());
    ctx->save_for_backward({x, wt, std::get<1>(r)});
    ctx->saved_data["activation"] = act;
    return std::get<0>(r);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto r = op_gated_backward(grads[0], saved[2], saved[0], saved[1], ctx->saved_data["activation"].toInt(), ctx->needs_input_grad(0),
                               ctx->needs_input_grad(1));
    torch::autograd::variable_list out{std::move(std::get<0>(r)), std::move(std::get<1>(r))};
    if (at::GradMode::is_enabled()) {            // create_graph: the gradients cannot be differentiated again, and say so on every way back
      auto refuses = std::make_shared<torch::autograd::Error>("gated_linear cannot be differentiated twice",
                                                              torch::autograd::collect_next_edges(grads[0], saved[0], saved[1]));
      for (const Tensor& t : out)
        if (t.defined()) torch::autograd::set_history(t, refuses);
    }
    out.emplace_back();
    return out;
  }
};
// h, recorded where autograd records
Tensor op_gated_linear_auto(const Tensor& x, const Tensor& wt, int64_t act, Tensor out) {
  if (!recording({&x, &wt})) return std::get<0>(op_gated_linear(x, wt, act, false, std::move(out)));
  require_no_tangent({&x, &wt}, "gated_linear");            // (forward mode is off inside the recorded function)
  TORCH_CHECK_VALUE(!out.defined(), "out cannot be given where a gradient is recorded");
  return GatedLinear::apply(x, wt, act);
}

void require_no_recording(std::initializer_list<const Tensor*> ts) {
  if (recording(ts)) throw std::runtime_error("linear_adapters has no backward pass: call it under torch.no_grad() or on detached tensors");
}
Tensor op_linear_adapters(const Tensor& x, const Tensor& wt, const Tensor& ids, const Tensor& a, const Tensor& b, const Tensor& scales, Tensor out) {
  require_no_tangent({&x, &wt, &a, &b, &scales, &out}, "linear_adapters");
  require_no_history(out);
  TORCH_CHECK_VALUE(x.dim() == 2, "x must have shape [rows, K], got ", shape_text(x));
  TORCH_CHECK_VALUE(wt.dim() == 2 && wt.size(1) == x.size(1), "wt must have shape [N, ", x.size(1), "], got ", shape_text(wt));
  const int64_t M = x.size(0), K = x.size(1), Nn = wt.size(0);
  TORCH_CHECK_VALUE(K >= 8 && K % 8 == 0 && Nn >= 8 && Nn % 8 == 0, "K and N must be positive multiples of 8, got ", K, " and ", Nn);
  TORCH_CHECK_VALUE(a.dim() == 3 && a.size(2) == K, "a must have shape [adapters, R, ", K, "], got ", shape_text(a));
  const int64_t n = a.size(0), R = a.size(1);
  TORCH_CHECK_VALUE(n >= 1, "a must hold at least one adapter");
  TORCH_CHECK_VALUE(R >= 8 && R % 8 == 0 && R <= 128, "the rank must be a multiple of 8 up to 128 (pad with zeros), got ", R);
  require_size(M, "rows"); require_size(K, "K"); require_size(n * Nn, "adapters x N"); require_size(n * R, "adapters x R");
  const c10::Device dev = x.device();
  require_matrix(x, at::kBFloat16, {M, K}, dev, "x");
  require_matrix(wt, at::kBFloat16, {Nn, K}, dev, "wt");
  require_matrix(a, at::kBFloat16, {n, R, K}, dev, "a");
  require_matrix(b, at::kBFloat16, {n, Nn, R}, dev, "b");
  require(ids, at::kInt, -1, "ids");
  TORCH_CHECK_VALUE(ids.dim() == 1 && ids.size(0) == M, "ids must have shape (", M, ",), got ", shape_text(ids));
  require_on(ids, dev, "ids");
  if (scales.defined()) {
    require(scales, at::kFloat, -1, "scales");
    TORCH_CHECK_VALUE(scales.dim() == 1 && scales.size(0) == n, "scales must have shape (", n, ",), got ", shape_text(scales));
    require_on(scales, dev, "scales");
  }
  if (out.defined()) {
    require_matrix(out, at::kBFloat16, {M, Nn}, dev, "out");
    require_apart(out, x, "x"); require_apart(out, wt, "wt"); require_apart(out, ids, "ids");
    require_apart(out, a, "a"); require_apart(out, b, "b");
    if (scales.defined()) require_apart(out, scales, "scales");
  }
  const c10::cuda::CUDAGuard guard(dev);
  const bool given = out.defined();
  if (!given) out = new_empty({M, Nn}, at::kBFloat16, dev);
  Tensor ws = new_empty({(int64_t)api.adapters_workspace((int)M, (int)R, (int)n)}, at::kByte, dev);
  ok(api.linear_adapters(x.data_ptr(), wt.data_ptr(), (const int*)ids.data_ptr(), a.data_ptr(), b.data_ptr(),
                         scales.defined() ? (const float*)scales.data_ptr() : nullptr, (int)M, (int)Nn, (int)K, (int)R, (int)n,
                         ws.mutable_data_ptr(), out.mutable_data_ptr(), stream_of(dev)), "fp4ar_linear_adapters");
  if (given) written(out);
  return out;
}

// ---- torch.ops.fp4ar.* (the schemas are defined in ops/allreduce.py) ----
Tensor lib_decode_sum(const std::vector<Tensor>& q, const std::vector<Tensor>& rs) { return op_decode_sum(q, rs, {}, false); }
Tensor lib_add_rms_norm(const Tensor& x, Tensor& residual, const Tensor& weight, double eps, double weight_bias) {
  return std::get<0>(op_norm(x, residual, weight, eps, weight_bias, FP4AR_EPI_NORM_BF16, 1.0, true, Tensor()));
}
Tensor lib_linear(const Tensor& x, const Tensor& wt, double gs) { return std::get<0>(op_gemm(x, wt, gs, false, Tensor())); }

Tensor lib_gated_linear(const Tensor& x, const Tensor& wt, int64_t act) { return std::get<0>(op_gated_linear(x, wt, act, false, Tensor())); }
std::tuple<Tensor, Tensor> lib_gated_linear_pre(const Tensor& x, const Tensor& wt, int64_t act) { return op_gated_linear(x, wt, act, true, Tensor()); }
std::tuple<Tensor, Tensor> lib_gated_linear_backward(const Tensor& dh, const Tensor& pre, const Tensor& x, const Tensor& wt, int64_t act, bool need_dx,
                                                     bool need_dw) {
  auto r = op_gated_backward(dh, pre, x, wt, act, need_dx, need_dw);
  const auto none = [&](Tensor& t) { if (!t.defined()) t = new_empty({0}, at::kBFloat16, x.device()); };
  none(std::get<0>(r));
  none(std::get<1>(r));
  return r;
}
Tensor lib_linear_adapters(const Tensor& x, const Tensor& wt, const Tensor& ids, const Tensor& a, const Tensor& b, const std::optional<Tensor>& scales) {
  return op_linear_adapters(x, wt, ids, a, b, scales ? *scales : Tensor(), Tensor());
}
// Its autograd kernel, on every device: without one torch's fallback would record the call and deliver no gradient.
Tensor lib_linear_adapters_autograd(c10::DispatchKeySet keys, const Tensor& x, const Tensor& wt, const Tensor& ids, const Tensor& a, const Tensor& b,
                                    const std::optional<Tensor>& scales) {
  const Tensor none;
  require_no_recording({&x, &wt, &a, &b, scales ? &*scales : &none});
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fp4ar::linear_adapters", "").typed<decltype(lib_linear_adapters)>();
  const at::AutoDispatchBelowAutograd below;
  return op.redispatch(keys & c10::after_autograd_keyset, x, wt, ids, a, b, scales);
}
// Autograd kernel of the two parts of the backward pass: they can be recorded (a gradient taken with create_graph=True, or a call of their
// own), and whoever differentiates them hears that their derivatives do not exist.  Without it torch's fallback would leave those
// out of the sums with no more than a warning.  (In Python it took 7 us of host time a call.)
void lib_refuse_gradients(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  torch::autograd::edge_list edges;
  if (at::GradMode::is_enabled()) {
    for (size_t n = op.schema().arguments().size(), i = stack->size() - n; i < stack->size(); i++)
      if ((*stack)[i].isTensor() && (*stack)[i].toTensor().requires_grad())
        edges.push_back(torch::autograd::impl::gradient_edge((*stack)[i].toTensor()));
  }
  {
    const at::AutoDispatchBelowAutograd below;
    op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
  }
  if (edges.empty()) return;
  const bool forward = op.schema().name() == "fp4ar::gated_linear_pre";
  auto refuses = std::make_shared<torch::autograd::Error>(forward ? "gated_linear_pre records no gradient: differentiate gated_linear"
                                                                  : "gated_linear cannot be differentiated twice", std::move(edges));
  for (size_t n = op.schema().returns().size(), i = stack->size() - n; i < stack->size(); i++) torch::autograd::set_history((*stack)[i].toTensor(), refuses);
}

// Between autograd and the kernels of any device, for the ops above: no tangent gets past here.
void lib_refuse_tangents(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  for (size_t n = op.schema().arguments().size(), i = stack->size() - n; i < stack->size(); i++)
    if ((*stack)[i].isTensor()) require_no_tangent({&(*stack)[i].toTensor()}, op.schema().name().c_str() + sizeof("fp4ar::") - 1);
  const at::AutoDispatchBelowADInplaceOrView below;
  op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
}

// ---- Python entry points: positional arguments only, the wrappers fill in the defaults ----
const Tensor& tensor_arg(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw torch::TypeError(std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
double double_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int64_t int_arg(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
void arity(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) throw torch::TypeError("expected " + std::to_string(want) + " arguments, got " + std::to_string(got));
}
PyObject* wrap2(Tensor a, Tensor b) {
  THPObjectPtr t(PyTuple_New(2));
  if (!t) throw python_error();
  PyTuple_SET_ITEM(t.get(), 0, THPVariable_Wrap(std::move(a)));
  PyTuple_SET_ITEM(t.get(), 1, THPVariable_Wrap(std::move(b)));
  return t.release();
}
struct NoGil {
  PyThreadState* s = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(s); }
};

PyObject* py_encode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 1);
  const Tensor& x = tensor_arg(a[0], "x");
  auto r = [&] { NoGil g; return op_encode(x); }();
  return wrap2(std::move(std::get<0>(r)), std::move(std::get<1>(r)));
  END_HANDLE_TH_ERRORS
}
PyObject* py_encode_static(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 2);
  const Tensor& x = tensor_arg(a[0], "x");
  const double gs = double_arg(a[1]);
  return THPVariable_Wrap([&] { NoGil g; return op_encode_static(x, gs); }());
  END_HANDLE_TH_ERRORS
}
template <class F>
void each(PyObject* seq, F&& f) {
  THPObjectPtr fast(PySequence_Fast(seq, "expected a sequence"));
  if (!fast) throw python_error();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast.get());
  for (Py_ssize_t i = 0; i < n; i++) f(PySequence_Fast_GET_ITEM(fast.get(), i));
}
// (qrows, row_scales or None, gs or None).  Only the static scales of sources without row scales are looked at: the entries
// of the others may be anything, None among them.
struct SourceArgs {
  std::vector<Tensor> q, rs;
  std::vector<double> gs;
  bool have_gs;
  SourceArgs(PyObject* const* a) : have_gs(a[2] != Py_None) {
    q.reserve(FP4AR_MAX_RANKS);
    each(a[0], [&](PyObject* o) { q.push_back(tensor_arg(o, "source")); });
    if (a[1] != Py_None) {
      rs.reserve(FP4AR_MAX_RANKS);
      each(a[1], [&](PyObject* o) { if (o == Py_None) rs.emplace_back(); else rs.push_back(tensor_arg(o, "row_scales")); });
    }
    if (!have_gs) return;
    gs.resize(q.size());
    for (size_t i = 0; i < q.size(); i++) {
      if (a[1] != Py_None && (i >= rs.size() || rs[i].defined())) continue;
      THPObjectPtr key(PyLong_FromSize_t(i)), item(key ? PyObject_GetItem(a[2], key.get()) : nullptr);
      if (!item) throw python_error();
      gs[i] = double_arg(item.get());
    }
  }
};
PyObject* py_decode_sum(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 3);
  const SourceArgs s(a);
  return THPVariable_Wrap([&] { NoGil g; return op_decode_sum(s.q, s.rs, s.gs, s.have_gs); }());
  END_HANDLE_TH_ERRORS
}
PyObject* py_reduce_reencode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 3);
  const SourceArgs s(a);
  auto r = [&] { NoGil g; return op_reduce_reencode(s.q, s.rs, s.gs, s.have_gs); }();
  return wrap2(std::move(std::get<0>(r)), std::move(std::get<1>(r)));
  END_HANDLE_TH_ERRORS
}
// (x, residual, weight, eps, weight_bias, epilogue, qscale, inplace_residual, out or None)
PyObject* py_add_rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 9);
  const Tensor &x = tensor_arg(a[0], "x"), &res = tensor_arg(a[1], "residual"), &w = tensor_arg(a[2], "weight");
  const double eps = double_arg(a[3]), wb = double_arg(a[4]), qs = double_arg(a[6]);
  const int64_t epi = int_arg(a[5]);
  const bool inplace = bool_arg(a[7]);
  Tensor out = a[8] == Py_None ? Tensor() : tensor_arg(a[8], "out");
  auto r = [&] { NoGil g; return op_norm(x, res, w, eps, wb, epi, qs, inplace, std::move(out)); }();
  return wrap2(std::move(std::get<0>(r)), std::move(std::get<1>(r)));
  END_HANDLE_TH_ERRORS
}
// (x, wt, gs, want_acc, out or None): q, or (q, acc)
PyObject* py_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 5);
  const Tensor &x = tensor_arg(a[0], "x"), &wt = tensor_arg(a[1], "wt");
  const double gs = double_arg(a[2]);
  const bool acc = bool_arg(a[3]);
  Tensor out = a[4] == Py_None ? Tensor() : tensor_arg(a[4], "out");
  auto r = [&] { NoGil g; return op_gemm(x, wt, gs, acc, std::move(out)); }();
  if (!acc) return THPVariable_Wrap(std::move(std::get<0>(r)));
  return wrap2(std::move(std::get<0>(r)), std::move(std::get<1>(r)));
  END_HANDLE_TH_ERRORS
}
PyObject* wrap_or_none(Tensor t) {
  if (t.defined()) return THPVariable_Wrap(std::move(t));
  Py_RETURN_NONE;
}
PyObject* wrap2_or_none(std::tuple<Tensor, Tensor> r) {
  THPObjectPtr t(PyTuple_New(2));
  if (!t) throw python_error();
  PyTuple_SET_ITEM(t.get(), 0, wrap_or_none(std::move(std::get<0>(r))));
  PyTuple_SET_ITEM(t.get(), 1, wrap_or_none(std::move(std::get<1>(r))));
  return t.release();
}
// (x, wt, activation, out or None): (h, pre)
PyObject* py_gated_linear_pre(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 4);
  const Tensor &x = tensor_arg(a[0], "x"), &wt = tensor_arg(a[1], "wt");
  const int64_t act = int_arg(a[2]);
  Tensor out = a[3] == Py_None ? Tensor() : tensor_arg(a[3], "out");
  return wrap2_or_none([&] { NoGil g; return op_gated_linear(x, wt, act, true, std::move(out)); }());
  END_HANDLE_TH_ERRORS
}
// (x, wt, activation, out or None): h, recorded where autograd records
PyObject* py_gated_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 4);
  const Tensor &x = tensor_arg(a[0], "x"), &wt = tensor_arg(a[1], "wt");
  const int64_t act = int_arg(a[2]);
  Tensor out = a[3] == Py_None ? Tensor() : tensor_arg(a[3], "out");
  return THPVariable_Wrap([&] { NoGil g; return op_gated_linear_auto(x, wt, act, std::move(out)); }());
  END_HANDLE_TH_ERRORS
}
// (dh, pre, x, wt, activation, need_dx, need_dw): (dx or None, dwt or None)
PyObject* py_gated_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 7);
  const Tensor &dh = tensor_arg(a[0], "dh"), &pre = tensor_arg(a[1], "pre"), &x = tensor_arg(a[2], "x"), &wt = tensor_arg(a[3], "wt");
  const int64_t act = int_arg(a[4]);
  const bool dx = bool_arg(a[5]), dw = bool_arg(a[6]);
  return wrap2_or_none([&] { NoGil g; return op_gated_backward(dh, pre, x, wt, act, dx, dw); }());
  END_HANDLE_TH_ERRORS
}
// (x, wt, ids, a, b, scales or None, out or None)
PyObject* py_linear_adapters(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 7);
  const Tensor &x = tensor_arg(p[0], "x"), &wt = tensor_arg(p[1], "wt"), &ids = tensor_arg(p[2], "ids"), &a = tensor_arg(p[3], "a"),
               &b = tensor_arg(p[4], "b");
  const Tensor scales = p[5] == Py_None ? Tensor() : tensor_arg(p[5], "scales");
  Tensor out = p[6] == Py_None ? Tensor() : tensor_arg(p[6], "out");
  require_no_recording({&x, &wt, &a, &b, &scales});
  return THPVariable_Wrap([&] { NoGil g; return op_linear_adapters(x, wt, ids, a, b, scales, std::move(out)); }());
  END_HANDLE_TH_ERRORS
}

// ---- fused calls of a context ----
// Holds what a call needs of an Fp4ArContext.  Its methods take the plain, valid call and return None for everything
// else (an argument that does not fit, a tensor subclass): the Python wrapper then goes through its own checks, which
// name what is wrong.
struct FrontContext {
  PyObject_HEAD
  fp4ar_ctx* ctx;
  int nranks, device, compute_only;
  int64_t max_rows;
};

inline const Tensor* plain(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }
inline bool on(const Tensor& t, int device) { return t.is_cuda() && t.device().index() == device; }
inline bool rows_ok(const Tensor* t, at::ScalarType dtype, int64_t rows, int64_t cols, int device) {
  return t && layout_ok(*t, dtype, cols) && t->size(0) == rows && on(*t, device);
}
inline bool get_int(PyObject* o, int& v) {
  if (!PyLong_Check(o)) return false;
  int over = 0;
  const long l = PyLong_AsLongAndOverflow(o, &over);
  v = (int)l;
  return !over && l == (long)v;
}
inline bool get_float(PyObject* o, float& v) {
  if (PyFloat_Check(o)) {
    v = (float)PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (!PyLong_CheckExact(o)) return false;
  const double d = PyLong_AsDouble(o);
  v = (float)d;
  if (d != -1.0 || !PyErr_Occurred()) return true;
  PyErr_Clear();                 // beyond a double: the Python wrapper raises it
  return false;
}

// The input (BF16 rows or NVFP4 rows with one positive scale per rank) and the options every call has.
bool call_input(const FrontContext* c, PyObject* x_, PyObject* gs, PyObject* algo, PyObject* mode, PyObject* teams, fp4ar_args& a,
                const Tensor*& x) {
  x = plain(x_);
  if (!x || !on(*x, c->device) || !x->is_contiguous() || x->dim() != 2 || x->size(0) > c->max_rows) return false;
  if (x->scalar_type() == at::kBFloat16 && x->size(1) == kHidden) a.input = FP4AR_IN_BF16;
  else if (x->scalar_type() == at::kByte && x->size(1) == kQRow) a.input = FP4AR_IN_NVFP4;
  else return false;
  for (float& g : a.gs) g = 1.0f;
  if (a.input == FP4AR_IN_NVFP4) {
    if (!PyList_Check(gs) && !PyTuple_Check(gs)) return false;
    if (PySequence_Fast_GET_SIZE(gs) != c->nranks) return false;
    for (int r = 0; r < c->nranks; r++)
      if (!get_float(PySequence_Fast_GET_ITEM(gs, r), a.gs[r]) || !(a.gs[r] > 0.0f)) return false;
  }
  if (!get_int(algo, a.algo) || !get_int(mode, a.mode) || !get_int(teams, a.tune[0])) return false;
  if (c->compute_only && a.mode != FP4AR_MODE_COMPUTE) return false;
  a.x = x->data_ptr();
  a.rows = (int)x->size(0);
  a.hidden = FP4AR_HIDDEN;
  return true;
}
int launch(const FrontContext* c, const fp4ar_args& a) {
  NoGil g;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)c->device);
  return api.launch(c->ctx, &a, stream_of(c10::Device(c10::kCUDA, (c10::DeviceIndex)c->device)));
}
void launched(int rc) {
  if (rc == FP4AR_OK) return;
  THPObjectPtr r(PyObject_CallFunction(check_rc, "is", rc, "fp4ar_launch"));
  if (!r) throw python_error();
}

// (x, out or None, gs or None, algo, mode, teams)
PyObject* ctx_all_reduce(PyObject* self, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 6);
  const FrontContext* c = (const FrontContext*)self;
  fp4ar_args a{};
  const Tensor* x;
  if (!call_input(c, p[0], p[2], p[3], p[4], p[5], a, x)) Py_RETURN_NONE;
  Tensor out;
  if (p[1] == Py_None) {
    out = new_empty({a.rows, kHidden}, at::kBFloat16, x->device());
  } else {
    if (!rows_ok(plain(p[1]), at::kBFloat16, a.rows, kHidden, c->device)) Py_RETURN_NONE;
    out = THPVariable_Unpack(p[1]);
  }
  a.out = out.mutable_data_ptr();
  launched(launch(c, a));
  if (p[1] != Py_None) written(out);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}
// (x, residual, weight, eps, weight_bias, epilogue, qscale, gs or None, algo, out or None, residual_out or None, mode, teams)
PyObject* ctx_block(PyObject* self, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 13);
  const FrontContext* c = (const FrontContext*)self;
  fp4ar_args a{};
  const Tensor* x;
  if (!call_input(c, p[0], p[7], p[8], p[11], p[12], a, x)) Py_RETURN_NONE;
  if (!get_float(p[3], a.eps) || !get_float(p[4], a.weight_bias) || !get_int(p[5], a.epilogue) || !get_float(p[6], a.qscale)) Py_RETURN_NONE;
  if (a.epilogue < FP4AR_EPI_NORM_BF16 || a.epilogue > FP4AR_EPI_NORM_MXFP8) Py_RETURN_NONE;
  const Tensor *res = plain(p[1]), *w = plain(p[2]);
  if (!rows_ok(res, at::kBFloat16, a.rows, kHidden, c->device)) Py_RETURN_NONE;
  if (!w || w->scalar_type() != at::kBFloat16 || w->numel() != kHidden || !w->is_contiguous() || !on(*w, c->device)) Py_RETURN_NONE;
  const Tensor* res_out = p[10] == Py_None ? res : plain(p[10]);
  if (res_out != res && !rows_ok(res_out, at::kBFloat16, a.rows, kHidden, c->device)) Py_RETURN_NONE;
  const bool bf16 = a.epilogue == FP4AR_EPI_NORM_BF16;
  const int64_t cols = bf16 ? kHidden : (a.epilogue == FP4AR_EPI_NORM_NVFP4 ? kQRow : kMxRow);
  const at::ScalarType dtype = bf16 ? at::kBFloat16 : at::kByte;
  Tensor out;
  if (p[9] == Py_None) {
    out = new_empty({a.rows, cols}, dtype, x->device());
  } else {
    if (!rows_ok(plain(p[9]), dtype, a.rows, cols, c->device)) Py_RETURN_NONE;
    out = THPVariable_Unpack(p[9]);
  }
  (bf16 ? a.out : a.outq) = out.mutable_data_ptr();
  a.res_in = res->data_ptr();
  a.res_out = res_out->mutable_data_ptr();
  a.weight = w->data_ptr();
  launched(launch(c, a));
  if (p[9] != Py_None) written(out);
  written(*res_out);
  return wrap2(std::move(out), *res_out);
  END_HANDLE_TH_ERRORS
}

PyObject* ctx_new(PyTypeObject* type, PyObject* args, PyObject*) {
  unsigned long long ptr;
  int nranks, device, compute_only;
  long long max_rows;
  if (!PyArg_ParseTuple(args, "KiLip", &ptr, &nranks, &max_rows, &device, &compute_only)) return nullptr;
  FrontContext* c = (FrontContext*)type->tp_alloc(type, 0);
  if (!c) return nullptr;
  c->ctx = (fp4ar_ctx*)(uintptr_t)ptr;
  c->nranks = nranks; c->device = device; c->compute_only = compute_only; c->max_rows = max_rows;
  return (PyObject*)c;
}
PyMethodDef ctx_methods[] = {
    {"all_reduce", (PyCFunction)(void (*)(void))ctx_all_reduce, METH_FASTCALL, nullptr},
    {"block", (PyCFunction)(void (*)(void))ctx_block, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyTypeObject ctx_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

// (library path, _native.check): binds the C interface
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 2);
  const char* path = PyUnicode_AsUTF8(a[0]);
  if (!path) throw python_error();
  void* lib = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!lib) throw std::runtime_error(std::string("cannot load ") + path + ": " + dlerror());
  const bool all = bind(lib, "fp4ar_launch", api.launch) && bind(lib, "fp4ar_last_cuda_error", api.last_error) &&
                   bind(lib, "fp4ar_encode", api.encode) && bind(lib, "fp4ar_encode_static", api.encode_static) &&
                   bind(lib, "fp4ar_decode_sum", api.decode_sum) && bind(lib, "fp4ar_reduce_reencode", api.reduce_reencode) &&
                   bind(lib, "fp4ar_add_rmsnorm", api.add_rmsnorm) && bind(lib, "fp4ar_gemm_nvfp4", api.gemm) &&
                   bind(lib, "fp4ar_gated_linear", api.gated_linear) && bind(lib, "fp4ar_gated_backward", api.gated_backward) &&
                   bind(lib, "fp4ar_adapters_workspace", api.adapters_workspace) && bind(lib, "fp4ar_linear_adapters", api.linear_adapters);
  if (!all) throw std::runtime_error(std::string(path) + " lacks a function of the C interface");
  Py_INCREF(a[1]);
  Py_XSETREF(check_rc, a[1]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define FP4AR_METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FP4AR_METHOD(bind), FP4AR_METHOD(encode), FP4AR_METHOD(encode_static), FP4AR_METHOD(decode_sum),
                         FP4AR_METHOD(reduce_reencode), FP4AR_METHOD(add_rmsnorm), FP4AR_METHOD(gemm), FP4AR_METHOD(gated_linear), FP4AR_METHOD(gated_linear_pre), FP4AR_METHOD(gated_backward),
                         FP4AR_METHOD(linear_adapters), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fp4ar_front", nullptr, -1, methods};

}  // namespace

TORCH_LIBRARY_IMPL(fp4ar, CUDA, m) {
  m.impl("encode", op_encode);
  m.impl("encode_static", op_encode_static);
  m.impl("decode_sum", lib_decode_sum);
  m.impl("add_rms_norm", lib_add_rms_norm);
  m.impl("linear_nvfp4", lib_linear);
  m.impl("gated_linear", lib_gated_linear);
  m.impl("gated_linear_pre", lib_gated_linear_pre);
  m.impl("gated_linear_backward", lib_gated_linear_backward);
  m.impl("linear_adapters", lib_linear_adapters);
}
TORCH_LIBRARY_IMPL(fp4ar, ADInplaceOrView, m) {
  for (const char* op : {"gated_linear", "gated_linear_pre", "gated_linear_backward", "linear_adapters"})
    m.impl(op, torch::CppFunction::makeFromBoxedFunction<&lib_refuse_tangents>());
}
TORCH_LIBRARY_IMPL(fp4ar, Autograd, m) {
  m.impl("linear_adapters", TORCH_FN(lib_linear_adapters_autograd));
  for (const char* op : {"gated_linear_pre", "gated_linear_backward"}) m.impl(op, torch::CppFunction::makeFromBoxedFunction<&lib_refuse_gradients>());
}

PyMODINIT_FUNC PyInit__fp4ar_front() {
  ctx_type.tp_name = "_fp4ar_front.Context";
  ctx_type.tp_basicsize = sizeof(FrontContext);
  ctx_type.tp_flags = Py_TPFLAGS_DEFAULT;
  ctx_type.tp_methods = ctx_methods;
  ctx_type.tp_new = ctx_new;
  if (PyType_Ready(&ctx_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  Py_INCREF(&ctx_type);
  if (PyModule_AddObject(m, "Context", (PyObject*)&ctx_type) < 0) return nullptr;
  return m;
}
