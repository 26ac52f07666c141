// Host side of the norm, the gated feed-forward block, the AdamW step, windowed
// attention, the scan's token step and the choice of tokens: a Python extension
// over the C ABI (include/thetascan_b200.h).
//
// These operators are called with few rows (a decoding step) or many small
// tensors (an optimizer step), where the host's share of a call exceeds the
// GPU's.  Checks of arguments, allocation of outputs and workspaces, the
// filling of the ABI's structs and the autograd nodes are therefore C++; a call
// takes 5-10 us instead of the 30-40 us of the same steps in Python.  Nothing
// is kept between calls.  Every function works on the current stream of the
// device of its tensors and returns without waiting.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <climits>
#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "../../include/thetascan_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kGroup = 128, kStateBlock = 256;

void check(int code) {
  if (code == TS_OK) return;
  char text[512];
  ts_b200_last_error(text, sizeof(text));
  TORCH_CHECK_VALUE(code != TS_ERR_VALUE, text);
  TORCH_CHECK_NOT_IMPLEMENTED(code != TS_ERR_NOT_IMPLEMENTED, text);
  TORCH_CHECK(false, text);
}

ts_stream_t current_stream(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// Forward-mode derivatives are not formed here: the result would have none, which reads as zero.
void refuse_tangent(const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
                              name, " carries a forward-mode derivative, which is not supported");
}

void require_cuda(const char* name, const Tensor& t, const Tensor& first) {
  refuse_tangent(name, t);
  TORCH_CHECK(t.is_cuda(), "b200 backend requires CUDA tensors (", name, " is on ", t.device(), ")");
  TORCH_CHECK_VALUE(t.device() == first.device(), name, " is on ", t.device(), ", x on ", first.device());
}

int dtype_code(const char* name, const Tensor& t) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name,
                    " must be float32 or bfloat16, got ", t.scalar_type());
  return t.scalar_type() == at::kFloat ? TS_DTYPE_F32 : TS_DTYPE_BF16;
}

void refuse_double_backward(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the gradient has no gradient (create_graph is not supported)");
}

// t [..., width] as rows with contiguous channels: a view where the strides allow one, else a copy.
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

// ------------------------------------------------------------------ norm

void norm_check(const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps) {
  require_cuda("x", x, x);
  require_cuda("weight", weight, x);
  dtype_code("x", x);
  dtype_code("weight", weight);
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 1 && weight.size(0) == x.size(-1), "weight ", weight.sizes(),
                    " does not match the last dimension of x ", x.sizes());
  if (residual) {
    require_cuda("residual", *residual, x);
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
                      "residual must have the shape and dtype of x (", x.sizes(), ", ", x.scalar_type(), "), got ",
                      residual->sizes(), ", ", residual->scalar_type());
  }
  TORCH_CHECK_VALUE(eps >= 0, "eps must be >= 0, got ", eps);
}

ts_norm_args norm_args(const Tensor& x2, const Tensor& weight, double eps) {
  ts_norm_args a = {};
  a.rows = x2.size(0);
  a.width = static_cast<int>(x2.size(1) > INT_MAX ? INT_MAX : x2.size(1));
  a.dtype = dtype_code("x", x2);
  a.weight_dtype = dtype_code("weight", weight);
  a.eps = static_cast<float>(eps);
  a.x = x2.data_ptr();
  a.x_stride = x2.stride(0);
  a.weight = weight.data_ptr();
  return a;
}

struct NormOut {
  Tensor y, sum, rstd, scales;
};

// kCodes: y receives e4m3 codes (group 0: a scale per row).  Checked arguments.
NormOut norm_run(const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps, bool keep, bool codes,
                 int64_t group) {
  const c10::cuda::CUDAGuard guard(x.device());
  NormOut o;
  o.y = at::empty(x.sizes(), codes ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
  if (residual) o.sum = at::empty(x.sizes(), x.options());
  const int64_t width = x.size(-1), rows = width ? x.numel() / width : 0;
  if (keep) o.rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  if (codes) {
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = group ? (width + group - 1) / group : 1;
    o.scales = at::empty(shape, x.options().dtype(at::kFloat));
  }
  if (x.numel() == 0) return o;
  const Tensor x2 = rows_of(x), w = weight.contiguous();
  Tensor r2;
  ts_norm_args a = norm_args(x2, w, eps);
  a.y = o.y.data_ptr();
  if (residual) {
    r2 = rows_of(*residual);
    a.residual = r2.data_ptr();
    a.residual_stride = r2.stride(0);
    a.sum = o.sum.data_ptr();
  }
  if (keep) a.rstd = o.rstd.data_ptr<float>();
  if (codes) {
    a.scales = o.scales.data_ptr<float>();
    a.group = static_cast<int>(group);
  }
  check(ts_b200_norm_fwd(&a, current_stream(x)));
  return o;
}

// (dx, dweight): dx is the gradient of x and of the residual; `sum` is the stored sum (x without a residual).
std::pair<Tensor, Tensor> norm_grads(const Tensor& dy, const Tensor& dsum, const Tensor& sum, const Tensor& weight,
                                     const Tensor& rstd, double eps) {
  norm_check(sum, OptTensor(dy), weight, eps);
  if (dsum.defined()) norm_check(sum, OptTensor(dsum), weight, eps);
  require_cuda("rstd", rstd, sum);
  TORCH_CHECK_VALUE(rstd.scalar_type() == at::kFloat && rstd.is_contiguous() &&
                        rstd.numel() * sum.size(-1) == sum.numel(),
                    "rstd must be contiguous float32, one value for each row of ", sum.sizes());
  const c10::cuda::CUDAGuard guard(sum.device());
  Tensor dx = at::empty(sum.sizes(), sum.options()), dweight = at::empty(weight.sizes(), weight.options());
  if (sum.numel() == 0) return {dx, dweight.zero_()};
  const Tensor s2 = rows_of(sum), w = weight.contiguous(), dy2 = rows_of(dy);
  Tensor ds2;
  ts_norm_args a = norm_args(s2, w, eps);
  a.rstd = rstd.data_ptr<float>();
  ts_norm_grad_args g = {};
  g.dy = dy2.data_ptr();
  g.dy_stride = dy2.stride(0);
  if (dsum.defined()) {
    ds2 = rows_of(dsum);
    g.dsum = ds2.data_ptr();
    g.dsum_stride = ds2.stride(0);
  }
  g.workspace_bytes = ts_b200_norm_bwd_workspace_bytes(&a);
  const Tensor ws = at::empty({static_cast<int64_t>(g.workspace_bytes)}, sum.options().dtype(at::kByte));
  g.dx = dx.data_ptr();
  g.dweight = dweight.data_ptr();
  g.workspace = ws.data_ptr();
  check(ts_b200_norm_bwd(&a, &g, current_stream(sum)));
  return {dx, dweight};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const Tensor& weight,
                               double eps) {
    NormOut o = norm_run(x, residual, weight, eps, true, false, 0);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["added"] = residual.has_value();
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({residual ? o.sum : x, weight, o.rstd});
    if (residual) return {o.y, o.sum};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("rms_norm");
    const variable_list saved = ctx->get_saved_variables();
    const bool added = ctx->saved_data["added"].toBool();
    const Tensor dsum = added ? grads[1] : Tensor();
    Tensor dx = dsum, dweight;
    if (grads[0].defined())
      std::tie(dx, dweight) = norm_grads(grads[0], dsum, saved[0], saved[1], saved[2],
                                         ctx->saved_data["eps"].toDouble());
    return {dx, added ? dx : Tensor(), dweight, Tensor()};
  }
};

// ------------------------------------------------------------------- ffn

int activation_code(const std::string& name) {
  if (name == "silu") return TS_FFN_SILU;
  if (name == "gelu") return TS_FFN_GELU;
  if (name == "relu2") return TS_FFN_RELU2;
  TORCH_CHECK_VALUE(false, "activation must be one of gelu, relu2, silu, got '", name, "'");
}

void ffn_check(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd) {
  const std::pair<const char*, const Tensor*> all[] = {{"x", &x}, {"w_gate", &wg}, {"w_up", &wu}, {"w_down", &wd}};
  for (const auto& [name, t] : all) {
    require_cuda(name, *t, x);
    TORCH_CHECK_VALUE(t->scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t->scalar_type());
  }
  TORCH_CHECK_VALUE(x.dim() >= 1 && wg.dim() == 2 && wg.sizes() == wu.sizes() && wg.size(1) == x.size(-1), "w_gate ",
                    wg.sizes(), " and w_up ", wu.sizes(), " must be [hidden, width] for x ", x.sizes());
  TORCH_CHECK_VALUE(wd.dim() == 2 && wd.size(1) == wg.size(0), "w_down ", wd.sizes(), " must be [width_out, hidden], w_gate is ",
                    wg.sizes());
  for (int64_t n : {wg.size(0), wg.size(1), wd.size(0)})
    TORCH_CHECK_NOT_IMPLEMENTED(n > 0 && n % 8 == 0 && n <= (1 << 20),
                                "gated_ffn: widths must be nonzero multiples of 8 (up to 2^20), got ", n);
}

// t [..., width] as rows with contiguous channels, a 16-byte aligned base and
// a row stride that is a multiple of 8: a view where t is one, else a copy.
struct Matrix {
  Tensor t;
  int64_t stride;
  explicit Matrix(const Tensor& from) : t(from.dim() == 2 ? from : from.reshape({-1, from.size(-1)})) {
    const bool one = t.size(0) == 1;
    if (t.stride(1) != 1 || (!one && (t.stride(0) % 8 || t.stride(0) < t.size(1))) ||
        reinterpret_cast<uintptr_t>(t.data_ptr()) % 16)
      t = t.clone(at::MemoryFormat::Contiguous);
    stride = one ? t.size(1) : t.stride(0);
  }
  void* ptr() const { return t.data_ptr(); }
};

struct FfnCall {
  Matrix x, wg, wu, wd;
  ts_ffn_args a = {};
  FfnCall(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, const Tensor& wd_, int activation)
      : x(x_), wg(wg_), wu(wu_), wd(wd_) {
    a.rows = x.t.size(0);
    a.width = static_cast<int>(x.t.size(1));
    a.hidden = static_cast<int>(wg.t.size(0));
    a.width_out = static_cast<int>(wd.t.size(0));
    a.activation = activation;
    a.x = x.ptr();
    a.w_gate = wg.ptr();
    a.w_up = wu.ptr();
    a.w_down = wd.ptr();
    a.x_stride = x.stride;
    a.w_gate_stride = wg.stride;
    a.w_up_stride = wu.stride;
    a.w_down_stride = wd.stride;
  }
  Tensor workspace(size_t bytes) {
    if (bytes == 0) {   // the size query refused the arguments
      char text[512];
      check(ts_b200_last_error(text, sizeof(text)));
    }
    Tensor ws = at::empty({static_cast<int64_t>(bytes)}, x.t.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = bytes;
    return ws;
  }
};

struct FfnOut {
  Tensor y, h, kept;
};

// bf16 parts that h is kept in.
int64_t h_parts(int64_t rows) { return rows <= TS_FFN_TWO_PART_ROWS ? 2 : 1; }

int64_t kept_bytes(int64_t rows, int64_t hidden) {
  return (rows + 31) / 32 * ((hidden + 31) / 32) * TS_FFN_KEPT_BLOCK;
}

FfnOut ffn_run(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int activation, bool keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  FfnOut o;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = wd.size(0);
  o.y = at::empty(shape, x.options());
  const int64_t rows = x.numel() / x.size(-1), hidden = wg.size(0);
  if (keep) {
    o.h = at::empty({h_parts(rows) * rows, hidden}, x.options());
    o.kept = at::empty({kept_bytes(rows, hidden)}, x.options().dtype(at::kByte));
  }
  if (x.numel() == 0) return o;
  FfnCall c(x, wg, wu, wd, activation);
  c.a.y = o.y.data_ptr();
  if (keep) {
    c.a.h = o.h.data_ptr();
    c.a.kept = o.kept.data_ptr();
  }
  const Tensor ws = c.workspace(ts_b200_ffn_fwd_workspace_bytes(&c.a));
  check(ts_b200_ffn_fwd(&c.a, current_stream(x)));
  return o;
}

// Gradients of x, w_gate, w_up, w_down; undefined where not wanted.
std::vector<Tensor> ffn_grads(const Tensor& dy, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                              const Tensor& h, const Tensor& kept, int activation, const std::vector<bool>& wanted) {
  ffn_check(x, wg, wu, wd);
  const int64_t rows = x.numel() / x.size(-1), hidden = wg.size(0);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor*>{"dy", &dy}, {"h", &h}, {"kept", &kept}})
    require_cuda(name, *t, x);
  TORCH_CHECK_VALUE(dy.scalar_type() == at::kBFloat16 && dy.dim() == x.dim() && dy.size(-1) == wd.size(0) &&
                        dy.numel() == rows * wd.size(0),
                    "dy must be bfloat16 and of the output's shape, got ", dy.scalar_type(), " ", dy.sizes());
  TORCH_CHECK_VALUE(h.scalar_type() == at::kBFloat16 && h.is_contiguous() && h.numel() == h_parts(rows) * rows * hidden &&
                        kept.scalar_type() == at::kByte && kept.is_contiguous() &&
                        kept.numel() == kept_bytes(rows, hidden),
                    "h and kept must be what the forward of these inputs kept");
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor* inputs[] = {&x, &wg, &wu, &wd};
  std::vector<Tensor> out(4);
  for (int i = 0; i < 4; ++i)
    if (wanted[i]) out[i] = at::empty(inputs[i]->sizes(), inputs[i]->options());
  if (x.numel() == 0) {
    for (Tensor& t : out)
      if (t.defined()) t.zero_();
    return out;
  }
  FfnCall c(x, wg, wu, wd, activation);
  const Matrix d(dy);
  c.a.h = h.data_ptr();
  c.a.kept = kept.data_ptr();
  const Tensor ws = c.workspace(ts_b200_ffn_bwd_workspace_bytes(&c.a));
  ts_ffn_grad_args g = {};
  g.dy = d.ptr();
  g.dy_stride = d.stride;
  void** to[] = {&g.dx, &g.dw_gate, &g.dw_up, &g.dw_down};
  for (int i = 0; i < 4; ++i) *to[i] = out[i].defined() ? out[i].data_ptr() : nullptr;
  check(ts_b200_ffn_bwd(&c.a, &g, current_stream(x)));
  return out;
}

struct FfnNode : torch::autograd::Function<FfnNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                        int64_t activation) {
    FfnOut o = ffn_run(x, wg, wu, wd, static_cast<int>(activation), true);
    ctx->saved_data["activation"] = activation;
    ctx->save_for_backward({x, wg, wu, wd, o.h, o.kept});
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("gated_ffn");
    const variable_list s = ctx->get_saved_variables();
    std::vector<bool> wanted(4);
    for (int i = 0; i < 4; ++i) wanted[i] = ctx->needs_input_grad(i);
    variable_list out = ffn_grads(grads[0], s[0], s[1], s[2], s[3], s[4], s[5],
                                  static_cast<int>(ctx->saved_data["activation"].toInt()), wanted);
    out.emplace_back();
    return out;
  }
};

// ----------------------------------------------------------------- adamw

// The tensors of a Python sequence.
std::vector<Tensor> tensors_of(PyObject* object, const char* what) {
  THPObjectPtr list(PySequence_Fast(object, what));
  if (!list) throw python_error();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list.get());
  std::vector<Tensor> out;
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PySequence_Fast_GET_ITEM(list.get(), i);
    TORCH_CHECK_TYPE(THPVariable_Check(item), "adamw: ", what, " must be tensors");
    out.push_back(THPVariable_Unpack(item));
  }
  return out;
}

// Whether the elements of t are those of `like` in their order: of its shape, or one of the two flat.
bool in_order(const Tensor& t, const Tensor& like) {
  return t.sizes() == like.sizes() || ((t.dim() == 1 || like.dim() == 1) && t.numel() == like.numel());
}

// Contiguous tensors of one dtype on the parameters' device, with the shapes of `like` or flat (`blocks`: a scale for
// each block).
void same(const std::vector<Tensor>& list, const std::vector<Tensor>& like, at::ScalarType type, bool blocks,
          const char* what) {
  TORCH_CHECK_VALUE(list.size() == like.size(), "adamw: ", like.size(), " parameters but ", list.size(), " ", what);
  for (size_t i = 0; i < list.size(); ++i) {
    const Tensor& t = list[i];
    const int64_t n = blocks ? (like[i].numel() + kStateBlock - 1) / kStateBlock : like[i].numel();
    TORCH_CHECK_VALUE(t.scalar_type() == type, "adamw: ", what, " must be ", type, ", got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.numel() == n, "adamw: ", what, " ", i, " has ", t.numel(), " elements, not ", n);
    TORCH_CHECK_VALUE(blocks || in_order(t, like[i]), "adamw: ", what, " ", i, " is ", t.sizes(), ", its parameter ",
                      like[i].sizes());
    TORCH_CHECK_VALUE(t.device() == like[0].device(), "adamw: ", what, " must be on the parameters' device");
    TORCH_CHECK_VALUE(t.is_contiguous(), "adamw: ", what, " must be contiguous");
  }
}

struct AdamW {
  std::vector<Tensor> params, grads, m, v, masters, m_scales, v_scales;
  std::vector<int64_t> ordinals;
  bool has_masters = false, has_scales = false;
  ts_adamw_args a = {};

  // One launch for the tensors `at` of one kind.
  void run(const std::vector<size_t>& at) {
    std::vector<ts_adamw_tensor> table(at.size());
    for (size_t k = 0; k < at.size(); ++k) {
      const size_t i = at[k];
      ts_adamw_tensor& t = table[k];
      t.param = params[i].data_ptr();
      t.grad = grads[i].data_ptr();
      t.master = has_masters ? masters[i].data_ptr<float>() : nullptr;
      t.exp_avg = m[i].data_ptr();
      t.exp_avg_sq = v[i].data_ptr();
      t.exp_avg_scale = has_scales ? m_scales[i].data_ptr<float>() : nullptr;
      t.exp_avg_sq_scale = has_scales ? v_scales[i].data_ptr<float>() : nullptr;
      t.n = params[i].numel();
      t.ordinal = static_cast<int>(ordinals[i]);
    }
    a.count = static_cast<int>(table.size());
    a.tensors = table.data();
    a.param_dtype = dtype_code("parameters", params[at[0]]);
    a.grad_dtype = dtype_code("gradients", grads[at[0]]);
    check(ts_b200_adamw(&a, current_stream(params[0])));
  }

  void step() {
    const size_t n = params.size();
    if (n == 0) return;
    for (const Tensor& p : params) {
      TORCH_CHECK(p.is_cuda(), "b200 backend requires CUDA tensors (a parameter is on ", p.device(), ")");
      dtype_code("parameters", p);
      TORCH_CHECK_VALUE(p.device() == params[0].device(), "adamw: parameters must be on one device");
      TORCH_CHECK_VALUE(p.is_contiguous(), "adamw: parameters must be contiguous");
    }
    TORCH_CHECK_VALUE(grads.size() == n, "adamw: ", n, " parameters but ", grads.size(), " gradients");
    for (size_t i = 0; i < n; ++i) {
      TORCH_CHECK_VALUE(!grads[i].is_sparse(), "adamw: sparse gradients are not supported");
      dtype_code("gradients", grads[i]);
      TORCH_CHECK_VALUE(in_order(grads[i], params[i]) && grads[i].device() == params[0].device(),
                        "adamw: gradient ", i, " does not match its parameter");
    }
    if (torch::autograd::ForwardADLevel::try_get_by_idx(0)) {
      for (const auto& list : {std::make_pair("a parameter", &params), std::make_pair("a gradient", &grads)})
        for (const Tensor& t : *list.second) refuse_tangent(list.first, t);
    }
    const c10::cuda::CUDAGuard guard(params[0].device());
    TORCH_CHECK(at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None,
                "adamw: a captured step would repeat its step count; call it outside the graph");
    for (Tensor& g : grads) g = g.contiguous();
    const bool eight = !m.empty() && m[0].scalar_type() == at::kFloat8_e4m3fn;
    const at::ScalarType state = eight ? at::kFloat8_e4m3fn : at::kFloat;
    same(m, params, state, false, "first moments");
    same(v, params, state, false, "second moments");
    TORCH_CHECK_VALUE(eight == has_scales, eight ? "adamw: 8-bit states need their scales" : "adamw: scales belong to 8-bit states");
    if (has_scales) {
      same(m_scales, params, at::kFloat, true, "first moments' scales");
      same(v_scales, params, at::kFloat, true, "second moments' scales");
    }
    if (has_masters) {
      same(masters, params, at::kFloat, false, "masters");
      for (const Tensor& p : params)
        TORCH_CHECK_VALUE(p.scalar_type() == at::kBFloat16, "adamw: masters belong to bfloat16 parameters");
    }
    TORCH_CHECK_VALUE(ordinals.size() == n, "adamw: ", n, " parameters but ", ordinals.size(), " ordinals");
    a.master = has_masters;
    a.state_bits = eight ? 8 : 32;
    // one launch for each kind of parameter and gradient
    std::vector<size_t> kinds[4];
    for (size_t i = 0; i < n; ++i)
      kinds[2 * (params[i].scalar_type() == at::kBFloat16) + (grads[i].scalar_type() == at::kBFloat16)].push_back(i);
    for (const auto& k : kinds)
      if (!k.empty()) run(k);
    // the parameters changed under autograd's eyes
    for (const Tensor& p : params)
      if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
  }
};

// ---------------------------------------------------------------- window

// t [batch, heads, tokens, dim] as the kernels read it: a view where its channels are contiguous and its base and
// strides are multiples of 16 bytes, else a copy.
Tensor streams_of(const Tensor& t) {
  bool fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(3) == 1;
  for (int i = 0; i < 3 && fits; ++i) {
    const int64_t s = t.stride(i);
    fits = t.size(i) == 1 || (s > 0 && s % 8 == 0 && s < (int64_t{1} << 38));
  }
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

void set_strides(long long (&to)[3], const Tensor& t) {
  // a dimension of one has no stride of its own
  for (int i = 0; i < 3; ++i) to[i] = t.size(i) > 1 ? t.stride(i) : (t.size(3) + 7) / 8 * 8;
}

void lengths_check(const char* name, const Tensor& lengths, int64_t batch, const Tensor& first) {
  require_cuda(name, lengths, first);
  TORCH_CHECK_VALUE(lengths.scalar_type() == at::kInt && lengths.is_contiguous() && lengths.dim() == 1 &&
                        lengths.size(0) == batch,
                    name, " must be contiguous int32 [", batch, "], got ", lengths.scalar_type(), " ", lengths.sizes());
}

void bf16_4d(const char* name, const Tensor& t, const Tensor& first) {
  require_cuda(name, t, first);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must be [batch, heads, tokens, head width], got ", t.sizes());
}

void window_check(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, double scale,
                  const OptTensor& lengths) {
  bf16_4d("q", q, q);
  bf16_4d("k", k, q);
  bf16_4d("v", v, q);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3) && k.size(2) >= q.size(2),
                    "k ", k.sizes(), " and v ", v.sizes(), " do not go with q ", q.sizes());
  TORCH_CHECK_VALUE(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "the ", q.size(1), " heads of q do not share the ",
                    k.size(1), " of k");
  TORCH_CHECK_NOT_IMPLEMENTED(q.size(3) >= 8 && q.size(3) <= 128 && q.size(3) % 8 == 0,
                              "window_attention: the head width must be a multiple of 8 up to 128, got ", q.size(3));
  TORCH_CHECK_VALUE(window >= 1 && sinks >= 0, "window must be >= 1 and sinks >= 0, got ", window, " and ", sinks);
  TORCH_CHECK_VALUE(std::isfinite(static_cast<float>(scale)) && static_cast<float>(scale) > 0,
                    "scale must be positive and finite, got ", scale);
  TORCH_CHECK_NOT_IMPLEMENTED(k.size(2) <= (1 << 30), "window_attention: more than 2^30 tokens");
  if (lengths) lengths_check("lengths", *lengths, q.size(0), q);
}

int clipped(int64_t n) { return static_cast<int>(n > (1 << 30) ? 1 << 30 : n); }

struct WindowCall {
  Tensor q, k, v;
  ts_window_args a = {};
  WindowCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t window, int64_t sinks, double scale,
             const OptTensor& lengths)
      : q(streams_of(q_)), k(streams_of(k_)), v(streams_of(v_)) {
    a.batch = clipped(q.size(0));
    a.heads = clipped(q.size(1));
    a.kv_heads = clipped(k.size(1));
    a.dim = static_cast<int>(q.size(3));
    a.q_tokens = static_cast<int>(q.size(2));
    a.kv_tokens = static_cast<int>(k.size(2));
    a.window = clipped(window);
    a.sinks = clipped(sinks);
    a.scale = static_cast<float>(scale);
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    set_strides(a.q_strides, q);
    set_strides(a.k_strides, k);
    set_strides(a.v_strides, v);
    a.lengths = lengths ? lengths->data_ptr<int>() : nullptr;
  }
};

// [batch, heads, tokens, dim] whose memory is [batch, tokens, heads, dim]: the heads of a token lie together, as the
// projections around an attention have them.  No view: autograd lets the result of a function be changed in place only then.
Tensor token_major(const Tensor& like) {
  const int64_t h = like.size(1), n = like.size(2), d = like.size(3);
  return at::empty_strided(like.sizes(), {n * h * d, d, h * d, 1}, like.options());
}

std::pair<Tensor, Tensor> window_run(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks,
                                     double scale, const OptTensor& lengths, bool keep) {
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor y = token_major(q);
  Tensor lse;
  if (keep) lse = at::empty({q.size(0), q.size(1), (q.size(2) + 127) / 128 * 128}, q.options().dtype(at::kFloat));
  if (q.numel() == 0) return {y, lse};
  WindowCall c(q, k, v, window, sinks, scale, lengths);
  c.a.y = y.data_ptr();
  set_strides(c.a.y_strides, y);
  if (keep) c.a.lse = lse.data_ptr<float>();
  check(ts_b200_window_fwd(&c.a, current_stream(q)));
  return {y, lse};
}

std::vector<Tensor> window_grads(const Tensor& dy_, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& y,
                                 const Tensor& lse, int64_t window, int64_t sinks, double scale, const OptTensor& lengths) {
  window_check(q, k, v, window, sinks, scale, lengths);
  bf16_4d("dy", dy_, q);
  bf16_4d("y", y, q);
  require_cuda("lse", lse, q);
  TORCH_CHECK_VALUE(dy_.sizes() == q.sizes() && y.sizes() == q.sizes(), "dy ", dy_.sizes(), " and y ", y.sizes(),
                    " must have the shape of q ", q.sizes());
  TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                        lse.numel() == q.size(0) * q.size(1) * ((q.size(2) + 127) / 128 * 128),
                    "lse must be what the forward of these inputs kept");
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor dq = token_major(q), dk = token_major(k), dv = token_major(v);
  if (q.numel() == 0) {
    dk.zero_();
    dv.zero_();
    return {dq, dk, dv};
  }
  WindowCall c(q, k, v, window, sinks, scale, lengths);
  const Tensor dy = streams_of(dy_), yy = streams_of(y);
  c.a.y = yy.data_ptr();
  set_strides(c.a.y_strides, yy);
  c.a.lse = lse.data_ptr<float>();
  ts_window_grad_args g = {};
  g.dy = dy.data_ptr();
  set_strides(g.dy_strides, dy);
  g.dq = dq.data_ptr();
  g.dk = dk.data_ptr();
  g.dv = dv.data_ptr();
  set_strides(g.dq_strides, dq);
  set_strides(g.dk_strides, dk);
  set_strides(g.dv_strides, dv);
  g.workspace_bytes = ts_b200_window_bwd_workspace_bytes(&c.a);
  if (g.workspace_bytes == 0) {   // the size query refused the arguments
    char text[512];
    check(ts_b200_last_error(text, sizeof(text)));
  }
  const Tensor ws = at::empty({static_cast<int64_t>(g.workspace_bytes)}, q.options().dtype(at::kByte));
  g.workspace = ws.data_ptr();
  check(ts_b200_window_bwd(&c.a, &g, current_stream(q)));
  return {dq, dk, dv};
}

struct WindowNode : torch::autograd::Function<WindowNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t window,
                        int64_t sinks, double scale, const OptTensor& lengths) {
    const auto [y, lse] = window_run(q, k, v, window, sinks, scale, lengths, true);
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    ctx->save_for_backward({q, k, v, y, lse, lengths ? *lengths : Tensor()});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("window_attention");
    const variable_list s = ctx->get_saved_variables();
    const variable_list g = window_grads(grads[0], s[0], s[1], s[2], s[3], s[4], ctx->saved_data["window"].toInt(),
                                         ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toDouble(),
                                         s[5].defined() ? OptTensor(s[5]) : OptTensor());
    return {g[0], g[1], g[2], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// What a kernel writes in place: its autograd version moves on.
void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void in_place_check(const char* name, const Tensor& t) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name, " is written in place and must not require a gradient");
  for (int64_t i = 0; i < t.dim(); ++i)
    TORCH_CHECK_VALUE(t.size(i) < 2 || t.stride(i) > 0, name, " is written in place and must not be an expanded view");
}

// The cache's part of the arguments; `k` and `v` are the new tokens.
ts_window_cache window_cache(const Tensor& k, const Tensor& v, const Tensor& keys, const Tensor& values,
                             const Tensor& lengths, int64_t sinks) {
  bf16_4d("k", k, k);
  bf16_4d("v", v, k);
  bf16_4d("keys", keys, k);
  bf16_4d("values", values, k);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "k ", k.sizes(), " and v ", v.sizes(), " must have one shape");
  TORCH_CHECK_VALUE(keys.sizes() == values.sizes() && keys.size(0) == k.size(0) && keys.size(1) == k.size(1) &&
                        keys.size(3) == k.size(3),
                    "a cache of ", keys.sizes(), " and ", values.sizes(), " does not go with k ", k.sizes());
  TORCH_CHECK_VALUE(sinks >= 0 && sinks < keys.size(2), "of the cache's ", keys.size(2), " slots, sinks must leave one, got ", sinks);
  TORCH_CHECK_NOT_IMPLEMENTED(k.size(3) >= 8 && k.size(3) <= 128 && k.size(3) % 8 == 0,
                              "window attention: the head width must be a multiple of 8 up to 128, got ", k.size(3));
  lengths_check("lengths", lengths, k.size(0), k);
  ts_window_cache c = {};
  for (const auto& [name, t] : {std::pair<const char*, const Tensor*>{"keys", &keys}, {"values", &values}}) {
    in_place_check(name, *t);
    bool fits = reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0 && t->stride(3) == 1;
    for (int i = 0; i < 3; ++i) fits = fits && (t->size(i) == 1 || t->stride(i) % 8 == 0);
    TORCH_CHECK_VALUE(fits, name, " must have contiguous channels, and a base and strides that are multiples of 16 bytes");
  }
  c.batch = clipped(k.size(0));
  c.kv_heads = clipped(k.size(1));
  c.dim = static_cast<int>(k.size(3));
  c.sinks = clipped(sinks);
  c.window = clipped(keys.size(2) - sinks);
  TORCH_CHECK_NOT_IMPLEMENTED(keys.size(2) <= (1 << 30), "window attention: more than 2^30 slots");
  c.keys = keys.data_ptr();
  c.values = values.data_ptr();
  set_strides(c.keys_strides, keys);
  set_strides(c.values_strides, values);
  c.lengths = lengths.data_ptr<int>();
  return c;
}

Tensor window_step_run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& keys, const Tensor& values,
                       const Tensor& lengths, int64_t sinks, double scale) {
  bf16_4d("q", q, k);
  TORCH_CHECK_VALUE(q.size(2) == 1 && k.size(2) == 1, "window_attention_step takes one token, got q ", q.sizes(), " and k ", k.sizes());
  TORCH_CHECK_VALUE(q.size(0) == k.size(0) && q.size(3) == k.size(3) && k.size(1) > 0 && q.size(1) % k.size(1) == 0, "q ",
                    q.sizes(), " does not go with k ", k.sizes());
  TORCH_CHECK_VALUE(std::isfinite(static_cast<float>(scale)) && static_cast<float>(scale) > 0,
                    "scale must be positive and finite, got ", scale);
  ts_window_step_args a = {};
  a.cache = window_cache(k, v, keys, values, lengths, sinks);
  const c10::cuda::CUDAGuard guard(k.device());
  Tensor y = at::empty(q.sizes(), q.options());
  if (q.numel() == 0) return y;
  const Tensor q4 = streams_of(q), k4 = streams_of(k), v4 = streams_of(v);
  a.heads = clipped(q.size(1));
  a.scale = static_cast<float>(scale);
  a.q = q4.data_ptr();
  a.k = k4.data_ptr();
  a.v = v4.data_ptr();
  for (const auto& [to, t] : {std::pair<long long*, const Tensor*>{a.q_strides, &q4}, {a.k_strides, &k4}, {a.v_strides, &v4}}) {
    long long s[3];
    set_strides(s, *t);
    to[0] = s[0];
    to[1] = s[1];
  }
  a.y = y.data_ptr();
  check(ts_b200_window_step(&a, current_stream(k)));
  changed(keys);
  changed(values);
  return y;
}

void window_extend_run(const Tensor& k, const Tensor& v, const Tensor& keys, const Tensor& values, const Tensor& lengths,
                       int64_t sinks, const OptTensor& fresh) {
  ts_window_extend_args a = {};
  a.cache = window_cache(k, v, keys, values, lengths, sinks);
  if (fresh) lengths_check("new", *fresh, k.size(0), k);
  TORCH_CHECK_NOT_IMPLEMENTED(k.size(2) <= (1 << 30), "window_cache_extend: more than 2^30 tokens");
  if (k.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(k.device());
  const Tensor k4 = streams_of(k), v4 = streams_of(v);
  a.tokens = static_cast<int>(k.size(2));
  a.k = k4.data_ptr();
  a.v = v4.data_ptr();
  set_strides(a.k_strides, k4);
  set_strides(a.v_strides, v4);
  a.fresh = fresh ? fresh->data_ptr<int>() : nullptr;
  check(ts_b200_window_extend(&a, current_stream(k)));
  changed(keys);
  changed(values);
}

// ------------------------------------------------------------- scan step

// Reads [views, batch, heads, 1, width]; the state changes in place.
Tensor scan_step_run(const Tensor& q, const Tensor& k, const Tensor& v, const std::vector<OptTensor>& retentions, bool unit,
                     const Tensor& state) {
  const std::pair<const char*, const Tensor*> all[] = {{"q", &q}, {"k", &k}, {"v", &v}, {"state", &state}};
  for (const auto& [name, t] : all) require_cuda(name, *t, q);
  TORCH_CHECK_NOT_IMPLEMENTED(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() &&
                                  (q.scalar_type() == at::kFloat || q.scalar_type() == at::kBFloat16),
                              "b200 scan step: q, k and v must all be bf16 or all float32, got ", q.scalar_type(), ", ",
                              k.scalar_type(), ", ", v.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(2) == 1 && k.sizes() == q.sizes() && v.dim() == 4 && v.size(0) == q.size(0) &&
                        v.size(1) == q.size(1) && v.size(2) == 1,
                    "b200 scan step: q and k must be [B,H,1,Dk] and v [B,H,1,Dv], got ", q.sizes(), ", ", k.sizes(), " and ",
                    v.sizes());
  const int64_t B = q.size(0), H = q.size(1), width = v.size(3) + unit, R = static_cast<int64_t>(retentions.size());
  TORCH_CHECK_NOT_IMPLEMENTED(R <= TS_MAX_RETENTIONS, "b200 scan step: at most ", TS_MAX_RETENTIONS, " retentions per call");
  TORCH_CHECK_NOT_IMPLEMENTED(q.size(3) >= 1 && q.size(3) <= 256 && width <= 256 && width > unit,
                              "b200 scan step: key and payload widths up to 256, got ", q.size(3), " and ", width);
  TORCH_CHECK_VALUE(state.scalar_type() == at::kFloat && state.is_contiguous() &&
                        state.sizes() == at::IntArrayRef({B, H, R, q.size(3), width}),
                    "b200 scan step: state must be contiguous f32 [", B, ",", H, ",", R, ",", q.size(3), ",", width, "], got ",
                    state.scalar_type(), " ", state.sizes());
  in_place_check("state", state);
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty({R, B, H, 1, width}, q.options());
  std::vector<Tensor> las;
  ts_scan_step_args a = {};
  for (int64_t i = 0; i < R; ++i) {
    if (!retentions[i]) continue;
    const Tensor& r = *retentions[i];
    require_cuda("retention", r, q);
    const bool gate = r.dim() == 4;
    TORCH_CHECK_VALUE(gate ? r.sizes() == at::IntArrayRef({B, H, 1, 1}) : r.numel() == H,
                      "b200 scan step: a retention is None, one entry per head or [B,H,1,1], got ", r.sizes());
    las.push_back(r.detach().reshape({-1}).to(at::kFloat).contiguous());
    a.log_alpha[i] = las.back().data_ptr<float>();
    a.log_alpha_batch[i] = gate ? H : 0;
  }
  if (out.numel() == 0) return out;
  auto rows = [](const Tensor& t) { return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous(); };
  const Tensor q4 = rows(q), k4 = rows(k), v4 = rows(v);
  a.batch = clipped(B);
  a.heads = clipped(H);
  a.dk = static_cast<int>(q.size(3));
  a.dv = static_cast<int>(width);
  a.v_append_unit = unit;
  a.dtype = dtype_code("q", q);
  a.q = q4.data_ptr();
  a.k = k4.data_ptr();
  a.v = v4.data_ptr();
  for (int i = 0; i < 2; ++i) {
    a.q_strides[i] = q4.stride(i);
    a.k_strides[i] = k4.stride(i);
    a.v_strides[i] = v4.stride(i);
  }
  a.n_retentions = static_cast<int>(R);
  a.state = state.data_ptr<float>();
  a.out = out.data_ptr();
  check(ts_b200_scan_step(&a, current_stream(q)));
  changed(state);
  return out;
}

// ---------------------------------------------------------------- sample

// A setting of the choice: a number for all rows, or a tensor with one for each.
struct Setting {
  Tensor rows;
  double value;
  Setting(const OptTensor& t, double value_, at::ScalarType type, const char* name, int64_t count, const Tensor& logits)
      : value(value_) {
    if (!t) return;
    require_cuda(name, *t, logits);
    TORCH_CHECK_VALUE(type == at::kInt ? at::isIntegralType(t->scalar_type(), false) : t->scalar_type() == type, name,
                      " must be a number or a tensor of ", type, ", got ", t->scalar_type());
    TORCH_CHECK_VALUE(t->numel() == count, name, " must have one value for each of the ", count, " rows, got ", t->sizes());
    // 64-bit integers end at the ones that 32 bits hold; an unsigned one above them is negative then, and as little of a
    // limit as it was
    rows = t->scalar_type() == type ? t->contiguous()
                                    : (t->element_size() > 4 ? t->to(at::kLong).clamp(INT_MIN, INT_MAX) : *t).to(type).contiguous();
  }
};

std::pair<Tensor, Tensor> sample_run(const Tensor& logits, const Tensor& uniform, const OptTensor& temperature,
                                     double temperature_value, const OptTensor& top_k, int64_t top_k_value,
                                     const OptTensor& top_p, double top_p_value, const OptTensor& min_p, double min_p_value,
                                     bool logprobs) {
  require_cuda("logits", logits, logits);
  require_cuda("uniform", uniform, logits);
  dtype_code("logits", logits);
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must be [..., vocabulary], got ", logits.sizes());
  const int64_t vocab = logits.size(-1), rows = logits.numel() / vocab;
  TORCH_CHECK_VALUE(uniform.scalar_type() == at::kFloat && uniform.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    "uniform must be float32 ", logits.sizes().slice(0, logits.dim() - 1), ", got ", uniform.scalar_type(), " ",
                    uniform.sizes());
  TORCH_CHECK_NOT_IMPLEMENTED(vocab <= (1 << 21) && rows <= (1 << 27), "sample_tokens: more than 2^21 tokens or 2^27 rows");
  TORCH_CHECK_VALUE(temperature || (temperature_value >= 0 && std::isfinite(temperature_value)),
                    "temperature must be >= 0 and finite, got ", temperature_value);
  TORCH_CHECK_VALUE(top_k || top_k_value >= 0, "top_k must be >= 1, got ", top_k_value);
  TORCH_CHECK_VALUE(top_p || (top_p_value > 0 && top_p_value <= 1), "top_p must be in (0, 1], got ", top_p_value);
  TORCH_CHECK_VALUE(min_p || (min_p_value >= 0 && min_p_value <= 1), "min_p must be in [0, 1], got ", min_p_value);
  const c10::cuda::CUDAGuard guard(logits.device());
  const Setting t(temperature, temperature_value, at::kFloat, "temperature", rows, logits),
      k(top_k, 0, at::kInt, "top_k", rows, logits), pp(top_p, top_p_value, at::kFloat, "top_p", rows, logits),
      mp(min_p, min_p_value, at::kFloat, "min_p", rows, logits);
  Tensor tokens = at::empty(uniform.sizes(), logits.options().dtype(at::kLong)), chances;
  if (logprobs) chances = at::empty(uniform.sizes(), logits.options().dtype(at::kFloat));
  if (rows == 0) return {tokens, chances};
  const Tensor x = rows_of(logits.detach()), u = uniform.contiguous();
  ts_sample_args a = {};
  a.rows = static_cast<int>(rows);
  a.vocab = static_cast<int>(vocab);
  a.dtype = dtype_code("logits", x);
  a.logits = x.data_ptr();
  a.row_stride = x.stride(0);
  a.uniform = u.data_ptr<float>();
  a.temperature = t.rows.defined() ? t.rows.data_ptr<float>() : nullptr;
  a.temperature_value = t.value;
  a.top_k = k.rows.defined() ? k.rows.data_ptr<int>() : nullptr;
  a.top_k_value = clipped(top_k_value);
  a.top_p = pp.rows.defined() ? pp.rows.data_ptr<float>() : nullptr;
  a.top_p_value = pp.value;
  a.min_p = mp.rows.defined() ? mp.rows.data_ptr<float>() : nullptr;
  a.min_p_value = mp.value;
  a.tokens = reinterpret_cast<long long*>(tokens.data_ptr<int64_t>());
  a.logprobs = logprobs ? chances.data_ptr<float>() : nullptr;
  check(ts_b200_sample(&a, current_stream(logits)));
  return {tokens, chances};
}

// ---------------------------------------------------------------- Python

const Tensor& tensor_arg(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
OptTensor optional_arg(PyObject* o, const char* name) {
  return o == Py_None ? OptTensor() : OptTensor(tensor_arg(o, name));
}
double double_arg(PyObject* o) {
  const double d = PyFloat_AsDouble(o);
  if (d == -1.0 && PyErr_Occurred()) throw python_error();
  return d;
}
int64_t int_arg(PyObject* o) {
  const long long i = PyLong_AsLongLong(o);
  if (i == -1 && PyErr_Occurred()) throw python_error();
  return i;
}
std::string text_arg(PyObject* o) {
  const char* s = PyUnicode_AsUTF8(o);
  if (!s) throw python_error();
  return s;
}
PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
PyObject* wrap_all(std::initializer_list<const Tensor*> list) {
  PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(list.size()));
  if (!tuple) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor* t : list) PyTuple_SET_ITEM(tuple, i++, wrap(*t));
  return tuple;
}
void count_args(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments, got ", n); }

bool needs_grad(std::initializer_list<const Tensor*> list) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : list)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// rms_norm(x, residual or None, weight, eps) -> y, or (y, sum) with a residual; with gradients
PyObject* py_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 4);
  const Tensor& x = tensor_arg(args[0], "x");
  const OptTensor r = optional_arg(args[1], "residual");
  const Tensor& w = tensor_arg(args[2], "weight");
  const double eps = double_arg(args[3]);
  norm_check(x, r, w, eps);
  const Tensor none, &added = r ? *r : none;
  if (needs_grad({&x, &w, &added})) {
    const variable_list out = NormNode::apply(x, r, w, eps);
    return r ? wrap_all({&out[0], &out[1]}) : wrap(out[0]);
  }
  const NormOut o = norm_run(x, r, w, eps, false, false, 0);
  return r ? wrap_all({&o.y, &o.sum}) : wrap(o.y);
  END_HANDLE_TH_ERRORS
}

// norm_fwd(x, residual, weight, eps, keep) -> (y, sum or None, rstd or None); no gradients
PyObject* py_norm_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 5);
  const Tensor& x = tensor_arg(args[0], "x");
  const OptTensor r = optional_arg(args[1], "residual");
  const Tensor& w = tensor_arg(args[2], "weight");
  const double eps = double_arg(args[3]);
  norm_check(x, r, w, eps);
  const NormOut o = norm_run(x, r, w, eps, args[4] == Py_True, false, 0);
  return wrap_all({&o.y, &o.sum, &o.rstd});
  END_HANDLE_TH_ERRORS
}

// norm_bwd(dy, dsum or None, sum, weight, rstd, eps) -> (dx, dweight)
PyObject* py_norm_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 6);
  const OptTensor dsum = optional_arg(args[1], "dsum");
  const auto [dx, dw] = norm_grads(tensor_arg(args[0], "dy"), dsum ? *dsum : Tensor(), tensor_arg(args[2], "sum"),
                                   tensor_arg(args[3], "weight"), tensor_arg(args[4], "rstd"), double_arg(args[5]));
  return wrap_all({&dx, &dw});
  END_HANDLE_TH_ERRORS
}

// rms_norm_8bit(x, residual or None, weight, eps, group or None) -> (codes, scales[, sum])
PyObject* py_rms_norm_8bit(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 5);
  const Tensor& x = tensor_arg(args[0], "x");
  const OptTensor r = optional_arg(args[1], "residual");
  const Tensor& w = tensor_arg(args[2], "weight");
  const double eps = double_arg(args[3]);
  const int64_t group = args[4] == Py_None ? 0 : int_arg(args[4]);
  norm_check(x, r, w, eps);
  TORCH_CHECK_VALUE(args[4] == Py_None || group == kGroup, "group must be None (one scale per row) or ", kGroup,
                    ", got ", group);
  const Tensor none, &added = r ? *r : none;
  TORCH_CHECK(!needs_grad({&x, &w, &added}), "rms_norm_8bit has no gradient: call it under torch.no_grad()");
  const NormOut o = norm_run(x, r, w, eps, false, true, group);
  return r ? wrap_all({&o.y, &o.scales, &o.sum}) : wrap_all({&o.y, &o.scales});
  END_HANDLE_TH_ERRORS
}

// gated_ffn(x, w_gate, w_up, w_down, activation) -> y; with gradients
PyObject* py_gated_ffn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 5);
  const Tensor &x = tensor_arg(args[0], "x"), &wg = tensor_arg(args[1], "w_gate"), &wu = tensor_arg(args[2], "w_up"),
               &wd = tensor_arg(args[3], "w_down");
  const int activation = activation_code(text_arg(args[4]));
  ffn_check(x, wg, wu, wd);
  if (needs_grad({&x, &wg, &wu, &wd})) return wrap(FfnNode::apply(x, wg, wu, wd, static_cast<int64_t>(activation)));
  return wrap(ffn_run(x, wg, wu, wd, activation, false).y);
  END_HANDLE_TH_ERRORS
}

// ffn_fwd(x, w_gate, w_up, w_down, activation, keep) -> (y, h or None, kept or None); no gradients
PyObject* py_ffn_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 6);
  const Tensor &x = tensor_arg(args[0], "x"), &wg = tensor_arg(args[1], "w_gate"), &wu = tensor_arg(args[2], "w_up"),
               &wd = tensor_arg(args[3], "w_down");
  const int activation = activation_code(text_arg(args[4]));
  ffn_check(x, wg, wu, wd);
  const FfnOut o = ffn_run(x, wg, wu, wd, activation, args[5] == Py_True);
  return wrap_all({&o.y, &o.h, &o.kept});
  END_HANDLE_TH_ERRORS
}

// ffn_bwd(dy, x, w_gate, w_up, w_down, h, kept, activation, wanted) -> four gradients or None
PyObject* py_ffn_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 9);
  THPObjectPtr list(PySequence_Fast(args[8], "wanted"));
  if (!list) throw python_error();
  count_args(PySequence_Fast_GET_SIZE(list.get()), 4);
  std::vector<bool> wanted(4);
  for (int i = 0; i < 4; ++i) wanted[i] = PySequence_Fast_GET_ITEM(list.get(), i) == Py_True;
  const std::vector<Tensor> g =
      ffn_grads(tensor_arg(args[0], "dy"), tensor_arg(args[1], "x"), tensor_arg(args[2], "w_gate"),
                tensor_arg(args[3], "w_up"), tensor_arg(args[4], "w_down"), tensor_arg(args[5], "h"),
                tensor_arg(args[6], "kept"), activation_code(text_arg(args[7])), wanted);
  return wrap_all({&g[0], &g[1], &g[2], &g[3]});
  END_HANDLE_TH_ERRORS
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, masters or None, m scales or None, v scales or None, ordinals or None,
//       step, lr, beta1, beta2, eps, weight_decay, seed)
PyObject* py_adamw(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 15);
  AdamW s;
  s.params = tensors_of(args[0], "parameters");
  s.grads = tensors_of(args[1], "gradients");
  s.m = tensors_of(args[2], "first moments");
  s.v = tensors_of(args[3], "second moments");
  s.has_masters = args[4] != Py_None;
  if (s.has_masters) s.masters = tensors_of(args[4], "masters");
  TORCH_CHECK_VALUE((args[5] == Py_None) == (args[6] == Py_None), "adamw: 8-bit states need the scales of both moments");
  s.has_scales = args[5] != Py_None;
  if (s.has_scales) {
    s.m_scales = tensors_of(args[5], "scales");
    s.v_scales = tensors_of(args[6], "scales");
  }
  if (args[7] == Py_None) {
    s.ordinals.resize(s.params.size());
    for (size_t i = 0; i < s.ordinals.size(); ++i) s.ordinals[i] = static_cast<int64_t>(i);
  } else {
    THPObjectPtr list(PySequence_Fast(args[7], "ordinals"));
    if (!list) throw python_error();
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(list.get()); ++i)
      s.ordinals.push_back(int_arg(PySequence_Fast_GET_ITEM(list.get(), i)));
  }
  s.a.step = int_arg(args[8]);
  s.a.lr = double_arg(args[9]);
  s.a.beta1 = double_arg(args[10]);
  s.a.beta2 = double_arg(args[11]);
  s.a.eps = double_arg(args[12]);
  s.a.weight_decay = double_arg(args[13]);
  s.a.seed = int_arg(args[14]);
  s.step();
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

double scale_arg(PyObject* o, const Tensor& q) {
  return o == Py_None ? 1.0 / std::sqrt(static_cast<double>(q.dim() > 0 ? std::max<int64_t>(q.size(-1), 1) : 1)) : double_arg(o);
}

// window_attention(q, k, v, window, sinks, scale or None, lengths or None) -> y; with gradients
PyObject* py_window_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 7);
  const Tensor &q = tensor_arg(args[0], "q"), &k = tensor_arg(args[1], "k"), &v = tensor_arg(args[2], "v");
  const int64_t window = int_arg(args[3]), sinks = int_arg(args[4]);
  const double scale = scale_arg(args[5], q);
  const OptTensor lengths = optional_arg(args[6], "lengths");
  window_check(q, k, v, window, sinks, scale, lengths);
  if (needs_grad({&q, &k, &v})) return wrap(WindowNode::apply(q, k, v, window, sinks, scale, lengths));
  return wrap(window_run(q, k, v, window, sinks, scale, lengths, false).first);
  END_HANDLE_TH_ERRORS
}

// window_fwd(q, k, v, window, sinks, scale, lengths or None, keep) -> (y, lse or None); no gradients
PyObject* py_window_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 8);
  const Tensor &q = tensor_arg(args[0], "q"), &k = tensor_arg(args[1], "k"), &v = tensor_arg(args[2], "v");
  const int64_t window = int_arg(args[3]), sinks = int_arg(args[4]);
  const double scale = scale_arg(args[5], q);
  const OptTensor lengths = optional_arg(args[6], "lengths");
  window_check(q, k, v, window, sinks, scale, lengths);
  const auto [y, lse] = window_run(q, k, v, window, sinks, scale, lengths, args[7] == Py_True);
  return wrap_all({&y, &lse});
  END_HANDLE_TH_ERRORS
}

// window_bwd(dy, q, k, v, y, lse, window, sinks, scale, lengths or None) -> (dq, dk, dv)
PyObject* py_window_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 10);
  const Tensor& q = tensor_arg(args[1], "q");
  const std::vector<Tensor> g =
      window_grads(tensor_arg(args[0], "dy"), q, tensor_arg(args[2], "k"), tensor_arg(args[3], "v"), tensor_arg(args[4], "y"),
                   tensor_arg(args[5], "lse"), int_arg(args[6]), int_arg(args[7]), scale_arg(args[8], q),
                   optional_arg(args[9], "lengths"));
  return wrap_all({&g[0], &g[1], &g[2]});
  END_HANDLE_TH_ERRORS
}

// window_step(q, k, v, keys, values, lengths, sinks, scale or None) -> y; keys and values change in place
PyObject* py_window_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 8);
  const Tensor &q = tensor_arg(args[0], "q"), &k = tensor_arg(args[1], "k"), &v = tensor_arg(args[2], "v");
  TORCH_CHECK(!needs_grad({&q, &k, &v}), "window_attention_step has no gradient: call it under torch.no_grad()");
  return wrap(window_step_run(q, k, v, tensor_arg(args[3], "keys"), tensor_arg(args[4], "values"),
                              tensor_arg(args[5], "lengths"), int_arg(args[6]), scale_arg(args[7], q)));
  END_HANDLE_TH_ERRORS
}

// window_extend(k, v, keys, values, lengths, sinks, new or None); keys and values change in place
PyObject* py_window_extend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 7);
  const Tensor &k = tensor_arg(args[0], "k"), &v = tensor_arg(args[1], "v");
  TORCH_CHECK(!needs_grad({&k, &v}), "window_cache_extend has no gradient: call it under torch.no_grad()");
  window_extend_run(k, v, tensor_arg(args[2], "keys"), tensor_arg(args[3], "values"), tensor_arg(args[4], "lengths"),
                    int_arg(args[5]), optional_arg(args[6], "new"));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// scan_step(q, k, v, retentions, append_unit, state, apart) -> reads [views, B, H, 1, width], or (apart) a tuple of each
// view's; the state changes in place
PyObject* py_scan_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 7);
  const Tensor &q = tensor_arg(args[0], "q"), &k = tensor_arg(args[1], "k"), &v = tensor_arg(args[2], "v");
  THPObjectPtr list(PySequence_Fast(args[3], "retentions"));
  if (!list) throw python_error();
  std::vector<OptTensor> retentions;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(list.get()); ++i) {
    retentions.push_back(optional_arg(PySequence_Fast_GET_ITEM(list.get(), i), "a retention"));
    if (retentions.back())
      TORCH_CHECK(!needs_grad({&*retentions.back()}), "linattn_views_step has no gradient: call it under torch.no_grad()");
  }
  TORCH_CHECK(!needs_grad({&q, &k, &v}), "linattn_views_step has no gradient: call it under torch.no_grad()");
  TORCH_CHECK_VALUE(!retentions.empty(), "b200 scan step: no retentions");
  const Tensor reads = scan_step_run(q, k, v, retentions, PyObject_IsTrue(args[4]) == 1, tensor_arg(args[5], "state"));
  if (PyObject_IsTrue(args[6]) != 1) return wrap(reads);
  THPObjectPtr tuple(PyTuple_New(static_cast<Py_ssize_t>(reads.size(0))));
  if (!tuple) throw python_error();
  for (int64_t i = 0; i < reads.size(0); ++i) PyTuple_SET_ITEM(tuple.get(), i, wrap(reads.select(0, i)));
  return tuple.release();
  END_HANDLE_TH_ERRORS
}

// sample(logits, uniform, temperature, top_k or None, top_p or None, min_p or None, logprobs) -> tokens, or (tokens, logprobs)
PyObject* py_sample(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 7);
  const Tensor& logits = tensor_arg(args[0], "logits");
  const bool logprobs = args[6] == Py_True;
  TORCH_CHECK(!logprobs || !needs_grad({&logits}), "sample_tokens: the log-probabilities have no gradient: call it under torch.no_grad()");
  auto tensor = [](PyObject* o, const char* name) { return THPVariable_Check(o) ? OptTensor(tensor_arg(o, name)) : OptTensor(); };
  auto number = [](PyObject* o, double off) { return o == Py_None || THPVariable_Check(o) ? off : double_arg(o); };
  const bool k_number = args[3] != Py_None && !THPVariable_Check(args[3]);
  const int64_t top_k = k_number ? int_arg(args[3]) : 0;
  TORCH_CHECK_VALUE(!k_number || top_k >= 1, "top_k must be >= 1, got ", top_k);
  const auto [tokens, chances] =
      sample_run(logits, tensor_arg(args[1], "uniform"), tensor(args[2], "temperature"), number(args[2], 1.0),
                 tensor(args[3], "top_k"), top_k, tensor(args[4], "top_p"), number(args[4], 1.0), tensor(args[5], "min_p"),
                 number(args[5], 0.0), logprobs);
  return logprobs ? wrap_all({&tokens, &chances}) : wrap(tokens);
  END_HANDLE_TH_ERRORS
}

#define TS_METHOD(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {TS_METHOD(rms_norm),  TS_METHOD(norm_fwd), TS_METHOD(norm_bwd), TS_METHOD(rms_norm_8bit),
                         TS_METHOD(gated_ffn), TS_METHOD(ffn_fwd),  TS_METHOD(ffn_bwd),  TS_METHOD(adamw),
                         TS_METHOD(window_attention), TS_METHOD(window_fwd), TS_METHOD(window_bwd), TS_METHOD(window_step),
                         TS_METHOD(window_extend), TS_METHOD(scan_step), TS_METHOD(sample),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host side of the operators whose calls are short.", -1,
                      methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
