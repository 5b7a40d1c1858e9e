// operators_torch.cpp -- the cell-training operators of libnca_b200 as differentiable torch
// operators (torch.ops.nca_b200.group_norm_act, gated_ffn, distill_loss, distill_loss_and_grad).
//
// Each operator checks its arguments (ValueError / TypeError with the argument's name), allocates
// outputs and workspace from torch's caching allocator, and enqueues on torch's current stream of
// the input's device.  The gradients are first-order and backward: a backward pass under
// create_graph=True and forward-mode tangents are refused instead of giving a derivative that is
// silently constant.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <array>
#include <cstdlib>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/nca_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* stream_of(const Tensor& t) {
  return reinterpret_cast<void*>(at::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

void check(int32_t status, const char* what) {
  TORCH_CHECK(status == NCA_OK, what, ": ", nca_b200_status_string(status), " (status ", status, ")");
}

int dtype_of(const Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return NCA_F32;
    case at::kBFloat16: return NCA_BF16;
    case at::kHalf: return NCA_F16;
    default: break;
  }
  TORCH_CHECK_TYPE(false, op, ": ", name, " must be float32, bfloat16 or float16, not ", t.scalar_type());
  return -1;
}

int act_of(const std::string& act, bool gated, const char* op) {
  if (act == "none" && !gated) return NCA_ACT_NONE;
  if (act == "relu") return NCA_ACT_RELU;
  if (act == "silu") return NCA_ACT_SILU;
  if (act == "gelu") return NCA_ACT_GELU;
  if (act == "sigmoid") return NCA_ACT_SIGMOID;
  TORCH_CHECK_VALUE(false, op, ": act must be ", gated ? "" : "'none', ", "'relu', 'silu', 'gelu' or 'sigmoid', not '",
                    act, "'");
  return -1;
}

void on_cuda(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), op, ": ", name, " must be a CUDA tensor (there is no CPU fallback)");
  TORCH_CHECK_VALUE(t.layout() == at::kStrided, op, ": ", name, " must be a dense tensor");
}
void same_device(const Tensor& t, const Tensor& ref, const char* op, const char* name) {
  on_cuda(t, op, name);
  TORCH_CHECK_VALUE(t.get_device() == ref.get_device(), op, ": ", name, " must be on ", ref.device(), ", not ",
                    t.device());
}
void first_order(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": the backward pass is not differentiable (create_graph=True)");
}
void no_tangent(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK_VALUE(!t.defined() || !t._fw_grad(0).defined(), op, ": ", name,
                    " carries a forward-mode tangent, and there is no forward-mode derivative");
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool any_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (wants_grad(*t)) return true;
  return false;
}
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
// Which inputs of an autograd function need a gradient.  Autograd numbers the tensors that were
// passed, without the absent ones.
struct Needs {
  std::array<bool, 8> need{};
  Needs(AutogradContext* ctx, std::initializer_list<Tensor> inputs) {
    size_t edge = 0, i = 0;
    for (const Tensor& t : inputs) need[i++] = t.defined() && ctx->needs_input_grad(edge++);
  }
  bool operator[](size_t i) const { return need[i]; }
};
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
size_t bytes_of(const Tensor& t) { return t.defined() ? (size_t)t.numel() : 0; }

// -------------------------------------------------------------------------------- group norm
// (N, ..., C) seen as samples x cells x channels: a view when the dimensions between collapse to
// one stride and the channels are adjacent, else a copy.
struct Cells {
  Tensor t;
  int64_t n = 0, cells = 0, stride_n = 0, stride_cell = 0;
};
bool collapse(const Tensor& t, int64_t first, int64_t last, int64_t* size, int64_t* stride) {
  int64_t n = 1, s = 0;
  for (int64_t i = first; i < last; ++i)
    if (t.size(i) == 0) {  // no cells, whatever the strides
      *size = *stride = 0;
      return true;
    }
  for (int64_t i = last - 1; i >= first; --i) {
    if (t.size(i) == 1) continue;
    if (n == 1) s = t.stride(i);
    else if (t.stride(i) != n * s) return false;
    n *= t.size(i);
  }
  *size = n;
  *stride = s;
  return true;
}
Cells cells_of(const Tensor& x, bool channels) {
  Cells c;
  c.t = x;
  const int64_t last = x.dim() - (channels ? 1 : 0);
  const bool adjacent = !channels || x.size(-1) <= 1 || x.stride(-1) == 1;
  if (!adjacent || !collapse(x, 1, last, &c.cells, &c.stride_cell)) {
    c.t = x.contiguous();
    collapse(c.t, 1, last, &c.cells, &c.stride_cell);
  }
  c.n = x.size(0);
  c.stride_n = x.size(0) > 1 ? c.t.stride(0) : c.cells * c.stride_cell;
  return c;
}

constexpr int64_t kMostChannels = 1ll << 30;  // the kernels' channel numbers, and those of a tile beyond, fit 32 bits
struct Norm {
  NcaNormDesc d{};
  static int unaligned(const Tensor& t) {
    return t.defined() && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 ? 1 : 0;
  }
  Cells x, mask, dy;
  Norm(const Tensor& xt, int64_t groups, const Tensor& weight, const Tensor& bias, double eps, int act,
       const Tensor& maskt) {
    x = cells_of(xt, true);
    d.n = x.n;
    d.cells = x.cells;
    d.channels = (int32_t)xt.size(-1);
    d.groups = (int32_t)groups;
    d.dtype = dtype_of(xt, "group_norm_act", "x");
    const Tensor& param = weight.defined() ? weight : bias;
    d.param_dtype = param.defined() ? dtype_of(param, "group_norm_act", "weight") : NCA_F32;
    d.act = act;
    d.eps = (float)eps;
    d.x_stride_n = x.stride_n;
    d.x_stride_cell = x.stride_cell;
    if (maskt.defined()) {
      mask = cells_of(maskt, false);
      d.masked = 1;
      d.mask_stride_n = mask.stride_n;
      d.mask_stride_cell = mask.stride_cell;
    }
  }
  Tensor workspace(bool backward, const Tensor& out) {
    size_t bytes = 0;
    d.unaligned = unaligned(x.t) | unaligned(out) | unaligned(dy.t);
    check(nca_b200_group_norm_workspace(&d, backward, &bytes), "nca_b200_group_norm_workspace");
    return scratch(bytes, x.t);
  }
};

std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, int64_t groups, const Tensor& weight, const Tensor& bias,
                                        double eps, int act, const Tensor& mask, bool save) {
  const c10::cuda::CUDAGuard guard(x.device());
  Norm n(x, groups, weight, bias, eps, act, mask);
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor stats = save ? at::empty({n.d.n, groups, 2}, x.options().dtype(at::kFloat)) : Tensor();
  Tensor ws = n.workspace(false, y);
  check(nca_b200_group_norm(&n.d, ptr(n.x.t), ptr(weight), ptr(bias), static_cast<const uint8_t*>(ptr(n.mask.t)),
                            mptr(y), static_cast<float*>(mptr(stats)), mptr(ws), bytes_of(ws), stream_of(x)),
        "nca_b200_group_norm");
  return {y, stats};
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t groups, const OptTensor& weight_,
                        const OptTensor& bias_, double eps, int64_t act, const OptTensor& mask_) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor weight = or_none(weight_), bias = or_none(bias_), mask = or_none(mask_);
    auto [y, stats] = norm_forward(x, groups, weight, bias, eps, (int)act, mask, true);
    ctx->save_for_backward({x, weight, bias, mask, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order("group_norm_act");
    no_tangent(grads[0], "group_norm_act", "the gradient");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &mask = saved[3], &stats = saved[4];
    const c10::cuda::CUDAGuard guard(x.device());
    Norm n(x, ctx->saved_data["groups"].toInt(), weight, bias, ctx->saved_data["eps"].toDouble(),
           (int)ctx->saved_data["act"].toInt(), mask);
    n.dy = cells_of(grads[0], true);
    n.d.dy_stride_n = n.dy.stride_n;
    n.d.dy_stride_cell = n.dy.stride_cell;
    Tensor dx, dw, db;
    const Needs needs(ctx, {x, weight, bias, mask});
    if (needs[0]) dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    if (needs[1]) dw = at::empty_like(weight, at::MemoryFormat::Contiguous);
    if (needs[2]) db = at::empty_like(bias, at::MemoryFormat::Contiguous);
    Tensor ws = n.workspace(true, dx);
    check(nca_b200_group_norm_backward(&n.d, ptr(n.x.t), ptr(weight), ptr(bias),
                                       static_cast<const uint8_t*>(ptr(n.mask.t)),
                                       static_cast<const float*>(ptr(stats)), ptr(n.dy.t), mptr(dx), mptr(dw),
                                       mptr(db), mptr(ws), bytes_of(ws), stream_of(x)),
          "nca_b200_group_norm_backward");
    return {dx, Tensor(), dw, db, Tensor(), Tensor(), Tensor()};
  }
};

Tensor group_norm_act(const Tensor& x, int64_t groups, const OptTensor& weight_, const OptTensor& bias_, double eps,
                      std::string act_, const OptTensor& mask_) {
  constexpr const char* op = "group_norm_act";
  on_cuda(x, op, "x");
  no_tangent(x, op, "x");
  dtype_of(x, op, "x");
  const int act = act_of(act_, false, op);
  TORCH_CHECK_VALUE(x.dim() >= 2, op, ": x must be (N, ..., C), not ", x.sizes());
  const int64_t c = x.size(-1);
  TORCH_CHECK_VALUE(c > 0 && groups > 0 && c % groups == 0, op, ": ", groups, " groups do not divide ", c, " channels");
  TORCH_CHECK_VALUE(c <= kMostChannels, op, ": at most ", kMostChannels, " channels, not ", c);
  TORCH_CHECK_VALUE(eps >= 0, op, ": eps must not be negative");
  Tensor weight = or_none(weight_), bias = or_none(bias_), mask = or_none(mask_);
  for (const auto& [t, name] : {std::pair<Tensor*, const char*>{&weight, "weight"}, {&bias, "bias"}}) {
    if (!t->defined()) continue;
    same_device(*t, x, op, name);
    no_tangent(*t, op, name);
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == c, op, ": ", name, " must have shape (", c, "), not ", t->sizes());
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type(), op, ": ", name,
                     " must be float32 or of x's type");
    if (!t->is_contiguous()) *t = t->contiguous();
  }
  if (weight.defined() && bias.defined())
    TORCH_CHECK_TYPE(weight.scalar_type() == bias.scalar_type(), op, ": weight and bias must have one type");
  if (mask.defined()) {
    same_device(mask, x, op, "mask");
    TORCH_CHECK_TYPE(mask.scalar_type() == at::kBool || mask.scalar_type() == at::kByte, op,
                     ": mask must be bool or uint8");
    TORCH_CHECK_VALUE(mask.sizes() == x.sizes().slice(0, x.dim() - 1), op, ": mask must have shape ",
                      x.sizes().slice(0, x.dim() - 1), ", not ", mask.sizes());
  }
  if (any_grad({&x, &weight, &bias})) 
    return NormFunction::apply(x, groups, optional(weight), optional(bias), eps, (int64_t)act, optional(mask));
  return std::get<0>(norm_forward(x, groups, weight, bias, eps, act, mask, false));
}

// -------------------------------------------------------------------------------- gated block
// Control words of the bounded waits, one set a device, kept for the process.  They record that a wait ran
// out; whichever thread asks first (operators.check()) reads and clears them, and `count` tells the others.
struct Failures {
  std::mutex m, asking;
  Tensor words;
  int64_t count = 0;  // times that a failure was read
  int32_t status = 0, detail = 0;  // the last
};
constexpr int kMostDevices = 64;
Failures& failures(const c10::Device& dev) {
  static auto& kept = *new std::array<Failures, kMostDevices>;  // never destroyed: CUDA may be gone by then
  TORCH_CHECK(dev.index() >= 0 && dev.index() < kMostDevices, "device index ", (int)dev.index());
  return kept[dev.index()];
}
// The failures that this thread knows of: those of its time, from its first call on.
int64_t& known_failures(const c10::Device& dev) {
  thread_local std::array<int64_t, kMostDevices> known = [] {
    std::array<int64_t, kMostDevices> a;
    a.fill(-1);
    return a;
  }();
  return known[dev.index()];
}
Tensor control_words(const c10::Device& dev) {
  Failures& f = failures(dev);
  std::lock_guard<std::mutex> lock(f.m);
  if (!f.words.defined()) {
    f.words = at::zeros({4}, at::TensorOptions().device(dev).dtype(at::kInt));
    at::cuda::getCurrentCUDAStream(dev.index()).synchronize();  // once: every stream finds them cleared
  }
  int64_t& known = known_failures(dev);
  if (known < 0) known = f.count;
  return f.words;
}
// Limit of any single wait inside a kernel, as ncas_b200.engine reads it.
int32_t timeout_ms() {
  static const int32_t ms = [] {
    const char* v = std::getenv("NCA_B200_TIMEOUT_MS");
    const int n = v ? std::atoi(v) : 0;
    return n > 0 ? n : 20000;
  }();
  return ms;
}

struct Gated {
  NcaGatedDesc d{};
  static void strides(int64_t* to, const Tensor& t) {
    to[0] = t.stride(0);
    to[1] = t.stride(1);
  }
  static int unaligned(const Tensor& t, int bit) {
    return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 ? 1 << bit : 0;
  }
  Gated(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int bias_dtype, int act) {
    d.rows = x.size(0);
    d.d_in = x.size(1);
    d.hidden = wg.size(0);
    d.d_out = wd.size(0);
    d.dtype = x.scalar_type() == at::kBFloat16 ? NCA_BF16 : NCA_F16;
    d.bias_dtype = bias_dtype;
    d.act = act;
    strides(d.x_stride, x);
    strides(d.w_gate_stride, wg);
    strides(d.w_up_stride, wu);
    strides(d.w_down_stride, wd);
    d.unaligned = unaligned(x, 0) | unaligned(wg, 1) | unaligned(wu, 2) | unaligned(wd, 3);
  }
  void set_dy(const Tensor& dy) {
    strides(d.dy_stride, dy);
    d.unaligned |= unaligned(dy, 4);
  }
};

std::tuple<Tensor, Tensor> gated_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                                         const Tensor& bg, const Tensor& bu, const Tensor& bd, int bias_dtype, int act,
                                         bool save) {
  const c10::cuda::CUDAGuard guard(x.device());
  Gated g(x, wg, wu, wd, bias_dtype, act);
  Tensor y = at::empty({x.size(0), wd.size(0)}, x.options());
  size_t bytes = 0;
  Tensor saved;
  if (save) {
    check(nca_b200_gated_saved_bytes(&g.d, &bytes), "nca_b200_gated_saved_bytes");
    saved = scratch(bytes, x);
  }
  check(nca_b200_gated_workspace(&g.d, 0, &bytes), "nca_b200_gated_workspace");
  Tensor ws = scratch(bytes, x), ctrl = control_words(x.device());
  check(nca_b200_gated_ffn(&g.d, ptr(x), ptr(wg), ptr(wu), ptr(wd), ptr(bg), ptr(bu), ptr(bd), mptr(y), mptr(saved),
                           mptr(ws), bytes_of(ws), static_cast<int32_t*>(mptr(ctrl)), timeout_ms(),
                           stream_of(x)),
        "nca_b200_gated_ffn");
  return {y, saved};
}

struct GatedFunction : torch::autograd::Function<GatedFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                        const OptTensor& bg_, const OptTensor& bu_, const OptTensor& bd_, int64_t bias_dtype,
                        int64_t act) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor bg = or_none(bg_), bu = or_none(bu_), bd = or_none(bd_);
    auto [y, saved] = gated_forward(x, wg, wu, wd, bg, bu, bd, (int)bias_dtype, (int)act, true);
    ctx->save_for_backward({x, wg, wu, wd, bg, bu, bd, saved});
    ctx->saved_data["bias_dtype"] = bias_dtype;
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order("gated_ffn");
    no_tangent(grads[0], "gated_ffn", "the gradient");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &wd = saved[3];
    const Tensor& dy = grads[0];
    const c10::cuda::CUDAGuard guard(x.device());
    Gated g(x, wg, wu, wd, (int)ctx->saved_data["bias_dtype"].toInt(), (int)ctx->saved_data["act"].toInt());
    g.set_dy(dy);
    Tensor out[7];
    const Needs needs(ctx, {saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6]});
    for (int i = 0; i < 7; ++i)
      if (needs[i])
        out[i] = at::empty(saved[i].sizes(), saved[i].options().memory_format(at::MemoryFormat::Contiguous));
    size_t bytes = 0;
    check(nca_b200_gated_workspace(&g.d, needs[4] || needs[5] ? 1 : 2, &bytes), "nca_b200_gated_workspace");
    Tensor ws = scratch(bytes, x), ctrl = control_words(x.device());
    check(nca_b200_gated_ffn_backward(&g.d, ptr(x), ptr(wg), ptr(wu), ptr(wd), ptr(saved[7]), ptr(dy), mptr(out[0]),
                                      mptr(out[1]), mptr(out[2]), mptr(out[3]), mptr(out[4]), mptr(out[5]),
                                      mptr(out[6]), mptr(ws), bytes_of(ws), static_cast<int32_t*>(mptr(ctrl)),
                                      timeout_ms(), stream_of(x)),
          "nca_b200_gated_ffn_backward");
    return {out[0], out[1], out[2], out[3], out[4], out[5], out[6], Tensor(), Tensor()};
  }
};

Tensor gated_ffn(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down,
                 const OptTensor& b_gate, const OptTensor& b_up, const OptTensor& b_down, std::string act_) {
  constexpr const char* op = "gated_ffn";
  on_cuda(x, op, "x");
  no_tangent(x, op, "x");
  const int act = act_of(act_, true, op);
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, op,
                   ": x must be bfloat16 or float16, not ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, op, ": x must be (..., d_in) with d_in > 0, not ", x.sizes());
  for (const auto& [t, name] : {std::pair<const Tensor*, const char*>{&w_gate, "w_gate"}, {&w_up, "w_up"},
                                {&w_down, "w_down"}}) {
    same_device(*t, x, op, name);
    no_tangent(*t, op, name);
    TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type(), op, ": ", name, " must be of x's type ", x.scalar_type(),
                     ", not ", t->scalar_type());
    TORCH_CHECK_VALUE(t->dim() == 2 && t->numel() > 0, op, ": ", name, " must be a non-empty matrix, not ", t->sizes());
  }
  const int64_t d = x.size(-1), f = w_gate.size(0), o = w_down.size(0);
  TORCH_CHECK_VALUE(w_gate.size(1) == d, op, ": w_gate must be (hidden, ", d, "), not ", w_gate.sizes());
  TORCH_CHECK_VALUE(w_up.sizes() == w_gate.sizes(), op, ": w_up must be ", w_gate.sizes(), ", not ", w_up.sizes());
  TORCH_CHECK_VALUE(w_down.size(1) == f, op, ": w_down must be (d_out, ", f, "), not ", w_down.sizes());
  Tensor b[3] = {or_none(b_gate), or_none(b_up), or_none(b_down)};
  const char* names[3] = {"b_gate", "b_up", "b_down"};
  const int64_t sizes[3] = {f, f, o};
  int bias_dtype = NCA_F32;
  const Tensor* first = nullptr;
  for (int i = 0; i < 3; ++i) {
    if (!b[i].defined()) continue;
    same_device(b[i], x, op, names[i]);
    no_tangent(b[i], op, names[i]);
    TORCH_CHECK_VALUE(b[i].dim() == 1 && b[i].size(0) == sizes[i], op, ": ", names[i], " must have shape (", sizes[i],
                      "), not ", b[i].sizes());
    TORCH_CHECK_TYPE(b[i].scalar_type() == at::kFloat || b[i].scalar_type() == x.scalar_type(), op, ": ", names[i],
                     " must be float32 or of x's type");
    TORCH_CHECK_TYPE(!first || first->scalar_type() == b[i].scalar_type(), op, ": the biases must have one type");
    first = &b[i];
    bias_dtype = dtype_of(b[i], op, names[i]);
    if (!b[i].is_contiguous()) b[i] = b[i].contiguous();
  }
  Tensor rows = x.dim() == 2 ? x : x.reshape({-1, d});
  Tensor y;
  if (any_grad({&x, &w_gate, &w_up, &w_down, &b[0], &b[1], &b[2]}))
    y = GatedFunction::apply(rows, w_gate, w_up, w_down, optional(b[0]), optional(b[1]), optional(b[2]),
                             (int64_t)bias_dtype, (int64_t)act);
  else
    y = std::get<0>(gated_forward(rows, w_gate, w_up, w_down, b[0], b[1], b[2], bias_dtype, act, false));
  if (x.dim() == 2) return y;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = o;
  return y.view(shape);
}

std::vector<int64_t> operators_status(const Tensor& like) {
  on_cuda(like, "operators_status", "like");
  const c10::cuda::CUDAGuard guard(like.device());
  const Tensor words = control_words(like.device());
  Failures& f = failures(like.device());
  std::lock_guard<std::mutex> one_at_a_time(f.asking);
  int32_t detail = 0;
  const int32_t s = nca_b200_ctrl_status(static_cast<int32_t*>(mptr(words)), &detail, stream_of(like));
  if (s != NCA_OK && s != NCA_ERR_TIMEOUT) return {s, detail};
  std::lock_guard<std::mutex> lock(f.m);
  if (s != NCA_OK) {
    ++f.count;
    f.status = s;
    f.detail = detail;
  }
  int64_t& known = known_failures(like.device());
  if (known == f.count) return {NCA_OK, 0};
  known = f.count;
  return {f.status, f.detail};
}

// ------------------------------------------------------------------------------- distillation
struct Distill {
  NcaDistillDesc d{};
  Tensor logits, teacher, index, weight;  // rows x classes, rows x top, rows x top, rows
};

Tensor rows_of(const Tensor& t, int64_t width) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});
  if (r.size(1) > 1 && r.stride(1) != 1) r = r.contiguous();
  return r;
}

Distill distill_args(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature,
                     const OptTensor& weight, const char* op) {
  on_cuda(logits, op, "logits");
  Distill a;
  a.d.dtype = dtype_of(logits, op, "logits");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) > 0, op,
                    ": logits must be (..., classes) with classes > 0, not ", logits.sizes());
  no_tangent(logits, op, "logits");
  same_device(teacher, logits, op, "teacher_logits");
  no_tangent(teacher, op, "teacher_logits");
  same_device(index, logits, op, "teacher_index");
  a.d.teacher_dtype = dtype_of(teacher, op, "teacher_logits");
  TORCH_CHECK_TYPE(index.scalar_type() == at::kInt || index.scalar_type() == at::kLong, op,
                   ": teacher_index must be int32 or int64, not ", index.scalar_type());
  TORCH_CHECK_VALUE(teacher.dim() == logits.dim() &&
                        teacher.sizes().slice(0, teacher.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
                    op, ": teacher_logits must be (..., top) with the leading sizes of logits ", logits.sizes(),
                    ", not ", teacher.sizes());
  TORCH_CHECK_VALUE(index.sizes() == teacher.sizes(), op, ": teacher_index must be ", teacher.sizes(), ", not ",
                    index.sizes());
  TORCH_CHECK_VALUE(teacher.size(-1) <= 4096, op, ": at most 4096 entries a row, not ", teacher.size(-1));
  const float tau = (float)temperature;
  TORCH_CHECK_VALUE(tau >= 1e-30f && tau <= 1e30f, op, ": temperature must lie between 1e-30 and 1e30, not ", temperature);
  TORCH_CHECK_VALUE(!teacher.requires_grad() || !at::GradMode::is_enabled(), op,
                    ": teacher_logits gets no gradient: detach it");
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < logits.dim(); ++i) rows *= logits.size(i);
  const int64_t top = teacher.size(-1);
  a.logits = rows ? rows_of(logits, logits.size(-1)) : logits;
  a.teacher = rows && top ? rows_of(teacher, top) : teacher;
  a.index = rows && top ? rows_of(index, top) : index;
  if (weight.has_value() && weight->defined()) {
    same_device(*weight, logits, op, "weight");
    no_tangent(*weight, op, "weight");
    TORCH_CHECK_TYPE(weight->scalar_type() == at::kFloat, op, ": weight must be float32");
    TORCH_CHECK_VALUE(weight->sizes() == logits.sizes().slice(0, logits.dim() - 1), op, ": weight must be ",
                      logits.sizes().slice(0, logits.dim() - 1), ", not ", weight->sizes());
    TORCH_CHECK_VALUE(!weight->requires_grad() || !at::GradMode::is_enabled(), op,
                      ": weight gets no gradient: detach it");
    a.weight = weight->reshape({-1}).contiguous();
  }
  a.d.rows = rows;
  a.d.classes = logits.size(-1);
  a.d.top = top;
  a.d.index_bits = index.scalar_type() == at::kInt ? 32 : 64;
  a.d.temperature = tau;
  a.d.logits_stride = rows > 1 ? a.logits.stride(0) : a.d.classes;
  a.d.teacher_stride = rows > 1 && top ? a.teacher.stride(0) : top;
  a.d.index_stride = rows > 1 && top ? a.index.stride(0) : top;
  return a;
}

Tensor distill_run(Distill& a, const Tensor& stats, const Tensor& dlogits) {
  Tensor loss = at::empty({a.d.rows}, a.logits.options().dtype(at::kFloat));
  size_t bytes = 0;
  check(nca_b200_distill_workspace(&a.d, &bytes), "nca_b200_distill_workspace");
  Tensor ws = scratch(bytes, a.logits);
  check(nca_b200_distill(&a.d, ptr(a.logits), ptr(a.teacher), ptr(a.index), static_cast<const float*>(ptr(a.weight)),
                         static_cast<float*>(mptr(loss)), static_cast<float*>(mptr(stats)), mptr(dlogits), mptr(ws),
                         bytes_of(ws), stream_of(a.logits)),
        "nca_b200_distill");
  return loss;
}

struct DistillFunction : torch::autograd::Function<DistillFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher, const Tensor& index,
                        double temperature, const OptTensor& weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(logits.device());
    Distill a = distill_args(logits, teacher, index, temperature, weight, "distill_loss");
    Tensor stats = at::empty({a.d.rows, 2}, logits.options().dtype(at::kFloat));
    Tensor loss = distill_run(a, stats, Tensor());
    ctx->save_for_backward({logits, teacher, index, or_none(weight), stats});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order("distill_loss");
    no_tangent(grads[0], "distill_loss", "the gradient");
    const auto saved = ctx->get_saved_variables();
    const Tensor& logits = saved[0];
    const c10::cuda::CUDAGuard guard(logits.device());
    Distill a = distill_args(logits, saved[1], saved[2], ctx->saved_data["temperature"].toDouble(), optional(saved[3]),
                             "distill_loss");
    Tensor grad = grads[0].to(at::kFloat);
    Tensor out = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
    check(nca_b200_distill_backward(&a.d, ptr(a.logits), ptr(a.teacher), ptr(a.index),
                                    static_cast<const float*>(ptr(a.weight)), static_cast<const float*>(ptr(saved[4])),
                                    static_cast<const float*>(ptr(grad)), a.d.rows > 1 ? grad.stride(0) : 0, mptr(out),
                                    stream_of(logits)),
          "nca_b200_distill_backward");
    return {out, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor reduced(const Tensor& loss, const std::string& reduction, const Tensor& logits, const char* op) {
  if (reduction == "sum") return loss.sum();
  if (reduction == "mean") return loss.mean();
  TORCH_CHECK_VALUE(reduction == "none", op, ": reduction must be 'none', 'sum' or 'mean', not '", reduction, "'");
  return loss.view(logits.sizes().slice(0, logits.dim() - 1));
}

Tensor distill_loss(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature,
                    const OptTensor& weight, std::string reduction) {
  Tensor loss;
  if (any_grad({&logits})) {
    distill_args(logits, teacher, index, temperature, weight, "distill_loss");  // the checks, before autograd
    loss = DistillFunction::apply(logits, teacher, index, temperature, weight);
  } else {
    Distill a = distill_args(logits, teacher, index, temperature, weight, "distill_loss");
    const c10::cuda::CUDAGuard guard(logits.device());
    loss = distill_run(a, Tensor(), Tensor());
  }
  return reduced(loss, reduction, logits, "distill_loss");
}

std::tuple<Tensor, Tensor> distill_loss_and_grad(const Tensor& logits_, const Tensor& teacher, const Tensor& index,
                                                 double temperature, const OptTensor& weight_, std::string reduction) {
  no_tangent(logits_, "distill_loss_and_grad", "logits");
  const Tensor logits = logits_.detach();
  at::NoGradGuard no_grad;
  Distill a = distill_args(logits, teacher, index, temperature, weight_, "distill_loss_and_grad");
  const c10::cuda::CUDAGuard guard(logits.device());
  if (reduction == "mean" && a.d.rows > 0)  // the mean's 1 / rows goes into the rows' weights
    a.weight = a.weight.defined() ? a.weight.div(at::Scalar((double)a.d.rows))
                                  : at::full({a.d.rows}, 1.0 / (double)a.d.rows, logits.options().dtype(at::kFloat));
  Tensor grad = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor loss = distill_run(a, Tensor(), grad);
  return {reduced(loss, reduction == "mean" && a.d.rows > 0 ? "sum" : reduction, logits, "distill_loss_and_grad"), grad};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nca_b200, m) {
  m.def("group_norm_act(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, str act, Tensor? mask) -> Tensor",
        &group_norm_act);
  m.def("gated_ffn(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, Tensor? b_gate, Tensor? b_up, Tensor? b_down, "
        "str act) -> Tensor",
        &gated_ffn);
  m.def("distill_loss(Tensor logits, Tensor teacher_logits, Tensor teacher_index, float temperature, Tensor? weight, "
        "str reduction) -> Tensor",
        &distill_loss);
  m.def("distill_loss_and_grad(Tensor logits, Tensor teacher_logits, Tensor teacher_index, float temperature, "
        "Tensor? weight, str reduction) -> (Tensor, Tensor)",
        &distill_loss_and_grad);
  m.def("operators_status(Tensor like) -> int[]", &operators_status);
}
