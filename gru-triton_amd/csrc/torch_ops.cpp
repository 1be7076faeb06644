// The torch side of the gated linear recurrence, the linear operator and AdamW: argument
// checks, allocations and autograd in C++ around the C ABI of libgruscan.so. A call of
// these operators takes the GPU a few microseconds at small sizes; from Python its checks,
// struct and autograd node took longer than that (a training step of the recurrence 93 us
// on the host, of which torch's engine is 45).
//
// Errors are ValueError (device, dtype, shape, arguments) and RuntimeError (HIP), as in
// the rest of the package.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <atomic>
#include <string>
#include <vector>

#include "../../include/gruscan.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kStateBlock = 256;  // elements that share a scale where moments are held in 8 bits

void raise_for(int64_t rc) {
  if (rc >= 0) return;
  TORCH_CHECK_VALUE(rc != GS_ERR_INVALID, gs_last_error());
  TORCH_CHECK(false, gs_last_error());
}

// The tensors' device made current, and torch's stream there.
struct On {
  c10::hip::OptionalHIPGuard guard;
  hipStream_t stream;
  explicit On(const Tensor& t) {
    const auto d = t.device();
    if (d.index() != c10::hip::current_device()) guard.set_index(d.index());
    stream = c10::hip::getCurrentHIPStream(d.index()).stream();
  }
};

template <typename T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

int dtype_of(const char* who, const char* name, const Tensor& t) {
  if (t.scalar_type() == torch::kFloat) return GS_DTYPE_F32;
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kBFloat16, who, ": ", name, " dtype must be float32 or bfloat16; got ",
                    t.scalar_type());
  return GS_DTYPE_BF16;
}

// A tangent of forward-mode differentiation would be lost without a word: the kernels read values
// alone, and a dual tensor need not require a gradient.
void check_no_tangent(const char* who, const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), who, ": forward-mode derivatives are not implemented; ", name,
                              " has a tangent");
}

void check_on(const char* who, const char* name, const Tensor& t, const Tensor& ref) {
  TORCH_CHECK_VALUE(t.is_cuda(), who, ": ", name, " must be a CUDA (HIP) tensor; got ", t.device());
  TORCH_CHECK_VALUE(t.device() == ref.device(), who, ": all tensors must be on ", ref.device(), "; ", name, " is on ",
                    t.device());
  check_no_tangent(who, name, t);
}

// Unit stride along the last dimension.
Tensor unit(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// A tensor written through its pointer counts as modified in place: autograd refuses graphs
// that saved it before, and what the package keeps per version of a weight is found anew.
void modified(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }
// Asked before the launch: a tensor made in inference mode has no version to count outside it.
void check_may_modify(const char* who, const char* name, const Tensor& t) {
  TORCH_CHECK(!t.is_inference() || c10::InferenceMode::is_enabled(), who, ": ", name,
              " was made in inference mode and cannot be updated in place outside it");
}

// A backward's results. Where a graph of them is asked for (create_graph), it goes on to
// `from`, which they were computed from, through an error for whoever asks for a second
// derivative: without it that derivative would lack their terms and nobody would know.
variable_list once(const char* who, variable_list grads, const variable_list& from) {
  if (!torch::GradMode::is_enabled()) return grads;
  const size_t n = grads.size();
  grads.insert(grads.end(), from.begin(), from.end());
  grads = torch::autograd::DelayedError(std::string(who) + ": second derivatives are not implemented",
                                        (int64_t)grads.size())(std::move(grads));
  grads.resize(n);
  return grads;
}

Tensor scratch(int64_t bytes, const Tensor& like) {
  raise_for(bytes);
  return bytes ? torch::empty({bytes}, like.options().dtype(torch::kByte)) : Tensor();
}

// ---- gated linear recurrence ---------------------------------------------------------

// The device's fault mirror, which a chained scan writes when a wait runs out (_lib.py holds
// them all). The first scan that needs it makes it, unless it is being captured, where no host
// memory may be allocated: that scan then reports by its NaNs alone.
constexpr int kMostDevices = 64;
std::atomic<uint32_t*> fault_words[kMostDevices];

uint32_t* fault_word(int64_t device) {
  if (device >= kMostDevices) return nullptr;
  uint32_t* word = fault_words[device].load(std::memory_order_acquire);
  if (word == nullptr && c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) {
    py::gil_scoped_acquire gil;
    word = reinterpret_cast<uint32_t*>(
        py::module_::import("gru_qat_amd._lib").attr("scan_fault_word")(device).cast<uintptr_t>());
    fault_words[device].store(word, std::memory_order_release);
  }
  return word;
}

void raise_scan_fault(const char* who, int64_t device) {
  const uint32_t* word = device < kMostDevices ? fault_words[device].load(std::memory_order_acquire) : nullptr;
  if (word == nullptr || *static_cast<const volatile uint32_t*>(word) == 0) return;
  py::gil_scoped_acquire gil;
  py::module_::import("gru_qat_amd._lib").attr("raise_scan_fault")(device, who);
}

// out as [T, B, H], batch rows outermost in memory where gi's are (batch_first).
std::tuple<Tensor, Tensor> glr_forward(const Tensor& gi, const Tensor& h0, const Tensor& reset, int64_t act,
                                       bool batch_first) {
  const int64_t T = gi.size(0), B = gi.size(1), H = gi.size(2) / 2;
  Tensor out = batch_first ? torch::empty({B, T, H}, gi.options()).transpose(0, 1) : torch::empty({T, B, H}, gi.options());
  Tensor h_last = torch::empty({B, H}, gi.options().dtype(torch::kFloat));
  gs_glr_args a{};
  a.gi = gi.data_ptr();
  a.h0 = ptr<float>(h0);
  a.reset = ptr<uint8_t>(reset);
  a.out = out.data_ptr();
  a.h_last = h_last.data_ptr<float>();
  a.T = T;
  a.B = B;
  a.H = H;
  a.sg_t = gi.stride(0);
  a.sg_b = gi.stride(1);
  a.sh0_b = h0.defined() ? h0.stride(0) : 0;
  a.sr_t = reset.defined() ? reset.stride(0) : 0;
  a.sr_b = reset.defined() ? reset.stride(1) : 0;
  a.so_t = out.stride(0);
  a.so_b = out.stride(1);
  a.dtype = gi.scalar_type() == torch::kFloat ? GS_DTYPE_F32 : GS_DTYPE_BF16;
  a.activation = (int32_t)act;
  const On on(gi);
  const Tensor buf = scratch(gs_glr_scratch_bytes(&a), gi);
  a.scratch = ptr<void>(buf);
  a.scratch_bytes = buf.defined() ? buf.numel() : 0;
  if (buf.defined()) a.fault_mirror = fault_word(gi.get_device());
  raise_for(gs_glr_fwd(&a, on.stream));
  return {out, h_last};  // the caching allocator keeps buf until the stream's work is done
}

struct GlrFunction : torch::autograd::Function<GlrFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gi, const OptTensor& h0, const OptTensor& reset,
                               int64_t act, bool batch_first) {
    auto [out, h_last] = glr_forward(gi, get(h0), get(reset), act, batch_first);
    ctx->save_for_backward({gi, get(h0), get(reset), out});
    ctx->saved_data["act"] = act;
    ctx->set_materialize_grads(false);
    return {out, h_last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &gi = saved[0], &h0 = saved[1], &reset = saved[2], &out = saved[3];
    Tensor dout = grads[0], dh = grads[1];
    if (!dout.defined() && !dh.defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    if (dout.defined()) check_no_tangent("gated_linear_scan", "the gradient of out", dout);
    if (dh.defined()) check_no_tangent("gated_linear_scan", "the gradient of h_T", dh);
    const int64_t T = out.size(0), B = out.size(1), H = out.size(2);
    dout = dout.defined() ? unit(dout) : torch::zeros({H}, out.options()).expand({T, B, H});
    if (dh.defined()) dh = dh.contiguous();
    Tensor dgi = out.stride(0) >= out.stride(1) ? torch::empty({T, B, 2 * H}, gi.options())
                                                : torch::empty({B, T, 2 * H}, gi.options()).transpose(0, 1);
    // needs_input_grad counts the tensors that were given
    Tensor dh0 = h0.defined() && ctx->needs_input_grad(1) ? torch::empty({B, H}, gi.options().dtype(torch::kFloat)) : Tensor();
    gs_glr_bwd_args a{};
    a.gi = gi.data_ptr();
    a.h0 = ptr<float>(h0);
    a.reset = ptr<uint8_t>(reset);
    a.out = out.data_ptr();
    a.dout = dout.data_ptr();
    a.dh_last = ptr<float>(dh);
    a.dgi = dgi.data_ptr();
    a.dh0 = ptr<float>(dh0);
    a.T = T;
    a.B = B;
    a.H = H;
    a.sg_t = gi.stride(0);
    a.sg_b = gi.stride(1);
    a.sh0_b = h0.defined() ? h0.stride(0) : 0;
    a.sr_t = reset.defined() ? reset.stride(0) : 0;
    a.sr_b = reset.defined() ? reset.stride(1) : 0;
    a.so_t = out.stride(0);
    a.so_b = out.stride(1);
    a.sd_t = dout.stride(0);
    a.sd_b = dout.stride(1);
    a.sdg_t = dgi.stride(0);
    a.sdg_b = dgi.stride(1);
    a.dtype = gi.scalar_type() == torch::kFloat ? GS_DTYPE_F32 : GS_DTYPE_BF16;
    a.activation = (int32_t)ctx->saved_data["act"].toInt();
    const On on(gi);
    const Tensor buf = scratch(gs_glr_bwd_scratch_bytes(&a), gi);
    a.scratch = ptr<void>(buf);
    a.scratch_bytes = buf.defined() ? buf.numel() : 0;
    if (buf.defined()) a.fault_mirror = fault_word(gi.get_device());
    raise_for(gs_glr_bwd(&a, on.stream));
    return once("gated_linear_scan", {dgi, dh0, Tensor(), Tensor(), Tensor()}, {gi, h0, grads[0], grads[1]});
  }
};

std::tuple<Tensor, Tensor> gated_linear_scan(Tensor gi, OptTensor h0, OptTensor reset, int64_t act, bool batch_first) {
  const char* who = "gated_linear_scan";
  check_on(who, "gi", gi, gi);
  dtype_of(who, "gi", gi);
  TORCH_CHECK_VALUE(gi.dim() == 3 && gi.size(2) > 0 && gi.size(2) % 2 == 0, who,
                    ": gi must be [T, B, 2H] with H > 0; got shape ", gi.sizes());
  if (batch_first) gi = gi.transpose(0, 1);
  const int64_t T = gi.size(0), B = gi.size(1), H = gi.size(2) / 2;
  TORCH_CHECK_VALUE(T > 0, "seq length T must be > 0; got T=", T);
  TORCH_CHECK_VALUE(B > 0, "batch size B must be > 0; got B=", B);
  bool grad = gi.requires_grad();
  if (h0.has_value()) {
    check_on(who, "h0", *h0, gi);
    TORCH_CHECK_VALUE(h0->scalar_type() == torch::kFloat && h0->dim() == 2 && h0->size(0) == B && h0->size(1) == H,
                      "h0 must be float32 of shape (B, H)=(", B, ", ", H, "); got ", h0->scalar_type(), " ", h0->sizes());
    grad = grad || h0->requires_grad();
    h0 = unit(*h0);
  }
  if (reset.has_value()) {
    check_on(who, "reset", *reset, gi);
    if (batch_first && reset->dim() == 2) reset = reset->transpose(0, 1);
    TORCH_CHECK_VALUE(reset->scalar_type() == torch::kBool && reset->dim() == 2 && reset->size(0) == T && reset->size(1) == B,
                      who, ": reset must be bool with one flag a step and row; got ", reset->scalar_type(), " ",
                      reset->sizes());
  }
  gi = unit(gi);
  raise_scan_fault(who, gi.get_device());
  Tensor out, h_last;
  if (grad && torch::GradMode::is_enabled()) {
    auto r = GlrFunction::apply(gi, h0, reset, act, batch_first);
    out = r[0];
    h_last = r[1];
  } else {
    std::tie(out, h_last) = glr_forward(gi, get(h0), get(reset), act, batch_first);
  }
  return {batch_first ? out.transpose(0, 1) : out, h_last};
}

Tensor gated_linear_step(const Tensor& gi_, const Tensor& state, const OptTensor& slots_, int64_t act) {
  const char* who = "gated_linear_step";
  check_on(who, "gi", gi_, gi_);
  gs_glr_step_args a{};
  a.dtype = dtype_of(who, "gi", gi_);
  TORCH_CHECK_VALUE(gi_.dim() == 2 && gi_.size(0) > 0 && gi_.size(1) > 0 && gi_.size(1) % 2 == 0, who,
                    ": gi must be [B, 2H] with B, H > 0; got shape ", gi_.sizes());
  const int64_t B = gi_.size(0), H = gi_.size(1) / 2;
  check_on(who, "state", state, gi_);
  TORCH_CHECK_VALUE(state.dim() == 2 && state.size(1) == H && state.size(0) > 0 && state.scalar_type() == torch::kFloat, who,
                    ": state must be float32 [S, H] with H=", H, "; got ", state.scalar_type(), " ", state.sizes());
  TORCH_CHECK_VALUE(state.stride(1) == 1 || H == 1, who,
                    ": state is updated in place and must have unit stride along H; got strides ", state.strides());
  check_may_modify(who, "state", state);
  Tensor slots;
  if (slots_.has_value()) {
    check_on(who, "slots", *slots_, gi_);
    TORCH_CHECK_VALUE(slots_->dim() == 1 && slots_->size(0) == B && slots_->scalar_type() == torch::kInt, who,
                      ": slots must be int32 [B]=[", B, "]; got ", slots_->scalar_type(), " ", slots_->sizes());
    slots = slots_->contiguous();
  } else {
    TORCH_CHECK_VALUE(state.size(0) >= B, who, ": ", state.size(0), " states for B=", B, " rows");
  }
  const Tensor gi = unit(gi_);
  Tensor out = torch::empty({B, H}, gi.options());
  a.gi = gi.data_ptr();
  a.state = static_cast<float*>(state.data_ptr());
  a.slots = ptr<int32_t>(slots);
  a.out = out.data_ptr();
  a.B = B;
  a.H = H;
  a.S = state.size(0);
  a.sg_b = gi.stride(0);
  a.ss = state.stride(0);
  a.so_b = H;
  a.activation = (int32_t)act;
  const On on(gi);
  raise_for(gs_glr_step(&a, on.stream));
  modified(state);
  return out;
}

// ---- linear --------------------------------------------------------------------------

Tensor linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, int64_t act,
                      const Tensor& pre) {
  gs_linear_args a{};
  a.M = x.size(0);
  a.N = w.size(0);
  a.K = x.size(1);
  Tensor y = torch::empty({a.M, a.N}, x.options());
  a.x = x.data_ptr();
  a.w = w.data_ptr();
  a.bias = ptr<void>(bias);
  a.residual = ptr<void>(residual);
  a.y = y.data_ptr();
  a.pre = ptr<void>(pre);
  a.sx = x.stride(0);
  a.sr = residual.defined() ? residual.stride(0) : 0;
  a.sy = a.N;
  a.dtype = x.scalar_type() == torch::kFloat ? GS_DTYPE_F32 : GS_DTYPE_BF16;
  a.activation = (int32_t)act;
  const On on(x);
  const Tensor buf = scratch(gs_linear_scratch_bytes(&a), x);
  a.scratch = ptr<void>(buf);
  a.scratch_bytes = buf.defined() ? buf.numel() : 0;
  raise_for(gs_linear_fwd(&a, on.stream));
  return y;
}

constexpr int64_t kHasBias = 256, kHasResidual = 512;  // beside the activation's number

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias,
                        const OptTensor& residual, int64_t act) {
    const auto kept = x.scalar_type() == torch::kFloat ? torch::kFloat : torch::kHalf;
    const Tensor pre = act != GS_ACT_NONE ? torch::empty({x.size(0), w.size(0)}, x.options().dtype(kept)) : Tensor();
    Tensor y = linear_forward(x, w, get(bias), get(residual), act, pre);
    ctx->save_for_backward({x, w, pre});
    ctx->saved_data["act"] = act | (bias.has_value() ? kHasBias : 0) | (residual.has_value() ? kHasResidual : 0);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &pre = saved[2];
    const int64_t given = ctx->saved_data["act"].toInt();
    const bool has_bias = (given & kHasBias) != 0;
    // needs_input_grad counts the tensors that were given
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = has_bias && ctx->needs_input_grad(2);
    const Tensor dres = (given & kHasResidual) && ctx->needs_input_grad(2 + has_bias) ? grads[0] : Tensor();
    if (!nx && !nw && !nb) return {Tensor(), Tensor(), Tensor(), dres, Tensor()};
    check_no_tangent("linear_act", "the output's gradient", grads[0]);
    const Tensor dy = unit(grads[0]);
    gs_linear_bwd_args a{};
    a.M = x.size(0);
    a.N = w.size(0);
    a.K = x.size(1);
    Tensor dx = nx ? torch::empty({a.M, a.K}, x.options()) : Tensor();
    Tensor dw = nw ? torch::empty({a.N, a.K}, x.options()) : Tensor();
    Tensor db = nb ? torch::empty({a.N}, x.options()) : Tensor();
    a.x = x.data_ptr();
    a.w = w.data_ptr();
    a.pre = ptr<void>(pre);
    a.dy = dy.data_ptr();
    a.dx = ptr<void>(dx);
    a.dw = ptr<void>(dw);
    a.dbias = ptr<void>(db);
    a.sx = x.stride(0);
    a.sdy = dy.stride(0);
    a.dtype = x.scalar_type() == torch::kFloat ? GS_DTYPE_F32 : GS_DTYPE_BF16;
    a.activation = (int32_t)(given & (kHasBias - 1));
    const On on(x);
    const Tensor buf = scratch(gs_linear_bwd_scratch_bytes(&a), x);
    a.scratch = ptr<void>(buf);
    a.scratch_bytes = buf.defined() ? buf.numel() : 0;
    raise_for(gs_linear_bwd(&a, on.stream));
    variable_list r = once("linear_act", {dx, dw, db, Tensor(), Tensor()}, {x, w, pre, grads[0]});
    r[3] = dres;
    return r;
  }
};

// [..., n] as rows of unit stride.
Tensor rows(const Tensor& t) { return unit(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }

Tensor linear_act(const Tensor& x, const Tensor& w, OptTensor bias, OptTensor residual, int64_t act) {
  const char* who = "linear_act";
  check_on(who, "x", x, x);
  dtype_of(who, "x", x);
  bool grad = x.requires_grad() || w.requires_grad();
  auto check = [&](const char* name, const Tensor& t) {
    check_on(who, name, t, x);
    TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type(), who, ": all tensors must be float32 or all bfloat16; ", name,
                      " is ", t.scalar_type(), ", x ", x.scalar_type());
  };
  check("weight", w);
  TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1), who,
                    ": weight must be [N, K] with K = x.shape[-1]; got x ", x.sizes(), ", weight ", w.sizes());
  TORCH_CHECK_VALUE(x.numel() > 0 && w.numel() > 0, who, ": x and weight must be non-empty; got x ", x.sizes(),
                    ", weight ", w.sizes());
  const int64_t N = w.size(0);
  if (bias.has_value()) {
    check("bias", *bias);
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == N, who, ": bias must be [", N, "]; got ", bias->sizes());
    grad = grad || bias->requires_grad();
    bias = bias->contiguous();
  }
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  if (residual.has_value()) {
    check("residual", *residual);
    TORCH_CHECK_VALUE(residual->sizes() == c10::IntArrayRef(shape), who, ": residual must be ", c10::IntArrayRef(shape),
                      "; got ", residual->sizes());
    grad = grad || residual->requires_grad();
    residual = rows(*residual);
  }
  const Tensor x2 = rows(x), w2 = w.contiguous();
  Tensor y = grad && torch::GradMode::is_enabled() ? LinearFunction::apply(x2, w2, bias, residual, act)
                                                   : linear_forward(x2, w2, get(bias), get(residual), act, Tensor());
  return shape.size() == 2 ? y : y.view(shape);
}

// ---- AdamW ---------------------------------------------------------------------------

typedef std::vector<Tensor> Tensors;

const Tensors* get(const std::optional<Tensors>& t) { return t.has_value() ? &*t : nullptr; }

// One contiguous tensor of counts[i] elements for each parameter, of type `kind`, on ref's device.
// `updated`: the step writes them.
void check_list(const char* name, const Tensors& ts, const std::vector<int64_t>& counts, torch::ScalarType kind,
                const Tensor& ref, bool updated = true) {
  const char* who = "adamw_step";
  // without a level of forward-mode differentiation no tensor has a tangent: asking each costs 30 ns where it is a view
  const bool dual = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
  TORCH_CHECK_VALUE(ts.size() == counts.size(), who, ": ", ts.size(), " tensors in ", name, " for ", counts.size(),
                    " parameters");
  for (size_t i = 0; i < ts.size(); ++i) {
    const Tensor& t = ts[i];
    TORCH_CHECK_VALUE(t.device() == ref.device(), who, ": every tensor must be on one CUDA (HIP) device, ", ref.device(),
                      "; ", name, "[", i, "] is on ", t.device());
    TORCH_CHECK_VALUE(t.scalar_type() == kind, who, ": ", name, "[", i, "] dtype must be ", kind, "; got ",
                      t.scalar_type());
    TORCH_CHECK_VALUE(t.numel() == counts[i], who, ": ", name, "[", i, "] must have ", counts[i], " elements; got shape ",
                      t.sizes());
    TORCH_CHECK_VALUE(t.is_contiguous(), who, ": ", name, "[", i, "] must be contiguous; got strides ", t.strides());
    if (dual) check_no_tangent(who, name, t);
    if (updated) check_may_modify(who, name, t);
  }
}

void adamw_step(const Tensors& params, Tensors grads, const Tensors& exp_avgs, const Tensors& exp_avg_sqs, int64_t step,
                double lr, double beta1, double beta2, double eps, double weight_decay,
                const std::optional<Tensors>& masters, const std::optional<Tensors>& exp_avg_scales,
                const std::optional<Tensors>& exp_avg_sq_scales, const OptTensor& grad_scale, int64_t rounding) {
  const char* who = "adamw_step";
  if (params.empty()) return;
  const Tensor& ref = params[0];
  TORCH_CHECK_VALUE(ref.is_cuda(), who, ": params must be CUDA (HIP) tensors; got ", ref.device());
  TORCH_CHECK_VALUE(exp_avg_scales.has_value() == exp_avg_sq_scales.has_value(), who,
                    ": exp_avg_scales and exp_avg_sq_scales belong together");
  const bool bytes = exp_avg_scales.has_value();
  gs_adamw_args a{};
  a.param_dtype = dtype_of(who, "params", ref);
  TORCH_CHECK_VALUE(!grads.empty(), who, ": 0 tensors in grads for ", params.size(), " parameters");
  a.grad_dtype = dtype_of(who, "grads", grads[0]);
  std::vector<int64_t> counts(params.size()), blocks(params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    counts[i] = params[i].numel();
    blocks[i] = (counts[i] + kStateBlock - 1) / kStateBlock;
  }
  for (Tensor& g : grads)
    if (!g.is_contiguous()) g = g.contiguous();
  check_list("params", params, counts, ref.scalar_type(), ref);
  check_list("grads", grads, counts, grads[0].scalar_type(), ref, false);
  check_list("exp_avgs", exp_avgs, counts, bytes ? torch::kChar : torch::kFloat, ref);
  check_list("exp_avg_sqs", exp_avg_sqs, counts, bytes ? torch::kByte : torch::kFloat, ref);
  if (bytes) {
    check_list("exp_avg_scales", *exp_avg_scales, blocks, torch::kFloat, ref);
    check_list("exp_avg_sq_scales", *exp_avg_sq_scales, blocks, torch::kFloat, ref);
  }
  if (masters.has_value()) {
    TORCH_CHECK_VALUE(a.param_dtype == GS_DTYPE_BF16, who, ": masters belong to bfloat16 parameters; got ",
                      ref.scalar_type());
    check_list("masters", *masters, counts, torch::kFloat, ref);
  }
  if (grad_scale.has_value()) {
    TORCH_CHECK_VALUE(grad_scale->device() == ref.device() && grad_scale->scalar_type() == torch::kFloat && grad_scale->numel() == 1,
                      who, ": grad_scale must be one float32 number on the parameters' device; got ",
                      grad_scale->scalar_type(), " ", grad_scale->sizes(), " on ", grad_scale->device());
    check_no_tangent(who, "grad_scale", *grad_scale);
  }
  std::vector<gs_adamw_tensor> table(params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    gs_adamw_tensor& t = table[i];
    t = gs_adamw_tensor{};
    t.param = params[i].data_ptr();
    t.grad = grads[i].data_ptr();
    t.exp_avg = exp_avgs[i].data_ptr();
    t.exp_avg_sq = exp_avg_sqs[i].data_ptr();
    if (bytes) {
      t.exp_avg_scale = static_cast<float*>((*exp_avg_scales)[i].data_ptr());
      t.exp_avg_sq_scale = static_cast<float*>((*exp_avg_sq_scales)[i].data_ptr());
    }
    if (masters.has_value()) t.master = static_cast<float*>((*masters)[i].data_ptr());
    t.n = counts[i];
  }
  a.tensors = table.data();
  a.count = (int64_t)table.size();
  a.lr = lr;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.weight_decay = weight_decay;
  a.step = step;
  a.grad_scale = grad_scale.has_value() ? static_cast<const float*>(grad_scale->data_ptr()) : nullptr;
  a.state_bits = bytes ? 8 : 32;
  a.has_master = masters.has_value();
  a.rounding = (int32_t)rounding;
  const On on(ref);
  raise_for(gs_adamw_step(&a, on.stream));
  for (const Tensors* ts : {&params, &exp_avgs, &exp_avg_sqs, get(masters), get(exp_avg_scales), get(exp_avg_sq_scales)})
    if (ts != nullptr)
      for (const Tensor& t : *ts) modified(t);
}

Tensor adamw_dequantize_state(const Tensor& codes, const Tensor& scales) {
  const char* who = "adamw_dequantize_state";
  const bool second = codes.scalar_type() == torch::kByte;
  TORCH_CHECK_VALUE(codes.is_cuda() && codes.is_contiguous() && (second || codes.scalar_type() == torch::kChar), who,
                    ": codes must be a contiguous int8 or uint8 CUDA (HIP) tensor; got ", codes.scalar_type(), " on ",
                    codes.device());
  const int64_t n = codes.numel();
  TORCH_CHECK_VALUE(scales.device() == codes.device() && scales.scalar_type() == torch::kFloat && scales.is_contiguous() &&
                        scales.numel() == (n + kStateBlock - 1) / kStateBlock,
                    who, ": scales must be ", (n + kStateBlock - 1) / kStateBlock, " contiguous float32 numbers on ",
                    codes.device(), "; got ", scales.scalar_type(), " ", scales.sizes(), " on ", scales.device());
  check_no_tangent(who, "scales", scales);
  Tensor out = torch::empty(codes.sizes(), codes.options().dtype(torch::kFloat));
  const On on(codes);
  raise_for(gs_adamw_dequantize(codes.data_ptr(), ptr<float>(scales), out.data_ptr<float>(), n, second, on.stream));
  return out;
}

}  // namespace

PYBIND11_MODULE(_ops, m) {
  m.def("abi_version", [] { return GS_ABI_VERSION; });
  m.def("gated_linear_scan", &gated_linear_scan, py::call_guard<py::gil_scoped_release>());
  m.def("gated_linear_step", &gated_linear_step, py::call_guard<py::gil_scoped_release>());
  m.def("linear_act", &linear_act, py::call_guard<py::gil_scoped_release>());
  m.def("adamw_step", &adamw_step, py::call_guard<py::gil_scoped_release>());
  m.def("adamw_dequantize_state", &adamw_dequantize_state, py::call_guard<py::gil_scoped_release>());
}
