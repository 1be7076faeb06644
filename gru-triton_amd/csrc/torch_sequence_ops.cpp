// The torch side of the operators over sequences of tokens: the causal convolution, the selective
// scan, the embedding and the token log probabilities. As torch_ops.cpp.
#include "torch_ops.h"

namespace {

int dtype_code(const Tensor& t) { return t.scalar_type() == torch::kFloat ? GS_DTYPE_F32 : GS_DTYPE_BF16; }

// [T, B, n] in the memory order that the call's other tensors have.
Tensor empty_steps(int64_t T, int64_t B, int64_t n, bool batch_first, const Tensor& like) {
  return batch_first ? torch::empty({B, T, n}, like.options()).transpose(0, 1) : torch::empty({T, B, n}, like.options());
}
Tensor zero_steps(const Tensor& like) { return torch::zeros({like.size(2)}, like.options()).expand_as(like); }

void check_same(const char* who, const char* name, const Tensor& t, const char* ref_name, const Tensor& ref) {
  check_on(who, name, t, ref);
  TORCH_CHECK_VALUE(t.scalar_type() == ref.scalar_type(), who, ": ", name, " must be of ", ref_name, "'s type, ",
                    ref.scalar_type(), "; got ", t.scalar_type());
}
void check_shape(const char* who, const char* name, const Tensor& t, c10::IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.sizes() == shape, who, ": ", name, " must be ", shape, "; got ", t.sizes());
}
void check_float(const char* who, const char* name, const Tensor& t, const Tensor& ref, c10::IntArrayRef shape) {
  check_on(who, name, t, ref);
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kFloat, who, ": ", name, " must be float32; got ", t.scalar_type());
  check_shape(who, name, t, shape);
}
OptTensor check_reset(const char* who, OptTensor reset, const Tensor& ref, int64_t T, int64_t B, bool batch_first) {
  if (!reset.has_value()) return reset;
  check_on(who, "reset", *reset, ref);
  if (batch_first && reset->dim() == 2) reset = reset->transpose(0, 1);
  TORCH_CHECK_VALUE(reset->scalar_type() == torch::kBool && reset->dim() == 2 && reset->size(0) == T && reset->size(1) == B,
                    who, ": reset must be bool with one flag a step and row; got ", reset->scalar_type(), " ", reset->sizes());
  return reset;
}
// A cache that a step updates in place, and the rows' slots in it.
Tensor check_cache(const char* who, const Tensor& state, const OptTensor& slots, const Tensor& x, int64_t B, int64_t d1, int64_t d2) {
  TORCH_CHECK_VALUE(state.dim() == 3 && state.size(0) > 0 && state.size(1) == d1 && state.size(2) == d2, who,
                    ": state must be [S, ", d1, ", ", d2, "]; got ", state.sizes());
  TORCH_CHECK_VALUE(state.stride(2) == 1 || d2 == 1, who, ": state is updated in place and its rows must be contiguous; got strides ",
                    state.strides());
  TORCH_CHECK_VALUE(state.stride(1) == d2 || d1 == 1, who, ": state is updated in place and its rows must be contiguous; got strides ",
                    state.strides());
  check_may_modify(who, "state", state);
  if (!slots.has_value()) {
    TORCH_CHECK_VALUE(state.size(0) >= B, who, ": ", state.size(0), " states for B=", B, " rows");
    return Tensor();
  }
  check_on(who, "slots", *slots, x);
  TORCH_CHECK_VALUE(slots->dim() == 1 && slots->size(0) == B && slots->scalar_type() == torch::kInt, who,
                    ": slots must be int32 [B]=[", B, "]; got ", slots->scalar_type(), " ", slots->sizes());
  return slots->contiguous();
}
void check_taps(const char* who, const Tensor& x, const Tensor& w, const OptTensor& bias, int64_t C) {
  check_same(who, "weight", w, "x", x);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == C && w.size(1) >= 2 && w.size(1) <= 4, who,
                    ": weight must be [C, W] with C=", C, " and W from 2 to 4; got ", w.sizes());
  if (!bias.has_value()) return;
  check_same(who, "bias", *bias, "x", x);
  check_shape(who, "bias", *bias, {C});
}

template <typename Args>
void set_reset(Args& a, const Tensor& reset) {
  a.reset = ptr<uint8_t>(reset);
  a.sr_t = reset.defined() ? reset.stride(0) : 0;
  a.sr_b = reset.defined() ? reset.stride(1) : 0;
}

// ---- causal convolution -----------------------------------------------------------------

std::tuple<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state,
                                        const Tensor& reset, int64_t act, bool batch_first) {
  gs_conv_args a{};
  a.T = x.size(0);
  a.B = x.size(1);
  a.C = x.size(2);
  a.W = w.size(1);
  Tensor y = empty_steps(a.T, a.B, a.C, batch_first, x), last = torch::empty({a.B, a.W - 1, a.C}, x.options());
  a.x = x.data_ptr();
  a.w = w.data_ptr();
  a.bias = ptr<void>(bias);
  a.state = ptr<void>(state);
  set_reset(a, reset);
  a.y = y.data_ptr();
  a.last = last.data_ptr();
  a.sx_t = x.stride(0);
  a.sx_b = x.stride(1);
  a.sy_t = y.stride(0);
  a.sy_b = y.stride(1);
  a.dtype = dtype_code(x);
  a.activation = (int32_t)act;
  const On on(x);
  raise_for(gs_conv_fwd(&a, on.stream));
  return {y, last};
}

struct ConvFunction : torch::autograd::Function<ConvFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias,
                               const OptTensor& state, const OptTensor& reset, int64_t act, bool batch_first) {
    auto [y, last] = conv_forward(x, w, get(bias), get(state), get(reset), act, batch_first);
    ctx->save_for_backward({x, w, get(bias), get(state), get(reset)});
    ctx->saved_data["act"] = act;
    ctx->saved_data["batch_first"] = batch_first;
    ctx->set_materialize_grads(false);
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* who = "causal_conv";
    check_capture(who);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &bias = saved[2], &state = saved[3], &reset = saved[4];
    Tensor dy = grads[0], dlast = grads[1];
    if (!dy.defined() && !dlast.defined()) return variable_list(7);
    if (dy.defined()) check_no_tangent(who, "the gradient of y", dy);
    if (dlast.defined()) check_no_tangent(who, "the gradient of the last inputs", dlast);
    dy = dy.defined() ? unit(dy) : zero_steps(x);
    if (dlast.defined()) dlast = dlast.contiguous();
    gs_conv_bwd_args a{};
    a.T = x.size(0);
    a.B = x.size(1);
    a.C = x.size(2);
    a.W = w.size(1);
    Tensor dx = empty_steps(a.T, a.B, a.C, ctx->saved_data["batch_first"].toBool(), x);
    Tensor dw = torch::empty_like(w), db = bias.defined() ? torch::empty_like(bias) : Tensor();
    Tensor dstate = state.defined() ? torch::empty_like(state) : Tensor();
    a.x = x.data_ptr();
    a.w = w.data_ptr();
    a.bias = ptr<void>(bias);
    a.state = ptr<void>(state);
    set_reset(a, reset);
    a.dy = dy.data_ptr();
    a.dlast = ptr<void>(dlast);
    a.dx = dx.data_ptr();
    a.dstate = ptr<void>(dstate);
    a.dw = dw.data_ptr();
    a.dbias = ptr<void>(db);
    a.sx_t = x.stride(0);
    a.sx_b = x.stride(1);
    a.sdy_t = dy.stride(0);
    a.sdy_b = dy.stride(1);
    a.sdx_t = dx.stride(0);
    a.sdx_b = dx.stride(1);
    a.dtype = dtype_code(x);
    a.activation = (int32_t)ctx->saved_data["act"].toInt();
    const On on(x);
    const Tensor buf = scratch(gs_conv_bwd_scratch_bytes(&a), x);
    a.scratch = ptr<void>(buf);
    a.scratch_bytes = buf.defined() ? buf.numel() : 0;
    raise_for(gs_conv_bwd(&a, on.stream));
    return once(who, {dx, dw, db, dstate, Tensor(), Tensor(), Tensor()}, {x, w, bias, state, grads[0], grads[1]});
  }
};

std::tuple<Tensor, Tensor> causal_conv(Tensor x, const Tensor& w, OptTensor bias, OptTensor state, OptTensor reset,
                                       int64_t act, bool batch_first) {
  const char* who = "causal_conv";
  check_on(who, "x", x, x);
  dtype_of(who, "x", x);
  TORCH_CHECK_VALUE(x.dim() == 3 && x.numel() > 0, who, ": x must be [T, B, C] and not empty; got shape ", x.sizes());
  if (batch_first) x = x.transpose(0, 1);
  const int64_t T = x.size(0), B = x.size(1), C = x.size(2);
  check_taps(who, x, w, bias, C);
  bool grad = x.requires_grad() || w.requires_grad() || (bias.has_value() && bias->requires_grad());
  if (bias.has_value()) bias = bias->contiguous();
  if (state.has_value()) {
    check_same(who, "state", *state, "x", x);
    check_shape(who, "state", *state, {B, w.size(1) - 1, C});
    grad = grad || state->requires_grad();
    state = state->contiguous();
  }
  reset = check_reset(who, reset, x, T, B, batch_first);
  x = unit(x);
  const Tensor w2 = w.contiguous();
  Tensor y, last;
  if (grad && torch::GradMode::is_enabled()) {
    auto r = ConvFunction::apply(x, w2, bias, state, reset, act, batch_first);
    y = r[0];
    last = r[1];
  } else {
    std::tie(y, last) = conv_forward(x, w2, get(bias), get(state), get(reset), act, batch_first);
  }
  return {batch_first ? y.transpose(0, 1) : y, last};
}

Tensor causal_conv_step(const Tensor& x_, const Tensor& w, const OptTensor& bias, const Tensor& state,
                        const OptTensor& slots_, int64_t act) {
  const char* who = "causal_conv_step";
  check_on(who, "x", x_, x_);
  dtype_of(who, "x", x_);
  TORCH_CHECK_VALUE(x_.dim() == 2 && x_.numel() > 0, who, ": x must be [B, C] and not empty; got shape ", x_.sizes());
  gs_conv_step_args a{};
  a.B = x_.size(0);
  a.C = x_.size(1);
  check_taps(who, x_, w, bias, a.C);
  a.W = w.size(1);
  check_same(who, "state", state, "x", x_);
  const Tensor slots = check_cache(who, state, slots_, x_, a.B, a.W - 1, a.C);
  const Tensor x = unit(x_), w2 = w.contiguous(), b2 = bias.has_value() ? bias->contiguous() : Tensor();
  Tensor y = torch::empty({a.B, a.C}, x.options());
  a.x = x.data_ptr();
  a.w = w2.data_ptr();
  a.bias = ptr<void>(b2);
  a.state = state.data_ptr();
  a.slots = ptr<int32_t>(slots);
  a.y = y.data_ptr();
  a.S = state.size(0);
  a.sx = x.stride(0);
  a.ss = state.stride(0);
  a.sy = a.C;
  a.dtype = dtype_code(x);
  a.activation = (int32_t)act;
  const On on(x);
  raise_for(gs_conv_step(&a, on.stream));
  modified(state);
  return y;
}

// ---- selective scan -------------------------------------------------------------------------

// What both directions of the scan read; undefined tensors were not given.
struct SsmInputs {
  Tensor u, delta, A, bm, cm, D, z, bias, h0, reset;
  template <typename Args>
  void set(Args& a) const {
    a.T = u.size(0);
    a.B = u.size(1);
    a.H = u.size(2);
    a.N = A.size(1);
    a.u = u.data_ptr();
    a.delta = delta.data_ptr();
    a.z = ptr<void>(z);
    a.bm = bm.data_ptr();
    a.cm = cm.data_ptr();
    a.A = static_cast<const float*>(A.data_ptr());
    a.D = ptr<float>(D);
    a.delta_bias = ptr<float>(bias);
    a.h0 = ptr<float>(h0);
    set_reset(a, reset);
    a.su_t = u.stride(0);
    a.su_b = u.stride(1);
    a.sdl_t = delta.stride(0);
    a.sdl_b = delta.stride(1);
    a.sz_t = z.defined() ? z.stride(0) : 0;
    a.sz_b = z.defined() ? z.stride(1) : 0;
    a.sb_t = bm.stride(0);
    a.sb_b = bm.stride(1);
    a.sc_t = cm.stride(0);
    a.sc_b = cm.stride(1);
    a.dtype = dtype_code(u);
  }
};

// y, h_T and, where `keep`, the states that the backward starts from.
std::tuple<Tensor, Tensor, Tensor> ssm_forward(const SsmInputs& in, bool batch_first, bool keep) {
  gs_ssm_args a{};
  in.set(a);
  const auto f32 = in.u.options().dtype(torch::kFloat);
  Tensor y = empty_steps(a.T, a.B, a.H, batch_first, in.u), h = torch::empty({a.B, a.H, a.N}, f32), saved;
  a.y = y.data_ptr();
  a.h_last = h.data_ptr<float>();
  a.sy_t = y.stride(0);
  a.sy_b = y.stride(1);
  const On on(in.u);
  if (keep) {
    const int64_t bytes = gs_ssm_saved_bytes(&a);
    raise_for(bytes);
    saved = torch::empty({bytes / 4}, f32);
    a.saved = saved.data_ptr<float>();
  }
  const Tensor buf = scratch(gs_ssm_scratch_bytes(&a), in.u);
  a.scratch = ptr<void>(buf);
  a.scratch_bytes = buf.defined() ? buf.numel() : 0;
  raise_for(gs_ssm_fwd(&a, on.stream));
  return {y, h, saved};
}

struct SsmFunction : torch::autograd::Function<SsmFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& bm,
                               const Tensor& cm, const OptTensor& D, const OptTensor& z, const OptTensor& bias,
                               const OptTensor& h0, const OptTensor& reset, bool batch_first) {
    auto [y, h, saved] = ssm_forward(SsmInputs{u, delta, A, bm, cm, get(D), get(z), get(bias), get(h0), get(reset)}, batch_first, true);
    ctx->save_for_backward({u, delta, A, bm, cm, get(D), get(z), get(bias), get(h0), get(reset), saved});
    ctx->saved_data["batch_first"] = batch_first;
    ctx->set_materialize_grads(false);
    return {y, h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* who = "selective_scan";
    check_capture(who);
    const auto s = ctx->get_saved_variables();
    const SsmInputs in{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9]};
    Tensor dy = grads[0], dh = grads[1];
    if (!dy.defined() && !dh.defined()) return variable_list(11);
    if (dy.defined()) check_no_tangent(who, "the gradient of y", dy);
    if (dh.defined()) check_no_tangent(who, "the gradient of h_T", dh);
    dy = dy.defined() ? unit(dy) : zero_steps(in.u);
    if (dh.defined()) dh = dh.contiguous();
    gs_ssm_bwd_args a{};
    in.set(a);
    const bool batch_first = ctx->saved_data["batch_first"].toBool();
    const auto like = [](const Tensor& t) { return t.defined() ? torch::empty_like(t, at::MemoryFormat::Contiguous) : Tensor(); };
    Tensor du = empty_steps(a.T, a.B, a.H, batch_first, in.u), dd = empty_steps(a.T, a.B, a.H, batch_first, in.u);
    Tensor dz = in.z.defined() ? empty_steps(a.T, a.B, a.H, batch_first, in.u) : Tensor();
    Tensor dbm = like(in.bm), dcm = like(in.cm), dA = like(in.A), dD = like(in.D), db = like(in.bias), dh0 = like(in.h0);
    a.saved = s[10].data_ptr<float>();
    a.dy = dy.data_ptr();
    a.dh_last = ptr<float>(dh);
    a.du = du.data_ptr();
    a.ddelta = dd.data_ptr();
    a.dz = ptr<void>(dz);
    a.dbm = dbm.data_ptr();
    a.dcm = dcm.data_ptr();
    a.dA = dA.data_ptr<float>();
    a.dD = ptr<float>(dD);
    a.ddelta_bias = ptr<float>(db);
    a.dh0 = ptr<float>(dh0);
    a.sdy_t = dy.stride(0);
    a.sdy_b = dy.stride(1);
    a.sdu_t = du.stride(0);
    a.sdu_b = du.stride(1);
    a.sdd_t = dd.stride(0);
    a.sdd_b = dd.stride(1);
    a.sdz_t = dz.defined() ? dz.stride(0) : 0;
    a.sdz_b = dz.defined() ? dz.stride(1) : 0;
    const On on(in.u);
    const Tensor buf = scratch(gs_ssm_bwd_scratch_bytes(&a), in.u);
    a.scratch = ptr<void>(buf);
    a.scratch_bytes = buf.defined() ? buf.numel() : 0;
    raise_for(gs_ssm_bwd(&a, on.stream));
    return once(who, {du, dd, dA, dbm, dcm, dD, dz, db, dh0, Tensor(), Tensor()},
                {in.u, in.delta, in.A, in.bm, in.cm, in.D, in.z, in.bias, in.h0, grads[0], grads[1]});
  }
};

// What the scan (dim 3) and the step (dim 2) check alike.
void check_ssm(const char* who, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& bm, const Tensor& cm,
               const OptTensor& D, const OptTensor& z, const OptTensor& bias, int64_t dim) {
  check_on(who, "u", u, u);
  dtype_of(who, "u", u);
  TORCH_CHECK_VALUE(u.dim() == dim && u.numel() > 0, who, ": u must be ", dim == 3 ? "[T, B, H]" : "[B, H]",
                    " and not empty; got shape ", u.sizes());
  const int64_t H = u.size(-1);
  check_same(who, "delta", delta, "u", u);
  check_shape(who, "delta", delta, u.sizes());
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(1) >= 1 && A.size(1) <= 32, who, ": A must be [H, N] with N from 1 to 32; got ", A.sizes());
  check_float(who, "A", A, u, {H, A.size(1)});
  std::vector<int64_t> shape(u.sizes().begin(), u.sizes().end());
  shape.back() = A.size(1);
  check_same(who, "B", bm, "u", u);
  check_shape(who, "B", bm, shape);
  check_same(who, "C", cm, "u", u);
  check_shape(who, "C", cm, shape);
  if (D.has_value()) check_float(who, "D", *D, u, {H});
  if (bias.has_value()) check_float(who, "delta_bias", *bias, u, {H});
  if (z.has_value()) {
    check_same(who, "z", *z, "u", u);
    check_shape(who, "z", *z, u.sizes());
  }
}
OptTensor whole(const OptTensor& t) { return t.has_value() ? OptTensor(t->contiguous()) : t; }

std::tuple<Tensor, Tensor> selective_scan(Tensor u, Tensor delta, const Tensor& A, Tensor bm, Tensor cm, const OptTensor& D,
                                          OptTensor z, const OptTensor& h0, const OptTensor& bias, OptTensor reset,
                                          bool batch_first) {
  const char* who = "selective_scan";
  check_ssm(who, u, delta, A, bm, cm, D, z, bias, 3);
  auto steps = [&](const Tensor& t) { return unit(batch_first ? t.transpose(0, 1) : t); };
  u = steps(u);
  delta = steps(delta);
  bm = steps(bm);
  cm = steps(cm);
  if (z.has_value()) z = steps(*z);
  const int64_t T = u.size(0), B = u.size(1);
  if (h0.has_value()) check_float(who, "h0", *h0, u, {B, u.size(2), A.size(1)});
  reset = check_reset(who, reset, u, T, B, batch_first);
  auto wants = [](const OptTensor& t) { return t.has_value() && t->requires_grad(); };
  const bool grad = torch::GradMode::is_enabled() && (u.requires_grad() || delta.requires_grad() || A.requires_grad() ||
                    bm.requires_grad() || cm.requires_grad() || wants(D) || wants(z) || wants(h0) || wants(bias));
  const Tensor A2 = A.contiguous();
  const OptTensor D2 = whole(D), h2 = whole(h0), b2 = whole(bias);
  Tensor y, h;
  if (grad) {
    auto r = SsmFunction::apply(u, delta, A2, bm, cm, D2, z, b2, h2, reset, batch_first);
    y = r[0];
    h = r[1];
  } else {
    Tensor none;
    std::tie(y, h, none) = ssm_forward(SsmInputs{u, delta, A2, bm, cm, get(D2), get(z), get(b2), get(h2), get(reset)}, batch_first, false);
  }
  return {batch_first ? y.transpose(0, 1) : y, h};
}

Tensor selective_step(const Tensor& u_, const Tensor& delta_, const Tensor& A_, const Tensor& bm_, const Tensor& cm_,
                      const Tensor& state, const OptTensor& slots_, const OptTensor& D_, const OptTensor& z_,
                      const OptTensor& bias_) {
  const char* who = "selective_step";
  check_ssm(who, u_, delta_, A_, bm_, cm_, D_, z_, bias_, 2);
  gs_ssm_step_args a{};
  a.B = u_.size(0);
  a.H = u_.size(1);
  a.N = A_.size(1);
  check_on(who, "state", state, u_);
  TORCH_CHECK_VALUE(state.scalar_type() == torch::kFloat, who, ": state must be float32; got ", state.scalar_type());
  const Tensor slots = check_cache(who, state, slots_, u_, a.B, a.H, a.N);
  const Tensor u = unit(u_), delta = unit(delta_), bm = unit(bm_), cm = unit(cm_), A = A_.contiguous();
  const Tensor z = z_.has_value() ? unit(*z_) : Tensor(), D = get(whole(D_)), bias = get(whole(bias_));
  Tensor y = torch::empty({a.B, a.H}, u.options());
  a.u = u.data_ptr();
  a.delta = delta.data_ptr();
  a.z = ptr<void>(z);
  a.bm = bm.data_ptr();
  a.cm = cm.data_ptr();
  a.A = static_cast<const float*>(A.data_ptr());
  a.D = ptr<float>(D);
  a.delta_bias = ptr<float>(bias);
  a.state = static_cast<float*>(state.data_ptr());
  a.slots = ptr<int32_t>(slots);
  a.y = y.data_ptr();
  a.S = state.size(0);
  a.su = u.stride(0);
  a.sdl = delta.stride(0);
  a.sz = z.defined() ? z.stride(0) : 0;
  a.sb = bm.stride(0);
  a.sc = cm.stride(0);
  a.ss = state.stride(0);
  a.sy = a.H;
  a.dtype = dtype_code(u);
  const On on(u);
  raise_for(gs_ssm_step(&a, on.stream));
  modified(state);
  return y;
}

// ---- embedding ------------------------------------------------------------------------------

int token_bits(const char* who, const Tensor& tokens) {
  if (tokens.scalar_type() == torch::kLong) return 64;
  TORCH_CHECK_VALUE(tokens.scalar_type() == torch::kInt, who, ": tokens must be int32 or int64; got ", tokens.scalar_type());
  return 32;
}

Tensor embedding_forward(const Tensor& tokens, const Tensor& w, double scale) {
  gs_embedding_args a{};
  a.M = tokens.numel();
  a.V = w.size(0);
  a.K = w.size(1);
  Tensor out = torch::empty({a.M, a.K}, w.options());
  a.tokens = tokens.data_ptr();
  a.w = w.data_ptr();
  a.out = out.data_ptr();
  a.so = a.K;
  a.scale = (float)scale;
  a.token_bits = token_bits("embedding", tokens);
  a.dtype = dtype_code(w);
  const On on(w);
  raise_for(gs_embedding_fwd(&a, on.stream));
  return out;
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& w, double scale) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["V"] = w.size(0);
    return embedding_forward(tokens, w, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* who = "embedding";
    check_capture(who);
    const Tensor tokens = ctx->get_saved_variables()[0];
    check_no_tangent(who, "the output's gradient", grads[0]);
    const Tensor dout = unit(grads[0]);
    gs_embedding_bwd_args a{};
    a.M = tokens.numel();
    a.V = ctx->saved_data["V"].toInt();
    a.K = dout.size(1);
    Tensor dw = torch::empty({a.V, a.K}, dout.options());
    // rows that share memory (an expanded gradient) are made apart
    const Tensor d2 = a.M > 1 && dout.stride(0) < a.K ? dout.contiguous() : dout;
    a.tokens = tokens.data_ptr();
    a.dout = d2.data_ptr();
    a.dw = dw.data_ptr();
    a.sdo = a.M > 1 ? d2.stride(0) : a.K;
    a.scale = (float)ctx->saved_data["scale"].toDouble();
    a.token_bits = token_bits(who, tokens);
    a.dtype = dtype_code(dout);
    const On on(dout);
    const Tensor buf = scratch(gs_embedding_bwd_scratch_bytes(&a), dout);
    a.scratch = ptr<void>(buf);
    a.scratch_bytes = buf.defined() ? buf.numel() : 0;
    raise_for(gs_embedding_bwd(&a, on.stream));
    return once(who, {Tensor(), dw, Tensor()}, {grads[0]});
  }
};

Tensor embedding(const Tensor& tokens, const Tensor& w, double scale) {
  const char* who = "embedding";
  check_on(who, "weight", w, w);
  dtype_of(who, "weight", w);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.numel() > 0, who, ": weight must be [V, K] and not empty; got ", w.sizes());
  check_on(who, "tokens", tokens, w);
  token_bits(who, tokens);
  TORCH_CHECK_VALUE(tokens.numel() > 0, who, ": tokens must not be empty; got shape ", tokens.sizes());
  std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
  shape.push_back(w.size(1));
  const Tensor flat = tokens.reshape({-1}).contiguous(), w2 = w.contiguous();
  Tensor out = w.requires_grad() && torch::GradMode::is_enabled() ? EmbeddingFunction::apply(flat, w2, scale)
                                                                   : embedding_forward(flat, w2, scale);
  return shape.size() == 2 ? out : out.view(shape);
}

// ---- token log probabilities ------------------------------------------------------------------

struct Probs {
  Tensor logprob, entropy, top_logprob, top_token, stats;
};
Probs logprobs_forward(const Tensor& x, const Tensor& tokens, int64_t top, bool keep) {
  gs_logprobs_args a{};
  a.M = x.size(0);
  a.V = x.size(1);
  a.top = top;
  const auto f32 = x.options().dtype(torch::kFloat);
  Probs r{torch::empty({a.M}, f32), torch::empty({a.M}, f32), torch::empty({a.M, top}, f32),
          torch::empty({a.M, top}, x.options().dtype(torch::kLong)), keep ? torch::empty({a.M, 2}, f32) : Tensor()};
  a.x = x.data_ptr();
  a.tokens = tokens.data_ptr();
  a.logprob = r.logprob.data_ptr<float>();
  a.entropy = r.entropy.data_ptr<float>();
  a.stats = ptr<float>(r.stats);
  a.top_logprob = r.top_logprob.data_ptr<float>();
  a.top_token = r.top_token.data_ptr<int64_t>();
  a.sx = x.stride(0);
  a.token_bits = token_bits("token_logprobs", tokens);
  a.dtype = dtype_code(x);
  const On on(x);
  const Tensor buf = scratch(gs_logprobs_scratch_bytes(&a), x);
  a.scratch = ptr<void>(buf);
  a.scratch_bytes = buf.defined() ? buf.numel() : 0;
  raise_for(gs_logprobs_fwd(&a, on.stream));
  return r;
}

struct LogprobsFunction : torch::autograd::Function<LogprobsFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& tokens, int64_t top) {
    Probs r = logprobs_forward(x, tokens, top, true);
    ctx->save_for_backward({x, tokens, r.entropy, r.stats});
    ctx->mark_non_differentiable({r.top_logprob, r.top_token});
    ctx->set_materialize_grads(false);
    return {r.logprob, r.entropy, r.top_logprob, r.top_token};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* who = "token_logprobs";
    check_capture(who);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &tokens = saved[1];
    Tensor dl = grads[0], de = grads[1];
    if (!dl.defined() && !de.defined()) return variable_list(3);
    if (dl.defined()) check_no_tangent(who, "the gradient of logprobs", dl);
    if (de.defined()) check_no_tangent(who, "the gradient of the entropy", de);
    if (dl.defined()) dl = dl.contiguous();
    if (de.defined()) de = de.contiguous();
    gs_logprobs_bwd_args a{};
    a.M = x.size(0);
    a.V = x.size(1);
    Tensor dx = torch::empty({a.M, a.V}, x.options());
    a.x = x.data_ptr();
    a.tokens = tokens.data_ptr();
    a.entropy = saved[2].data_ptr<float>();
    a.stats = saved[3].data_ptr<float>();
    a.dlogprob = ptr<float>(dl);
    a.dentropy = ptr<float>(de);
    a.dx = dx.data_ptr();
    a.sx = x.stride(0);
    a.sdx = a.V;
    a.token_bits = token_bits(who, tokens);
    a.dtype = dtype_code(x);
    const On on(x);
    raise_for(gs_logprobs_bwd(&a, on.stream));
    return once(who, {dx, Tensor(), Tensor()}, {x, grads[0], grads[1]});
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t top) {
  const char* who = "token_logprobs";
  check_on(who, "logits", logits, logits);
  dtype_of(who, "logits", logits);
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.numel() > 0, who, ": logits must be [..., V] and not empty; got shape ", logits.sizes());
  check_on(who, "tokens", tokens, logits);
  token_bits(who, tokens);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  check_shape(who, "tokens", tokens, lead);
  TORCH_CHECK_VALUE(top >= 0 && top <= 32 && top <= logits.size(-1), who, ": top must be 0 to 32 and at most V=", logits.size(-1),
                    "; got ", top);
  const Tensor x = rows(logits), flat = tokens.reshape({-1}).contiguous();
  Probs r;
  if (logits.requires_grad() && torch::GradMode::is_enabled()) {
    auto v = LogprobsFunction::apply(x, flat, top);
    r = Probs{v[0], v[1], v[2], v[3], Tensor()};
  } else {
    r = logprobs_forward(x, flat, top, false);
  }
  if (lead.size() == 1) return {r.logprob, r.entropy, r.top_logprob, r.top_token};
  std::vector<int64_t> with_top(lead.begin(), lead.end());
  with_top.push_back(top);
  return {r.logprob.view(lead), r.entropy.view(lead), r.top_logprob.view(with_top), r.top_token.view(with_top)};
}

}  // namespace

void bind_sequence_ops(py::module_& m) {
  m.def("causal_conv", &causal_conv, py::call_guard<py::gil_scoped_release>());
  m.def("causal_conv_step", &causal_conv_step, py::call_guard<py::gil_scoped_release>());
  m.def("selective_scan", &selective_scan, py::call_guard<py::gil_scoped_release>());
  m.def("selective_step", &selective_step, py::call_guard<py::gil_scoped_release>());
  m.def("embedding", &embedding, py::call_guard<py::gil_scoped_release>());
  m.def("token_logprobs", &token_logprobs, py::call_guard<py::gil_scoped_release>());
}
