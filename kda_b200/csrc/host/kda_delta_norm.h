// Part of kda_torch.cpp (included inside its namespace): the chunked gated delta rule with one decay per head, and the norms around a block.

// Every tensor of a call lies on `dev`: the kernels take addresses.
void require_device(const at::Device& dev, std::initializer_list<std::pair<const char*, const Tensor*>> ts) {
  for (const auto& [name, t] : ts) KDA_REQUIRE(!t->defined() || t->device() == dev, PyExc_ValueError, "kda_b200: `", name, "` is on ", t->device(), ", expected ", dev);
}
Tensor known(const Tensor& t) { return !t.defined() || known_dtype(t) ? dense(t) : f32(t); }      // bf16 and float32 as they are, other types as float32
std::optional<Tensor> some(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
Tensor as_type(const Tensor& t, int64_t type) { return t.defined() && static_cast<int64_t>(t.scalar_type()) != type ? t.to(static_cast<at::ScalarType>(type)) : t; }
int64_t type_of(const Tensor& t) { return t.defined() ? static_cast<int64_t>(t.scalar_type()) : 0; }
// Gradients are computed by kernels that autograd does not see into: asked for a graph of them, it would find nothing there.
void no_second_derivative(const char* what) { TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "kda_b200: ", what, " has no second derivative (create_graph=True)"); }

// ======================================================================================================================
// chunked gated delta rule
// ======================================================================================================================
struct DeltaCall {
  Tensor q, k, v, g, beta, h0, cu;
  std::optional<double> scale;
  bool output_final = false, l2norm = false, transposed = false;
  int slices = 0;
};
struct DeltaSaved { Tensor q, k, v, g, beta, h0, cu, ws; };
struct DeltaOpts { double scale = 1.0; bool output_final = false, l2norm = false; int slices = 0; };

kda_delta_args delta_args(const DeltaSaved& s, const DeltaOpts& o, bool save) {
  kda_delta_args a{};
  a.q = ptr(s.q); a.k = ptr(s.k); a.v = ptr(s.v); a.g = ptr(s.g); a.beta = ptr(s.beta); a.h0 = ptr<float>(s.h0); a.cu_seqlens = ptr<int32_t>(s.cu);
  a.workspace = ptr(s.ws); a.workspace_bytes = static_cast<size_t>(s.ws.numel());
  a.tokens = s.q.size(0) * s.q.size(1);
  a.N = static_cast<int32_t>(s.cu.defined() ? s.cu.numel() - 1 : s.q.size(0)); a.H = static_cast<int32_t>(s.v.size(2)); a.HQ = static_cast<int32_t>(s.q.size(2));
  a.K = static_cast<int32_t>(s.q.size(3)); a.V = static_cast<int32_t>(s.v.size(3)); a.io_dtype = dtype_code(s.q);
  a.g_dtype = dtype_code(s.g); a.beta_dtype = dtype_code(s.beta); a.use_qk_l2norm = o.l2norm; a.save_for_backward = save; a.scan_slices = o.slices;
  a.scale = static_cast<float>(o.scale);
  return a;
}

std::pair<Tensor, Tensor> delta_forward(DeltaSaved& s, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const Tensor& h0, const Tensor& cu,
                                        const DeltaOpts& o, bool save) {
  const at::Device dev = q.device();
  const c10::cuda::CUDAGuard guard(dev);
  s = {aligned(dense(q), true), aligned(dense(k), true), aligned(dense(v), true), known(g), known(beta), aligned(dense(h0), true), cu, Tensor()};
  const int64_t tokens = q.size(0) * q.size(1), N = cu.defined() ? cu.numel() - 1 : q.size(0), H = v.size(2), K = q.size(3), V = v.size(3);
  s.ws = bytes(kda_delta_chunk_workspace_bytes(tokens, static_cast<int32_t>(N), static_cast<int32_t>(H), static_cast<int32_t>(K), static_cast<int32_t>(V), save), dev);
  const Tensor out = empty(v.sizes(), v.scalar_type(), dev), ht = o.output_final ? empty({N, H, K, V}, at::kFloat, dev) : Tensor();
  kda_delta_args a = delta_args(s, o, save);
  a.o = ptr(out);
  a.ht = ptr<float>(ht);
  check_rc(kda_delta_chunk_fwd(&a, stream_of(dev)), "kda_delta_chunk_fwd");
  if (checked_mode() && tokens > 0 && N > 0) check_chunk_status(s.ws, "kda_delta_chunk_fwd");
  return {out, ht};
}

class DeltaFunction : public torch::autograd::Function<DeltaFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const std::optional<Tensor>& h0,
                               const std::optional<Tensor>& cu, const DeltaOpts& o) {
    DeltaSaved s;
    auto [out, ht] = delta_forward(s, q, k, v, g, beta, h0.value_or(Tensor()), cu.value_or(Tensor()), o, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({s.q, s.k, s.v, s.g, s.beta, s.h0, s.cu, s.ws});
    ctx->saved_data["opts"] = static_cast<int64_t>(o.output_final | o.l2norm << 1 | static_cast<int64_t>(o.slices) << 8);
    ctx->saved_data["scale"] = o.scale;
    ctx->saved_data["g"] = type_of(g);
    ctx->saved_data["beta"] = type_of(beta);
    if (o.output_final) return {out, ht};
    return {out};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("chunk_gated_delta");
    const variable_list t = ctx->get_saved_variables();
    const DeltaSaved s{t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7]};
    const int64_t f = ctx->saved_data["opts"].toInt();
    const DeltaOpts o{ctx->saved_data["scale"].toDouble(), (f & 1) != 0, (f & 2) != 0, static_cast<int>(f >> 8)};
    const at::Device dev = s.q.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor d_o = grads[0].defined() ? aligned(dense(as_type(grads[0], type_of(s.v))), true) : at::zeros_like(s.v);
    const Tensor d_ht = grads.size() > 1 ? aligned(f32(grads[1]), true) : Tensor();
    const Tensor dq = empty(s.q.sizes(), s.q.scalar_type(), dev), dk = empty(s.k.sizes(), s.k.scalar_type(), dev), dv = empty(s.v.sizes(), s.v.scalar_type(), dev);
    const Tensor dg = empty(s.g.sizes(), s.g.scalar_type(), dev), dbeta = empty(s.beta.sizes(), s.beta.scalar_type(), dev);
    const Tensor dh0 = s.h0.defined() ? empty(s.h0.sizes(), at::kFloat, dev) : Tensor();
    kda_delta_args a = delta_args(s, o, true);
    const Tensor bws = bytes(kda_delta_chunk_bwd_workspace_bytes(a.tokens, a.N, a.H, a.HQ, a.K, a.V), dev);
    a.d_o = ptr(d_o); a.d_ht = ptr<float>(d_ht); a.dq = ptr(dq); a.dk = ptr(dk); a.dv = ptr(dv); a.dg = ptr(dg); a.dbeta = ptr(dbeta); a.dh0 = ptr<float>(dh0);
    a.bwd_workspace = ptr(bws); a.bwd_workspace_bytes = static_cast<size_t>(bws.numel());
    check_rc(kda_delta_chunk_bwd(&a, stream_of(dev)), "kda_delta_chunk_bwd");
    if (checked_mode() && a.tokens > 0 && a.N > 0) check_chunk_status(s.ws, "kda_delta_chunk_bwd");
    return {dq, dk, dv, as_type(dg, ctx->saved_data["g"].toInt()), as_type(dbeta, ctx->saved_data["beta"].toInt()), dh0, Tensor(), Tensor()};
  }
};

// bf16, heads of multiples of eight columns up to 128.  Returns false for a call that takes another path.
bool chunk_delta(DeltaCall& c, Tensor& o, Tensor& ht) {
  const Sizes s = check_common(c.q, c.k, c.v, c.g, c.beta, c.h0, c.cu, true);
  const at::Device dev = c.q.device();
  require_device(dev, {{"k", &c.k}, {"v", &c.v}, {"g", &c.g}, {"beta", &c.beta}, {"initial_state", &c.h0}});
  KDA_REQUIRE(!has_tangent({&c.q, &c.k, &c.v, &c.g, &c.beta, &c.h0}), PyExc_NotImplementedError, "kda_b200: chunk_gated_delta has no forward-mode derivative (jvp)");
  const int64_t N = c.cu.defined() ? c.cu.numel() - 1 : s.B;
  const int64_t rows = c.transposed ? s.V : s.K, cols = c.transposed ? s.K : s.V;
  KDA_REQUIRE(!c.cu.defined() || (c.cu.dim() == 1 && c.cu.numel() >= 1), PyExc_ValueError, "cu_seqlens must be [N + 1], got ", c.cu.sizes());
  KDA_REQUIRE(!c.h0.defined() || (c.h0.sizes() == at::IntArrayRef{N, s.H, rows, cols}), PyExc_ValueError, "initial_state must have shape [", N, ", ", s.H, ", ", rows, ", ", cols,
              "], got ", c.h0.sizes());
  if (c.q.scalar_type() != at::kBFloat16 || s.K > 128 || s.V > 128 || s.K % 8 || s.V % 8) return false;
  const DeltaOpts opt{c.scale ? *c.scale : 1.0 / std::sqrt(static_cast<double>(s.K)), c.output_final, c.l2norm, c.slices};
  if (c.transposed && c.h0.defined()) c.h0 = c.h0.transpose(-1, -2);
  const Tensor cu = i32(c.cu, dev);
  if (wants_grad({&c.q, &c.k, &c.v, &c.g, &c.beta, &c.h0})) {
    const variable_list r = DeltaFunction::apply(c.q, c.k, c.v, c.g, c.beta, some(c.h0), some(cu), opt);
    o = r[0];
    if (r.size() > 1) ht = r[1];
  } else {
    DeltaSaved saved;
    std::tie(o, ht) = delta_forward(saved, c.q, c.k, c.v, c.g, c.beta, c.h0, cu, opt, false);
  }
  if (c.transposed && ht.defined()) ht = ht.transpose(-1, -2).contiguous();
  return true;
}

// ======================================================================================================================
// norms
// ======================================================================================================================
struct NormShape { int64_t rows, cols; };
NormShape norm_shape(const Tensor& x) {
  KDA_REQUIRE(x.is_cuda(), PyExc_RuntimeError, "kda_b200 runs on CUDA (sm_100a) tensors only; there is no CPU path");
  KDA_REQUIRE(x.dim() >= 1 && x.size(-1) > 0, PyExc_ValueError, "kda_b200: x must have a last dimension of at least one column, got ", x.sizes());
  const int64_t cols = x.size(-1);
  KDA_REQUIRE(cols <= 8192, PyExc_NotImplementedError, "kda_b200: the norm kernels take up to 8192 columns, got ", cols);
  KDA_REQUIRE(known_dtype(x), PyExc_NotImplementedError, "kda_b200: the norm kernels take bfloat16 and float32, got ", x.scalar_type());
  return {x.numel() / cols, cols};
}
void check_param(const Tensor& t, const char* name, int64_t cols) {
  if (!t.defined()) return;
  KDA_REQUIRE(t.dim() == 1 && t.size(0) == cols, PyExc_ValueError, "kda_b200: `", name, "` must have shape [", cols, "], got ", t.sizes());
  KDA_REQUIRE(known_dtype(t), PyExc_NotImplementedError, "kda_b200: `", name, "` must be bfloat16 or float32, got ", t.scalar_type());
}
int code_or(const Tensor& t) { return t.defined() ? dtype_code(t) : KDA_FP32; }

void check_norm_status(const char* what) {
  uint32_t st = 0;
  check_rc(kda_norm_status(&st), "kda_norm_status");
  if (!st) return;
  GilAcquire gil;
  PyErr_SetString(g_kda_error ? g_kda_error : PyExc_RuntimeError, cat(what, ": device status ", st, " (a bounded wait gave up); the outputs are incomplete").c_str());
  throw_current_python_error();
}

class GatedNormFunction : public torch::autograd::Function<GatedNormFunction> {
 public:
  static kda_norm_args args(const Tensor& x, const Tensor& gate, const Tensor& w, double eps, int act) {
    kda_norm_args a{};
    a.x = ptr(x); a.gate = ptr(gate); a.weight = ptr(w);
    a.cols = static_cast<int32_t>(x.size(-1)); a.rows = x.numel() / a.cols;
    a.io_dtype = dtype_code(x); a.gate_dtype = dtype_code(gate); a.weight_dtype = code_or(w); a.activation = act; a.eps = static_cast<float>(eps);
    return a;
  }
  static Tensor run(const Tensor& x, const Tensor& gate, const Tensor& w, double eps, int act) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor y = empty(x.sizes(), x.scalar_type(), x.device());
    kda_norm_args a = args(x, gate, w, eps, act);
    a.y = ptr(y);
    check_rc(kda_gated_norm_fwd(&a, stream_of(x.device())), "kda_gated_norm_fwd");
    if (checked_mode()) check_norm_status("kda_gated_norm_fwd");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& gate_, const std::optional<Tensor>& w_, double eps, int64_t act) {
    const Tensor x = dense(x_), gate = dense(gate_), w = dense(w_.value_or(Tensor()));
    ctx->save_for_backward({x, gate, w});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    return run(x, gate, w, eps, static_cast<int>(act));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("gated_rms_norm");
    const variable_list t = ctx->get_saved_variables();
    const Tensor &x = t[0], &gate = t[1], &w = t[2];
    const at::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor dy = dense(as_type(grads[0], type_of(x)));
    const Tensor dx = empty(x.sizes(), x.scalar_type(), dev), dz = empty(gate.sizes(), gate.scalar_type(), dev);
    const Tensor dw = w.defined() && ctx->needs_input_grad(2) ? empty(w.sizes(), w.scalar_type(), dev) : Tensor();
    kda_norm_args a = args(x, gate, w, ctx->saved_data["eps"].toDouble(), static_cast<int>(ctx->saved_data["act"].toInt()));
    a.dy = ptr(dy); a.dx = ptr(dx); a.dgate = ptr(dz); a.dweight = ptr(dw);
    Tensor ws;
    if (dw.defined()) {
      ws = bytes(kda_norm_bwd_workspace_bytes(a.rows, a.cols, 1), dev);
      a.workspace = ptr(ws); a.workspace_bytes = static_cast<size_t>(ws.numel());
    }
    check_rc(kda_gated_norm_bwd(&a, stream_of(dev)), "kda_gated_norm_bwd");
    if (checked_mode()) check_norm_status("kda_gated_norm_bwd");
    return {dx, dz, dw, Tensor(), Tensor()};
  }
};

Tensor gated_norm(const Tensor& x, const Tensor& gate, const Tensor& w, double eps, int act) {
  const NormShape s = norm_shape(x);
  require_device(x.device(), {{"gate", &gate}, {"weight", &w}});
  KDA_REQUIRE(gate.sizes() == x.sizes(), PyExc_ValueError, "kda_b200: gate must have x's shape ", x.sizes(), ", got ", gate.sizes());
  KDA_REQUIRE(known_dtype(gate), PyExc_NotImplementedError, "kda_b200: the norm kernels take bfloat16 and float32, got a gate of ", gate.scalar_type());
  check_param(w, "weight", s.cols);
  KDA_REQUIRE(!has_tangent({&x, &gate, &w}), PyExc_NotImplementedError, "kda_b200: gated_rms_norm has no forward-mode derivative (jvp)");
  if (wants_grad({&x, &gate, &w})) return GatedNormFunction::apply(x, gate, some(w), eps, static_cast<int64_t>(act));
  return GatedNormFunction::run(dense(x), dense(gate), dense(w), eps, act);
}

class ResidualNormFunction : public torch::autograd::Function<ResidualNormFunction> {
 public:
  static kda_norm_args args(const Tensor& x, const Tensor& res, const Tensor& w, const Tensor& post, const Tensor& scale, double value, double eps) {
    kda_norm_args a{};
    a.x = ptr(x); a.residual = ptr(res); a.weight = ptr(w); a.post_weight = ptr(post); a.scale = ptr(scale);
    a.cols = static_cast<int32_t>(x.size(-1)); a.rows = x.numel() / a.cols;
    a.io_dtype = dtype_code(x); a.residual_dtype = dtype_code(res); a.weight_dtype = dtype_code(w); a.post_dtype = code_or(post); a.scale_dtype = code_or(scale);
    a.eps = static_cast<float>(eps); a.scale_value = static_cast<float>(value);
    return a;
  }
  static std::pair<Tensor, Tensor> run(const Tensor& x, const Tensor& res, const Tensor& w, const Tensor& post, const Tensor& scale, double value, double eps) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor y = empty(x.sizes(), x.scalar_type(), x.device()), r = empty(res.sizes(), res.scalar_type(), x.device());
    kda_norm_args a = args(x, res, w, post, scale, value, eps);
    a.y = ptr(y);
    a.r = ptr(r);
    check_rc(kda_residual_norm_fwd(&a, stream_of(x.device())), "kda_residual_norm_fwd");
    if (checked_mode()) check_norm_status("kda_residual_norm_fwd");
    return {y, r};
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& x_, const Tensor& res_, const Tensor& w_, const std::optional<Tensor>& post_, const std::optional<Tensor>& scale_,
                               double value, double eps) {
    const Tensor x = dense(x_), res = dense(res_), w = dense(w_), post = dense(post_.value_or(Tensor())), scale = dense(scale_.value_or(Tensor()));
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, res, w, post, scale});
    ctx->saved_data["value"] = value;
    ctx->saved_data["eps"] = eps;
    auto [y, r] = run(x, res, w, post, scale, value, eps);
    return {y, r};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("residual_rms_norm");
    const variable_list t = ctx->get_saved_variables();
    const Tensor &x = t[0], &res = t[1], &w = t[2], &post = t[3], &scale = t[4];
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(7);
    const at::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor dy = dense(as_type(grads[0], type_of(x))), dr = dense(as_type(grads[1], type_of(res)));
    auto sum = [&](const Tensor& p, size_t i) { return p.defined() && ctx->needs_input_grad(i) ? empty(p.sizes(), p.scalar_type(), dev) : Tensor(); };
    const Tensor dx = empty(x.sizes(), x.scalar_type(), dev), dres = ctx->needs_input_grad(1) ? empty(res.sizes(), res.scalar_type(), dev) : Tensor();
    const Tensor dw = sum(w, 2), dpost = sum(post, 3), dscale = sum(scale, post.defined() ? 4 : 3);      // (only tensors that are there are counted)
    kda_norm_args a = args(x, res, w, post, scale, ctx->saved_data["value"].toDouble(), ctx->saved_data["eps"].toDouble());
    a.dy = ptr(dy); a.dr = ptr(dr); a.dx = ptr(dx); a.dresidual = ptr(dres); a.dweight = ptr(dw); a.dpost_weight = ptr(dpost); a.dscale = ptr(dscale);
    Tensor ws;
    if (dw.defined() || dpost.defined() || dscale.defined()) {
      ws = bytes(kda_norm_bwd_workspace_bytes(a.rows, a.cols, 2), dev);
      a.workspace = ptr(ws); a.workspace_bytes = static_cast<size_t>(ws.numel());
    }
    check_rc(kda_residual_norm_bwd(&a, stream_of(dev)), "kda_residual_norm_bwd");
    if (checked_mode()) check_norm_status("kda_residual_norm_bwd");
    return {dx, dres, dw, dpost, dscale, Tensor(), Tensor()};
  }
};

std::pair<Tensor, Tensor> residual_norm(const Tensor& x, const Tensor& res, const Tensor& w, const Tensor& scale, double value, const Tensor& post, double eps) {
  const NormShape s = norm_shape(x);
  require_device(x.device(), {{"residual", &res}, {"weight", &w}, {"scale", &scale}, {"post_weight", &post}});
  KDA_REQUIRE(res.sizes() == x.sizes(), PyExc_ValueError, "kda_b200: residual must have x's shape ", x.sizes(), ", got ", res.sizes());
  KDA_REQUIRE(known_dtype(res), PyExc_NotImplementedError, "kda_b200: the norm kernels take bfloat16 and float32, got a residual of ", res.scalar_type());
  check_param(w, "weight", s.cols);
  check_param(post, "post_weight", s.cols);
  check_param(scale, "scale", s.cols);
  KDA_REQUIRE(!has_tangent({&x, &res, &w, &scale, &post}), PyExc_NotImplementedError, "kda_b200: residual_rms_norm has no forward-mode derivative (jvp)");
  if (wants_grad({&x, &res, &w, &scale, &post})) {
    const variable_list r = ResidualNormFunction::apply(x, res, w, some(post), some(scale), value, eps);
    return {r[0], r[1]};
  }
  return ResidualNormFunction::run(dense(x), dense(res), dense(w), dense(post), dense(scale), value, eps);
}
