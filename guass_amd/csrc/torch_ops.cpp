// torch_ops.cpp - the feed-forward operators as torch operators (torch.ops.guass_amd.*): argument checks, outputs,
// workspaces and autograd around the C ABI of libgaussfield.so.  In C++ because a small call is all latency: the
// backward runs on autograd's own thread, where the same work in Python took 40 us more (64 x 1280 dropout, forward and
// backward: 96 us from Python, 48 us of them autograd's own).
#include "torch_common.h"

namespace {

void check_seed(const MaybeTensor& seed, const Tensor& x) {
  if (present(seed))
    TORCH_CHECK(seed->scalar_type() == at::kLong && seed->numel() == 1 && seed->device() == x.device(),
                "a seed tensor must be one int64 element on x's device");
}

gf_dropout make_dropout(double p, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset) {
  return {p, (uint64_t)seed, present(seed_tensor) ? (const uint64_t*)seed_tensor->data_ptr() : nullptr, (uint64_t)offset};
}

// ------------------------------------------------------------------------------- dropout

void check_dropout(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& seed) {
  check_first(x);
  if (present(residual)) {
    check_like(*residual, "residual", x);
    TORCH_CHECK(residual->sym_sizes() == x.sym_sizes(), "residual must have x's shape ", x.sym_sizes(), " (got ", residual->sym_sizes(), ")");
  }
  check_seed(seed, x);
}

Tensor dropout_forward(const Tensor& x, const MaybeTensor& residual, double p, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset) {
  check_dropout(x, residual, seed_tensor);
  const gf_dropout d = make_dropout(p, seed, seed_tensor, offset);
  Tensor y = at::empty_like(x, at::MemoryFormat::Contiguous);
  if (y.numel() == 0) return y;
  const c10::DeviceGuard guard(x.device());
  const Rows a(x.dim() ? x : x.view({1}));
  std::optional<Rows> r;
  if (present(residual)) r.emplace(x.dim() ? *residual : residual->view({1}));
  check_rc(gf_dropout_add(dtype_of(x), &d, a.rows, a.cols, a.data(), a.ld, r ? r->data() : nullptr, r ? r->ld : 0, y.data_ptr(), a.cols,
                          stream_of(x)),
           "gf_dropout_add");
  return y;
}

Tensor call_dropout_forward(const Tensor& x, const MaybeTensor& residual, double p, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("guass_amd::dropout_forward", "").typed<decltype(dropout_forward)>();
  return op.call(x, residual, p, seed, seed_tensor, offset);
}

struct DropoutAdd : torch::autograd::Function<DropoutAdd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual, double p, int64_t seed,
                        const MaybeTensor& seed_tensor, int64_t offset) {
    ctx->saved_data["rng"] = std::make_tuple(p, seed, offset);
    ctx->saved_data["residual"] = present(residual);
    if (present(seed_tensor)) ctx->save_for_backward({*seed_tensor});
    return call_dropout_forward(x, residual, p, seed, seed_tensor, offset);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto [p, seed, offset] = ctx->saved_data["rng"].to<std::tuple<double, int64_t, int64_t>>();
    const bool want_x = ctx->needs_input_grad(0), want_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1);
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    const bool again = dy.requires_grad();
    Tensor dx;
    if (want_x) dx = call_dropout_forward(dy, std::nullopt, p, seed, saved.empty() ? MaybeTensor() : saved[0], offset);
    return once({dx, want_r ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, "dropout_add", again);
  }
};

Tensor dropout_add(const Tensor& x, const MaybeTensor& residual, double p, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset) {
  check_dropout(x, residual, seed_tensor);
  check_no_tangent("dropout_add", x, residual);
  if (at::GradMode::is_enabled() && (wants(x) || wants(residual))) return DropoutAdd::apply(x, residual, p, seed, seed_tensor, offset);
  return call_dropout_forward(x, residual, p, seed, seed_tensor, offset);
}

// ------------------------------------------------------------------------ linear and gated

void check_linear(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual, int64_t activation,
                  const MaybeTensor& seed) {
  check_first(x);
  check_like(weight, "weight", x);
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2, "x must have shape [..., in_features] and weight two dimensions");
  const auto rows = weight.sym_size(0), cols = weight.sym_size(1);  // symbolic in a trace
  TORCH_CHECK(rows != 0 && cols != 0, "weight must not be empty");
  TORCH_CHECK(activation == GF_ACT_NONE || rows % 2 == 0, "a gated weight must have an even number of rows: the value's, then the gate's");
  TORCH_CHECK(x.sym_size(-1) == cols, "x has ", x.sym_size(-1), " features, weight takes ", cols);
  if (present(bias)) {
    check_like(*bias, "bias", x);
    TORCH_CHECK(bias->dim() == 1 && bias->sym_size(0) == rows, "bias must have shape [", rows, "]");
  }
  if (present(residual)) {
    check_like(*residual, "residual", x);
    auto want = x.sym_sizes().vec();
    want.back() = rows;
    TORCH_CHECK(residual->sym_sizes() == c10::SymIntArrayRef(want), "residual must have shape ", c10::SymIntArrayRef(want), " (got ",
                residual->sym_sizes(), ")");
  }
  check_seed(seed, x);
}

struct Products {
  Rows x, weight;
  gf_ff_args args{};
  Products(const Tensor& x_, const Tensor& weight_, int64_t activation, const gf_dropout& d) : x(x_), weight(weight_) {
    args.dtype = dtype_of(x_);
    args.activation = (int32_t)activation;
    args.rows = x.rows, args.in_features = x.cols;
    args.out_features = weight.rows / (activation == GF_ACT_NONE ? 1 : 2);
    args.x = x.data(), args.ldx = x.ld, args.weight = weight.data(), args.ldw = weight.ld;
    args.dropout = d;
  }
  // on the current stream, with a workspace of torch's allocator on that stream
  void run(bool backward) {
    const size_t bytes = gf_ff_workspace_bytes(&args, backward);
    Tensor workspace;
    if (bytes) workspace = at::empty({(int64_t)bytes}, x.t.options().dtype(at::kByte));
    void* const p = bytes ? workspace.data_ptr() : nullptr;
    if (backward)
      check_rc(gf_ff_backward(&args, p, bytes, stream_of(x.t)), "gf_ff_backward");
    else
      check_rc(gf_ff_forward(&args, p, bytes, stream_of(x.t)), "gf_ff_forward");
  }
};

// y, and what the backward needs of the products (undefined for a linear product or if not to be saved)
std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual,
                                          int64_t activation, double p_drop, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset,
                                          bool save) {
  check_linear(x, weight, bias, residual, activation, seed_tensor);
  const gf_dropout d = make_dropout(p_drop, seed, seed_tensor, offset);
  auto shape = x.sizes().vec();
  shape.back() = weight.size(0) / (activation == GF_ACT_NONE ? 1 : 2);
  Tensor y = at::empty(shape, x.options()), saved, b;
  if (y.numel() == 0) {
    if (save && activation != GF_ACT_NONE) saved = at::empty({0}, x.options().dtype(at::kByte));  // as a trace has it
    return {y, saved};
  }
  const c10::DeviceGuard guard(x.device());
  Products p(x, weight, activation, d);
  if (save && activation != GF_ACT_NONE) {
    saved = at::empty({(int64_t)gf_ff_saved_bytes(&p.args)}, x.options().dtype(at::kByte));
    p.args.saved = saved.data_ptr();
  }
  p.args.y = y.data_ptr();
  if (present(bias)) b = bias->contiguous(), p.args.bias = b.data_ptr();
  std::optional<Rows> r;
  if (present(residual)) r.emplace(*residual), p.args.residual = r->data(), p.args.ldr = r->ld;
  p.run(false);
  return {y, saved};
}

std::tuple<Tensor, Tensor> call_linear_forward(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual,
                                               int64_t activation, double p, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset,
                                               bool save) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("guass_amd::linear_forward", "").typed<decltype(linear_forward)>();
  return op.call(x, weight, bias, residual, activation, p, seed, seed_tensor, offset, save);
}

// The gradients of x, weight and bias that are wanted.
std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& x, const Tensor& weight, const MaybeTensor& saved, const Tensor& dy,
                                                   int64_t activation, double p_drop, int64_t seed, const MaybeTensor& seed_tensor,
                                                   int64_t offset, bool want_x, bool want_w, bool want_b) {
  check_linear(x, weight, std::nullopt, std::nullopt, activation, seed_tensor);
  check_like(dy, "dy", x);
  auto want = x.sizes().vec();
  want.back() = weight.size(0) / (activation == GF_ACT_NONE ? 1 : 2);
  TORCH_CHECK(dy.sizes() == at::IntArrayRef(want), "dy must have shape ", at::IntArrayRef(want), " (got ", dy.sizes(), ")");
  const gf_dropout d = make_dropout(p_drop, seed, seed_tensor, offset);
  const bool some = dy.numel() != 0;  // no rows: every sum is empty
  auto make = [&](at::IntArrayRef shape) { return some ? at::empty(shape, x.options()) : at::zeros(shape, x.options()); };
  Tensor dx, dw, db;
  if (want_x) dx = make(x.sizes());
  if (want_w) dw = make(weight.sizes());
  if (want_b) db = make(weight.sizes().slice(0, 1));
  if (!some || !(want_x || want_w || want_b)) return {dx, dw, db};
  const c10::DeviceGuard guard(x.device());
  Products p(x, weight, activation, d);
  const Rows g(dy);
  p.args.dy = g.data(), p.args.lddy = g.ld;
  if (activation != GF_ACT_NONE) {
    TORCH_CHECK(present(saved) && saved->is_cuda() && saved->is_contiguous() && saved->nbytes() >= gf_ff_saved_bytes(&p.args),
                "saved must be what the forward with save=True returned");
    p.args.saved = saved->data_ptr();
  }
  if (want_x) p.args.dx = dx.data_ptr();
  if (want_w) p.args.dweight = dw.data_ptr();
  if (want_b) p.args.dbias = db.data_ptr();
  p.run(true);
  return {dx, dw, db};
}

std::tuple<Tensor, Tensor, Tensor> call_linear_backward(const Tensor& x, const Tensor& weight, const MaybeTensor& saved, const Tensor& dy,
                                                        int64_t activation, double p, int64_t seed, const MaybeTensor& seed_tensor,
                                                        int64_t offset, bool want_x, bool want_w, bool want_b) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("guass_amd::linear_backward", "").typed<decltype(linear_backward)>();
  return op.call(x, weight, saved, dy, activation, p, seed, seed_tensor, offset, want_x, want_w, want_b);
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual,
                        int64_t activation, double p, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset) {
    const bool save = wants(x) || wants(weight) || wants(bias);
    auto [y, saved] = call_linear_forward(x, weight, bias, residual, activation, p, seed, seed_tensor, offset, save);
    ctx->save_for_backward({x, weight, saved, present(seed_tensor) ? *seed_tensor : Tensor()});
    ctx->saved_data["call"] = std::make_tuple(activation, p, seed, offset);
    ctx->saved_data["inputs"] = std::make_tuple(present(bias), present(residual), wants(bias));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto [activation, p, seed, offset] = ctx->saved_data["call"].to<std::tuple<int64_t, double, int64_t, int64_t>>();
    const auto [has_bias, has_residual, trains_bias] = ctx->saved_data["inputs"].to<std::tuple<bool, bool, bool>>();
    // what this backward is for: of the inputs that train, those that it was asked for (edges are the tensors that are there)
    const bool wx = ctx->needs_input_grad(0), ww = ctx->needs_input_grad(1), wb = has_bias && ctx->needs_input_grad(2),
               wr = has_residual && ctx->needs_input_grad(2 + has_bias);
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    // what the gradients depend on: a gated product's on the bias too, by value and gate
    const bool again = dy.requires_grad() || saved[0].requires_grad() || saved[1].requires_grad() || (activation != GF_ACT_NONE && trains_bias);
    auto [dx, dw, db] = call_linear_backward(saved[0], saved[1], maybe(saved[2]), dy, activation, p, seed, maybe(saved[3]), offset, wx, ww, wb);
    return once({dx, dw, db, wr ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()},
                activation == GF_ACT_NONE ? "linear_dropout_add" : "gated_linear", again);
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual, int64_t activation, double p,
              int64_t seed, const MaybeTensor& seed_tensor, int64_t offset) {
  check_linear(x, weight, bias, residual, activation, seed_tensor);
  check_no_tangent(activation == GF_ACT_NONE ? "linear_dropout_add" : "gated_linear", x, MaybeTensor(weight), bias, residual);
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias) || wants(residual)))
    return Linear::apply(x, weight, bias, residual, activation, p, seed, seed_tensor, offset);
  return std::get<0>(call_linear_forward(x, weight, bias, residual, activation, p, seed, seed_tensor, offset, false));
}

// ------------------------------------------------------------------------------ autocast

// As torch's linear: the operands in autocast's type.  A residual of that type is added by the kernels; another one after them,
// by torch's rules (a float32 residual stream stays one).
Tensor linear_autocast(const Tensor& x, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& residual, int64_t activation,
                       double p, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset) {
  const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
  const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
  auto cast = [&](const Tensor& t) { return at::autocast::cached_cast(type, t, at::kCUDA); };
  const bool fused = !present(residual) || residual->scalar_type() == type;
  const Tensor y = linear(cast(x), cast(weight), present(bias) ? MaybeTensor(cast(*bias)) : bias, fused ? residual : MaybeTensor(), activation, p,
                          seed, seed_tensor, offset);
  return fused ? y : *residual + y;
}

// As torch's dropout: in x's own type, and the sum by torch's rules where the residual's is another.
Tensor dropout_add_autocast(const Tensor& x, const MaybeTensor& residual, double p, int64_t seed, const MaybeTensor& seed_tensor, int64_t offset) {
  const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
  if (!present(residual) || residual->scalar_type() == x.scalar_type()) return dropout_add(x, residual, p, seed, seed_tensor, offset);
  return *residual + dropout_add(x, std::nullopt, p, seed, seed_tensor, offset);
}

}  // namespace

TORCH_LIBRARY_IMPL(guass_amd, Autocast, m) {
  m.impl("dropout_add", dropout_add_autocast);
  m.impl("linear", linear_autocast);
}

TORCH_LIBRARY(guass_amd, m) {
  // what a user calls: checks and autograd around the operators below
  m.def("dropout_add(Tensor x, Tensor? residual, float p, int seed, Tensor? seed_tensor, int offset) -> Tensor", dropout_add);
  m.def("linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int activation, float p, int seed, Tensor? seed_tensor, "
        "int offset) -> Tensor", linear);
  // the launches by themselves, without autograd: what a HIP graph captures, and what a trace (torch.compile) holds
  m.def("dropout_forward(Tensor x, Tensor? residual, float p, int seed, Tensor? seed_tensor, int offset) -> Tensor");
  m.def("linear_forward(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int activation, float p, int seed, Tensor? seed_tensor, "
        "int offset, bool save) -> (Tensor, Tensor)");
  m.def("linear_backward(Tensor x, Tensor weight, Tensor? saved, Tensor dy, int activation, float p, int seed, Tensor? seed_tensor, "
        "int offset, bool want_x, bool want_weight, bool want_bias) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(guass_amd, CUDA, m) {
  m.impl("dropout_forward", dropout_forward);
  m.impl("linear_forward", linear_forward);
  m.impl("linear_backward", linear_backward);
}

TORCH_LIBRARY_IMPL(guass_amd, Autograd, m) {
  for (const char* name : {"dropout_forward", "linear_forward", "linear_backward"}) m.impl(name, torch::CppFunction::makeFallthrough());
}
