// torch_block_ops.cpp - the norms around a block and products with 4-bit weights as torch operators, as torch_ops.cpp has the
// feed-forward operators.
#include "torch_common.h"

#include <array>
#include <string>
#include <vector>

namespace {

// -------------------------------------------------------------------------------- norms

// gate, scale or shift: a row for each group of x's rows, or (ld 0) one for all.
struct Shared {
  std::optional<Rows> m;
  int64_t group_rows = 0;  // 0: for all rows
  const void* data() const { return m ? m->data() : nullptr; }
  int64_t ld() const { return group_rows ? m->ld : 0; }
};

// [cols], or x's sizes with ones behind the first few.
Shared shared_of(const MaybeTensor& t, const char* name, const Tensor& x) {
  Shared s;
  if (!present(t)) return s;
  check_like(*t, name, x);
  bool ok = t->dim() >= 1 && t->size(-1) == x.size(-1) && (t->dim() == 1 || t->dim() == x.dim());
  int64_t own = 0;  // leading dimensions that are t's own
  if (ok && t->dim() > 1) {
    for (int64_t i = 0; i + 1 < x.dim(); ++i)
      if (t->size(i) != 1) own = i + 1;
    for (int64_t i = 0; i < own; ++i) ok = ok && t->size(i) == x.size(i);
  }
  TORCH_CHECK(ok, name, " must have shape [", x.size(-1), "] or x's, ", x.sizes(), ", with ones behind its first dimensions (got ", t->sizes(), ")");
  s.m.emplace(*t);
  if (own) {
    s.group_rows = 1;
    for (int64_t i = own; i + 1 < x.dim(); ++i) s.group_rows *= x.size(i);
  }
  return s;
}

void check_vector(const MaybeTensor& t, const char* name, const Tensor& x) {
  if (!present(t)) return;
  check_like(*t, name, x);
  TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), name, " must have shape [", x.size(-1), "] (got ", t->sizes(), ")");
}

void check_same(const MaybeTensor& t, const char* name, const Tensor& x) {
  if (!present(t)) return;
  check_like(*t, name, x);
  TORCH_CHECK(t->sizes() == x.sizes(), name, " must have x's shape ", x.sizes(), " (got ", t->sizes(), ")");
}

#define NORM_PARAMETERS                                                                                                              \
  const Tensor &x, const MaybeTensor &residual, const MaybeTensor &weight, const MaybeTensor &bias, const MaybeTensor &gate,          \
      double gate_value, double residual_scale, int64_t kind, double eps, const MaybeTensor &next_weight, const MaybeTensor &next_bias, \
      const MaybeTensor &scale, const MaybeTensor &shift, int64_t next_kind, double next_eps
#define NORM_ARGUMENTS \
  x, residual, weight, bias, gate, gate_value, residual_scale, kind, eps, next_weight, next_bias, scale, shift, next_kind, next_eps

// The call as the C ABI takes it, with the tensors that it points into.  A residual that is not read (a backward without a next norm) has x's
// place.
struct NormCall {
  Rows x;
  std::optional<Rows> residual;
  std::array<Tensor, 4> vectors;
  Shared gate, scale, shift;
  gf_norm_args a{};
  explicit NormCall(NORM_PARAMETERS, bool reads_residual = true) : x(x) {
    a.dtype = dtype_of(x), a.kind = (int32_t)kind, a.next_kind = (int32_t)next_kind;
    a.rows = this->x.rows, a.cols = this->x.cols;
    a.eps = eps, a.next_eps = next_eps, a.gate_value = gate_value, a.residual_scale = residual_scale;
    a.x = this->x.data(), a.ldx = this->x.ld;
    check_same(residual, "residual", x);
    if (present(residual) && reads_residual)
      this->residual.emplace(*residual), a.residual = this->residual->data(), a.ldr = this->residual->ld;
    else if (present(residual))
      a.residual = a.x, a.ldr = a.ldx;
    const MaybeTensor* const from[] = {&weight, &bias, &next_weight, &next_bias};
    const void** const to[] = {&a.weight, &a.bias, &a.next_weight, &a.next_bias};
    const char* const names[] = {"weight", "bias", present(residual) ? "next_weight" : "weight", present(residual) ? "next_bias" : "bias"};
    for (int i = 0; i < 4; ++i) {
      check_vector(*from[i], names[i], x);
      if (present(*from[i])) vectors[i] = (*from[i])->contiguous(), *to[i] = vectors[i].data_ptr();
    }
    this->gate = shared_of(gate, "gate", x), this->scale = shared_of(scale, "scale", x), this->shift = shared_of(shift, "shift", x);
    a.gate = this->gate.data(), a.ld_gate = this->gate.ld();
    a.scale = this->scale.data(), a.ld_scale = this->scale.ld();
    a.shift = this->shift.data(), a.ld_shift = this->shift.ld();
    a.group_rows = 0;
    for (const Shared* s : {&this->gate, &this->scale, &this->shift}) {
      if (s->group_rows == 0) continue;
      TORCH_CHECK(a.group_rows == 0 || a.group_rows == s->group_rows, "gate, scale and shift must be shared by the same rows, or by all");
      a.group_rows = s->group_rows;
    }
    if (a.group_rows == 0) a.group_rows = std::max<int64_t>(a.rows, 1);
  }
};

void check_norm(const Tensor& x) {
  check_first(x);
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
}

// (stream, normed), undefined where there is none
std::tuple<Tensor, Tensor> block_norm_forward(NORM_PARAMETERS, bool want_stream) {
  check_norm(x);
  const c10::DeviceGuard guard(x.device());
  Tensor stream, normed;
  if (present(residual) && want_stream) stream = at::empty(x.sizes(), x.options());
  if (next_kind != GF_NORM_NONE) normed = at::empty(x.sizes(), x.options());
  NormCall c(NORM_ARGUMENTS);
  if (c.x.rows == 0 && c.x.cols != 0) return {stream, normed};  // an empty residual has no address
  if (stream.defined()) c.a.stream = stream.data_ptr();
  if (normed.defined()) c.a.normed = normed.data_ptr();
  check_rc(gf_norm_forward(&c.a, stream_of(x)), "gf_norm_forward");
  return {stream, normed};
}

// Which gradients are wanted, by bit, in the order in which they are returned.
enum Want { kX, kResidual, kWeight, kBias, kGate, kNextWeight, kNextBias, kScale, kShift, kWants };

using NormGrads = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

NormGrads block_norm_backward(NORM_PARAMETERS, const MaybeTensor& dstream, const MaybeTensor& dnormed, int64_t wants) {
  check_norm(x);
  const c10::DeviceGuard guard(x.device());
  check_same(dstream, "dstream", x), check_same(dnormed, "dnormed", x);
  const MaybeTensor* const like[kWants] = {nullptr, &residual, &weight, &bias, &gate, &next_weight, &next_bias, &scale, &shift};
  const bool next = present(dnormed);  // else the stream's gradient alone: the next norm's parameters have zeros
  std::array<Tensor, kWants> grads;
  void* at_[kWants] = {};
  for (int i = 0; i < kWants; ++i) {
    if (!(wants >> i & 1) || (i != kX && !present(*like[i]))) continue;
    const auto sizes = i == kX ? x.sizes() : (*like[i])->sizes();
    const bool zero = x.numel() == 0 || (!next && i >= kNextWeight) || (!next && !present(dstream));
    grads[i] = zero ? at::zeros(sizes, x.options()) : at::empty(sizes, x.options());
    if (!zero) at_[i] = grads[i].data_ptr();
  }
  if (x.numel() != 0 && (next || present(dstream))) {
    const MaybeTensor none;
    NormCall c(x, residual, weight, bias, gate, gate_value, residual_scale, kind, eps, next ? next_weight : none, next ? next_bias : none,
               next ? scale : none, next ? shift : none, next ? next_kind : (int64_t)GF_NORM_NONE, next_eps, next);
    std::optional<Rows> ds, dh;
    if (present(dstream)) ds = dstream->is_same(x) ? c.x : Rows(*dstream), c.a.dstream = ds->data(), c.a.ld_dstream = ds->ld;
    if (next) dh.emplace(*dnormed), c.a.dnormed = dh->data(), c.a.ld_dnormed = dh->ld;
    c.a.dx = at_[kX], c.a.dresidual = at_[kResidual], c.a.dweight = at_[kWeight], c.a.dbias = at_[kBias], c.a.dgate = at_[kGate];
    c.a.dnext_weight = at_[kNextWeight], c.a.dnext_bias = at_[kNextBias], c.a.dscale = at_[kScale], c.a.dshift = at_[kShift];
    const size_t bytes = gf_norm_workspace_bytes(&c.a);
    Tensor workspace;
    if (bytes) workspace = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    check_rc(gf_norm_backward(&c.a, bytes ? workspace.data_ptr() : nullptr, bytes, stream_of(x)), "gf_norm_backward");
  }
  return {grads[0], grads[1], grads[2], grads[3], grads[4], grads[5], grads[6], grads[7], grads[8]};
}

std::tuple<Tensor, Tensor> call_norm_forward(NORM_PARAMETERS, bool want_stream) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("guass_amd::block_norm_forward", "").typed<decltype(block_norm_forward)>();
  return op.call(NORM_ARGUMENTS, want_stream);
}

NormGrads call_norm_backward(NORM_PARAMETERS, const MaybeTensor& dstream, const MaybeTensor& dnormed, int64_t wants) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("guass_amd::block_norm_backward", "").typed<decltype(block_norm_backward)>();
  return op.call(NORM_ARGUMENTS, dstream, dnormed, wants);
}

const char* norm_name(bool branch, bool next) { return !branch ? "norm" : next ? "gate_add_norm" : "gate_add"; }

// What a gradient is made of besides the outputs' gradients, by Want's bits, where the next norm has one (`next`) and where the stream has
// alone: then the residual goes into none, and x only through a norm or into what is summed with it.
int64_t made_of(int i, bool next, bool normed) {
  if (next) {
    const int64_t stream = 1 << kX | 1 << kResidual | 1 << kWeight | 1 << kBias | 1 << kGate;
    switch (i) {
      case kNextWeight: return stream | 1 << kScale;
      case kNextBias: return 1 << kScale;
      case kScale: return stream | 1 << kNextWeight | 1 << kNextBias;
      case kShift: return 0;
      default: return stream | 1 << kNextWeight | 1 << kScale;
    }
  }
  const int64_t row = normed ? 1 << kX : 0;
  switch (i) {
    case kX: return row | 1 << kWeight | 1 << kGate;
    case kWeight: return row | 1 << kGate;
    case kBias: return 1 << kGate;
    case kGate: return 1 << kX | 1 << kWeight | 1 << kBias;
    default: return 0;
  }
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
  // the positions of the tensors among forward's arguments
  static constexpr int kAt[kWants] = {0, 1, 2, 3, 4, 9, 10, 11, 12};
  static variable_list forward(AutogradContext* ctx, NORM_PARAMETERS) {
    const bool branch = present(residual), next = next_kind != GF_NORM_NONE;
    auto [stream, normed] = call_norm_forward(NORM_ARGUMENTS, true);
    const MaybeTensor first(x);
    const MaybeTensor* const inputs[kWants] = {&first, &residual, &weight, &bias, &gate, &next_weight, &next_bias, &scale, &shift};
    // x and the residual only where a gradient is made of them: they are as large as the stream, and the caller may write them
    int64_t there = 0, needs = next ? 1 << kX | 1 << kResidual : 0;
    for (int i = 0; i < kWants; ++i) {
      if (!present(*inputs[i])) continue;
      there |= int64_t(1) << i;
      if (!next && wants(*inputs[i])) needs |= made_of(i, false, kind != GF_NORM_NONE);
    }
    variable_list saved(kWants);
    for (int i = 0; i < kWants; ++i)
      if ((there >> i & 1) && (i > kResidual || (needs >> i & 1))) saved[i] = **inputs[i];
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["call"] = std::make_tuple(gate_value, residual_scale, kind, eps, next_kind, next_eps, there);
    ctx->set_materialize_grads(false);
    if (!branch) return {normed};
    return next ? variable_list{stream, normed} : variable_list{stream};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto [gate_value, residual_scale, kind, eps, next_kind, next_eps, there] =
        ctx->saved_data["call"].to<std::tuple<double, double, int64_t, double, int64_t, double, int64_t>>();
    auto s = ctx->get_saved_variables();
    const bool branch = there >> kResidual & 1, next = next_kind != GF_NORM_NONE;
    const Tensor dstream = branch ? grads[0] : Tensor(), dnormed = next ? grads[branch ? 1 : 0] : Tensor();
    int64_t wants = 0, train = 0;
    for (int i = 0, edge = 0; i < kWants; ++i) {
      if (!(there >> i & 1)) continue;
      if (ctx->needs_input_grad(edge++)) wants |= int64_t(1) << i;  // edges are the tensors that are there
      if (s[i].defined() && s[i].requires_grad()) train |= int64_t(1) << i;
    }
    variable_list out(15);
    if (!dstream.defined() && !dnormed.defined()) return out;
    // an unscaled residual that only gate_add has seen: its gradient is the stream's
    const bool same = !next && residual_scale == 1.0 && (wants >> kResidual & 1);
    if (same) wants &= ~(int64_t(1) << kResidual);
    NormGrads g;
    if (wants) {
      if (!next) {  // what is not read needs a shape only
        for (const int i : {kX, kResidual})
          if (!s[i].defined()) s[i] = dstream;
      }
      g = call_norm_backward(s[kX], maybe(s[kResidual]), maybe(s[kWeight]), maybe(s[kBias]), maybe(s[kGate]), gate_value, residual_scale, kind, eps,
                             maybe(s[kNextWeight]), maybe(s[kNextBias]), maybe(s[kScale]), maybe(s[kShift]), next_kind, next_eps, maybe(dstream),
                             maybe(dnormed), wants);
    }
    const auto& [g0, g1, g2, g3, g4, g5, g6, g7, g8] = g;
    const Tensor* const all[kWants] = {&g0, &g1, &g2, &g3, &g4, &g5, &g6, &g7, &g8};
    // those that depend on what trains refuse a second derivative
    const bool linear = (dstream.defined() && dstream.requires_grad()) || (dnormed.defined() && dnormed.requires_grad());
    variable_list refusing(kWants);
    bool again = false;
    for (int i = 0; i < kWants; ++i) {
      const bool depends = all[i]->defined() && (linear || (made_of(i, dnormed.defined(), kind != GF_NORM_NONE) & train));
      (depends ? refusing[i] : out[kAt[i]]) = *all[i];
      again = again || depends;
    }
    refusing = once(std::move(refusing), norm_name(branch, next), again);
    for (int i = 0; i < kWants; ++i)
      if (refusing[i].defined()) out[kAt[i]] = refusing[i];
    if (same) out[kAt[kResidual]] = dstream;
    return out;
  }
};

// (stream, normed), undefined where there is none
std::tuple<Tensor, Tensor> block_norm(NORM_PARAMETERS) {
  check_norm(x);
  const bool branch = present(residual), next = next_kind != GF_NORM_NONE;
  check_no_tangent(norm_name(branch, next), x, residual, weight, bias, gate, next_weight, next_bias, scale, shift);
  const bool grad = wants(x) || wants(residual) || wants(weight) || wants(bias) || wants(gate) || wants(next_weight) || wants(next_bias) ||
                    wants(scale) || wants(shift);
  if (!at::GradMode::is_enabled() || !grad) return call_norm_forward(NORM_ARGUMENTS, true);
  variable_list out = BlockNorm::apply(NORM_ARGUMENTS);
  if (!branch) return {Tensor(), out[0]};
  return {out[0], next ? out[1] : Tensor()};
}

// As torch's layer_norm: in 32 bits.
std::tuple<Tensor, Tensor> block_norm_autocast(NORM_PARAMETERS) {
  const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
  auto cast = [](const Tensor& t) { return at::autocast::cached_cast(at::kFloat, t, at::kCUDA); };
  auto maybe_cast = [&](const MaybeTensor& t) { return present(t) ? MaybeTensor(cast(*t)) : t; };
  return block_norm(cast(x), maybe_cast(residual), maybe_cast(weight), maybe_cast(bias), maybe_cast(gate), gate_value, residual_scale, kind, eps,
                    maybe_cast(next_weight), maybe_cast(next_bias), maybe_cast(scale), maybe_cast(shift), next_kind, next_eps);
}

// ------------------------------------------------------------------------ 4-bit weights

constexpr int64_t kTileCodes = 1024, kTileScales = 64;  // bytes of a tile of 16 rows x 128 columns

// codes and scales as the kernels read them
struct Packed {
  Tensor codes, scales;
  Packed(const Tensor& c, const Tensor& s, int64_t rows, int64_t cols, c10::Device device) : codes(c), scales(s) {
    TORCH_CHECK(c.scalar_type() == at::kByte && s.scalar_type() == at::kByte, "codes and scales must be uint8");
    TORCH_CHECK(c.device() == device && s.device() == device, "all tensors must be on the same device (got ", device, ", ", c.device(), " and ",
                s.device(), ")");
    const int64_t bands = (rows + 15) / 16, across = (cols + 127) / 128, codes_of[] = {bands, across, kTileCodes}, scales_of[] = {bands, across, kTileScales};
    TORCH_CHECK(rows >= 0 && cols > 0 && c.sizes() == at::IntArrayRef(codes_of) && s.sizes() == at::IntArrayRef(scales_of), "a weight [", rows, ", ", cols,
                "] has tiles of codes [", bands, ", ", across, ", 1024] and scales [", bands, ", ", across, ", 64] (got ", c.sizes(), " and ", s.sizes(), ")");
    if (!codes.is_contiguous() || (uintptr_t)codes.data_ptr() % 16 != 0) codes = codes.clone(at::MemoryFormat::Contiguous);
    if (!scales.is_contiguous() || (uintptr_t)scales.data_ptr() % 4 != 0) scales = scales.clone(at::MemoryFormat::Contiguous);
  }
};

std::tuple<Tensor, Tensor> q4_quantize(const Tensor& weight) {
  TORCH_CHECK(weight.is_cuda(), "weight must be a CUDA tensor");
  const auto t = weight.scalar_type();
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "weight must be float32, bfloat16 or float16 (got ", type_name(t), ")");
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) > 0, "weight must have two dimensions, the second not empty");
  const c10::DeviceGuard guard(weight.device());
  const int64_t rows = weight.size(0), cols = weight.size(1), bands = (rows + 15) / 16, across = (cols + 127) / 128;
  const auto bytes = weight.options().dtype(at::kByte);
  Tensor codes = at::empty({bands, across, kTileCodes}, bytes), scales = at::empty({bands, across, kTileScales}, bytes);
  if (rows == 0) return {codes, scales};
  const Rows w(weight);
  check_rc(gf_q4_quantize(dtype_of(weight), rows, cols, w.data(), w.ld, codes.data_ptr(), scales.data_ptr(), stream_of(weight)), "gf_q4_quantize");
  return {codes, scales};
}

Tensor q4_dequantize(const Tensor& codes, const Tensor& scales, int64_t rows, int64_t cols, at::ScalarType dtype) {
  TORCH_CHECK(codes.is_cuda(), "codes must be a CUDA tensor");
  TORCH_CHECK(dtype == at::kFloat || dtype == at::kBFloat16 || dtype == at::kHalf, "dtype must be float32, bfloat16 or float16 (got ", type_name(dtype), ")");
  const c10::DeviceGuard guard(codes.device());
  const Packed p(codes, scales, rows, cols, codes.device());
  Tensor weight = at::empty({rows, cols}, codes.options().dtype(dtype));
  if (rows == 0) return weight;
  check_rc(gf_q4_dequantize(dtype_of(weight), rows, cols, p.codes.data_ptr(), p.scales.data_ptr(), weight.data_ptr(), stream_of(codes)),
           "gf_q4_dequantize");
  return weight;
}

struct Q4Call {
  Packed w;
  gf_q4_args a{};
  Q4Call(const Tensor& like, const Tensor& codes, const Tensor& scales, int64_t out, int64_t cols, int64_t rows, int64_t activation)
      : w(codes, scales, out, cols, like.device()) {
    a.dtype = dtype_of(like), a.activation = (int32_t)activation;
    a.rows = rows, a.in_features = cols, a.out_features = out / (activation == GF_ACT_NONE ? 1 : 2);
    a.codes = w.codes.data_ptr(), a.scales = w.scales.data_ptr();
  }
  void run(bool backward, const Tensor& like) {
    const size_t bytes = gf_q4_workspace_bytes(&a, backward);
    Tensor workspace;
    if (bytes) workspace = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
    void* const p = bytes ? workspace.data_ptr() : nullptr;
    if (backward)
      check_rc(gf_q4_backward(&a, p, bytes, stream_of(like)), "gf_q4_backward");
    else
      check_rc(gf_q4_forward(&a, p, bytes, stream_of(like)), "gf_q4_forward");
  }
};

void check_q4(const Tensor& x, const MaybeTensor& bias, const MaybeTensor& residual, int64_t rows, int64_t cols, int64_t activation) {
  check_first(x);
  TORCH_CHECK(x.dim() >= 1, "x must have shape [..., in_features]");
  TORCH_CHECK(cols > 0 && rows > 0, "weight must not be empty");
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
}

// y, and what the backward needs of a gated product (undefined for a linear one or if not to be saved)
std::tuple<Tensor, Tensor> q4_forward(const Tensor& x, const Tensor& codes, const Tensor& scales, const MaybeTensor& bias, const MaybeTensor& residual,
                                      int64_t rows, int64_t cols, int64_t activation, bool save) {
  check_q4(x, bias, residual, rows, cols, activation);
  const c10::DeviceGuard guard(x.device());
  const Rows r(x);
  Q4Call c(x, codes, scales, rows, cols, r.rows, activation);
  auto shape = x.sizes().vec();
  shape.back() = c.a.out_features;
  Tensor y = at::empty(shape, x.options()), saved, b;
  save = save && activation != GF_ACT_NONE;
  if (save) saved = at::empty({r.rows ? (int64_t)gf_q4_saved_bytes(&c.a) : 0}, x.options().dtype(at::kByte));
  if (r.rows == 0) return {y, saved};
  c.a.x = r.data(), c.a.ldx = r.ld, c.a.y = y.data_ptr();
  if (save) c.a.saved = saved.data_ptr();
  if (present(bias)) b = bias->contiguous(), c.a.bias = b.data_ptr();
  std::optional<Rows> res;
  if (present(residual)) res.emplace(*residual), c.a.residual = res->data(), c.a.ldr = res->ld;
  c.run(false, x);
  return {y, saved};
}

// The gradients of x and bias that are wanted.
std::tuple<Tensor, Tensor> q4_backward(const Tensor& dy, const Tensor& codes, const Tensor& scales, const MaybeTensor& saved, int64_t rows, int64_t cols,
                                       int64_t activation, bool want_x, bool want_b) {
  check_first(dy);
  TORCH_CHECK(dy.dim() >= 1, "dy must have at least one dimension");
  const c10::DeviceGuard guard(dy.device());
  TORCH_CHECK(rows > 0 && dy.size(-1) == rows / (activation == GF_ACT_NONE ? 1 : 2), "dy has ", dy.size(-1), " features, weight ", rows, " rows");
  const Rows g(dy);
  Q4Call c(dy, codes, scales, rows, cols, g.rows, activation);
  auto shape = dy.sizes().vec();
  shape.back() = cols;
  auto make = [&](at::IntArrayRef s) { return g.rows ? at::empty(s, dy.options()) : at::zeros(s, dy.options()); };
  Tensor dx, db;
  if (want_x) dx = make(shape);
  if (want_b) db = make({rows});
  if (g.rows == 0 || !(want_x || want_b)) return {dx, db};
  c.a.dy = g.data(), c.a.lddy = g.ld;
  if (activation != GF_ACT_NONE) {
    TORCH_CHECK(present(saved) && saved->is_cuda() && saved->is_contiguous() && saved->nbytes() >= gf_q4_saved_bytes(&c.a),
                "saved must be what the forward with save=True returned");
    c.a.saved = saved->data_ptr();
  }
  if (want_x) c.a.dx = dx.data_ptr();
  if (want_b) c.a.dbias = db.data_ptr();
  c.run(true, dy);
  return {dx, db};
}

std::tuple<Tensor, Tensor> call_q4_forward(const Tensor& x, const Tensor& codes, const Tensor& scales, const MaybeTensor& bias,
                                           const MaybeTensor& residual, int64_t rows, int64_t cols, int64_t activation, bool save) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("guass_amd::q4_forward", "").typed<decltype(q4_forward)>();
  return op.call(x, codes, scales, bias, residual, rows, cols, activation, save);
}

std::tuple<Tensor, Tensor> call_q4_backward(const Tensor& dy, const Tensor& codes, const Tensor& scales, const MaybeTensor& saved, int64_t rows, int64_t cols,
                                            int64_t activation, bool want_x, bool want_b) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("guass_amd::q4_backward", "").typed<decltype(q4_backward)>();
  return op.call(dy, codes, scales, saved, rows, cols, activation, want_x, want_b);
}

const char* q4_name(int64_t activation) { return activation == GF_ACT_NONE ? "quantized_linear" : "quantized_gated_linear"; }

struct Q4Linear : torch::autograd::Function<Q4Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& codes, const Tensor& scales, const MaybeTensor& bias,
                        const MaybeTensor& residual, int64_t rows, int64_t cols, int64_t activation) {
    auto [y, saved] = call_q4_forward(x, codes, scales, bias, residual, rows, cols, activation, wants(x) || wants(bias));
    ctx->save_for_backward({codes, scales, saved});
    ctx->saved_data["call"] = std::make_tuple(rows, cols, activation, present(bias), present(residual), wants(x) || wants(bias));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto [rows, cols, activation, has_bias, has_residual, trains] =
        ctx->saved_data["call"].to<std::tuple<int64_t, int64_t, int64_t, bool, bool, bool>>();
    // edges are the tensors that are there: x, codes, scales, bias, residual
    const bool wx = ctx->needs_input_grad(0), wb = has_bias && ctx->needs_input_grad(3), wr = has_residual && ctx->needs_input_grad(3 + has_bias);
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    // what the gradients depend on: of a gated product x and bias too, by value and gate
    const bool again = dy.requires_grad() || (activation != GF_ACT_NONE && trains);
    auto [dx, db] = call_q4_backward(dy, saved[0], saved[1], maybe(saved[2]), rows, cols, activation, wx, wb);
    variable_list out = once({dx, Tensor(), Tensor(), db, Tensor(), Tensor(), Tensor(), Tensor()}, q4_name(activation), again);
    if (wr) out[4] = dy;
    return out;
  }
};

Tensor q4_linear(const Tensor& x, const Tensor& codes, const Tensor& scales, const MaybeTensor& bias, const MaybeTensor& residual, int64_t rows, int64_t cols,
                 int64_t activation) {
  check_q4(x, bias, residual, rows, cols, activation);
  check_no_tangent(q4_name(activation), x, bias, residual);
  if (at::GradMode::is_enabled() && (wants(x) || wants(bias) || wants(residual)))
    return Q4Linear::apply(x, codes, scales, bias, residual, rows, cols, activation);
  return std::get<0>(call_q4_forward(x, codes, scales, bias, residual, rows, cols, activation, false));
}

// As torch's linear: x and bias in autocast's type, and a residual of another type added by torch's rules.
Tensor q4_linear_autocast(const Tensor& x, const Tensor& codes, const Tensor& scales, const MaybeTensor& bias, const MaybeTensor& residual,
                          int64_t rows, int64_t cols, int64_t activation) {
  const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
  const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
  auto cast = [&](const Tensor& t) { return at::autocast::cached_cast(type, t, at::kCUDA); };
  const bool fused = !present(residual) || residual->scalar_type() == type;
  const Tensor y = q4_linear(cast(x), codes, scales, present(bias) ? MaybeTensor(cast(*bias)) : bias, fused ? residual : MaybeTensor(), rows, cols, activation);
  return fused ? y : *residual + y;
}

}  // namespace

TORCH_LIBRARY_IMPL(guass_amd, Autocast, m) {
  m.impl("block_norm", block_norm_autocast);
  m.impl("q4_linear", q4_linear_autocast);
}

#define NORM_SCHEMA                                                                                                                    \
  "Tensor x, Tensor? residual, Tensor? weight, Tensor? bias, Tensor? gate, float gate_value, float residual_scale, int kind, float eps, " \
  "Tensor? next_weight, Tensor? next_bias, Tensor? scale, Tensor? shift, int next_kind, float next_eps"

TORCH_LIBRARY_FRAGMENT(guass_amd, m) {
  // what a user calls: checks and autograd around the operators below
  m.def("block_norm(" NORM_SCHEMA ") -> (Tensor, Tensor)", block_norm);
  m.def("q4_linear(Tensor x, Tensor codes, Tensor scales, Tensor? bias, Tensor? residual, int rows, int cols, int activation) -> Tensor", q4_linear);
  // the launches by themselves, without autograd: what a HIP graph captures, and what a trace (torch.compile) holds
  m.def("block_norm_forward(" NORM_SCHEMA ", bool want_stream) -> (Tensor, Tensor)");
  m.def("block_norm_backward(" NORM_SCHEMA ", Tensor? dstream, Tensor? dnormed, int wants) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, "
        "Tensor, Tensor)");
  m.def("q4_quantize(Tensor weight) -> (Tensor, Tensor)");
  m.def("q4_dequantize(Tensor codes, Tensor scales, int rows, int cols, ScalarType dtype) -> Tensor");
  m.def("q4_forward(Tensor x, Tensor codes, Tensor scales, Tensor? bias, Tensor? residual, int rows, int cols, int activation, bool save) -> (Tensor, Tensor)");
  m.def("q4_backward(Tensor dy, Tensor codes, Tensor scales, Tensor? saved, int rows, int cols, int activation, bool want_x, bool want_b) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(guass_amd, CUDA, m) {
  m.impl("block_norm_forward", block_norm_forward);
  m.impl("block_norm_backward", block_norm_backward);
  m.impl("q4_quantize", q4_quantize);
  m.impl("q4_dequantize", q4_dequantize);
  m.impl("q4_forward", q4_forward);
  m.impl("q4_backward", q4_backward);
}

TORCH_LIBRARY_IMPL(guass_amd, Autograd, m) {
  for (const char* name : {"block_norm_forward", "block_norm_backward", "q4_forward", "q4_backward"}) m.impl(name, torch::CppFunction::makeFallthrough());
}
