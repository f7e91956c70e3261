// norms.hip - gfx950 kernels and C ABI of what stands before and after a block: its norm (modulated by a sample's scale and
// shift), and the way back into the stream with a gate and the residual's scale, each alone or both in one pass.
//
//   k_norm_forward   s = rho r + g (n(x) w + b), h = (n'(s) w' + b')(1 + scale) + shift; either half alone
//   k_norm_backward  the rows' gradients, and per chunk of rows the column sums that the parameters' come from
//   k_norm_finish    the chunks' sums into the parameters' gradients
//   k_norm_join      those of several slabs of groups added
//
// A row is read once into registers, its statistics and all that follows are computed there in 32 bits, and each output is rounded
// once: a fused pass gives h of the unrounded s.  Nothing is kept for the backward but the inputs: it makes s and both statistics
// again from what it reads anyway.  No atomics: every sum has one order.
#include "elements.h"

namespace {

// What the kernels read and write; a matrix as in gf_norm_args.
template <typename T>
struct Norms {
  int64_t rows, group_rows;
  int32_t cols, kind, next_kind;
  float eps, next_eps, gate_value, residual_scale, inverse;  // inverse: 1 / cols
  const T *x, *residual, *weight, *bias, *gate, *next_weight, *next_bias, *scale, *shift;
  int64_t ldx, ldr, ld_gate, ld_scale, ld_shift;
  T *stream, *normed;
  const T *dstream, *dnormed;
  int64_t ld_dstream, ld_dnormed;
  T *dx, *dresidual, *dweight, *dbias, *dgate, *dnext_weight, *dnext_bias, *dscale, *dshift;
};

// The sum of v over the L lanes of a row.  Past a wave the waves' sums meet in LDS: `slot` alternates between two places, so that
// one barrier a sum is enough (whoever writes a place again has passed the next sum's barrier, as have all that read it).
template <int L>
struct Sum {
  float (*part)[L > 64 ? L / 64 : 1];
  int slot = 0;
  __device__ float operator()(float v) {
#pragma unroll
    for (int i = (L < 64 ? L : 64) / 2; i > 0; i /= 2) v += __shfl_xor(v, i);
    if constexpr (L > 64) {
      if ((threadIdx.x & 63) == 0) part[slot][threadIdx.x / 64] = v;
      __syncthreads();
      v = 0.0f;
#pragma unroll
      for (int i = 0; i < L / 64; ++i) v += part[slot][i];
      slot ^= 1;
    }
    return v;
  }
};

// A row of L lanes: lane `lane` holds the groups of 8 columns (g L + lane).  Elements past the row are zero.
template <int L, int G>
struct Place {
  int lane, cols;
  __device__ int col(int g) const { return (g * L + lane) * 8; }
  __device__ int count(int g) const {
    const int n = cols - col(g);
    return n < 0 ? 0 : n < 8 ? n : 8;
  }
  template <typename T>
  __device__ void load(float v[G][8], const T* row) const {
#pragma unroll
    for (int g = 0; g < G; ++g) load8(v[g], row + col(g), count(g) == 8, count(g));
  }
  template <typename T>
  __device__ void store(T* row, const float v[G][8]) const {
#pragma unroll
    for (int g = 0; g < G; ++g) store8(row + col(g), v[g], count(g) == 8, count(g));
  }
  // v times (plus) a vector of parameters
  template <typename T, typename F>
  __device__ void apply(float v[G][8], const T* p, F f) const {
    if (p == nullptr) return;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float w[8];
      load8(w, p + col(g), count(g) == 8, count(g));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[g][j] = f(v[g][j], w[j]);
    }
  }
};

// x becomes n(x), zero past the row; returns 1 / deviation (rms: 1 / root mean square).  The mean first, then the squares of what is
// left: both from registers, so nothing cancels.
template <int L, int G>
__device__ inline float normalise(float x[G][8], int kind, float eps, float inverse, const Place<L, G>& at, Sum<L>& sum) {
  float v = 0.0f;
  if (kind == GF_NORM_LAYER) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) v += x[g][j];
    const float mean = sum(v) / (float)at.cols;  // a row of one value has that mean
    v = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int n = at.count(g);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[g][j] -= mean;
      if (n < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j >= n) x[g][j] = 0.0f;
      }
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < 8; ++j) v = __builtin_fmaf(x[g][j], x[g][j], v);
  const float rstd = 1.0f / sqrtf(__builtin_fmaf(sum(v), inverse, eps));
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < 8; ++j) x[g][j] *= rstd;
  return rstd;
}

// The gradient of x from that of n(x), in place: rstd (g - mean g - n(x) mean(g n(x))), without mean g for rms; zero past the row.
template <int L, int G>
__device__ inline void through_norm(float g_[G][8], const float n_[G][8], int kind, float rstd, float inverse, const Place<L, G>& at,
                                    Sum<L>& sum) {
  float a = 0.0f, b = 0.0f;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < 8; ++j) a += g_[g][j], b = __builtin_fmaf(g_[g][j], n_[g][j], b);
  a = kind == GF_NORM_LAYER ? sum(a) * inverse : 0.0f;
  b = sum(b) * inverse;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int n = at.count(g);
#pragma unroll
    for (int j = 0; j < 8; ++j) g_[g][j] = rstd * (g_[g][j] - __builtin_fmaf(n_[g][j], b, a));
    if (n < 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j >= n) g_[g][j] = 0.0f;
    }
  }
}

constexpr auto kTimes = [](float v, float w) { return v * w; };
constexpr auto kPlus = [](float v, float w) { return v + w; };
constexpr auto kTimesOnePlus = [](float v, float w) { return __builtin_fmaf(v, w, v); };

// v (n(x), or x itself) becomes g (v w + b).
template <typename T, int L, int G>
__device__ inline void branch(const Norms<T>& a, const Place<L, G>& at, float v[G][8], int64_t group) {
  at.apply(v, a.weight, kTimes);
  at.apply(v, a.bias, kPlus);
  if (a.gate != nullptr) {
    at.apply(v, a.gate + group * a.ld_gate, kTimes);
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[g][j] *= a.gate_value;
  }
}

// The gradient of g (v w + b), in place, into that of v.
template <typename T, int L, int G>
__device__ inline void through_branch(const Norms<T>& a, const Place<L, G>& at, float v[G][8], int64_t group) {
  at.apply(v, a.weight, kTimes);
  if (a.gate != nullptr) {
    at.apply(v, a.gate + group * a.ld_gate, kTimes);
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[g][j] *= a.gate_value;
  }
}

// Forward, L lanes a row.  BRANCH: s from x and the residual; NEXT: h from s (without BRANCH, from x).
template <typename T, int L, int G, bool BRANCH, bool NEXT>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_norm_forward(Norms<T> a) {
  constexpr int kAtOnce = L < 256 ? 256 / L : 1;
  __shared__ float part[2][L > 64 ? L / 64 : 1];
  Sum<L> sum{part};
  const Place<L, G> at{(int)threadIdx.x % L, a.cols};
  for (int64_t row = (int64_t)blockIdx.x * kAtOnce + threadIdx.x / L; row < a.rows; row += (int64_t)gridDim.x * kAtOnce) {
    const int64_t group = (uint32_t)row / (uint32_t)a.group_rows;
    float v[G][8];
    at.load(v, a.x + row * a.ldx);
    if constexpr (BRANCH) {
      float r[G][8];
      at.load(r, a.residual + row * a.ldr);
      if (a.kind != GF_NORM_NONE) normalise<L, G>(v, a.kind, a.eps, a.inverse, at, sum);
      branch(a, at, v, group);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[g][j] = __builtin_fmaf(a.residual_scale, r[g][j], v[g][j]);
      if (a.stream != nullptr) at.store(a.stream + row * a.cols, v);
    }
    if constexpr (NEXT) {
      normalise<L, G>(v, a.next_kind, a.next_eps, a.inverse, at, sum);
      at.apply(v, a.next_weight, kTimes);
      at.apply(v, a.next_bias, kPlus);
      if (a.scale != nullptr) at.apply(v, a.scale + group * a.ld_scale, kTimesOnePlus);
      if (a.shift != nullptr) at.apply(v, a.shift + group * a.ld_shift, kPlus);
      at.store(a.normed + row * a.cols, v);
    }
  }
}

// Column sums of a chunk of rows, per element: of ds, ds n(x), dh, dh n'(s).
constexpr int kSums = 4;

// Backward, by chunks of rows of one group each (`chunks` a group, `all` together).  SUMS: the column sums too, into parts [chunk][kSums][width].
template <typename T, int L, int G, bool BRANCH, bool NEXT, bool SUMS>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_norm_backward(Norms<T> a, int64_t chunk_rows, int64_t chunks, int64_t all, float* parts,
                                                                      int64_t width) {
  constexpr int kAtOnce = L < 256 ? 256 / L : 1;
  __shared__ float part[2][L > 64 ? L / 64 : 1];
  __shared__ float meet[SUMS && kAtOnce > 1 ? kAtOnce : 1][SUMS && kAtOnce > 1 ? L * G * 8 : 1];
  Sum<L> sum{part};
  const int sub = threadIdx.x / L;
  const Place<L, G> at{(int)threadIdx.x % L, a.cols};
  for (int64_t chunk = blockIdx.x; chunk < all; chunk += gridDim.x) {
    const int64_t group = chunk / chunks, first = (chunk % chunks) * chunk_rows;
    const int64_t begin = group * a.group_rows + first;
    const int64_t end = group * a.group_rows + (first + chunk_rows < a.group_rows ? first + chunk_rows : a.group_rows);
    float sums[SUMS ? kSums : 1][G][8] = {};
    auto add = [&](int k, const float d[G][8], const float n[G][8]) {
      if constexpr (SUMS) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int j = 0; j < 8; ++j) sums[k][g][j] += d[g][j], sums[k + 1][g][j] = __builtin_fmaf(d[g][j], n[g][j], sums[k + 1][g][j]);
      }
    };
    for (int64_t row = begin + sub; row < end; row += kAtOnce) {
      float x[G][8], d[G][8];
      if (NEXT || SUMS || a.kind != GF_NORM_NONE) at.load(x, a.x + row * a.ldx);
      float rstd = 1.0f;
      if constexpr (BRANCH && !NEXT) {
        at.load(d, a.dstream + row * a.ld_dstream);
        if (a.kind != GF_NORM_NONE) rstd = normalise<L, G>(x, a.kind, a.eps, a.inverse, at, sum);
      }
      if constexpr (NEXT) {
        at.load(d, a.dnormed + row * a.ld_dnormed);
        float s[BRANCH ? G : 1][8], ds[BRANCH ? G : 1][8];
        if constexpr (BRANCH) {
          float r[G][8];
          at.load(r, a.residual + row * a.ldr);
          if (a.dstream != nullptr) at.load(ds, a.dstream + row * a.ld_dstream);
          if (a.kind != GF_NORM_NONE) rstd = normalise<L, G>(x, a.kind, a.eps, a.inverse, at, sum);
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[g][j] = x[g][j];
          branch(a, at, s, group);
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[g][j] = __builtin_fmaf(a.residual_scale, r[g][j], s[g][j]);
        }
        float(*n)[8] = BRANCH ? s : x;
        const float next_rstd = normalise<L, G>(n, a.next_kind, a.next_eps, a.inverse, at, sum);
        add(2, d, n);
        at.apply(d, a.next_weight, kTimes);
        if (a.scale != nullptr) at.apply(d, a.scale + group * a.ld_scale, kTimesOnePlus);
        through_norm<L, G>(d, n, a.next_kind, next_rstd, a.inverse, at, sum);
        if constexpr (BRANCH) {
          if (a.dstream != nullptr) {
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
              for (int j = 0; j < 8; ++j) d[g][j] += ds[g][j];
          }
        }
      }
      if constexpr (BRANCH) {
        add(0, d, x);
        if (a.dresidual != nullptr) {
          float t[G][8];
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 8; ++j) t[g][j] = a.residual_scale * d[g][j];
          at.store(a.dresidual + row * a.cols, t);
        }
        if (a.dx != nullptr) {
          through_branch(a, at, d, group);
          if (a.kind != GF_NORM_NONE) through_norm<L, G>(d, x, a.kind, rstd, a.inverse, at, sum);
        }
      }
      if (a.dx != nullptr) at.store(a.dx + row * a.cols, d);
    }
    if constexpr (SUMS) {
#pragma unroll
      for (int k = BRANCH ? 0 : 2; k < (NEXT ? kSums : 2); ++k) {
        float* const out = parts + ((int64_t)chunk * kSums + k) * width;
        if constexpr (kAtOnce == 1) {
          for (int g = 0; g < G; ++g)
            if (at.count(g) > 0) store8(out + at.col(g), sums[k][g], true, 8);
        } else {
          __syncthreads();
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 8; ++j) meet[sub][at.col(g) + j] = sums[k][g][j];
          __syncthreads();
          for (int c = threadIdx.x; c < a.cols; c += 256) {
            float v = meet[0][c];
#pragma unroll
            for (int i = 1; i < kAtOnce; ++i) v += meet[i][c];
            out[c] = v;
          }
        }
      }
    }
  }
}

// The chunks' sums into gradients: 32 columns a workgroup, the branch's (z = 0) or the next norm's.  With S0 = sum d, S1 = sum d n of a
// group, w, b the half's weight and bias and f its factor (the gate; 1 + scale):
//   of the factor  w S1 + b S0;   of the shift  S0;   of w  sum over groups of f S1;   of b  sum over groups of f S0.
// 32 half-waves share out the groups, several of them one group where there are fewer; a slab (y) is a range of groups, and what is shared
// by all groups goes to `partial` [slab][half][4][width] (of the weight, the bias, the factor, the shift) where there are several slabs.
template <typename T>
struct Half {
  const T *weight, *bias, *factor;
  int64_t ld_factor, ld_shift;
  float one, value;  // the factor is one + factor[], or `value`
  T *dweight, *dbias, *dfactor, *dshift;
};

template <typename T>
__global__ __launch_bounds__(1024) void k_norm_finish(Half<T> branch, Half<T> next, int half0, int32_t cols, int64_t groups, int64_t chunks,
                                                      const float* parts, int64_t width, int team, float* partial) {
  __shared__ float meet[4][32][32];
  const int lane = threadIdx.x & 31, member = threadIdx.x >> 5, half = half0 + blockIdx.z;
  const Half<T>& h = half == 0 ? branch : next;
  const int64_t c = blockIdx.x * 32ll + lane;
  const bool in = c < cols;
  const int64_t slab = (groups + gridDim.y - 1) / gridDim.y, g0 = blockIdx.y * slab, g1 = g0 + slab < groups ? g0 + slab : groups;
  const int teams = 32 / team, of = member % team;
  const float w = in && h.weight != nullptr ? (float)h.weight[c] : 1.0f, b = in && h.bias != nullptr ? (float)h.bias[c] : 0.0f;
  float dw = 0.0f, db = 0.0f, df = 0.0f, dsh = 0.0f;
  for (int64_t base = g0; base < g1; base += teams) {
    const int64_t g = base + member / team;
    float s0 = 0.0f, s1 = 0.0f;
    if (in && g < g1) {
#pragma unroll 4
      for (int64_t i = of; i < chunks; i += team) {
        const float* p = parts + ((g * chunks + i) * kSums + 2 * half) * width + c;
        s0 += p[0], s1 += p[width];
      }
    }
    if (team > 1) {
      __syncthreads();
      meet[0][member][lane] = s0, meet[1][member][lane] = s1;
      __syncthreads();
      if (of == 0) {
        for (int i = 1; i < team; ++i) s0 += meet[0][member + i][lane], s1 += meet[1][member + i][lane];
      }
    }
    if (in && g < g1 && of == 0) {
      const float f = h.factor != nullptr ? h.one + (float)h.factor[g * h.ld_factor + c] : h.value;
      dw = __builtin_fmaf(f, s1, dw), db = __builtin_fmaf(f, s0, db);
      const float own = __builtin_fmaf(w, s1, b * s0);
      if (h.dfactor != nullptr) {
        if (h.ld_factor != 0) h.dfactor[g * cols + c] = (T)own;
        else df += own;
      }
      if (h.dshift != nullptr) {
        if (h.ld_shift != 0) h.dshift[g * cols + c] = (T)s0;
        else dsh += s0;
      }
    }
  }
  __syncthreads();
  meet[0][member][lane] = dw, meet[1][member][lane] = db, meet[2][member][lane] = df, meet[3][member][lane] = dsh;
  __syncthreads();
  if (member >= 4 || !in) return;
  float v = 0.0f;
  for (int i = 0; i < 32; i += team) v += meet[member][i][lane];
  if (partial != nullptr) {
    partial[((int64_t)blockIdx.y * 2 + half) * 4 * width + member * width + c] = v;
    return;
  }
  T* const out = member == 0 ? h.dweight : member == 1 ? h.dbias : member == 2 ? (h.ld_factor == 0 ? h.dfactor : nullptr) : h.ld_shift == 0 ? h.dshift : nullptr;
  if (out != nullptr) out[c] = (T)v;
}

template <typename T>
__global__ __launch_bounds__(256) void k_norm_join(Half<T> branch, Half<T> next, int half0, int32_t cols, int64_t slabs, const float* partial,
                                                   int64_t width) {
  const int half = half0 + blockIdx.z, which = blockIdx.y;
  const Half<T>& h = half == 0 ? branch : next;
  const int64_t c = blockIdx.x * 256ll + threadIdx.x;
  T* const out = which == 0 ? h.dweight : which == 1 ? h.dbias : which == 2 ? (h.ld_factor == 0 ? h.dfactor : nullptr) : h.ld_shift == 0 ? h.dshift : nullptr;
  if (c >= cols || out == nullptr) return;
  float v = 0.0f;
#pragma unroll 4
  for (int64_t i = 0; i < slabs; ++i) v += partial[(i * 2 + half) * 4 * width + which * width + c];
  out[c] = (T)v;
}

// ------------------------------------------------------------------------------------------
// Host.

constexpr int kMaxCols = 16384;

int check_args(const gf_norm_args* a) {
  if (a == nullptr) return fail(GF_E_INVALID_ARGUMENT, "args must not be NULL");
  GF_TRY(check_dtype(a->dtype));
  for (const int32_t kind : {a->kind, a->next_kind})
    if (kind < GF_NORM_NONE || kind > GF_NORM_RMS) return fail(GF_E_INVALID_ARGUMENT, "unknown norm %d", (int)kind);
  if (a->rows < 0 || a->rows > kMaxSize) return fail(GF_E_INVALID_ARGUMENT, "rows negative or too large");
  if (a->cols < 1 || a->cols > kMaxCols) return fail(GF_E_INVALID_ARGUMENT, "cols must lie in [1, %d] (got %lld)", kMaxCols, (long long)a->cols);
  if (a->group_rows < 1 || a->rows % a->group_rows != 0) return fail(GF_E_INVALID_ARGUMENT, "group_rows must divide rows");
  for (const double eps : {a->eps, a->next_eps})
    if (!(eps >= 0.0 && eps <= 1e30)) return fail(GF_E_INVALID_ARGUMENT, "eps must be finite and not negative");
  if (a->residual == nullptr && (a->kind != GF_NORM_NONE || a->gate != nullptr || a->next_kind == GF_NORM_NONE))
    return fail(GF_E_INVALID_ARGUMENT, "without a residual there is the next norm only");
  if (a->kind == GF_NORM_NONE && (a->weight != nullptr || a->bias != nullptr))
    return fail(GF_E_INVALID_ARGUMENT, "a branch without a norm takes no weight or bias");
  if (a->next_kind == GF_NORM_NONE && (a->next_weight != nullptr || a->next_bias != nullptr || a->scale != nullptr || a->shift != nullptr))
    return fail(GF_E_INVALID_ARGUMENT, "without a next norm there is no weight, bias, scale or shift of it");
  return GF_OK;
}

int check_inputs(const gf_norm_args& a) {
  const int size = size_of(a.dtype);
  const int64_t groups = a.rows / a.group_rows;
  GF_TRY(check_matrix("x", a.x, a.rows, a.ldx, a.cols, size));
  if (a.residual != nullptr) GF_TRY(check_matrix("residual", a.residual, a.rows, a.ldr, a.cols, size));
  const struct { const char* name; const void* p; int64_t ld; } shared[] = {{"gate", a.gate, a.ld_gate}, {"scale", a.scale, a.ld_scale}, {"shift", a.shift, a.ld_shift}};
  for (const auto& m : shared)
    if (m.p != nullptr) GF_TRY(check_matrix(m.name, m.p, m.ld == 0 ? 1 : groups, m.ld == 0 ? a.cols : m.ld, a.cols, size));
  const struct { const char* name; const void* p; } vectors[] = {
      {"weight", a.weight}, {"bias", a.bias}, {"next_weight", a.next_weight}, {"next_bias", a.next_bias}};
  for (const auto& v : vectors)
    if (v.p != nullptr) GF_TRY(check_matrix(v.name, v.p, 1, a.cols, a.cols, size));
  return GF_OK;
}

template <typename T>
Norms<T> make_norms(const gf_norm_args& a) {
  Norms<T> n{};
  n.rows = a.rows, n.group_rows = a.group_rows, n.cols = (int32_t)a.cols, n.kind = a.kind, n.next_kind = a.next_kind;
  n.eps = (float)a.eps, n.next_eps = (float)a.next_eps, n.gate_value = (float)a.gate_value, n.residual_scale = (float)a.residual_scale;
  n.inverse = (float)(1.0 / (double)a.cols);
  n.x = (const T*)a.x, n.residual = (const T*)a.residual, n.weight = (const T*)a.weight, n.bias = (const T*)a.bias, n.gate = (const T*)a.gate;
  n.next_weight = (const T*)a.next_weight, n.next_bias = (const T*)a.next_bias, n.scale = (const T*)a.scale, n.shift = (const T*)a.shift;
  n.ldx = a.ldx, n.ldr = a.ldr, n.ld_gate = a.ld_gate, n.ld_scale = a.ld_scale, n.ld_shift = a.ld_shift;
  n.stream = (T*)a.stream, n.normed = (T*)a.normed;
  n.dstream = (const T*)a.dstream, n.dnormed = (const T*)a.dnormed, n.ld_dstream = a.ld_dstream, n.ld_dnormed = a.ld_dnormed;
  n.dx = (T*)a.dx, n.dresidual = (T*)a.dresidual, n.dweight = (T*)a.dweight, n.dbias = (T*)a.dbias, n.dgate = (T*)a.dgate;
  n.dnext_weight = (T*)a.dnext_weight, n.dnext_bias = (T*)a.dnext_bias, n.dscale = (T*)a.dscale, n.dshift = (T*)a.dshift;
  return n;
}

template <int L, int G>
struct Lanes {
  static constexpr int lanes = L, groups = G;
};

// How many lanes take a row, and how many groups of 8 columns each.
template <typename F>
int with_lanes(int64_t cols, F f) {
  if (cols <= 128) return f(Lanes<16, 1>());
  if (cols <= 512) return f(Lanes<64, 1>());
  if (cols <= 1024) return f(Lanes<64, 2>());
  if (cols <= 1536) return f(Lanes<64, 3>());
  if (cols <= 2048) return f(Lanes<256, 1>());
  if (cols <= 4096) return f(Lanes<256, 2>());
  if (cols <= 6144) return f(Lanes<256, 3>());
  return f(Lanes<1024, 2>());
}

template <typename F>
int with_halves(const gf_norm_args& a, F f) {
  using Yes = std::true_type;
  using No = std::false_type;
  if (a.residual == nullptr) return f(No(), Yes());
  return a.next_kind == GF_NORM_NONE ? f(Yes(), No()) : f(Yes(), Yes());
}

bool wants_sums(const gf_norm_args& a) {
  return a.dweight || a.dbias || a.dgate || a.dnext_weight || a.dnext_bias || a.dscale || a.dshift;
}

int backward(const gf_norm_args& a, Arena& ws, bool run, hipStream_t s) {
  const int64_t groups = a.rows / a.group_rows, width = round_up(a.cols, 8);
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_lanes(a.cols, [&](auto lanes) {
      constexpr int L = lanes.lanes, G = lanes.groups, kThreads = L < 256 ? 256 : L, kAtOnce = kThreads / L;
      return with_halves(a, [&](auto branch, auto next) {
        constexpr bool kBranch = branch.value, kNext = next.value;
        const bool sums = wants_sums(a);
        const int64_t want = std::max<int64_t>((sums ? 512 : 4096) / groups, 1);
        const int64_t cut = std::min(want, (a.group_rows + kAtOnce - 1) / kAtOnce), chunk_rows = (a.group_rows + cut - 1) / cut;
        const int64_t chunks = (a.group_rows + chunk_rows - 1) / chunk_rows, all = groups * chunks;
        const int64_t slabs = groups <= 256 ? 1 : std::min<int64_t>((groups + 127) / 128, 64);
        float* const parts = sums ? (float*)ws.take(all * kSums * width * 4) : nullptr;
        float* const partial = sums && slabs > 1 ? (float*)ws.take(slabs * 8 * width * 4) : nullptr;
        GF_RUN {
          const Norms<T> n = make_norms<T>(a);
          const unsigned grid = (unsigned)std::min<int64_t>(all, 1 << 20);
          if (sums)
            k_norm_backward<T, L, G, kBranch, kNext, true><<<grid, kThreads, 0, s>>>(n, chunk_rows, chunks, all, parts, width);
          else
            k_norm_backward<T, L, G, kBranch, kNext, false><<<grid, kThreads, 0, s>>>(n, chunk_rows, chunks, all, nullptr, 0);
          GF_LAUNCH_CHECK("k_norm_backward");
          if (sums) {
            const Half<T> b{n.weight, n.bias, n.gate, n.ld_gate, 0, 0.0f, n.gate_value, n.dweight, n.dbias, n.dgate, nullptr};
            const Half<T> f{n.next_weight, n.next_bias, n.scale, n.ld_scale, n.ld_shift, 1.0f, 1.0f, n.dnext_weight, n.dnext_bias, n.dscale, n.dshift};
            int team = 1;
            while (team < 32 && team * 2 * groups <= 32) team *= 2;
            const int half0 = kBranch ? 0 : 1, halves = (kBranch ? 1 : 0) + (kNext ? 1 : 0);
            k_norm_finish<T><<<dim3((unsigned)((a.cols + 31) / 32), (unsigned)slabs, halves), 1024, 0, s>>>(b, f, half0, n.cols, groups, chunks, parts,
                                                                                                         width, team, partial);
            GF_LAUNCH_CHECK("k_norm_finish");
            if (partial != nullptr) {
              k_norm_join<T><<<dim3((unsigned)((a.cols + 255) / 256), 4, halves), 256, 0, s>>>(b, f, half0, n.cols, slabs, partial, width);
              GF_LAUNCH_CHECK("k_norm_join");
            }
          }
        }
        return (int)GF_OK;
      });
    });
  });
}

}  // namespace

extern "C" {

int gf_norm_forward(const gf_norm_args* args, void* stream) {
  GF_TRY(check_args(args));
  const gf_norm_args& a = *args;
  if (a.rows == 0) return GF_OK;
  GF_TRY(check_inputs(a));
  const int size = size_of(a.dtype);
  if (a.residual == nullptr && a.stream != nullptr) return fail(GF_E_INVALID_ARGUMENT, "a norm alone has no stream to write");
  if (a.stream != nullptr) GF_TRY(check_matrix("stream", a.stream, a.rows, a.cols, a.cols, size));
  if (a.next_kind != GF_NORM_NONE)
    GF_TRY(check_matrix("normed", a.normed, a.rows, a.cols, a.cols, size));
  else if (a.stream == nullptr)
    return fail(GF_E_INVALID_ARGUMENT, "stream must not be NULL");
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_lanes(a.cols, [&](auto lanes) {
      constexpr int L = lanes.lanes, G = lanes.groups, kThreads = L < 256 ? 256 : L, kAtOnce = kThreads / L;
      return with_halves(a, [&](auto branch, auto next) {
        const unsigned grid = (unsigned)std::min<int64_t>((a.rows + kAtOnce - 1) / kAtOnce, 8192);
        k_norm_forward<T, L, G, branch.value, next.value><<<grid, kThreads, 0, (hipStream_t)stream>>>(make_norms<T>(a));
        GF_LAUNCH_CHECK("k_norm_forward");
        return (int)GF_OK;
      });
    });
  });
}

size_t gf_norm_workspace_bytes(const gf_norm_args* args) {
  if (check_args(args) != GF_OK || args->rows == 0) return 0;
  Arena count{nullptr};
  return backward(*args, count, false, nullptr) == GF_OK ? count.used : 0;
}

int gf_norm_backward(const gf_norm_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  GF_TRY(check_args(args));
  const gf_norm_args& a = *args;
  if (a.rows == 0) return fail(GF_E_INVALID_ARGUMENT, "a backward needs rows");
  GF_TRY(check_inputs(a));
  const int size = size_of(a.dtype);
  if (a.residual == nullptr) {
    if (a.dstream != nullptr || a.dresidual != nullptr || a.dweight != nullptr || a.dbias != nullptr || a.dgate != nullptr)
      return fail(GF_E_INVALID_ARGUMENT, "without a residual there is the next norm only");
  }
  if (a.next_kind != GF_NORM_NONE)
    GF_TRY(check_matrix("dnormed", a.dnormed, a.rows, a.ld_dnormed, a.cols, size));
  else if (a.dnext_weight != nullptr || a.dnext_bias != nullptr || a.dscale != nullptr || a.dshift != nullptr)
    return fail(GF_E_INVALID_ARGUMENT, "without a next norm there is no weight, bias, scale or shift of it");
  if (a.dstream != nullptr || a.next_kind == GF_NORM_NONE) GF_TRY(check_matrix("dstream", a.dstream, a.rows, a.ld_dstream, a.cols, size));
  const struct { const char* name; const void* p; const void* of; } grads[] = {
      {"dgate", a.dgate, a.gate}, {"dscale", a.dscale, a.scale}, {"dshift", a.dshift, a.shift}, {"dweight", a.dweight, a.weight},
      {"dbias", a.dbias, a.bias}, {"dnext_weight", a.dnext_weight, a.next_weight}, {"dnext_bias", a.dnext_bias, a.next_bias}};
  for (const auto& g : grads) {
    if (g.p != nullptr && g.of == nullptr) return fail(GF_E_INVALID_ARGUMENT, "%s without its parameter", g.name);
    if ((uintptr_t)g.p % size != 0) return fail(GF_E_INVALID_ARGUMENT, "%s is not aligned to its type", g.name);
  }
  if (a.dx != nullptr) GF_TRY(check_matrix("dx", a.dx, a.rows, a.cols, a.cols, size));
  if (a.dresidual != nullptr) GF_TRY(check_matrix("dresidual", a.dresidual, a.rows, a.cols, a.cols, size));
  Arena count{nullptr}, ws{(uint8_t*)workspace};
  GF_TRY(backward(a, count, false, nullptr));
  GF_TRY(check_workspace(count.used, workspace, workspace_bytes));
  return backward(a, ws, true, (hipStream_t)stream);
}

}  // extern "C"
