// feedforward.hip - gfx950 kernels and C ABI of the feed-forward block around the adapted linears:
// dropout from a counter, the gated projection and the projection back, each with its backward.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../include/gaussfield.h"
#include "error.h"

namespace {

using bf16 = __bf16;
using f16 = _Float16;

template <typename... A>
int fail(int code, const char* fmt, A... a) {
  char msg[512];
  snprintf(msg, sizeof(msg), fmt, a...);
  return gf_set_error(code, msg);
}
int fail(int code, const char* msg) { return gf_set_error(code, msg); }

#define FF_LAUNCH_CHECK(name)                                                                    \
  do {                                                                                           \
    hipError_t e_ = hipGetLastError();                                                           \
    if (e_ != hipSuccess) return fail(GF_E_HIP, "launch of %s failed: %s", name, hipGetErrorString(e_)); \
  } while (0)

// ------------------------------------------------------------------------------------------
// Dropout.

struct Drop {
  uint32_t threshold;  // round(p 2^16): half-words below it are dropped; 0: nothing is
  float scale;         // 2^16 / (2^16 - threshold)
  uint32_t k0, k1, c2, c3;
  const uint64_t* key;  // where the key is read from instead, or NULL
};

__device__ inline void load_key(Drop& d) {
  if (d.key != nullptr) {
    const uint64_t k = *d.key;
    d.k0 = (uint32_t)k;
    d.k1 = (uint32_t)(k >> 32);
  }
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// each round multiplies two counter words by constants and crosses the products' halves.
// One block gives the 8 half-words of the 8 elements [8 group, 8 group + 8) of a row.
__device__ inline void random_block(const Drop& d, uint32_t row, uint32_t group, uint32_t out[4]) {
  uint32_t c0 = group, c1 = row, c2 = d.c2, c3 = d.c3, k0 = d.k0, k1 = d.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0, out[1] = c1, out[2] = c2, out[3] = c3;
}

__device__ inline float dropped(const Drop& d, const uint32_t bits[4], int j, float v) {
  const uint32_t h = (bits[j >> 1] >> (16 * (j & 1))) & 0xffffu;
  return h >= d.threshold ? v * d.scale : 0.0f;
}

// residual + drop(x), 8 elements of a row a thread.
template <typename T>
__global__ __launch_bounds__(256) void k_dropout(Drop d, int64_t rows, int64_t cols, const T* x, int64_t ldx, const T* res,
                                                 int64_t ldr, T* y, int64_t ldy) {
  load_key(d);
  const int64_t groups = (cols + 7) / 8, total = rows * groups;
  for (int64_t g = blockIdx.x * 256ll + threadIdx.x; g < total; g += gridDim.x * 256ll) {
    const int64_t row = g / groups, group = g % groups;
    uint32_t bits[4];
    random_block(d, (uint32_t)row, (uint32_t)group, bits);
    const int n = cols - 8 * group < 8 ? (int)(cols - 8 * group) : 8;
    for (int j = 0; j < n; ++j) {
      const int64_t c = 8 * group + j;
      float v = dropped(d, bits, j, (float)x[row * ldx + c]);
      if (res != nullptr) v += (float)res[row * ldr + c];
      y[row * ldy + c] = (T)v;
    }
  }
}

// ------------------------------------------------------------------------------------------
// Activations: act(g), and with it act'(g).

template <int ACT>
__device__ inline float activation(float g, float* slope) {
  if constexpr (ACT == GF_ACT_SILU) {  // g s, s = 1 / (1 + e^-g); s' = s (1 - s)
    const float s = 1.0f / (1.0f + expf(-g));
    if (slope != nullptr) *slope = s + g * s * (1.0f - s);
    return g * s;
  } else if constexpr (ACT == GF_ACT_GELU) {  // g Phi(g); Phi' = e^(-g^2/2) / sqrt(2 pi)
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * g);
    if (slope != nullptr) *slope = cdf + g * (0.39894228040143268f * expf(-0.5f * g * g));
    return g * cdf;
  } else {  // (1 + tanh u) / 2 = 1 / (1 + e^-2u), u = sqrt(2/pi) (g + 0.044715 g^3)
    const float u2 = 1.5957691216057308f * g * (1.0f + 0.044715f * g * g);
    const float s = 1.0f / (1.0f + expf(-u2));
    if (slope != nullptr) *slope = s + g * s * (1.0f - s) * (1.5957691216057308f * (1.0f + 3.0f * 0.044715f * g * g));
    return g * s;
  }
}

template <int ACT>
using ActTag = std::integral_constant<int, ACT>;

// ------------------------------------------------------------------------------------------
// Products.  C[m, n] = sum over k of A(m, k) B(n, k), both operands by their strides, in tiles of 64 x 64
// through LDS in 32 bits.

struct Operand {
  const void* p;
  int64_t row, k;  // strides in elements
};

struct Epilogue {
  void* out;  // [M, N], contiguous (gated: [M, N / 2])
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* saved;  // gated: the value's plane, then the gate's, [M, saved_ld]
  int64_t saved_ld;
  Drop drop;
};

constexpr int kTile = 64, kStep = 16;

// B2: the second weight half's rows begin at row `second` of B (gated), and C is drop(value * act(gate)).
template <typename T, int ACT>
__global__ __launch_bounds__(256) void k_product(int64_t M, int64_t N, int64_t K, Operand A, Operand B, int64_t second,
                                                 Epilogue e) {
  constexpr int H = ACT == GF_ACT_NONE ? 1 : 2;
  __shared__ float sa[kStep][kTile + 4], sb[H][kStep][kTile + 4];
  const int64_t m0 = (int64_t)blockIdx.x * kTile, n0 = (int64_t)blockIdx.y * kTile;
  const int t = threadIdx.x, tm = t / 16 * 4, tn = t % 16 * 4;
  float acc[H][4][4] = {};
  const T *a = (const T*)A.p, *b = (const T*)B.p;
  for (int64_t k0 = 0; k0 < K; k0 += kStep) {
    for (int i = t; i < kTile * kStep; i += 256) {
      const int r = A.k == 1 ? i / kStep : i % kTile, k = A.k == 1 ? i % kStep : i / kTile;
      sa[k][r] = m0 + r < M && k0 + k < K ? (float)a[(m0 + r) * A.row + (k0 + k) * A.k] : 0.0f;
    }
    for (int i = t; i < kTile * kStep; i += 256) {
      const int r = B.k == 1 ? i / kStep : i % kTile, k = B.k == 1 ? i % kStep : i / kTile;
      for (int h = 0; h < H; ++h)
        sb[h][k][r] = n0 + r < N && k0 + k < K ? (float)b[(n0 + r + h * second) * B.row + (k0 + k) * B.k] : 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < kStep; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
          for (int h = 0; h < H; ++h) acc[h][i][j] += sa[k][tm + i] * sb[h][k][tn + j];
    __syncthreads();
  }
  load_key(e.drop);
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + tm + i;
    if (m >= M) break;
    uint32_t bits[4];
    if (e.drop.threshold != 0) random_block(e.drop, (uint32_t)m, (uint32_t)((n0 + tn) / 8), bits);
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tn + j;
      if (n >= N) break;
      float v = acc[0][i][j];
      if (e.bias != nullptr) v += (float)((const T*)e.bias)[n];
      if constexpr (ACT != GF_ACT_NONE) {
        float g = acc[H - 1][i][j];
        if (e.bias != nullptr) g += (float)((const T*)e.bias)[second + n];
        if (e.saved != nullptr) {
          ((T*)e.saved)[m * e.saved_ld + n] = (T)v;
          ((T*)e.saved)[(M + m) * e.saved_ld + n] = (T)g;
        }
        v *= activation<ACT>(g, nullptr);
      }
      if (e.drop.threshold != 0) v = dropped(e.drop, bits, (int)(n % 8), v);
      if (e.residual != nullptr) v += (float)((const T*)e.residual)[m * e.ldr + n];
      ((T*)e.out)[m * N + n] = (T)v;
    }
  }
}

// dz [rows, ld]: the gradient of x W^T + b from dy (gated: the value's columns, then the gate's).
template <typename T, int ACT>
__global__ __launch_bounds__(256) void k_dz(Drop d, int64_t rows, int64_t out, const T* dy, int64_t lddy, const T* saved,
                                            int64_t saved_ld, T* dz, int64_t ld) {
  load_key(d);
  const int64_t groups = (out + 7) / 8, total = rows * groups;
  for (int64_t q = blockIdx.x * 256ll + threadIdx.x; q < total; q += gridDim.x * 256ll) {
    const int64_t row = q / groups, group = q % groups;
    uint32_t bits[4];
    if (d.threshold != 0) random_block(d, (uint32_t)row, (uint32_t)group, bits);
    const int n = out - 8 * group < 8 ? (int)(out - 8 * group) : 8;
    for (int j = 0; j < n; ++j) {
      const int64_t c = 8 * group + j;
      float v = (float)dy[row * lddy + c];
      if (d.threshold != 0) v = dropped(d, bits, j, v);
      if constexpr (ACT == GF_ACT_NONE) {
        dz[row * ld + c] = (T)v;
      } else {
        const float value = (float)saved[row * saved_ld + c], gate = (float)saved[(rows + row) * saved_ld + c];
        float slope;
        const float a = activation<ACT>(gate, &slope);
        dz[row * ld + c] = (T)(v * a);
        dz[row * ld + out + c] = (T)(v * value * slope);
      }
    }
  }
}

// Column sums of dz, one column a thread, rows in order.
template <typename T>
__global__ __launch_bounds__(256) void k_column_sums(int64_t rows, int64_t cols, const T* dz, int64_t ld, T* out) {
  const int64_t c = blockIdx.x * 256ll + threadIdx.x;
  if (c >= cols) return;
  float s = 0.0f;
  for (int64_t r = 0; r < rows; ++r) s += (float)dz[r * ld + c];
  out[c] = (T)s;
}

// ------------------------------------------------------------------------------------------
// Host.

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

int size_of(int32_t dtype) { return dtype == GF_DTYPE_F32 ? 4 : 2; }

int check_dropout(const gf_dropout* d) {
  if (d == nullptr) return fail(GF_E_INVALID_ARGUMENT, "dropout must not be NULL");
  if (!(d->p >= 0.0 && d->p <= 1.0)) return fail(GF_E_INVALID_ARGUMENT, "dropout p must lie in [0, 1]");
  return GF_OK;
}

Drop make_drop(const gf_dropout& d) {
  Drop r;
  r.threshold = (uint32_t)std::floor(d.p * 65536.0 + 0.5);
  r.scale = r.threshold >= 65536u ? 0.0f : (float)(65536.0 / (65536.0 - r.threshold));
  r.k0 = (uint32_t)d.seed, r.k1 = (uint32_t)(d.seed >> 32);
  r.c2 = (uint32_t)d.offset, r.c3 = (uint32_t)(d.offset >> 32);
  r.key = d.seed_device;
  return r;
}

constexpr int64_t kMaxSize = INT32_MAX;

int check_matrix(const char* name, const void* p, int64_t ld, int64_t width, int size) {
  if (p == nullptr) return fail(GF_E_INVALID_ARGUMENT, "%s must not be NULL", name);
  if (ld < width) return fail(GF_E_INVALID_ARGUMENT, "%s: row stride %lld is below its width %lld", name, (long long)ld, (long long)width);
  if ((uintptr_t)p % size != 0) return fail(GF_E_INVALID_ARGUMENT, "%s is not aligned to its type", name);
  return GF_OK;
}

#define FF_CHECK(expr)                 \
  do {                                 \
    if (int rc_ = (expr)) return rc_;  \
  } while (0)

int check_dtype(int32_t dtype) {
  if (dtype < GF_DTYPE_F32 || dtype > GF_DTYPE_F16) return fail(GF_E_INVALID_ARGUMENT, "unknown dtype %d", (int)dtype);
  return GF_OK;
}

int check_shape(const gf_ff_args* a) {
  if (a == nullptr) return fail(GF_E_INVALID_ARGUMENT, "args must not be NULL");
  FF_CHECK(check_dtype(a->dtype));
  if (a->activation < GF_ACT_NONE || a->activation > GF_ACT_SILU)
    return fail(GF_E_INVALID_ARGUMENT, "unknown activation %d", (int)a->activation);
  if (a->rows < 0 || a->in_features <= 0 || a->out_features <= 0)
    return fail(GF_E_INVALID_ARGUMENT, "rows must not be negative and in_features and out_features must be positive");
  if (a->rows > kMaxSize || a->in_features > kMaxSize / 2 || a->out_features > kMaxSize / 4)
    return fail(GF_E_INVALID_ARGUMENT, "rows, in_features or out_features too large");
  return check_dropout(&a->dropout);
}

int64_t weight_rows(const gf_ff_args* a) { return a->out_features * (a->activation == GF_ACT_NONE ? 1 : 2); }
int64_t saved_ld(const gf_ff_args* a) { return round_up(a->out_features, 8); }

template <typename F>
int with_dtype(int32_t dtype, F f) {
  switch (dtype) {
    case GF_DTYPE_F32: return f(float());
    case GF_DTYPE_BF16: return f(bf16());
    default: return f(f16());
  }
}

template <typename F>
int with_activation(int32_t act, F f) {
  switch (act) {
    case GF_ACT_NONE: return f(ActTag<GF_ACT_NONE>());
    case GF_ACT_GELU: return f(ActTag<GF_ACT_GELU>());
    case GF_ACT_GELU_TANH: return f(ActTag<GF_ACT_GELU_TANH>());
    default: return f(ActTag<GF_ACT_SILU>());
  }
}

unsigned blocks_for(int64_t threads) { return (unsigned)std::min<int64_t>(std::max<int64_t>((threads + 255) / 256, 1), 8192); }

template <typename T, int ACT>
int product(int64_t M, int64_t N, int64_t K, Operand A, Operand B, int64_t second, const Epilogue& e, hipStream_t s) {
  if (M == 0 || N == 0) return GF_OK;
  const int64_t tiles_n = (N + kTile - 1) / kTile;
  if (tiles_n > 65535) return fail(GF_E_INVALID_ARGUMENT, "in_features or out_features too large");
  k_product<T, ACT><<<dim3((unsigned)((M + kTile - 1) / kTile), (unsigned)tiles_n), 256, 0, s>>>(M, N, K, A, B, second, e);
  FF_LAUNCH_CHECK("k_product");
  return GF_OK;
}

}  // namespace

extern "C" {

int gf_dropout_add(int32_t dtype, const gf_dropout* dropout, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                   const void* residual, int64_t ldr, void* y, int64_t ldy, void* stream) {
  FF_CHECK(check_dtype(dtype));
  FF_CHECK(check_dropout(dropout));
  if (rows < 0 || cols < 0 || rows > kMaxSize || cols > kMaxSize) return fail(GF_E_INVALID_ARGUMENT, "rows or cols negative or too large");
  if (rows == 0 || cols == 0) return GF_OK;
  FF_CHECK(check_matrix("x", x, ldx, cols, size_of(dtype)));
  FF_CHECK(check_matrix("y", y, ldy, cols, size_of(dtype)));
  if (residual != nullptr) FF_CHECK(check_matrix("residual", residual, ldr, cols, size_of(dtype)));
  const Drop d = make_drop(*dropout);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_dropout<T><<<blocks_for(rows * ((cols + 7) / 8)), 256, 0, (hipStream_t)stream>>>(d, rows, cols, (const T*)x, ldx, (const T*)residual, ldr,
                                                                      (T*)y, ldy);
    FF_LAUNCH_CHECK("k_dropout");
    return (int)GF_OK;
  });
}

size_t gf_ff_saved_bytes(const gf_ff_args* args) {
  if (check_shape(args) != GF_OK || args->activation == GF_ACT_NONE) return 0;
  return (size_t)(2 * args->rows * saved_ld(args) * size_of(args->dtype));
}

size_t gf_ff_workspace_bytes(const gf_ff_args* args, int32_t backward) {
  if (check_shape(args) != GF_OK || !backward) return 0;
  return (size_t)(args->rows * round_up(weight_rows(args), 8) * size_of(args->dtype));
}

int gf_ff_forward(const gf_ff_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  FF_CHECK(check_shape(args));
  const gf_ff_args a = *args;
  if (a.rows == 0) return GF_OK;
  const int size = size_of(a.dtype);
  FF_CHECK(check_matrix("x", a.x, a.ldx, a.in_features, size));
  FF_CHECK(check_matrix("weight", a.weight, a.ldw, a.in_features, size));
  FF_CHECK(check_matrix("y", a.y, a.out_features, a.out_features, size));
  if (a.residual != nullptr) {
    if (a.activation != GF_ACT_NONE) return fail(GF_E_INVALID_ARGUMENT, "a gated product takes no residual");
    FF_CHECK(check_matrix("residual", a.residual, a.ldr, a.out_features, size));
  }
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_activation(a.activation, [&](auto act) {
      Epilogue e{a.y, a.bias, a.residual, a.ldr, a.saved, saved_ld(&a), make_drop(a.dropout)};
      return product<T, act.value>(a.rows, a.out_features, a.in_features, {a.x, a.ldx, 1}, {a.weight, a.ldw, 1}, a.out_features, e,
                                   (hipStream_t)stream);
    });
  });
}

int gf_ff_backward(const gf_ff_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  FF_CHECK(check_shape(args));
  const gf_ff_args a = *args;
  const int size = size_of(a.dtype);
  FF_CHECK(check_matrix("x", a.x, a.ldx, a.in_features, size));
  FF_CHECK(check_matrix("weight", a.weight, a.ldw, a.in_features, size));
  FF_CHECK(check_matrix("dy", a.dy, a.lddy, a.out_features, size));
  if (a.activation != GF_ACT_NONE) FF_CHECK(check_matrix("saved", a.saved, 1, 1, 16));
  if (workspace_bytes < gf_ff_workspace_bytes(args, 1) || (workspace == nullptr && workspace_bytes != 0))
    return fail(GF_E_WORKSPACE, "workspace too small");
  const hipStream_t s = (hipStream_t)stream;
  const int64_t wr = weight_rows(&a), ld = round_up(wr, 8);
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_activation(a.activation, [&](auto act) {
      T* dz = (T*)workspace;
      k_dz<T, act.value><<<blocks_for(a.rows * ((a.out_features + 7) / 8)), 256, 0, s>>>(
          make_drop(a.dropout), a.rows, a.out_features, (const T*)a.dy, a.lddy, (const T*)a.saved, saved_ld(&a), dz, ld);
      FF_LAUNCH_CHECK("k_dz");
      Epilogue e{};
      if (a.dx != nullptr) {
        e.out = a.dx;
        FF_CHECK((product<T, GF_ACT_NONE>(a.rows, a.in_features, wr, {dz, ld, 1}, {a.weight, 1, a.ldw}, 0, e, s)));
      }
      if (a.dweight != nullptr) {
        e.out = a.dweight;
        FF_CHECK((product<T, GF_ACT_NONE>(wr, a.in_features, a.rows, {dz, 1, ld}, {a.x, 1, a.ldx}, 0, e, s)));
      }
      if (a.dbias != nullptr) {
        k_column_sums<T><<<(unsigned)((wr + 255) / 256), 256, 0, s>>>(a.rows, wr, dz, ld, (T*)a.dbias);
        FF_LAUNCH_CHECK("k_column_sums");
      }
      return (int)GF_OK;
    });
  });
}

}  // extern "C"
