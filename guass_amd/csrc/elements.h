// elements.h - what the kernels on rows of 16- and 32-bit elements share (feedforward.hip, norms.hip, quantized.hip): loads and
// stores of 8 elements, activations, and on the host the checks of arguments, the choice of a type and workspaces.
#ifndef GF_ELEMENTS_H_
#define GF_ELEMENTS_H_

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

#define GF_LAUNCH_CHECK(name)                                                                    \
  do {                                                                                           \
    hipError_t e_ = hipGetLastError();                                                           \
    if (e_ != hipSuccess) return fail(GF_E_HIP, "launch of %s failed: %s", name, hipGetErrorString(e_)); \
  } while (0)

// 8 consecutive elements in 32 bits: 16 bytes (two times 16) a lane at whatever alignment, which global memory takes,
// or where they are not `all` there the first n, one by one.
template <typename T, int N>
using Vec = T __attribute__((ext_vector_type(N), aligned(sizeof(T))));

template <typename T>
__device__ inline void load8(float v[8], const T* p, bool all, int n) {
  constexpr int W = 16 / sizeof(T);
  if (all) {
#pragma unroll
    for (int i = 0; i < 8; i += W) {
      const Vec<T, W> t = *(const Vec<T, W>*)(p + i);
#pragma unroll
      for (int j = 0; j < W; ++j) v[i + j] = (float)t[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.0f;
  }
}

template <typename T>
__device__ inline void store8(T* p, const float v[8], bool all, int n) {
  constexpr int W = 16 / sizeof(T);
  if (all) {
#pragma unroll
    for (int i = 0; i < 8; i += W) {
      Vec<T, W> t;
#pragma unroll
      for (int j = 0; j < W; ++j) t[j] = (T)v[i + j];
      *(Vec<T, W>*)(p + i) = t;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)v[j];
  }
}

// ------------------------------------------------------------------------------------------
// Activations: act(g), and with it act'(g).  Exponentials and reciprocals are the hardware's (1 unit in the last place).

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

// Phi(-a) e^(a^2/2) for a >= 0 as t Q(t), t = 1 / (1 + p a): p and Q fitted (least squares reweighted to the largest
// relative error) over a in [0, 14]: good to 1.4e-7 with p and Q as floats, and to 3.7e-7 as evaluated in 32 bits (7.4e-7 if
// the reciprocal is a unit off); past that Phi(-a) is below the smallest float.
__device__ inline float normal_tail(float a) {
  const float t = rcp_fast(__builtin_fmaf(0.3045656383f, a, 1.0f));
  float q = 0.0367617272f;
  q = __builtin_fmaf(q, t, -0.153960079f);
  q = __builtin_fmaf(q, t, 0.188459948f);
  q = __builtin_fmaf(q, t, -0.0401414931f);
  q = __builtin_fmaf(q, t, 0.122078776f);
  q = __builtin_fmaf(q, t, 0.103001416f);
  q = __builtin_fmaf(q, t, 0.122335792f);
  q = __builtin_fmaf(q, t, 0.121463954f);
  return q * t;
}

constexpr float kLog2e = 1.4426950408889634f;

template <int ACT>
__device__ inline float activation(float g, float* slope) {
  if constexpr (ACT == GF_ACT_GELU) {  // g Phi(g); Phi' = e^(-g^2/2) / sqrt(2 pi)
    const float e = exp2_fast(-0.5f * kLog2e * g * g), tail = normal_tail(fabsf(g)) * e;
    const float cdf = g < 0.0f ? tail : 1.0f - tail;
    if (slope != nullptr) *slope = __builtin_fmaf(0.39894228040143268f * g, e, cdf);
    return g * cdf;
  } else if constexpr (ACT == GF_ACT_SILU) {  // g s, s = 1 / (1 + e^-g); s' = s (1 - s)
    const float s = rcp_fast(1.0f + exp2_fast(-kLog2e * g));
    if (slope != nullptr) *slope = __builtin_fmaf(g * s, 1.0f - s, s);
    return g * s;
  } else {  // (1 + tanh u) / 2 = 1 / (1 + e^-2u), u = sqrt(2/pi) (g + 0.044715 g^3)
    constexpr float c = 1.5957691216057308f;
    const float sq = fminf(0.044715f * g * g, 1e30f);  // finite: where it would not be, s (1 - s) is 0
    const float s = rcp_fast(1.0f + exp2_fast(-c * kLog2e * g * (1.0f + sq)));
    if (slope != nullptr) *slope = __builtin_fmaf(g * s * (1.0f - s), c * __builtin_fmaf(3.0f, sq, 1.0f), s);
    return g * s;
  }
}

template <int ACT>
using ActTag = std::integral_constant<int, ACT>;

// ------------------------------------------------------------------------------------------
// Host.

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

int size_of(int32_t dtype) { return dtype == GF_DTYPE_F32 ? 4 : 2; }

constexpr int64_t kMaxSize = INT32_MAX;
// Elements of a matrix, its row stride's gaps among them: more than a memory has, and 64 bits hold the bytes of all that is
// made of one (planes, parts: at most 2^7 bytes an element).
constexpr int64_t kMaxElements = int64_t(1) << 48;

int check_matrix(const char* name, const void* p, int64_t rows, int64_t ld, int64_t width, int size) {
  if (p == nullptr) return fail(GF_E_INVALID_ARGUMENT, "%s must not be NULL", name);
  if (rows > 1 && ld > kMaxElements / rows) return fail(GF_E_INVALID_ARGUMENT, "%s: too large", name);
  if (ld < width) return fail(GF_E_INVALID_ARGUMENT, "%s: row stride %lld is below its width %lld", name, (long long)ld, (long long)width);
  if ((uintptr_t)p % size != 0) return fail(GF_E_INVALID_ARGUMENT, "%s is not aligned to its type", name);
  return GF_OK;
}

int check_workspace(size_t need, const void* workspace, size_t bytes) {
  if (bytes < need || (need != 0 && workspace == nullptr))
    return fail(GF_E_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? bytes : size_t(0), need);
  if ((uintptr_t)workspace % 16 != 0) return fail(GF_E_INVALID_ARGUMENT, "workspace is not 16-byte aligned");
  return GF_OK;
}

#define GF_TRY(expr)                   \
  do {                                 \
    if (int rc_ = (expr)) return rc_;  \
  } while (0)

int check_dtype(int32_t dtype) {
  if (dtype < GF_DTYPE_F32 || dtype > GF_DTYPE_F16) return fail(GF_E_INVALID_ARGUMENT, "unknown dtype %d", (int)dtype);
  return GF_OK;
}

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

// Hands out a workspace from its start; without one it only counts.
struct Arena {
  uint8_t* base;
  size_t used = 0;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (size_t)round_up(bytes, 256);
    return p;
  }
};

#define GF_RUN if (run)  // nothing is launched while the workspace is counted

}  // namespace

#endif  // GF_ELEMENTS_H_
