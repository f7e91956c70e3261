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
// Products.  C[m, n] = sum over k of P(m, k) Q(n, k) on the matrix cores, accumulated in 32 bits.
//
// A workgroup computes a BM x BN tile, WM x WN waves a TM x TN part each, in steps of 64 along k.  An operand is
// either K-contiguous (its row in memory is a row of the tile: x and W forward, dz in dx) or row-contiguous
// (memory's rows are the steps of k: W in dx, dz and x in dW); nothing is transposed in memory:
//   K-contiguous   LDS [row][64 k], fragments by 16-byte reads;
//   row-contiguous LDS [64 k][row], fragments by the transposing 8-byte reads, 4 k of a column a lane.
// Both go from memory to LDS without registers, 16 bytes a lane, double-buffered.  Such a load writes LDS linearly
// by lane, so the bank swizzle permutes which 16 bytes of memory a lane asks for instead.
//
// Rows past the matrix are clamped to its last one: they only reach outputs that are not stored.  Steps past K ask
// for an address past the buffer's end, which reads as zero, in both operands, so that nothing is multiplied with
// what lies behind a row (it may be a NaN).
//
// Q's rows are the matrix instruction's rows, of which a lane holds 4 consecutive ones of each 8; they are assigned
// so that a lane ends up with 8 consecutive n of one m: one 16-byte store, one block of random bits.

using half8 = short __attribute__((ext_vector_type(8)));
using half4 = short __attribute__((ext_vector_type(4)));
using bf16x8 = bf16 __attribute__((ext_vector_type(8)));
using f16x8 = f16 __attribute__((ext_vector_type(8)));
using f32x16 = float __attribute__((ext_vector_type(16)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using lds_ptr = __attribute__((address_space(3))) void*;

template <typename T>
__device__ inline f32x16 mfma(half8 a, half8 b, f32x16 c) {
  if constexpr (std::is_same_v<T, f16>)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A matrix in memory: rows of `ld` elements, 16-byte aligned, `width` (a multiple of 8) of them readable.  32-bit
// matrices come as three such planes of bfloat16 (k_split), `plane` elements apart.
struct Matrix {
  const void* p;
  int64_t ld, plane;
  int32_t width;
};

struct Epilogue {
  void* out;  // [M, N], contiguous
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* saved;  // gated: the value's plane, then the gate's, [M, saved_ld]
  int64_t saved_ld;
  float* partial;  // not NULL: sums for k_join instead of all of the above, [split][M][N (gated: 2 N), whole groups of 8]
  int32_t vec;     // out, bias and residual can be read and written 16 bytes at a time
  Drop drop;
};

struct Shape {
  int64_t M, N, K;      // N: output columns (gated: the value's)
  int32_t tiles_m, tiles_n;
  int32_t splits;       // workgroups along k, `steps` steps of 64 each (the last: what is left)
  int32_t steps;
};

constexpr int kStep = 64;

// n within 32 of the matrix instruction's row r = 8 a + 4 h + e
__device__ inline int row_of(int r) { return 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3); }

template <typename T>
__device__ inline void load8(float v[8], const T* p, bool vec, int n) {
  if (vec) {
    if constexpr (sizeof(T) == 2) {
      using V = T __attribute__((ext_vector_type(8)));
      const V t = *(const V*)p;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
    } else {
      const f32x4 a = ((const f32x4*)p)[0], b = ((const f32x4*)p)[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.0f;
  }
}

template <typename T>
__device__ inline void store8(T* p, const float v[8], bool vec, int n) {
  if (vec) {
    if constexpr (sizeof(T) == 2) {
      using V = T __attribute__((ext_vector_type(8)));
      V t;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = (T)v[j];
      *(V*)p = t;
    } else {
      ((f32x4*)p)[0] = f32x4{v[0], v[1], v[2], v[3]};
      ((f32x4*)p)[1] = f32x4{v[4], v[5], v[6], v[7]};
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)v[j];
  }
}

// What follows the sums: 8 consecutive columns n.. of row m (gated: the value's in v, the gate's in g).
// WHOLE: all 8 are inside and everything can be read and written 16 bytes at a time.
template <typename T, int ACT, bool WHOLE>
__device__ inline void finish(const Epilogue& e, const Drop& drop, int64_t M, int64_t N, int64_t m, int64_t n, float v[8],
                              float g[8]) {
  const int left = N - n < 8 ? (int)(N - n) : 8;
  const bool vec = WHOLE || (e.vec && left == 8);
  if (e.bias != nullptr) {
    float b[8];
    load8(b, (const T*)e.bias + n, vec, left);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += b[j];
    if constexpr (ACT != GF_ACT_NONE) {
      load8(b, (const T*)e.bias + N + n, vec, left);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] += b[j];
    }
  }
  if constexpr (ACT != GF_ACT_NONE) {
    if (e.saved != nullptr) {  // its rows are padded to whole groups of 8
      store8((T*)e.saved + m * e.saved_ld + n, v, true, 8);
      store8((T*)e.saved + (M + m) * e.saved_ld + n, g, true, 8);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= activation<ACT>(g[j], nullptr);
  }
  if (drop.threshold != 0) {
    uint32_t bits[4];
    random_block(drop, (uint32_t)m, (uint32_t)(n >> 3), bits);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = dropped(drop, bits, j, v[j]);
  }
  if (e.residual != nullptr) {
    float r[8];
    load8(r, (const T*)e.residual + m * e.ldr + n, vec, left);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += r[j];
  }
  store8((T*)e.out + m * N + n, v, vec, left);
}

// One operand's way from memory into LDS.  ROWS: its rows of the tile.  HALF: the tile takes HALF rows of the value,
// HALF of the gate and so on (0: consecutive rows).
template <bool KC, int ROWS, int THREADS, int HALF>
struct Stage {
  static constexpr int kBytes = ROWS * kStep * 2;
  static constexpr int kLoads = kBytes / (THREADS * 16);  // a lane's loads a step
  static_assert(kBytes % (THREADS * 16) == 0 && ROWS % 64 == 0 && HALF % 8 == 0);

  uint32_t off[kLoads];
  int32_t k_of[kLoads];  // the first k (of the step's 64) of each load
  const uint8_t* base;
  int64_t gate, advance;  // bytes to the gate's rows; bytes a step

  __device__ void init(const Matrix& a, int64_t row0, int64_t rows, int64_t second) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    base = (const uint8_t*)a.p + (KC ? row0 * a.ld : row0) * 2;
    gate = second * a.ld * 2;
    advance = (KC ? kStep : kStep * a.ld) * 2;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int piece = (wave * kLoads + i) * 64 + lane;  // the 16 bytes of LDS that the lane fills
      if constexpr (KC) {
        const int r = piece / 8, chunk = (piece % 8) ^ swizzle(r);
        int64_t row = HALF ? r / (2 * HALF + !HALF) * HALF + r % (HALF + !HALF) : r;
        row = row < rows - row0 ? row : rows - row0 - 1;
        off[i] = (uint32_t)((row * a.ld + chunk * 8) * 2);
        k_of[i] = chunk * 8;
      } else {
        const int k = piece / (ROWS / 8), chunk = (piece % (ROWS / 8)) ^ swizzle(k);
        const int64_t last = a.width - row0 - 8, col = chunk * 8 < last ? chunk * 8 : last;
        off[i] = (uint32_t)((k * a.ld + col) * 2);
        k_of[i] = k;
      }
    }
  }

  // Which 16 bytes of an LDS row hold which: their number is xored with this.  K-contiguous: rows that row_of gives
  // 8 consecutive lanes differ in it.  Row-contiguous: the 4 k that 16 lanes read differ in their 32 bytes.
  __device__ static int swizzle(int r) {
    return KC ? (r & 3) | ((r >> 3) & 1) << 2 : (r & (ROWS / 16 - 1) & 7) << 1;
  }

  __device__ void seek(int64_t steps) { base += steps * advance; }

  template <bool CUT>
  __device__ void load(uint8_t* lds, int64_t left) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int piece = wave * kLoads + i;  // a wave's 1024 bytes
      const uint8_t* b = base;
      if constexpr (HALF != 0) b += (piece * 8 / HALF) % 2 ? gate : 0;
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)b, 0, 0x80000000, 0x00020000);
      const uint32_t o = CUT && k_of[i] >= left ? 0x80000000u : off[i];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(lds + piece * 1024), 16, o, 0, 0, 0);
    }
  }

  // The fragment of 32 rows from `row` on and 16 k from 16 s on: lane l has row row_of(l % 32) and 8 k from 8 (l / 32) on.
  __device__ static half8 fragment(const uint8_t* lds, int row, int s) {
    const int lane = threadIdx.x & 63;
    if constexpr (KC) {
      const int r = row_of(lane & 31);
      return *(const half8*)(lds + row * 128 + r * 128 + (((2 * s + (lane >> 5)) ^ swizzle(r)) << 4));
    } else {
      // 16 lanes read 4 k of 16 rows, a lane 4 rows of one k, and get 4 k of one row each
      const int i = lane & 15, q = 4 * ((lane >> 4) & 1) + (i & 3);  // q: which 4 matrix-instruction rows
      const int r = row + row_of(4 * q);
      half4 part[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = 16 * s + 8 * (lane >> 5) + 4 * u + (i >> 2);
        part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) half4*)(lds + k * ROWS * 2 + (((r >> 3) ^ swizzle(k)) << 4) + (r & 7) * 2));
      }
      return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Planes of a 32-bit matrix times planes of another: a = a0 + a1 + a2 exactly, 8 bits each, so the six products down to
// 2^-16 of a0 b0 leave out 3 2^-24 of a b.  Smallest first.
__device__ constexpr int kPlaneP[6] = {2, 0, 1, 1, 0, 0}, kPlaneQ[6] = {0, 2, 1, 0, 1, 0};

// One step of a workgroup: the loads of a later step into `to`, the products of this one out of `from`.  The two are
// different LDS arrays and said to be (__restrict__): otherwise the compiler waits for the loads before it reads.
template <typename T, typename SP, typename SQ, int TM, int TN, typename Load>
__device__ __forceinline__ void step(uint8_t* __restrict__ to, const uint8_t* __restrict__ from, bool more, Load& load, int wm, int wn,
                                     f32x16 (&acc)[TN / 32][TM / 32]) {
  if (more) load(to);
#pragma unroll
  for (int s = 0; s < kStep / 16; ++s) {
    half8 fp[TM / 32], fq[TN / 32];
#pragma unroll
    for (int i = 0; i < TM / 32; ++i) fp[i] = SP::fragment(from, wm + 32 * i, s);
#pragma unroll
    for (int j = 0; j < TN / 32; ++j) fq[j] = SQ::fragment(from + SP::kBytes, wn + 32 * j, s);
#pragma unroll
    for (int j = 0; j < TN / 32; ++j)
#pragma unroll
      for (int i = 0; i < TM / 32; ++i) acc[j][i] = mfma<T>(fq[j], fp[i], acc[j][i]);
  }
}

// All of this wave's LDS reads are done and all but its last `loads` loads are in LDS; then all waves'.
template <int LOADS>
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (LOADS & 15) | (LOADS >> 4) << 14);  // vmcnt(LOADS) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, bool PKC, bool QKC, int ACT, int WM, int WN, int TM, int TN, int STAGES>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_product(Shape sh, Matrix p, Matrix q, int64_t second, Epilogue e) {
  constexpr bool kGated = ACT != GF_ACT_NONE;
  constexpr int kThreads = WM * WN * 64, BM = WM * TM, BN = WN * TN, BO = kGated ? BN / 2 : BN;
  constexpr int kPlanes = std::is_same_v<T, float> ? 6 : 1;
  using SP = Stage<PKC, BM, kThreads, 0>;
  using SQ = Stage<QKC, BN, kThreads, kGated ? TN / 2 : 0>;
  constexpr int kBytes = SP::kBytes + SQ::kBytes, kLoads = SP::kLoads + SQ::kLoads;
  __shared__ __attribute__((aligned(1024))) uint8_t lds0[kBytes], lds1[kBytes], lds2[STAGES > 2 ? kBytes : 1024];

  // Workgroups go round the 8 dies by their number; a die gets consecutive tiles, in groups of 8 tile rows, so that
  // its cache sees the same rows of P and of Q again.
  const int tiles = sh.tiles_m * sh.tiles_n, die = blockIdx.x & 7, each = tiles >> 3, more = tiles & 7;
  const int tile = die * each + (die < more ? die : more) + (blockIdx.x >> 3);
  const int group = tile / (8 * sh.tiles_n), in_group = tile % (8 * sh.tiles_n);
  const int height = sh.tiles_m - 8 * group < 8 ? sh.tiles_m - 8 * group : 8;
  const int64_t m0 = (int64_t)(8 * group + in_group % height) * BM, n0 = (int64_t)(in_group / height) * BO;
  const int step0 = blockIdx.y * sh.steps, all = (int)((sh.K + kStep - 1) / kStep);
  const int steps = all - step0 < sh.steps ? all - step0 : sh.steps;

  SP sp;
  SQ sq;
  sp.init(p, m0, sh.M, 0);
  sq.init(q, n0, sh.N, second);
  sp.seek(step0);
  sq.seek(step0);
  const uint8_t *p_base = sp.base, *q_base = sq.base;

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wm = wave % WM * TM, wn = wave / WM * TN;
  f32x16 acc[TN / 32][TM / 32] = {};

  int64_t left = sh.K - (int64_t)step0 * kStep;  // k from the next load's first on
  int loaded = 0, plane = 0;                     // steps of this plane product loaded; which it is
  auto load = [&](uint8_t* to) {
    if constexpr (kPlanes > 1) {
      if (loaded == 0) {
        sp.base = p_base + kPlaneP[plane] * p.plane * 2;
        sq.base = q_base + kPlaneQ[plane] * q.plane * 2;
        left = sh.K - (int64_t)step0 * kStep;
      }
    }
    if (left >= kStep) {
      sp.template load<false>(to, left);
      sq.template load<false>(to + SP::kBytes, left);
    } else {
      sp.template load<true>(to, left);
      sq.template load<true>(to + SP::kBytes, left);
    }
    sp.seek(1);
    sq.seek(1);
    left -= kStep;
    if (++loaded == steps) loaded = 0, ++plane;
  };

  const int total = steps * kPlanes;
  if constexpr (STAGES == 2) {
    load(lds0);
    int t = 0;
    for (; t + 1 < total; t += 2) {
      meet<0>();
      step<T, SP, SQ, TM, TN>(lds1, lds0, true, load, wm, wn, acc);
      meet<0>();
      step<T, SP, SQ, TM, TN>(lds0, lds1, t + 2 < total, load, wm, wn, acc);
    }
    if (t < total) {
      meet<0>();
      step<T, SP, SQ, TM, TN>(lds1, lds0, false, load, wm, wn, acc);
    }
  } else {
    load(lds0);
    if (total > 1) load(lds1);
    int t = 0;
    for (; t + 4 < total; t += 3) {
      meet<kLoads>();
      step<T, SP, SQ, TM, TN>(lds2, lds0, true, load, wm, wn, acc);
      meet<kLoads>();
      step<T, SP, SQ, TM, TN>(lds0, lds1, true, load, wm, wn, acc);
      meet<kLoads>();
      step<T, SP, SQ, TM, TN>(lds1, lds2, true, load, wm, wn, acc);
    }
    // 1 to 4 steps are left, two of them loaded
    for (bool first = true; t < total; t += 3, first = false) {
      meet<0>();
      step<T, SP, SQ, TM, TN>(lds2, lds0, t + 2 < total, load, wm, wn, acc);
      if (t + 1 >= total) break;
      meet<0>();
      step<T, SP, SQ, TM, TN>(lds0, lds1, t + 3 < total, load, wm, wn, acc);
      if (t + 2 >= total) break;
      meet<0>();
      step<T, SP, SQ, TM, TN>(lds1, lds2, false, load, wm, wn, acc);
    }
  }

  // Lane l has, of each 32 x 32, row m = row_of(l % 32) and columns 16 h + 8 (l / 32) .. + 8 for h = 0, 1.
  Drop drop = e.drop;
  load_key(drop);
  constexpr int kOut = kGated ? TN / 64 : TN / 32;
#pragma unroll
  for (int i = 0; i < TM / 32; ++i) {
    const int64_t m = m0 + wm + 32 * i + row_of(lane & 31);
    if (m >= sh.M) continue;
#pragma unroll
    for (int j = 0; j < kOut; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t n = n0 + (kGated ? wn / 2 : wn) + 32 * j + 16 * h + 8 * (lane >> 5);
        if (n >= sh.N) continue;
        float v[8], g[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          v[r] = acc[j][i][8 * h + r];
          if constexpr (kGated) g[r] = acc[kOut + j][i][8 * h + r];
        }
        if (e.partial != nullptr) {
          const int64_t width = (sh.N + 7) / 8 * 8;
          float* out = e.partial + ((int64_t)blockIdx.y * sh.M + m) * width * (kGated ? 2 : 1) + n;
          store8(out, v, true, 8);
          if constexpr (kGated) store8(out + width, g, true, 8);
        } else {
          finish<T, ACT, true>(e, drop, sh.M, sh.N, m, n, v, g);
        }
      }
  }
}

// The products' parts, added in their order.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void k_join(Shape sh, Epilogue e) {
  constexpr bool kGated = ACT != GF_ACT_NONE;
  Drop drop = e.drop;
  load_key(drop);
  const int64_t groups = (sh.N + 7) / 8, width = groups * 8 * (kGated ? 2 : 1);
  for (int64_t t = blockIdx.x * 256ll + threadIdx.x; t < sh.M * groups; t += gridDim.x * 256ll) {
    const int64_t m = t / groups, n = t % groups * 8;
    float v[8] = {}, g[8] = {}, part[8];
    for (int s = 0; s < sh.splits; ++s) {
      const float* in = e.partial + ((int64_t)s * sh.M + m) * width + n;
      load8(part, in, true, 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += part[j];
      if constexpr (kGated) {
        load8(part, in + groups * 8, true, 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] += part[j];
      }
    }
    finish<T, ACT, false>(e, drop, sh.M, sh.N, m, n, v, g);
  }
}

// ------------------------------------------------------------------------------------------
// Operands that the products cannot read in place: 32-bit matrices into three bfloat16 planes, and 16-bit ones whose
// rows are not whole, aligned groups of 16 bytes into rows that are.  Columns past the matrix become zero.

// x = its 3 x 8 leading bits, by truncation: x - a0 and x - a0 - a1 are exact.  An infinity or a NaN stays in a0.
__device__ inline void split(float x, bf16 out[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t top = __builtin_bit_cast(uint32_t, x) & 0xffff0000u;
    const bool finite = (top & 0x7f800000u) != 0x7f800000u;
    out[i] = __builtin_bit_cast(bf16, (uint16_t)((__builtin_bit_cast(uint32_t, x) | (finite ? 0u : (__builtin_bit_cast(uint32_t, x) & 0xffffu) ? 0x10000u : 0u)) >> 16));
    x = finite ? x - __builtin_bit_cast(float, top) : 0.0f;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_pack(int64_t rows, int64_t cols, const T* x, int64_t ldx, int32_t vec, void* out,
                                              int64_t ld, int64_t plane) {
  const int64_t groups = ld / 8;
  for (int64_t t = blockIdx.x * 256ll + threadIdx.x; t < rows * groups; t += gridDim.x * 256ll) {
    const int64_t row = t / groups, c = t % groups * 8;
    const int n = cols - c < 8 ? (int)(cols - c) : 8;
    float v[8];
    load8(v, x + row * ldx + c, vec && n == 8, n);
    if constexpr (std::is_same_v<T, float>) {
      bf16x8 o[3];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bf16 s[3];
        split(v[j], s);
        o[0][j] = s[0], o[1][j] = s[1], o[2][j] = s[2];
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) *(bf16x8*)((bf16*)out + i * plane + row * ld + c) = o[i];
    } else {
      store8((T*)out + row * ld + c, v, true, 8);
    }
  }
}

// dz: the gradient of x W^T + b from dy (gated: the value's columns, then the gate's), as the products read it
// ([rows, ld], in planes for 32 bits, zero past its columns), and its columns' sums: a workgroup takes 256 columns of dy
// and `chunk` rows, 8 columns a thread in 8 interleaved rows, and leaves its sums in `sums` [row chunk][columns of dz].
template <typename T, int ACT>
__global__ __launch_bounds__(256) void k_dz(Drop d, int64_t rows, int64_t out, int64_t chunk, const T* dy, int64_t lddy, int32_t vec,
                                            const T* saved, int64_t saved_ld, void* dz, int64_t ld, int64_t plane, float* sums) {
  constexpr bool kGated = ACT != GF_ACT_NONE;
  constexpr int H = kGated ? 2 : 1;
  __shared__ float part[H][8][256 + 8];
  load_key(d);
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int64_t c = (blockIdx.x * 32ll + lane) * 8, width = H * out;
  const int n = c >= out ? 0 : out - c < 8 ? (int)(out - c) : 8;
  float sum[H][8] = {};
  if (n > 0) {
    const int64_t end = (blockIdx.y + 1) * chunk < rows ? (blockIdx.y + 1) * chunk : rows;
    for (int64_t row = blockIdx.y * chunk + line; row < end; row += 8) {
      float g[H][8];
      load8(g[0], dy + row * lddy + c, vec && n == 8, n);
      if (d.threshold != 0) {
        uint32_t bits[4];
        random_block(d, (uint32_t)row, (uint32_t)(c >> 3), bits);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[0][j] = dropped(d, bits, j, g[0][j]);
      }
      if constexpr (kGated) {
        float value[8], gate[8];
        load8(value, saved + row * saved_ld + c, true, 8);
        load8(gate, saved + (rows + row) * saved_ld + c, true, 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float slope;
          const float a = activation<ACT>(gate[j], &slope), v = g[0][j];
          g[0][j] = v * a;
          g[1][j] = v * value[j] * slope;
        }
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= n) g[h][j] = 0.0f;
          sum[h][j] += g[h][j];
        }
        if (dz == nullptr) continue;
        // the last columns' store also clears what follows them, up to ld
        const int64_t at = row * ld + h * out + c;
        const bool last = h == H - 1 && c + 8 >= out;
        const int put = last ? (int)(ld - h * out - c) : n;
        const bool whole = out % 8 == 0;
        if constexpr (std::is_same_v<T, float>) {
          bf16 s[8][3];
#pragma unroll
          for (int j = 0; j < 8; ++j) split(g[h][j], s[j]);
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            bf16* to = (bf16*)dz + i * plane + at;
            if (whole) {
              bf16x8 o;
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = s[j][i];
              *(bf16x8*)to = o;
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (j < put) to[j] = s[j][i];
              for (int j = 8; j < put; ++j) to[j] = (bf16)0.0f;
            }
          }
        } else {
          store8((T*)dz + at, g[h], whole, put);
          for (int j = 8; j < put; ++j) ((T*)dz)[at + j] = (T)0.0f;
        }
      }
    }
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int j = 0; j < 8; ++j) part[h][line][lane * 8 + j] = sum[h][j];
  __syncthreads();
  const int64_t col = blockIdx.x * 256ll + threadIdx.x;
  if (col >= out) return;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part[h][i][threadIdx.x];
    sums[blockIdx.y * width + h * out + col] = s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_join_sums(int64_t chunks, int64_t cols, const float* sums, T* out) {
  const int64_t c = blockIdx.x * 256ll + threadIdx.x;
  if (c >= cols) return;
  float s = 0.0f;
  for (int64_t i = 0; i < chunks; ++i) s += sums[i * cols + c];
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

int check_workspace(size_t need, const void* workspace, size_t bytes) {
  if (bytes < need || (need != 0 && workspace == nullptr))
    return fail(GF_E_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? bytes : size_t(0), need);
  if ((uintptr_t)workspace % 16 != 0) return fail(GF_E_INVALID_ARGUMENT, "workspace is not 16-byte aligned");
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

bool aligned(const void* p, int64_t ld, int size) { return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0; }

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

#define FF_RUN if (run)  // nothing is launched while the workspace is counted

// x as a product reads it: itself where it can be, else packed.
template <typename T>
int operand(Arena& ws, bool run, const void* x, int64_t rows, int64_t cols, int64_t ld, hipStream_t s, Matrix* out) {
  constexpr bool kSplit = std::is_same_v<T, float>;
  if (!kSplit && aligned(x, ld, 2) && cols % 8 == 0) {
    *out = {x, ld, 0, (int32_t)cols};
    return GF_OK;
  }
  const int64_t width = round_up(cols, 8), plane = rows * width;
  *out = {ws.take(plane * 2 * (kSplit ? 3 : 1)), width, plane, (int32_t)width};
  FF_RUN {
    k_pack<T><<<blocks_for(rows * width / 8), 256, 0, s>>>(rows, cols, (const T*)x, ld, aligned(x, ld, sizeof(T)),
                                                           (void*)out->p, width, plane);
    FF_LAUNCH_CHECK("k_pack");
  }
  return GF_OK;
}

constexpr int kUnits = 256;  // compute units

template <typename T, bool PKC, bool QKC, int ACT, int WM, int WN, int TM, int TN, int STAGES>
int product_tiled(Arena& ws, bool run, int64_t M, int64_t N, int64_t K, const Matrix& p, const Matrix& q, int64_t second, Epilogue e,
                  hipStream_t s) {
  constexpr int BM = WM * TM, BO = WN * TN / (ACT == GF_ACT_NONE ? 1 : 2);
  Shape sh{M, N, K, 0, 0, 1, 0};
  const int64_t tm = (M + BM - 1) / BM, tn = (N + BO - 1) / BO, steps = (K + kStep - 1) / kStep;
  if (tm * tn > (int64_t(1) << 30)) return fail(GF_E_INVALID_ARGUMENT, "rows, in_features or out_features too large");
  sh.tiles_m = (int32_t)tm, sh.tiles_n = (int32_t)tn;
  // Fewer tiles than compute units: the steps are split among workgroups, at least 4 each, until there are two
  // workgroups a unit.
  int64_t splits = 1;
  if (tm * tn < kUnits) splits = std::max<int64_t>(std::min<int64_t>(2 * kUnits / (tm * tn), steps / 4), 1);
  sh.steps = (int32_t)((steps + splits - 1) / splits);
  sh.splits = (int32_t)((steps + sh.steps - 1) / sh.steps);
  e.partial = nullptr;
  // Columns that are not whole, aligned groups of 8 are left to k_join too.
  const bool join = sh.splits > 1 || N % 8 != 0 || !e.vec;
  if (join) e.partial = (float*)ws.take(sh.splits * M * round_up(N, 8) * (ACT == GF_ACT_NONE ? 1 : 2) * 4);
  FF_RUN {
    k_product<T, PKC, QKC, ACT, WM, WN, TM, TN, STAGES><<<dim3((unsigned)(tm * tn), (unsigned)sh.splits), WM * WN * 64, 0, s>>>(sh, p, q, second, e);
    FF_LAUNCH_CHECK("k_product");
    if (join) {
      k_join<T, ACT><<<blocks_for(M * ((N + 7) / 8)), 256, 0, s>>>(sh, e);
      FF_LAUNCH_CHECK("k_join");
    }
  }
  return GF_OK;
}

template <typename T, bool PKC, bool QKC, int ACT>
int product(Arena& ws, bool run, int64_t M, int64_t N, int64_t K, const Matrix& p, const Matrix& q, int64_t second, const Epilogue& e,
            hipStream_t s) {
  // a load's 32-bit offset spans a tile's rows (K-contiguous) or a step's (row-contiguous)
  if (std::max(p.ld, q.ld) * 2 * 256 >= (int64_t(1) << 31)) return fail(GF_E_INVALID_ARGUMENT, "row stride too large");
  return product_tiled<T, PKC, QKC, ACT, 2, 2, 64, 64, 2>(ws, run, M, N, K, p, q, second, e, s);
}

int32_t vec_ok(const gf_ff_args& a, const void* out) {
  const int size = size_of(a.dtype);
  return aligned(out, a.out_features, size) && (a.bias == nullptr || aligned(a.bias, a.out_features, size)) &&
         (a.residual == nullptr || aligned(a.residual, a.ldr, size));
}

// The forward's launches, or (run false) its workspace.
int forward(const gf_ff_args& a, Arena& ws, bool run, hipStream_t s) {
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_activation(a.activation, [&](auto act) {
      Matrix x, w;
      FF_CHECK(operand<T>(ws, run, a.x, a.rows, a.in_features, a.ldx, s, &x));
      FF_CHECK(operand<T>(ws, run, a.weight, weight_rows(&a), a.in_features, a.ldw, s, &w));
      const Epilogue e{a.y, a.bias, a.residual, a.ldr, a.saved, saved_ld(&a), nullptr, vec_ok(a, a.y), make_drop(a.dropout)};
      return product<T, true, true, act.value>(ws, run, a.rows, a.out_features, a.in_features, x, w, a.out_features, e, s);
    });
  });
}

int backward(const gf_ff_args& a, Arena& ws, bool run, hipStream_t s) {
  const int64_t wr = weight_rows(&a), out = a.out_features;
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_activation(a.activation, [&](auto act) {
      constexpr int ACT = act.value;
      constexpr bool kSplit = std::is_same_v<T, float>;
      const Drop drop = make_drop(a.dropout);
      const bool products = a.dx != nullptr || a.dweight != nullptr;
      Matrix dz{};
      // linear, nothing dropped: dz is dy
      const bool same = ACT == GF_ACT_NONE && drop.threshold == 0;
      if (same && products) FF_CHECK(operand<T>(ws, run, a.dy, a.rows, out, a.lddy, s, &dz));
      const bool make = products && !same;
      if (make) {
        dz.ld = round_up(wr, 8), dz.plane = a.rows * dz.ld, dz.width = (int32_t)dz.ld;
        dz.p = ws.take(dz.plane * 2 * (kSplit ? 3 : 1));
      }
      if (make || a.dbias != nullptr) {
        // rows in chunks of at least 32 until there are about 4 workgroups a compute unit
        const int64_t across = (out + 255) / 256;
        int64_t chunks = std::max<int64_t>(std::min<int64_t>(4 * kUnits / across, a.rows / 32), 1);
        const int64_t chunk = (a.rows + chunks - 1) / chunks;
        chunks = (a.rows + chunk - 1) / chunk;
        float* sums = a.dbias != nullptr ? (float*)ws.take(chunks * wr * 4) : nullptr;
        FF_RUN {
          k_dz<T, ACT><<<dim3((unsigned)across, (unsigned)chunks), 256, 0, s>>>(
              drop, a.rows, out, chunk, (const T*)a.dy, a.lddy, aligned(a.dy, a.lddy, sizeof(T)), (const T*)a.saved, saved_ld(&a),
              make ? (void*)dz.p : nullptr, dz.ld, dz.plane, sums);
          FF_LAUNCH_CHECK("k_dz");
          if (sums != nullptr) {
            k_join_sums<T><<<(unsigned)((wr + 255) / 256), 256, 0, s>>>(chunks, wr, sums, (T*)a.dbias);
            FF_LAUNCH_CHECK("k_join_sums");
          }
        }
      }
      Epilogue e{};
      if (a.dx != nullptr) {
        Matrix w;
        FF_CHECK(operand<T>(ws, run, a.weight, wr, a.in_features, a.ldw, s, &w));
        e.out = a.dx, e.vec = aligned(a.dx, a.in_features, sizeof(T));
        FF_CHECK((product<T, true, false, GF_ACT_NONE>(ws, run, a.rows, a.in_features, wr, dz, w, 0, e, s)));
      }
      if (a.dweight != nullptr) {
        Matrix x;
        FF_CHECK(operand<T>(ws, run, a.x, a.rows, a.in_features, a.ldx, s, &x));
        e.out = a.dweight, e.vec = aligned(a.dweight, a.in_features, sizeof(T));
        FF_CHECK((product<T, false, false, GF_ACT_NONE>(ws, run, wr, a.in_features, a.rows, dz, x, 0, e, s)));
      }
      return (int)GF_OK;
    });
  });
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

size_t gf_ff_workspace_bytes(const gf_ff_args* args, int32_t is_backward) {
  if (check_shape(args) != GF_OK || args->rows == 0) return 0;
  Arena count{nullptr};
  const int rc = is_backward ? backward(*args, count, false, nullptr) : forward(*args, count, false, nullptr);
  return rc == GF_OK ? count.used : 0;
}

int gf_ff_forward(const gf_ff_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  FF_CHECK(check_shape(args));
  const gf_ff_args& a = *args;
  if (a.rows == 0) return GF_OK;
  const int size = size_of(a.dtype);
  FF_CHECK(check_matrix("x", a.x, a.ldx, a.in_features, size));
  FF_CHECK(check_matrix("weight", a.weight, a.ldw, a.in_features, size));
  FF_CHECK(check_matrix("y", a.y, a.out_features, a.out_features, size));
  if (a.residual != nullptr) {
    if (a.activation != GF_ACT_NONE) return fail(GF_E_INVALID_ARGUMENT, "a gated product takes no residual");
    FF_CHECK(check_matrix("residual", a.residual, a.ldr, a.out_features, size));
  }
  if (a.saved != nullptr) FF_CHECK(check_matrix("saved", a.saved, 1, 1, 16));
  Arena count{nullptr}, ws{(uint8_t*)workspace};
  FF_CHECK(forward(a, count, false, nullptr));
  FF_CHECK(check_workspace(count.used, workspace, workspace_bytes));
  return forward(a, ws, true, (hipStream_t)stream);
}

int gf_ff_backward(const gf_ff_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  FF_CHECK(check_shape(args));
  const gf_ff_args& a = *args;
  const int size = size_of(a.dtype);
  FF_CHECK(check_matrix("x", a.x, a.ldx, a.in_features, size));
  FF_CHECK(check_matrix("weight", a.weight, a.ldw, a.in_features, size));
  FF_CHECK(check_matrix("dy", a.dy, a.lddy, a.out_features, size));
  if (a.activation != GF_ACT_NONE) FF_CHECK(check_matrix("saved", a.saved, 1, 1, 16));
  if (a.rows == 0) return fail(GF_E_INVALID_ARGUMENT, "a backward needs rows");
  Arena count{nullptr}, ws{(uint8_t*)workspace};
  FF_CHECK(backward(a, count, false, nullptr));
  FF_CHECK(check_workspace(count.used, workspace, workspace_bytes));
  return backward(a, ws, true, (hipStream_t)stream);
}

}  // extern "C"
