// quantized.hip - gfx950 kernels and C ABI of weights in 4 bits: a weight into codes and scales, back, and products with it.
//
//   k_quantize    groups of 32 of a row: a power of two for a scale, and the nearest of the 16 values e2m1 has
//   k_dequantize  the values that codes and scales stand for, in a type of 16 or 32 bits
//   k_q4_few      the product of at most 64 rows: codes straight into the matrix instructions' operands
//
// A group's scale being a power of two, a weight's value is exact in bfloat16 (sign, 2 bits of fraction), and in float16 as long as the
// scale is not extreme: the matrix cores get it without a rounding of its own.  The hardware turns two codes into two values of a
// scale in one instruction.  More rows than 64 go through k_dequantize and the feed-forward products (feedforward.hip), forward
// and backward: the weight is frozen, so a backward has the inputs' gradient only.
#include "elements.h"

namespace {

constexpr int kGroup = 32;  // elements of a scale

using f32x2 = float __attribute__((ext_vector_type(2)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using bf16x2 = bf16 __attribute__((ext_vector_type(2)));
using f16x2 = f16 __attribute__((ext_vector_type(2)));
using bf16x8 = bf16 __attribute__((ext_vector_type(8)));
using f16x8 = f16 __attribute__((ext_vector_type(8)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

// 2^(byte - 127); 255 is NaN.
__device__ inline float scale_of(uint32_t byte) {
  const uint32_t bits = byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23;
  return __builtin_bit_cast(float, bits);
}

// ------------------------------------------------------------------------------------------
// 4 lanes a group, 8 elements each.  The scale 2^e: e the least with max <= 7 * 2^e, so that what lies between 6 and 7 goes to 6, as near
// as a next value 8 would let it; from the bits of the largest magnitude m 2^p, 1 <= m < 2: e = p - 2 up to m = 1.75, else p - 1.  Within
// [-125, 125], where every value is a normal number of 32 bits.  A group with an infinity or a NaN gets the scale NaN.
template <typename T>
__global__ __launch_bounds__(256) void k_quantize(int64_t rows, int64_t cols, int64_t groups, const T* __restrict__ w, int64_t ldw,
                                                  uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t all = rows * groups * 4;
  for (int64_t t = blockIdx.x * 256ll + threadIdx.x; t < all; t += gridDim.x * 256ll) {  // whole groups: 256 and `all` are multiples of 4
    const int64_t row = t / (groups * 4), q = t % (groups * 4), c = q * 8;
    const int n = cols - c >= 8 ? 8 : cols - c > 0 ? (int)(cols - c) : 0;
    float v[8];
    load8(v, w + row * ldw + c, n == 8, n);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
    most = max(most, (uint32_t)__shfl_xor((int)most, 1));
    most = max(most, (uint32_t)__shfl_xor((int)most, 2));
    int e = (int)(most >> 23) - 127 - ((most & 0x7fffffu) <= 0x600000u ? 2 : 1);
    e = e < -125 ? -125 : e > 125 ? 125 : e;
    const bool finite = most < 0x7f800000u;
    const float inverse = finite ? __builtin_bit_cast(float, (uint32_t)(127 - e) << 23) : 0.0f;
    uint32_t code = 0;
    if (finite) {
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[0] * inverse, v[1] * inverse, 1.0f, 0);
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[2] * inverse, v[3] * inverse, 1.0f, 1);
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[4] * inverse, v[5] * inverse, 1.0f, 2);
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[6] * inverse, v[7] * inverse, 1.0f, 3);
    }
    *(uint32_t*)(codes + row * groups * 16 + q * 4) = code;
    if ((q & 3) == 0) scales[row * groups + q / 4] = finite ? (uint8_t)(e + 127) : (uint8_t)255;
  }
}

// 8 values a thread, times their scale in 32 bits and rounded to T.
template <typename T>
__global__ __launch_bounds__(256) void k_dequantize(int64_t rows, int64_t cols, int64_t groups, const uint8_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, T* __restrict__ w) {
  const int64_t across = (cols + 7) / 8, all = rows * across;
  for (int64_t t = blockIdx.x * 256ll + threadIdx.x; t < all; t += gridDim.x * 256ll) {
    const int64_t row = t / across, q = t % across, c = q * 8;
    const int n = cols - c >= 8 ? 8 : (int)(cols - c);
    const uint32_t code = *(const uint32_t*)(codes + row * groups * 16 + q * 4);
    const float scale = scale_of(scales[row * groups + q / 4]);
    const f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 3)};
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j / 2][j % 2] * scale;
    store8(w + row * cols + c, v, n == 8, n);
  }
}

// ------------------------------------------------------------------------------------------

// 8 codes times a scale as an operand of the matrix instructions.
template <typename T>
__device__ inline Vec<T, 8> operand8(uint32_t code, float scale) {
  Vec<T, 8> v;
  if constexpr (std::is_same_v<T, bf16>) {
    const bf16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 3)};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j / 2][j % 2];
  } else if constexpr (std::is_same_v<T, f16>) {
    const f16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, scale, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, scale, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, scale, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, scale, 3)};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j / 2][j % 2];
  } else {
    const f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, scale, 3)};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j / 2][j % 2];
  }
  return v;
}

template <typename T>
struct Few {
  int64_t M, N, K, groups;
  const T* x;
  int64_t ldx;
  const uint8_t *codes, *scales;
  const T *bias, *residual;
  int64_t ldr;
  T* y;
};

// The product of at most 16 G rows.  A workgroup takes 16 output columns (gated: 16 of the value's and of the gate's), its waves
// interleaved chunks of 4 groups along k.  A lane loads 16 bytes, one group of W's row (lane % 16), which are the operands of 4
// matrix instructions 16 x 16 x 32: k may be summed in any order as long as x's operands have the same one, so lane / 16 chooses a group
// of the chunk and the instruction 8 elements in each.  32-bit operands are multiplied as such (16 x 16 x 4).  The waves' sums meet in LDS.
template <typename T, int ACT, int G>
__global__ __launch_bounds__(1024) void k_q4_few(Few<T> a) {
  constexpr int H = ACT == GF_ACT_NONE ? 1 : 2;
  __shared__ float sums[16][H][G][16][16 + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t n0 = blockIdx.x * 16ll;
  const int64_t n = n0 + (lane & 15) < a.N ? n0 + (lane & 15) : a.N - 1;
  const uint8_t *pc[H], *ps[H];
  const T* px[G];
#pragma unroll
  for (int h = 0; h < H; ++h) pc[h] = a.codes + (n + h * a.N) * a.groups * 16, ps[h] = a.scales + (n + h * a.N) * a.groups;
#pragma unroll
  for (int g = 0; g < G; ++g) px[g] = a.x + (16 * g + (lane & 15) < a.M ? 16 * g + (lane & 15) : a.M - 1) * a.ldx;
  f32x4 acc[H][G] = {};
  for (int64_t at = (int64_t)wave * 4 + (lane >> 4); at - (lane >> 4) < a.groups; at += waves * 4) {
    const bool in = at < a.groups;
    u32x4 code[H];
    float scale[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      code[h] = in ? *(const u32x4*)(pc[h] + at * 16) : u32x4{0, 0, 0, 0};
      scale[h] = in ? scale_of(ps[h][at]) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t k = at * 32 + j * 8;
      const int left = a.K - k >= 8 ? 8 : a.K - k > 0 ? (int)(a.K - k) : 0;
      Vec<T, 8> x[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (left == 8) {
          x[g] = *(const Vec<T, 8>*)(px[g] + k);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[g][i] = i < left ? px[g][k + i] : (T)0.0f;
        }
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const Vec<T, 8> w = operand8<T>(code[h][j], scale[h]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if constexpr (std::is_same_v<T, float>) {
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[h][g] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i], x[g][i], acc[h][g], 0, 0, 0);
          } else if constexpr (std::is_same_v<T, f16>) {
            acc[h][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x[g]), acc[h][g], 0, 0, 0);
          } else {
            acc[h][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x[g]), acc[h][g], 0, 0, 0);
          }
        }
      }
    }
  }
  // Lane l has row l % 16 of each 16 and columns 4 (l / 16) .. + 4.
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][h][g][lane & 15][4 * (lane >> 4) + r] = acc[h][g][r];
  __syncthreads();
  for (int t = threadIdx.x; t < G * 256; t += blockDim.x) {
    const int64_t m = t / 16, col = n0 + t % 16;
    if (m >= a.M || col >= a.N) continue;
    float v[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      v[h] = 0.0f;
      for (int i = 0; i < waves; ++i) v[h] += sums[i][h][t / 256][t / 16 % 16][t % 16];
      if (a.bias != nullptr) v[h] += (float)a.bias[col + h * a.N];
    }
    if constexpr (H == 2) v[0] *= activation<ACT>(v[1], nullptr);
    if (a.residual != nullptr) v[0] += (float)a.residual[m * a.ldr + col];
    a.y[m * a.N + col] = (T)v[0];
  }
}

// ------------------------------------------------------------------------------------------
// Host.

int64_t groups_of(int64_t cols) { return (cols + kGroup - 1) / kGroup; }
int64_t weight_rows(const gf_q4_args& a) { return a.out_features * (a.activation == GF_ACT_NONE ? 1 : 2); }

int check_weight(int64_t rows, int64_t cols, const void* codes, const void* scales) {
  if (rows < 0 || cols <= 0 || rows > kMaxSize || cols > kMaxSize / 2) return fail(GF_E_INVALID_ARGUMENT, "rows or cols of the weight negative or too large");
  if (rows != 0 && round_up(cols, kGroup) > kMaxElements / rows) return fail(GF_E_INVALID_ARGUMENT, "weight: too large");
  if (rows == 0) return GF_OK;
  if (codes == nullptr || scales == nullptr) return fail(GF_E_INVALID_ARGUMENT, "codes and scales must not be NULL");
  if ((uintptr_t)codes % 16 != 0) return fail(GF_E_INVALID_ARGUMENT, "codes must be 16-byte aligned");
  return GF_OK;
}

int check_args(const gf_q4_args* a) {
  if (a == nullptr) return fail(GF_E_INVALID_ARGUMENT, "args must not be NULL");
  GF_TRY(check_dtype(a->dtype));
  if (a->activation < GF_ACT_NONE || a->activation > GF_ACT_SILU) return fail(GF_E_INVALID_ARGUMENT, "unknown activation %d", (int)a->activation);
  if (a->rows < 0 || a->in_features <= 0 || a->out_features <= 0)
    return fail(GF_E_INVALID_ARGUMENT, "rows must not be negative and in_features and out_features must be positive");
  if (a->rows > kMaxSize || a->in_features > kMaxSize / 2 || a->out_features > kMaxSize / 4)
    return fail(GF_E_INVALID_ARGUMENT, "rows, in_features or out_features too large");
  if (std::max(a->rows, weight_rows(*a)) * round_up(a->in_features, kGroup) > kMaxElements || a->rows * weight_rows(*a) > kMaxElements)
    return fail(GF_E_INVALID_ARGUMENT, "rows, in_features or out_features too large");
  for (const int64_t ld : {a->ldx, a->ldr, a->lddy})
    if (ld > kMaxElements || ld < -kMaxElements) return fail(GF_E_INVALID_ARGUMENT, "row stride too large");
  return GF_OK;
}

// The same product with the weight's values, as the feed-forward entries take it.
gf_ff_args dense(const gf_q4_args& a, const void* weight) {
  gf_ff_args f{};
  f.dtype = a.dtype, f.activation = a.activation, f.rows = a.rows, f.in_features = a.in_features, f.out_features = a.out_features;
  f.x = a.x, f.ldx = a.ldx, f.weight = weight, f.ldw = a.in_features, f.bias = a.bias, f.residual = a.residual, f.ldr = a.ldr;
  f.y = a.y, f.saved = a.saved, f.dy = a.dy, f.lddy = a.lddy, f.dx = a.dx, f.dbias = a.dbias;
  return f;
}

bool few(const gf_q4_args& a) { return a.rows <= 64 && a.saved == nullptr; }

template <typename T>
int dequantize(int64_t rows, int64_t cols, const void* codes, const void* scales, void* out, hipStream_t s) {
  const int64_t groups = groups_of(cols);
  k_dequantize<T><<<blocks_for(rows * ((cols + 7) / 8)), 256, 0, s>>>(rows, cols, groups, (const uint8_t*)codes, (const uint8_t*)scales, (T*)out);
  GF_LAUNCH_CHECK("k_dequantize");
  return GF_OK;
}

// The values of the weight at the workspace's start, then the feed-forward entry's own.
int through_dense(const gf_q4_args& a, bool is_backward, Arena& ws, bool run, hipStream_t s) {
  void* const weight = ws.take(weight_rows(a) * a.in_features * size_of(a.dtype));
  const gf_ff_args f = dense(a, run ? weight : (void*)256);  // its alignment counts
  const size_t bytes = gf_ff_workspace_bytes(&f, is_backward);
  void* const rest = ws.take((int64_t)bytes);
  GF_RUN {
    GF_TRY(with_dtype(a.dtype, [&](auto t) { return dequantize<decltype(t)>(weight_rows(a), a.in_features, a.codes, a.scales, weight, s); }));
    return is_backward ? gf_ff_backward(&f, rest, bytes, s) : gf_ff_forward(&f, rest, bytes, s);
  }
  return GF_OK;
}

int run_few(const gf_q4_args& a, hipStream_t s) {
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_activation(a.activation, [&](auto act) {
      constexpr int ACT = act.value;
      const int64_t groups = groups_of(a.in_features);
      const Few<T> f{a.rows, a.out_features, a.in_features, groups, (const T*)a.x, a.ldx, (const uint8_t*)a.codes, (const uint8_t*)a.scales, (const T*)a.bias,
                     (const T*)a.residual, a.ldr, (T*)a.y};
      const dim3 grid((unsigned)((a.out_features + 15) / 16));
      const unsigned threads = groups >= 16 * 4 ? 1024 : 512;
      auto* kernel = a.rows <= 16 ? k_q4_few<T, ACT, 1> : a.rows <= 32 ? k_q4_few<T, ACT, 2> : k_q4_few<T, ACT, 4>;
      kernel<<<grid, threads, 0, s>>>(f);
      GF_LAUNCH_CHECK("k_q4_few");
      return (int)GF_OK;
    });
  });
}

}  // namespace

extern "C" {

int gf_q4_quantize(int32_t dtype, int64_t rows, int64_t cols, const void* weight, int64_t ldw, void* codes, void* scales, void* stream) {
  GF_TRY(check_dtype(dtype));
  GF_TRY(check_weight(rows, cols, codes, scales));
  if (rows == 0) return GF_OK;
  GF_TRY(check_matrix("weight", weight, rows, ldw, cols, size_of(dtype)));
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t groups = groups_of(cols);
    k_quantize<T><<<blocks_for(rows * groups * 4), 256, 0, (hipStream_t)stream>>>(rows, cols, groups, (const T*)weight, ldw, (uint8_t*)codes,
                                                                                 (uint8_t*)scales);
    GF_LAUNCH_CHECK("k_quantize");
    return (int)GF_OK;
  });
}

int gf_q4_dequantize(int32_t dtype, int64_t rows, int64_t cols, const void* codes, const void* scales, void* weight, void* stream) {
  GF_TRY(check_dtype(dtype));
  GF_TRY(check_weight(rows, cols, codes, scales));
  if (rows == 0) return GF_OK;
  GF_TRY(check_matrix("weight", weight, rows, cols, cols, size_of(dtype)));
  return with_dtype(dtype, [&](auto t) { return dequantize<decltype(t)>(rows, cols, codes, scales, weight, (hipStream_t)stream); });
}

size_t gf_q4_saved_bytes(const gf_q4_args* args) {
  if (check_args(args) != GF_OK) return 0;
  const gf_ff_args f = dense(*args, (void*)256);
  return gf_ff_saved_bytes(&f);
}

size_t gf_q4_workspace_bytes(const gf_q4_args* args, int32_t backward) {
  if (check_args(args) != GF_OK || args->rows == 0 || (!backward && few(*args))) return 0;
  Arena count{nullptr};
  return through_dense(*args, backward != 0, count, false, nullptr) == GF_OK ? count.used : 0;
}

int gf_q4_forward(const gf_q4_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  GF_TRY(check_args(args));
  const gf_q4_args& a = *args;
  if (a.rows == 0) return GF_OK;
  const int size = size_of(a.dtype);
  GF_TRY(check_weight(weight_rows(a), a.in_features, a.codes, a.scales));
  GF_TRY(check_matrix("x", a.x, a.rows, a.ldx, a.in_features, size));
  GF_TRY(check_matrix("y", a.y, a.rows, a.out_features, a.out_features, size));
  if (a.bias != nullptr) GF_TRY(check_matrix("bias", a.bias, 1, weight_rows(a), weight_rows(a), size));
  if (a.residual != nullptr) {
    if (a.activation != GF_ACT_NONE) return fail(GF_E_INVALID_ARGUMENT, "a gated product takes no residual");
    GF_TRY(check_matrix("residual", a.residual, a.rows, a.ldr, a.out_features, size));
  }
  if (a.saved != nullptr) GF_TRY(check_matrix("saved", a.saved, 1, 1, 1, 16));
  if (few(a)) return run_few(a, (hipStream_t)stream);
  Arena count{nullptr}, ws{(uint8_t*)workspace};
  GF_TRY(through_dense(a, false, count, false, nullptr));
  GF_TRY(check_workspace(count.used, workspace, workspace_bytes));
  return through_dense(a, false, ws, true, (hipStream_t)stream);
}

int gf_q4_backward(const gf_q4_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  GF_TRY(check_args(args));
  const gf_q4_args& a = *args;
  if (a.rows == 0) return fail(GF_E_INVALID_ARGUMENT, "a backward needs rows");
  const int size = size_of(a.dtype);
  GF_TRY(check_weight(weight_rows(a), a.in_features, a.codes, a.scales));
  GF_TRY(check_matrix("dy", a.dy, a.rows, a.lddy, a.out_features, size));
  if (a.activation != GF_ACT_NONE) GF_TRY(check_matrix("saved", a.saved, 1, 1, 1, 16));
  Arena count{nullptr}, ws{(uint8_t*)workspace};
  gf_q4_args b = a;
  b.x = a.dy, b.ldx = a.in_features;  // the weight's gradient is not asked for, so x is not read
  GF_TRY(through_dense(b, true, count, false, nullptr));
  GF_TRY(check_workspace(count.used, workspace, workspace_bytes));
  return through_dense(b, true, ws, true, (hipStream_t)stream);
}

}  // extern "C"
