// quantized.hip - gfx950 kernels and C ABI of weights in 4 bits: a weight into codes and scales, back, and products with it.
//
//   k_quantize    groups of 32 of a row: a power of two for a scale, and the nearest of the 16 values e2m1 has
//   k_dequantize  the values that codes and scales stand for, in a type of 16 or 32 bits
//   k_q4_few      the product of few rows: codes straight into the matrix instructions' operands
//   k_column_sums, k_column_join  a linear product's bias's gradient
//
// A group's scale being a power of two, a weight's value is exact in bfloat16 (sign, 2 bits of fraction), and in float16 as long as the
// scale is not extreme: the matrix cores get it without a rounding of its own.  The hardware turns two codes into two values of a
// scale in one instruction.  More rows go through k_dequantize and the feed-forward products (feedforward.hip), forward
// and backward: the weight is frozen, so a backward has the inputs' gradient only.
//
// Times at the kernels are medians within whole passes on two states in turn, under a profiler; those that compare two forms are of one call
// repeated, whose inputs the caches may partly hold.
#include "elements.h"

namespace {

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
// The layout: tiles of 16 rows x 128 columns, a band of 16 rows after another, a tile as k_q4_few's lanes take it.  A word holds 8 codes,
// the first lowest; lane q * 16 + row of a tile has the four words of columns 32 j + 8 q (j = 0..3) side by side: what it multiplies by in
// four matrix instructions, whose operands are 8 columns from each sixteen lanes.  So a wave reads a tile as 1024 bytes in a row.  The
// tile's scales: a word a row, a byte for each group of 32.  Codes past the matrix are zero.

constexpr int kTileCodes = 1024, kTileScales = 64;

// Where word `w` (columns 8 w..) of a row lies within its tile, in words.
__device__ inline int word_of(int row, int w) { return ((w & 3) * 16 + row) * 4 + (w >> 2); }

// A tile a workgroup and turn: 16 lanes a row, 8 elements each, four lanes a group.  The scale 2^e: e the least with max <= 7 * 2^e, so that
// what lies between 6 and 7 goes to 6, as near as a next value 8 would let it; from the bits of the largest magnitude m 2^p, 1 <= m < 2:
// e = p - 2 up to m = 1.75, else p - 1.  Within [-125, 125], where every value is a normal number of 32 bits.  A group with an infinity or a
// NaN gets the scale NaN.  The words change places in LDS, so that both sides of memory are read and written in a row.  Bound by memory: 10240 x
// 1280 in 32 bits 11 us (5.4 TB/s); repeated, 8192 x 8192 in bfloat16 33 us (5.1 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void k_quantize(int64_t rows, int64_t cols, int64_t across, int64_t tiles, const T* __restrict__ w, int64_t ldw,
                                                  uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  __shared__ uint32_t words[2][256];
  const int r = threadIdx.x >> 4, q = threadIdx.x & 15;
  int slot = 0;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, slot ^= 1) {
    const int64_t row = tile / across * 16 + r, c = tile % across * 128 + q * 8;
    const int n = row >= rows || cols <= c ? 0 : cols - c >= 8 ? 8 : (int)(cols - c);
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
    words[slot][word_of(r, q)] = code;  // the other half is read in the turn before, whose barrier lies behind
    if ((q & 3) == 0) scales[tile * kTileScales + r * 4 + q / 4] = finite ? (uint8_t)(e + 127) : (uint8_t)255;
    __syncthreads();
    codes[tile * (kTileCodes / 4) + threadIdx.x] = words[slot][threadIdx.x];
  }
}

// A tile a workgroup and turn, 8 values a thread, times their scale in 32 bits and rounded to T.  The next tile's words are on their way
// while one is written.  Bound by memory: 10240 x 1280 into bfloat16 9.0 us (3.7 TB/s), into 32 bits 13 us (4.5 TB/s); repeated, 8192 x 8192
// into bfloat16 34 us (5.0 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void k_dequantize(int64_t rows, int64_t cols, int64_t across, int64_t tiles, const uint32_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, T* __restrict__ w) {
  __shared__ uint32_t words[2][256];
  const int r = threadIdx.x >> 4, q = threadIdx.x & 15;
  int slot = 0;
  uint32_t word = 0, byte = 0;
  auto fetch = [&](int64_t tile) {
    word = codes[tile * (kTileCodes / 4) + threadIdx.x], byte = scales[tile * kTileScales + r * 4 + q / 4];
  };
  if (blockIdx.x < tiles) fetch(blockIdx.x);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, slot ^= 1) {
    const int64_t row = tile / across * 16 + r, c = tile % across * 128 + q * 8;
    const int n = row >= rows || cols <= c ? 0 : cols - c >= 8 ? 8 : (int)(cols - c);
    words[slot][threadIdx.x] = word;
    const float scale = scale_of(byte);
    if (tile + gridDim.x < tiles) fetch(tile + gridDim.x);
    __syncthreads();
    const uint32_t code = words[slot][word_of(r, q)];
    const f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 3)};
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j / 2][j % 2] * scale;
    if (n > 0) store8(w + row * cols + c, v, n == 8, n);
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
  int64_t M, N, K, across;  // across: tiles of a band
  const T* x;
  int64_t ldx;
  const uint8_t *codes, *scales;
  const T *bias, *residual;
  int64_t ldr;
  T* y;
  int act;
};

// The product of 16 G rows a workgroup (y).  It takes 16 NT output columns (gated: as many of the value's and of the gate's), its waves
// the tiles along k in turn, and the waves' sums meet in LDS.  Bound by reading the codes, so two tiles of them are under way at a time, and by x,
// which every workgroup reads: NT halves that where there are columns enough.
//
// x's operands are 8 columns of row lane % 16 from each sixteen lanes.  Loaded as such, neighbouring lanes would ask for different lines
// of memory, 64 a load.  Of more than 4 rows a wave loads them row by row, 16 lanes and 256 bytes each, and passes them through its own
// piece of LDS, 16 bytes at a time, at place p ^ row of a row's 16 so that neither side's lanes meet in a bank.  The hardware keeps a wave's
// LDS operations in their order, so it takes no barrier of the workgroup; that the compiler keeps it, a fence says.  Up to 4 rows (DIRECT)
// the lanes that have one load it themselves.  32-bit operands are multiplied as such (16 x 16 x 4).
template <typename T, int G>
constexpr int kFewWaves = G == 1 ? 16 : G * (int)sizeof(T) >= 16 ? 4 : 8;  // as registers allow

// What lanes of a wave have written to LDS before, others of it read after, and the other way round.  No instruction.
__device__ __attribute__((always_inline)) inline void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

template <typename T, int H, int G, int NT, bool DIRECT>
__global__ __launch_bounds__((kFewWaves<T, G> * 64)) void k_q4_few(Few<T> a) {
  constexpr int R = H * NT, W = kFewWaves<T, G>, S = (int)sizeof(T), E = 16 / S, P = 8 * S;  // P pieces of E elements in a row of a tile
  constexpr int kSums = W * R * G * 16 * 17 * 4, kStage = DIRECT ? 0 : W * G * 16 * P * 16;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kSums > kStage ? kSums : kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, quarter = lane >> 4;
  const int64_t n0 = blockIdx.x * (16ll * NT), m0 = blockIdx.y * (16ll * G);
  a.M -= m0, a.x += m0 * a.ldx, a.y += m0 * a.N, a.residual += a.residual != nullptr ? m0 * a.ldr : 0;
  using Piece = Vec<T, E>;
  const uint8_t *pc[R], *ps[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t n = n0 + r / H * 16 + (lane & 15);
    const int64_t row = (n < a.N ? n : a.N - 1) + r % H * a.N;
    pc[r] = a.codes + row / 16 * a.across * kTileCodes + (quarter * 16 + row % 16) * 16;
    ps[r] = a.scales + row / 16 * a.across * kTileScales + row % 16 * 4;
  }
  const int64_t whole = a.K / 128;  // tiles
  f32x4 acc[R][G] = {};
  struct Codes {
    u32x4 words[R];
    uint32_t scales[R];  // of the four groups, a byte each
  };
  auto load = [&](Codes& c, int64_t at) {
#pragma unroll
    for (int r = 0; r < R; ++r) c.words[r] = *(const u32x4*)(pc[r] + at * kTileCodes), c.scales[r] = *(const uint32_t*)(ps[r] + at * kTileScales);
  };
  // x's part of a tile: 16 G rows of P pieces, 64 / P rows a load
  constexpr int kLoads = DIRECT ? 4 * 8 / E : G * P / 4;
  struct Part {
    Piece x[kLoads];
  };
  auto x_row = [&](int i) { return DIRECT ? lane & 15 : i * (64 / P) + lane / P; };
  auto x_col = [&](int i) { return DIRECT ? i / (8 / E) * 32 + quarter * 8 + i % (8 / E) * E : lane % P * E; };
  auto load_x = [&](Part& c, int64_t at) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      c.x[i] = (T)0.0f;
      if (x_row(i) < a.M) c.x[i] = *(const Piece*)(a.x + x_row(i) * a.ldx + at * 128 + x_col(i));
    }
  };
  uint8_t* const stage = lds + wave * (kStage / W);
  // the next tile's part of x is asked for once this one's has left its registers
  auto multiply = [&](const Codes& c, Part& part, int64_t next) {
    const Part here = part;
    if constexpr (!DIRECT) {
      wave_fence();  // the tile before is read
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        *(Piece*)__builtin_assume_aligned(stage + (x_row(i) * P + ((lane % P) ^ (x_row(i) % 16 * (P / 16)))) * 16, 16) = here.x[i];
      wave_fence();
    }
    if (next < whole) load_x(part, next);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Vec<T, 8> b[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int h = 0; h < 8 / E; ++h) {
          const int m = g * 16 + (lane & 15), p = (j * 4 + quarter) * (8 / E) + h;
          const Piece v = DIRECT ? here.x[j * (8 / E) + h] : *(const Piece*)__builtin_assume_aligned(stage + (m * P + (p ^ (m % 16 * (P / 16)))) * 16, 16);
#pragma unroll
          for (int e = 0; e < E; ++e) b[g][h * E + e] = v[e];
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Vec<T, 8> w = operand8<T>(c.words[r][j], scale_of(c.scales[r] >> 8 * j & 255u));
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if constexpr (std::is_same_v<T, float>) {
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[r][g] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i], b[g][i], acc[r][g], 0, 0, 0);
          } else if constexpr (std::is_same_v<T, f16>) {
            acc[r][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, b[g]), acc[r][g], 0, 0, 0);
          } else {
            acc[r][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, b[g]), acc[r][g], 0, 0, 0);
          }
        }
      }
    }
  };
  Codes c[2];
  Part part;
  if (wave < a.across) load(c[0], wave);
  if (wave + waves < a.across) load(c[1], wave + waves);
  if (wave < whole) load_x(part, wave);
  int64_t at = wave;
  for (; at < whole; at += waves) {
    multiply(c[0], part, at + waves);
    c[0] = c[1];
    if (at + 2 * waves < a.across) load(c[1], at + 2 * waves);
  }
  if (at < a.across) {  // the part of a tile, at the wave whose turn it is
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      for (int e = 0; e < E; ++e) {
        const int64_t k = at * 128 + x_col(i) + e;
        part.x[i][e] = x_row(i) < a.M && k < a.K ? a.x[x_row(i) * a.ldx + k] : (T)0.0f;
      }
    multiply(c[0], part, whole);
  }
  // Lane l has row l % 16 of each 16 and columns 4 (l / 16) .. + 4.
  auto sums = (float(*)[R][G][16][17])lds;
  if constexpr (!DIRECT) __syncthreads();  // the staged rows are read
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][r][g][lane & 15][4 * quarter + i] = acc[r][g][i];
  __syncthreads();
  for (int t = threadIdx.x; t < NT * G * 256; t += blockDim.x) {
    const int64_t m = t / 16 % (16 * G), col = n0 + t / (256 * G) * 16 + t % 16;
    if (m >= a.M || col >= a.N) continue;
    float v[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      v[h] = 0.0f;
      for (int i = 0; i < waves; ++i) v[h] += sums[i][t / (256 * G) * H + h][m / 16][m % 16][t % 16];
      if (a.bias != nullptr) v[h] += (float)a.bias[col + h * a.N];
    }
    if constexpr (H == 2)
      v[0] *= a.act == GF_ACT_GELU   ? activation<GF_ACT_GELU>(v[1], nullptr)
              : a.act == GF_ACT_SILU ? activation<GF_ACT_SILU>(v[1], nullptr)
                                     : activation<GF_ACT_GELU_TANH>(v[1], nullptr);
    if (a.residual != nullptr) v[0] += (float)a.residual[m * a.ldr + col];
    a.y[m * a.N + col] = (T)v[0];
  }
}

// ------------------------------------------------------------------------------------------
// The bias's gradient of a linear product, the columns' sums of dy: 8 columns a thread, a chunk of rows a workgroup (y), then the chunks in
// their order.  Bound by reading dy: 8192 x 10240 in bfloat16 41 + 5 us in a training pass (3.7 TB/s), repeated 34 in all (5.0 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void k_column_sums(int64_t rows, int64_t cols, int64_t chunk, const T* __restrict__ dy, int64_t ld, float* __restrict__ sums,
                                                     int64_t width) {
  const int64_t c = (blockIdx.x * 256ll + threadIdx.x) * 8, begin = blockIdx.y * chunk, end = begin + chunk < rows ? begin + chunk : rows;
  if (c >= cols) return;
  const int n = cols - c >= 8 ? 8 : (int)(cols - c);
  float s[8] = {};
  int64_t row = begin;
  if (n == 8) {
    constexpr int kAtOnce = 8, E = 16 / sizeof(T);
    using V = Vec<T, E>;
    for (; row + kAtOnce <= end; row += kAtOnce) {
      V v[kAtOnce][8 / E];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int h = 0; h < 8 / E; ++h) v[i][h] = *(const V*)(dy + (row + i) * ld + c + h * E);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += (float)v[i][j / E][j % E];
    }
  }
  for (; row < end; ++row) {
    float v[8];
    load8(v, dy + row * ld + c, n == 8, n);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += v[j];
  }
  store8(sums + blockIdx.y * width + c, s, true, 8);
}

template <typename T>
__global__ __launch_bounds__(256) void k_column_join(int64_t chunks, int64_t cols, const float* __restrict__ sums, int64_t width, T* __restrict__ out) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t i = line; i < chunks; i += 8) s += sums[i * width + c];
  }
  part[line][lane] = s;
  __syncthreads();
  if (line != 0 || c >= cols) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += part[i][lane];
  out[c] = (T)s;
}

// ------------------------------------------------------------------------------------------
// Host.

int64_t bands_of(int64_t rows) { return (rows + 15) / 16; }
int64_t across_of(int64_t cols) { return (cols + 127) / 128; }
// 8 workgroups a unit: 10240 x 1280 into bfloat16, repeated, 7.7 us (16384 workgroups, a tile each: 8.2; 1024: 8.3)
unsigned tile_blocks(int64_t tiles) { return (unsigned)std::min<int64_t>(tiles, 2048); }
int64_t weight_rows(const gf_q4_args& a) { return a.out_features * (a.activation == GF_ACT_NONE ? 1 : 2); }

int check_weight(int64_t rows, int64_t cols, const void* codes, const void* scales) {
  if (rows < 0 || cols <= 0 || rows > kMaxSize || cols > kMaxSize / 2) return fail(GF_E_INVALID_ARGUMENT, "rows or cols of the weight negative or too large");
  if (rows != 0 && round_up(cols, 128) > kMaxElements / rows) return fail(GF_E_INVALID_ARGUMENT, "weight: too large");
  if (rows == 0) return GF_OK;
  if (codes == nullptr || scales == nullptr) return fail(GF_E_INVALID_ARGUMENT, "codes and scales must not be NULL");
  if ((uintptr_t)codes % 16 != 0 || (uintptr_t)scales % 4 != 0)
    return fail(GF_E_INVALID_ARGUMENT, "codes must be 16-byte aligned, scales 4-byte");
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
  if (std::max(a->rows, weight_rows(*a)) * round_up(a->in_features, 128) > kMaxElements || a->rows * weight_rows(*a) > kMaxElements)
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

// By the codes up to 128 rows, 64 at a time, whatever the size: one border, where either way loses somewhere.  128 rows, through the values
// and by the codes, repeated: in bfloat16 8192 -> 8192 66 and 40 us, 1280 -> 5120 gated 31 and 19, 320 -> 2560 gated 12 and 16; in 32 bits 332 and 197, 62
// and 66, 28 and 25: of these six, small gated weights lose 4 us by the codes.
bool few(const gf_q4_args& a) { return a.rows <= 128 && a.saved == nullptr; }

template <typename T>
int dequantize(int64_t rows, int64_t cols, const void* codes, const void* scales, void* out, hipStream_t s) {
  const int64_t across = across_of(cols), tiles = bands_of(rows) * across;
  k_dequantize<T><<<tile_blocks(tiles), 256, 0, s>>>(rows, cols, across, tiles, (const uint32_t*)codes, (const uint8_t*)scales, (T*)out);
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

// A workgroup a unit, since every chunk is read back to be joined: repeated, 8192 x 10240 34 us, 8192 x 1280 8.4 and 1000 x 5120 7.9; with
// four 35, 14 and 9.0.  Not compared within a training pass.
int column_sums(const gf_q4_args& a, Arena& ws, bool run, hipStream_t s) {
  const int64_t across = (a.out_features + 2047) / 2048, width = round_up(a.out_features, 8);
  const int64_t want = std::max<int64_t>(std::min<int64_t>(256 / across, a.rows / 8), 1), chunk = (a.rows + want - 1) / want, chunks = (a.rows + chunk - 1) / chunk;
  float* const sums = (float*)ws.take(chunks * width * 4);
  GF_RUN return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    k_column_sums<T><<<dim3((unsigned)across, (unsigned)chunks), 256, 0, s>>>(a.rows, a.out_features, chunk, (const T*)a.dy, a.lddy, sums, width);
    GF_LAUNCH_CHECK("k_column_sums");
    k_column_join<T><<<(unsigned)((a.out_features + 31) / 32), 256, 0, s>>>(chunks, a.out_features, sums, width, (T*)a.dbias);
    GF_LAUNCH_CHECK("k_column_join");
    return (int)GF_OK;
  });
  return GF_OK;
}

// A linear product's bias by its own kernel; the rest through the weight's values.
int backward(const gf_q4_args& a, Arena& ws, bool run, hipStream_t s) {
  gf_q4_args b = a;
  b.x = a.dy, b.ldx = a.in_features;  // the weight's gradient is not asked for, so x is not read
  if (a.activation == GF_ACT_NONE) {
    if (a.dbias != nullptr) GF_TRY(column_sums(a, ws, run, s));
    b.dbias = nullptr;
    if (a.dx == nullptr) return GF_OK;
  }
  return through_dense(b, true, ws, run, s);
}

template <typename T, int H, int G, bool DIRECT>
int launch_few(const Few<T>& f, bool wide, hipStream_t s) {
  // 32 columns a workgroup where that still makes one for each of 256 compute units: of 8192 -> 8192 in bfloat16, repeated, one row takes 10.6 us
  // (16 columns: 11.8), 64 rows 22.6 (36).  16 waves up to a workgroup a unit, else 8, of which two are at work on a unit: 5120 -> 1280 4.5 us
  // (8 waves: 5.3), 4096 -> 14336 9.6 (16: 11.3), 1280 -> 5120 gated 5.1 (16: 5.9).
  const int64_t cols = wide ? 32 : 16, groups = (f.N + cols - 1) / cols;
  const unsigned waves = (unsigned)std::min<int64_t>(f.across, std::min(kFewWaves<T, G>, groups <= 256 ? 16 : 8));
  const unsigned blocks = (unsigned)((f.M + 16 * G - 1) / (16 * G));
  if constexpr (H == 1) {
    if (wide) {
      k_q4_few<T, 1, G, 2, DIRECT><<<dim3((unsigned)groups, blocks), waves * 64, 0, s>>>(f);
      GF_LAUNCH_CHECK("k_q4_few");
      return GF_OK;
    }
  }
  k_q4_few<T, H, G, 1, DIRECT><<<dim3((unsigned)groups, blocks), waves * 64, 0, s>>>(f);
  GF_LAUNCH_CHECK("k_q4_few");
  return GF_OK;
}

int run_few(const gf_q4_args& a, hipStream_t s) {
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    const Few<T> f{a.rows, a.out_features, a.in_features, across_of(a.in_features), (const T*)a.x, a.ldx, (const uint8_t*)a.codes, (const uint8_t*)a.scales,
                   (const T*)a.bias, (const T*)a.residual, a.ldr, (T*)a.y, a.activation};
    const bool wide = a.activation == GF_ACT_NONE && f.N >= 32 * 256;
    auto run = [&](auto halves) {
      constexpr int H = halves.value;
      if (f.M <= 4) return launch_few<T, H, 1, true>(f, wide, s);
      if (f.M <= 16) return launch_few<T, H, 1, false>(f, wide, s);
      if (f.M <= 32) return launch_few<T, H, 2, false>(f, wide, s);
      return launch_few<T, H, 4, false>(f, wide, s);
    };
    return a.activation == GF_ACT_NONE ? run(std::integral_constant<int, 1>()) : run(std::integral_constant<int, 2>());
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
    const int64_t across = across_of(cols), tiles = bands_of(rows) * across;
    k_quantize<T><<<tile_blocks(tiles), 256, 0, (hipStream_t)stream>>>(rows, cols, across, tiles, (const T*)weight, ldw, (uint32_t*)codes, (uint8_t*)scales);
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

size_t gf_q4_workspace_bytes(const gf_q4_args* args, int32_t is_backward) {
  if (check_args(args) != GF_OK || args->rows == 0 || (!is_backward && few(*args))) return 0;
  Arena count{nullptr};
  const int rc = is_backward ? backward(*args, count, false, nullptr) : through_dense(*args, false, count, false, nullptr);
  return rc == GF_OK ? count.used : 0;
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
  if (a.dx != nullptr) GF_TRY(check_matrix("dx", a.dx, a.rows, a.in_features, a.in_features, size));
  if (a.dbias != nullptr) GF_TRY(check_matrix("dbias", a.dbias, 1, weight_rows(a), weight_rows(a), size));
  Arena count{nullptr}, ws{(uint8_t*)workspace};
  GF_TRY(backward(a, count, false, nullptr));
  GF_TRY(check_workspace(count.used, workspace, workspace_bytes));
  return backward(a, ws, true, (hipStream_t)stream);
}

}  // extern "C"
