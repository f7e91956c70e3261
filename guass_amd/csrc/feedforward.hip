// feedforward.hip - gfx950 kernels and C ABI of the feed-forward block around the adapted linears:
// dropout from a counter, the gated projection and the projection back, each with its backward.
//
//   k_dropout   residual + drop(x)
//   k_few       the forward of at most 64 rows: W read once, no LDS for operands
//   k_product   every other product, on the matrix cores, its epilogue fused (bias, activation, dropout, residual)
//   k_join      adds the parts of a product that was split along k, with the same epilogue
//   k_dz        the products' gradient from dy (dropout and activation undone) and its column sums
//   k_peak      that gradient's largest element, for its scale (gated, float16)
//   k_pack      32-bit operands into three bfloat16 planes, unaligned 16-bit ones into aligned rows
//   k_join_sums the column sums' chunks
//
// Forward: k_few, or (k_pack,) k_product (, k_join).  Backward: (k_peak,) k_dz (, k_join_sums) (, k_pack), k_product for dx and for
// dW (, k_join each).  No atomics: every sum has one order, so a call's results depend on its inputs alone.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <type_traits>
#include <utility>

#include "elements.h"

namespace {

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
// each round multiplies two counter words by constants and crosses the products' halves.  Its 20 wide products are what it
// costs, so a block serves 8 elements with 16 bits each: of p that is less than 2^-17 off, and the scale is that of the
// share really kept.
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

__device__ inline bool kept(const Drop& d, const uint32_t bits[4], int j) {
  return ((bits[j >> 1] >> (16 * (j & 1))) & 0xffffu) >= d.threshold;
}

__device__ inline float dropped(const Drop& d, const uint32_t bits[4], int j, float v) { return kept(d, bits, j) ? v * d.scale : 0.0f; }

// residual + drop(x), 8 elements of a row a thread and turn.  A thread's next group is a fixed number of groups on, whole
// rows and a rest of columns, so that nothing is divided in the loop.  Bound by memory: 32768 x 2560 bfloat16 60 us a pass
// (5.6 TB/s); 64 x 1280 3 us, a launch.
template <typename T, bool RESIDUAL>
__global__ __launch_bounds__(256) void k_dropout(Drop d, int64_t rows, int64_t cols, const T* __restrict__ x, int64_t ldx,
                                                 const T* __restrict__ res, int64_t ldr, T* __restrict__ y, int64_t ldy) {
  load_key(d);
  const uint32_t groups = (uint32_t)((cols + 7) / 8);
  const int64_t first = blockIdx.x * 256ll + threadIdx.x, all = gridDim.x * 256ll;
  int64_t row = first / groups;
  uint32_t group = (uint32_t)(first % groups);
  const int64_t row_step = all / groups;
  const uint32_t group_step = (uint32_t)(all % groups);
  while (row < rows) {
    const int64_t c = 8ll * group;
    const int n = cols - c < 8 ? (int)(cols - c) : 8;
    float v[8], r[8];
    load8(v, x + row * ldx + c, n == 8, n);
    if constexpr (RESIDUAL) load8(r, res + row * ldr + c, n == 8, n);
    if (d.threshold != 0) {
      uint32_t bits[4];
      random_block(d, (uint32_t)row, group, bits);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = dropped(d, bits, j, v[j]);
    }
    if constexpr (RESIDUAL)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += r[j];
    store8(y + row * ldy + c, v, n == 8, n);
    row += row_step, group += group_step;
    if (group >= groups) group -= groups, ++row;
  }
}

// ------------------------------------------------------------------------------------------
// Products.  C[m, n] = sum over k of P(m, k) Q(n, k) on the matrix cores, accumulated in 32 bits.
//
// A workgroup computes a BM x BN tile, WM x WN waves a TM x TN part each, in steps of 64 (32) along k.  An operand is
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
// so that a lane ends up with 8 consecutive n of one m.
//
// 4096 x 4096 x 8192 in bfloat16 takes 203 us (1.35 PFLOP/s) from operands the caches hold, in all three layouts, and 173 us of
// zeros, whose power leaves a higher clock; 223 us from memory.  Of 8192 x 1280 -> 5120 gated the forward takes 241 to 248 us
// (0.89 PFLOP/s; 294 MB written), dx 202 to 211, dW 184 to 193, by the card.  There the matrix cores are busy for 43, 51 and
// 58% of the cycles, at 1.8 to 1.9 GHz: what fills the rest (each round's first loads, operands from memory, the rounds' stores at
// the same time) was not taken apart.  32 bits:
// 4096 x 4096 x 2048 284 to 344 us by the layouts (0.20 to 0.24 PFLOP/s, six times that on the matrix cores).

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
// matrices come as three such planes of bfloat16 (k_pack, k_dz), `plane` elements apart.
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
  void* saved;  // gated: see Saved
  int64_t saved_ld;
  float* partial;  // not NULL: sums for k_join instead of all of the above, [split][M][N (gated: 2 N), whole groups of 8]
  Drop drop;
  float scale = 1.0f;  // of the sums of a product without activation, before everything else
  const float* scale_at = nullptr;  // where it is read from instead, or NULL
};

__device__ inline float scale_of(const Epilogue& e) { return e.scale_at != nullptr ? *e.scale_at : e.scale; }

struct Shape {
  int64_t M, N, K;      // N: output columns (gated: the value's)
  int32_t tiles_m, tiles_n;
  int32_t splits;       // workgroups along k, `steps` steps of 64 each (the last: what is left)
  int32_t steps;
};

// k that a step takes, and planes that an operand has: 32-bit operands come in three planes and a step of half the length.
template <typename T>
constexpr int kStep = std::is_same_v<T, float> ? 32 : 64;
template <typename T>
constexpr int kPlanes = std::is_same_v<T, float> ? 3 : 1;

// n within 32 of the matrix instruction's row r = 8 a + 4 h + e
__device__ inline int row_of(int r) { return 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3); }

// What a gated forward leaves for its backward: value and gate of [rows, ld], ld whole groups of 8.  In 32 bits two
// planes of floats.  For 16-bit tensors floats of fewer bits, 12 significant ones (bfloat16) or 16 (float16): the upper
// 16 bits of the float in two planes, the bits below them of value and gate together in a third.  A rounding to the
// tensors' own type here would count in dx and dW as much as the two that are needed, of dz and of the result itself
// (1.7 instead of 1.4 roundings); the third plane costs a quarter (half) more bytes than that.  Written past the caches:
// nobody reads it before the backward (16384 x 320 -> 1280: 74 -> 60 us, 8192 x 1280 -> 5120: 252 -> 244 us).
template <typename T>
struct Saved {
  static constexpr bool kFloat = std::is_same_v<T, float>;
  static constexpr int kExtra = std::is_same_v<T, bf16> ? 4 : 8;  // bits below the upper 16
  using Low = std::conditional_t<kExtra == 4, uint8_t, uint16_t>;
  static constexpr int64_t kBytes = kFloat ? 8 : 4 + sizeof(Low);  // an element

  void* p;
  int64_t rows, ld;

  __device__ Vec<uint16_t, 8>* high(int64_t row, int64_t col) const { return (Vec<uint16_t, 8>*)((uint16_t*)p + row * ld + col); }
  __device__ Vec<Low, 8>* low(int64_t row, int64_t col) const { return (Vec<Low, 8>*)((Low*)((uint16_t*)p + 2 * rows * ld) + row * ld + col); }

  // to the nearest, halves up; a NaN as it is, or its bits could carry into the sign
  __device__ static uint32_t rounded(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return x == x ? b + (0x8000u >> kExtra) : b;
  }

  __device__ void put(int64_t row, int64_t col, const float v[8], const float g[8]) const {
    if constexpr (kFloat) {
#pragma unroll
      for (int u = 0; u < 8; u += 4) {
        __builtin_nontemporal_store(f32x4{v[u], v[u + 1], v[u + 2], v[u + 3]}, (f32x4*)((float*)p + row * ld + col + u));
        __builtin_nontemporal_store(f32x4{g[u], g[u + 1], g[u + 2], g[u + 3]}, (f32x4*)((float*)p + (rows + row) * ld + col + u));
      }
    } else {
      Vec<uint16_t, 8> a, b;
      Vec<Low, 8> l;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t x = rounded(v[j]), y = rounded(g[j]);
        a[j] = (uint16_t)(x >> 16), b[j] = (uint16_t)(y >> 16);
        l[j] = (Low)((x & 0xffffu) >> (16 - kExtra) | ((y & 0xffffu) >> (16 - kExtra)) << kExtra);
      }
      __builtin_nontemporal_store(a, high(row, col));
      __builtin_nontemporal_store(b, high(rows + row, col));
      __builtin_nontemporal_store(l, low(row, col));
    }
  }

  __device__ void get(int64_t row, int64_t col, float v[8], float g[8]) const {
    if constexpr (kFloat) {
#pragma unroll
      for (int u = 0; u < 8; u += 4) {
        const f32x4 a = __builtin_nontemporal_load((const f32x4*)((const float*)p + row * ld + col + u));
        const f32x4 b = __builtin_nontemporal_load((const f32x4*)((const float*)p + (rows + row) * ld + col + u));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[u + j] = a[j], g[u + j] = b[j];
      }
    } else {
      const Vec<uint16_t, 8> a = __builtin_nontemporal_load(high(row, col)), b = __builtin_nontemporal_load(high(rows + row, col));
      const Vec<Low, 8> l = __builtin_nontemporal_load(low(row, col));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = __builtin_bit_cast(float, (uint32_t)a[j] << 16 | (l[j] & ((1u << kExtra) - 1)) << (16 - kExtra));
        g[j] = __builtin_bit_cast(float, (uint32_t)b[j] << 16 | (uint32_t)(l[j] >> kExtra) << (16 - kExtra));
      }
    }
  }
};

// What follows the sums: 8 consecutive columns n.. of row m (gated: the value's in v, the gate's in g).
// WHOLE: all 8 are inside.
template <typename T, int ACT, bool WHOLE>
__device__ inline void finish(const Epilogue& e, const Drop& drop, float scale, int64_t M, int64_t N, int64_t m, int64_t n, float v[8],
                              float g[8]) {
  const int left = N - n < 8 ? (int)(N - n) : 8;
  const bool all = WHOLE || left == 8;
  if constexpr (ACT == GF_ACT_NONE)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= scale;
  if (e.bias != nullptr) {
    float b[8];
    load8(b, (const T*)e.bias + n, all, left);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += b[j];
    if constexpr (ACT != GF_ACT_NONE) {
      load8(b, (const T*)e.bias + N + n, all, left);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] += b[j];
    }
  }
  if constexpr (ACT != GF_ACT_NONE) {
    if (e.saved != nullptr) Saved<T>{e.saved, M, e.saved_ld}.put(m, n, v, g);
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
    load8(r, (const T*)e.residual + m * e.ldr + n, all, left);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += r[j];
  }
  store8((T*)e.out + m * N + n, v, all, left);
}

// One operand's way from memory into LDS.  ROWS: its rows of the tile.  HALF: the tile takes HALF rows of the value,
// HALF of the gate and so on (0: consecutive rows).  STEP k in each of PLANES planes.
template <bool KC, int ROWS, int WAVES, int HALF, int STEP, int PLANES>
struct Stage {
  static constexpr int kPlaneBytes = ROWS * STEP * 2, kBytes = PLANES * kPlaneBytes;
  static constexpr int kPieces = kBytes / 1024, kPlanePieces = kPlaneBytes / 1024;  // one load of a wave each
  static constexpr int kLoads = (kPieces + WAVES - 1) / WAVES;
  static constexpr int kReads = (KC ? 1 : 2) * PLANES;  // LDS reads for 32 rows and 16 k
  static constexpr int kRowBytes = KC ? STEP * 2 : ROWS * 2, kChunks = kRowBytes / 16;
  static_assert(kPlaneBytes % 1024 == 0 && (HALF * STEP * 2) % 1024 == 0);

  uint32_t off[kLoads];
  int32_t k_of[kLoads];  // the first k (of the step's) of each load
  const uint8_t* base;
  int64_t gate, plane, advance;  // bytes to the gate's rows, to the next plane, to the next step

  __device__ void init(const Matrix& a, int64_t row0, int64_t rows, int64_t second) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    base = (const uint8_t*)a.p + (KC ? row0 * a.ld : row0) * 2;
    gate = second * a.ld * 2;
    plane = a.plane * 2;
    advance = (KC ? STEP : STEP * a.ld) * 2;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = ((i * WAVES + wave) % kPlanePieces) * 64 + lane;  // the 16 bytes of the LDS plane that the lane fills
      const int r = at / kChunks, chunk = (at % kChunks) ^ swizzle(r);
      if constexpr (KC) {
        int64_t row = HALF ? r / (2 * HALF + !HALF) * HALF + r % (HALF + !HALF) : r;
        row = row < rows - row0 ? row : rows - row0 - 1;
        off[i] = (uint32_t)((row * a.ld + chunk * 8) * 2);
        k_of[i] = chunk * 8;
      } else {
        const int64_t last = a.width - row0 - 8, col = chunk * 8 < last ? chunk * 8 : last;
        off[i] = (uint32_t)((r * a.ld + col) * 2);
        k_of[i] = r;
      }
    }
  }

  // Which 16 bytes of an LDS row hold which: their number is xored with this.  LDS has 64 banks of 4 bytes.
  // K-contiguous: 16 lanes read the same k of 16 rows together; rows that begin at the same bank differ in it.
  // Row-contiguous: 32 lanes read 64 bytes of 4 consecutive k together, which go to different quarters of the banks;
  // rows of an odd number of 64 bytes do so by themselves.
  __device__ static int swizzle(int r) {
    if constexpr (KC) return STEP == 64 ? (r >> 1) & 7 : (r >> 2) & 3;
    return ROWS % 128 == 0 ? (r & 3) << 2 : ROWS % 64 == 0 ? (r & 2) << 1 : 0;
  }

  __device__ void seek(int64_t steps) { base += steps * advance; }

  // left: how many of the k from here on are the matrix's
  __device__ void load(uint8_t* lds, int offset, int left) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int piece = i * WAVES + wave;
      if ((i + 1) * WAVES > kPieces && piece >= kPieces) break;
      const uint8_t* b = base;
      if constexpr (PLANES > 1) b += piece / kPlanePieces * plane;
      if constexpr (HALF != 0) b += piece % kPlanePieces * 1024 / (HALF * STEP * 2) % 2 ? gate : 0;
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)b, 0, 0x80000000, 0x00020000);
      const uint32_t o = k_of[i] < left ? off[i] : 0x80000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(lds + (uint32_t)(offset + piece * 1024)), 16, o, 0, 0, 0);
    }
  }

  // The fragment of 32 rows from `row` on and 16 k from 16 s on: lane l has row row_of(l % 32) and 8 k from 8 (l / 32) on.
  __device__ static half8 fragment(const uint8_t* lds, int offset, int row, int s) {
    const int lane = threadIdx.x & 63;
    if constexpr (KC) {
      const int r = row_of(lane & 31);
      return *(const half8*)(lds + (uint32_t)(offset + (row + r) * kRowBytes + (((2 * s + (lane >> 5)) ^ swizzle(r)) << 4)));
    } else {
      // 16 lanes read 4 k of 16 rows, a lane 4 rows of one k, and get 4 k of one row each
      const int i = lane & 15, r = row + row_of(16 * ((lane >> 4) & 1) + 4 * (i & 3)), k = 8 * (lane >> 5) + (i >> 2);
      const int at = offset + k * kRowBytes + (((r >> 3) ^ swizzle(k)) << 4) + (r & 7) * 2;  // swizzle(k): of k % 4 alone
      half4 part[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) half4*)(lds + (uint32_t)(at + (16 * s + 4 * u) * kRowBytes)));
      return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }

  template <int COUNT>
  __device__ static void fragments(const uint8_t* lds, int offset, int row, int s, half8 (&out)[PLANES][COUNT]) {
#pragma unroll
    for (int c = 0; c < PLANES; ++c)
#pragma unroll
      for (int i = 0; i < COUNT; ++i) out[c][i] = fragment(lds, offset + c * kPlaneBytes, row + 32 * i, s);
  }
};

// Planes of a 32-bit matrix times planes of another: a = a0 + a1 + a2 exactly, 8 bits each by truncation, so a1 is up to
// 2^-7 of a and a2 up to 2^-15.  The six products that are taken leave out a1 b2 + a2 b1 + a2 b2: at most 8 2^-24 of a b,
// 0.7 2^-24 on average, always towards zero.  Smallest first.
constexpr int kPlaneP[6] = {2, 0, 1, 1, 0, 0}, kPlaneQ[6] = {0, 2, 1, 0, 1, 0};

// This wave's LDS reads are done and its loads are in LDS; then all waves'.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A wave's LDS writes before are seen by its reads after (and the other way round).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// For the scheduler: a product, then its share of the LDS reads and of the loads, and so on.
template <int PRODUCTS, int READS, int LOADS, int I = 0>
__device__ __forceinline__ void interleave() {
  if constexpr (I < PRODUCTS) {
    constexpr int r = READS * (I + 1) / PRODUCTS - READS * I / PRODUCTS, l = LOADS * (I + 1) / PRODUCTS - LOADS * I / PRODUCTS;
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (r > 0) __builtin_amdgcn_sched_group_barrier(0x100, r, 0);
    if constexpr (l > 0) __builtin_amdgcn_sched_group_barrier(0x020, l, 0);
    interleave<PRODUCTS, READS, LOADS, I + 1>();
  }
}

// One step of a workgroup.  Its first fragments are in slot 0 already; those of 16 k more are read while the matrix
// cores work on the ones before, the next step's first ones too (NEXT), so that nobody waits behind the barrier.  Where
// the barrier is passed, `cur` has been read by all and takes the loads of the step after next (LOAD).
// cur and nxt are different LDS arrays, and every access is one offset from one of them: what the compiler cannot tell
// apart by that, it waits for all loads before reading.
template <typename T, typename SP, typename SQ, int TM, int TN, bool NEXT, bool LOAD, int S = 0, typename Load>
__device__ __forceinline__ void step(uint8_t* cur, const uint8_t* nxt, Load& load, int wm, int wn,
                                     half8 (&fp)[2][kPlanes<T>][TM / 32], half8 (&fq)[2][kPlanes<T>][TN / 32],
                                     f32x16 (&acc)[TN / 32][TM / 32]) {
  if constexpr (S < kStep<T> / 16) {
    constexpr bool kLast = S + 1 == kStep<T> / 16;
    constexpr int kReads = kLast && !NEXT ? 0 : SP::kReads * (TM / 32) + SQ::kReads * (TN / 32), kTimes = kPlanes<T> == 1 ? 1 : 6;
    if constexpr (!kLast) {
      SP::template fragments<TM / 32>(cur, 0, wm, S + 1, fp[~S & 1]);
      SQ::template fragments<TN / 32>(cur, SP::kBytes, wn, S + 1, fq[~S & 1]);
    } else if constexpr (NEXT) {
      meet();
      if constexpr (LOAD) load(cur);
      SP::template fragments<TM / 32>(nxt, 0, wm, 0, fp[~S & 1]);
      SQ::template fragments<TN / 32>(nxt, SP::kBytes, wn, 0, fq[~S & 1]);
    }
#pragma unroll
    for (int c = 0; c < kTimes; ++c)
#pragma unroll
      for (int j = 0; j < TN / 32; ++j)
#pragma unroll
        for (int i = 0; i < TM / 32; ++i)
          acc[j][i] = mfma<T>(fq[S & 1][kTimes == 1 ? 0 : kPlaneQ[c]][j], fp[S & 1][kTimes == 1 ? 0 : kPlaneP[c]][i], acc[j][i]);
    interleave<TM / 32 * (TN / 32) * kTimes, kReads, kLast && LOAD ? SP::kLoads + SQ::kLoads : 0>();
    step<T, SP, SQ, TM, TN, NEXT, LOAD, S + 1>(cur, nxt, load, wm, wn, fp, fq, acc);
  }
}

template <typename T, bool PKC, bool QKC, int ACT, int WM, int WN, int TM, int TN>
constexpr int kStageBytes = (WM * TM + WN * TN) * kStep<T> * 2 * kPlanes<T>;

// Waves a SIMD: by how many workgroups' double buffers the 160 KB of LDS hold, one or two.
template <typename T, bool PKC, bool QKC, int ACT, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM * WN * 64, WM * WN / (kStageBytes<T, PKC, QKC, ACT, WM, WN, TM, TN> * 2 > 80 * 1024 ? 4 : 2)) void k_product(
    Shape sh, Matrix p, Matrix q, int64_t second, Epilogue e) {
  constexpr bool kGated = ACT != GF_ACT_NONE;
  constexpr int kThreads = WM * WN * 64, BM = WM * TM, BN = WN * TN, BO = kGated ? BN / 2 : BN, kK = kStep<T>;
  using SP = Stage<PKC, BM, WM * WN, 0, kK, kPlanes<T>>;
  using SQ = Stage<QKC, BN, WM * WN, kGated ? TN / 2 : 0, kK, kPlanes<T>>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds0[SP::kBytes + SQ::kBytes], lds1[SP::kBytes + SQ::kBytes];

  // Workgroups go round the 8 dies by their number; a die gets consecutive tiles, in groups of 8 tile rows, so that
  // its cache sees the same rows of P and of Q again.
  const int tiles = sh.tiles_m * sh.tiles_n, die = blockIdx.x & 7, each = tiles >> 3, more = tiles & 7;
  const int tile = die * each + (die < more ? die : more) + (blockIdx.x >> 3);
  const int group = tile / (8 * sh.tiles_n), in_group = tile % (8 * sh.tiles_n);
  const int height = sh.tiles_m - 8 * group < 8 ? sh.tiles_m - 8 * group : 8;
  const int64_t m0 = (int64_t)(8 * group + in_group % height) * BM, n0 = (int64_t)(in_group / height) * BO;
  const int step0 = blockIdx.y * sh.steps, all = (int)((sh.K + kK - 1) / kK);
  const int steps = all - step0 < sh.steps ? all - step0 : sh.steps;

  SP sp;
  SQ sq;
  sp.init(p, m0, sh.M, 0);
  sq.init(q, n0, sh.N, second);
  sp.seek(step0);
  sq.seek(step0);

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wm = wave % WM * TM, wn = wave / WM * TN;
  f32x16 acc[TN / 32][TM / 32] = {};

  int left = (int)(sh.K - (int64_t)step0 * kK);  // k from the next load's first on; none: loads read nothing and fill with zeros
  auto load = [&](uint8_t* to) {
    sp.load(to, 0, left);
    sq.load(to, SP::kBytes, left);
    sp.seek(1);
    sq.seek(1);
    left -= kK;
  };

  half8 fp[2][kPlanes<T>][TM / 32], fq[2][kPlanes<T>][TN / 32];
  load(lds0);
  meet();
  load(lds1);
  SP::template fragments<TM / 32>(lds0, 0, wm, 0, fp[0]);
  SQ::template fragments<TN / 32>(lds0, SP::kBytes, wn, 0, fq[0]);
  int after = steps - 1;  // steps after the one to be done
  for (; after >= 2; after -= 2) {
    step<T, SP, SQ, TM, TN, true, true>(lds0, lds1, load, wm, wn, fp, fq, acc);
    step<T, SP, SQ, TM, TN, true, true>(lds1, lds0, load, wm, wn, fp, fq, acc);
  }
  if (after == 1) step<T, SP, SQ, TM, TN, true, false>(lds0, lds1, load, wm, wn, fp, fq, acc);
  step<T, SP, SQ, TM, TN, false, false>(after == 1 ? lds1 : lds0, lds0, load, wm, wn, fp, fq, acc);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the loads past the end have filled theirs while the LDS is still ours

  // Lane l has, of each 32 x 32, row m = row_of(l % 32) and columns 16 h + 8 (l / 32) .. + 8 for h = 0, 1.  Stored like
  // that a line of memory would be written in as many parts as it has 32 bytes, so a wave's 32 rows and at most 64
  // columns (gated: 64 of each half) go through its part of LDS and come out row by row, 8 columns a lane.
  // LDS rows of 16-byte pieces, whose number is xored with the row's against bank conflicts.
  constexpr int kOut = kGated ? TN / 64 : TN / 32, kBlock = kOut < 2 ? kOut : 2, kWidth = kBlock * 32 * (kGated ? 2 : 1);
  static_assert(WM * WN * 32 * kWidth * 4 <= 2 * (SP::kBytes + SQ::kBytes));
  constexpr int kHalf = (SP::kBytes + SQ::kBytes) / (32 * kWidth * 4);  // waves whose part is in lds0
  float* const part = (float*)(wave < kHalf ? lds0 : lds1) + (wave < kHalf ? wave : wave - kHalf) * 32 * kWidth;
  auto piece = [&](int row, int col) { return (f32x4*)(part + row * kWidth + (((col >> 2) ^ (row & (kWidth / 4 - 1) & 15)) << 2)); };
  Drop drop = e.drop;
  load_key(drop);
  const float scale = scale_of(e);
  meet();  // everyone has read lds0 and lds1
#pragma unroll
  for (int i = 0; i < TM / 32; ++i) {
#pragma unroll
    for (int j0 = 0; j0 < kOut; j0 += kBlock) {
      const int blocks = kOut - j0 < kBlock ? kOut - j0 : kBlock;
#pragma unroll
      for (int b = 0; b < blocks; ++b)
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // 4 columns each
          const int row = row_of(lane & 31), col = 32 * b + 16 * (u >> 1) + 8 * (lane >> 5) + 4 * (u & 1);
          *piece(row, col) = f32x4{acc[j0 + b][i][4 * u], acc[j0 + b][i][4 * u + 1], acc[j0 + b][i][4 * u + 2], acc[j0 + b][i][4 * u + 3]};
          if constexpr (kGated) {
            const f32x16& g = acc[kOut + j0 + b][i];
            *piece(row, kWidth / 2 + col) = f32x4{g[4 * u], g[4 * u + 1], g[4 * u + 2], g[4 * u + 3]};
          }
        }
      wave_sync();
#pragma unroll 1
      for (int t = lane; t < 32 * 4 * blocks; t += 64) {
        const int row = t / (4 * blocks), col = t % (4 * blocks) * 8;
        const int64_t m = m0 + wm + 32 * i + row, n = n0 + (kGated ? wn / 2 : wn) + 32 * j0 + col;
        if (m >= sh.M || n >= sh.N) continue;
        float v[8], g[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 x = *piece(row, col + 4 * u);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[4 * u + r] = x[r];
          if constexpr (kGated) {
            const f32x4 y = *piece(row, kWidth / 2 + col + 4 * u);
#pragma unroll
            for (int r = 0; r < 4; ++r) g[4 * u + r] = y[r];
          }
        }
        if (e.partial != nullptr) {
          const int64_t width = (sh.N + 7) / 8 * 8;
          float* out = e.partial + ((int64_t)blockIdx.y * sh.M + m) * width * (kGated ? 2 : 1) + n;
          store8(out, v, true, 8);
          if constexpr (kGated) store8(out + width, g, true, 8);
        } else if (n + 8 <= sh.N) {
          finish<T, ACT, true>(e, drop, scale, sh.M, sh.N, m, n, v, g);
        } else {
          finish<T, ACT, false>(e, drop, scale, sh.M, sh.N, m, n, v, g);
        }
      }
      wave_sync();
    }
  }
}

// The forward product of at most 16 G rows: bound by reading W once, so nothing of it goes through LDS.  A workgroup takes 16
// output columns (gated: 16 of the value's and of the gate's), its waves interleaved chunks of 64 bytes along k; a lane
// loads 16 bytes of W's row (lane % 16) and of x's straight into the matrix instruction's operands, at whatever
// alignment.  32-bit operands are multiplied as such (16 x 16 x 4).  The waves' sums meet in LDS.  One row of
// 1280 -> 5120 gated in bfloat16: 9.4 us for 26 MB (320 workgroups; 5 chunks a wave, four of them asked for together: two trips
// to memory one after the other), 5120 -> 1280 8.8 us for 13 MB (80 workgroups on 256 units; 10 chunks a wave: up to four
// trips).  The weights come from the last cache where the same call repeats.
template <typename T, int ACT, int G>
__global__ __launch_bounds__(1024) void k_few(int64_t M, int64_t N, int64_t K, const T* __restrict__ x, int64_t ldx,
                                              const T* __restrict__ w, int64_t ldw, Epilogue e) {
  constexpr int H = ACT == GF_ACT_NONE ? 1 : 2, E = 16 / sizeof(T), kChunk = 4 * E, kAhead = G > 2 ? 2 : 4;
  using V = Vec<T, E>;
  __shared__ float sums[16][H][G][16][16 + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t n0 = blockIdx.x * 16ll, at = (lane >> 4) * E;
  const int64_t n = n0 + (lane & 15) < N ? n0 + (lane & 15) : N - 1;
  const T *pw[H], *px[G];
#pragma unroll
  for (int h = 0; h < H; ++h) pw[h] = w + (n + h * N) * ldw + at;
#pragma unroll
  for (int g = 0; g < G; ++g) px[g] = x + (16 * g + (lane & 15) < M ? 16 * g + (lane & 15) : M - 1) * ldx + at;

  f32x4 acc[H][G] = {};
  auto multiply = [&](const V* a, const V* b) {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if constexpr (std::is_same_v<T, float>) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[h][g] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[h][i], b[g][i], acc[h][g], 0, 0, 0);
        } else if constexpr (std::is_same_v<T, f16>) {
          acc[h][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a[h]), __builtin_bit_cast(f16x8, b[g]), acc[h][g], 0, 0, 0);
        } else {
          acc[h][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[h]), __builtin_bit_cast(bf16x8, b[g]), acc[h][g], 0, 0, 0);
        }
      }
  };
  const int chunks = (int)(K / kChunk);  // whole ones
  int c = wave;
  for (; c + (kAhead - 1) * waves < chunks; c += kAhead * waves) {
    V a[kAhead][H], b[kAhead][G];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
#pragma unroll
      for (int h = 0; h < H; ++h) a[u][h] = *(const V*)(pw[h] + (int64_t)(c + u * waves) * kChunk);
#pragma unroll
      for (int g = 0; g < G; ++g) b[u][g] = *(const V*)(px[g] + (int64_t)(c + u * waves) * kChunk);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) multiply(a[u], b[u]);
  }
  for (; c <= chunks; c += waves) {  // the rest, and the part of a chunk
    const int64_t k = (int64_t)c * kChunk;
    const int64_t left = K - k - at;
    if (K - k <= 0) break;
    V a[H], b[G];
    if (c < chunks) {
#pragma unroll
      for (int h = 0; h < H; ++h) a[h] = *(const V*)(pw[h] + k);
#pragma unroll
      for (int g = 0; g < G; ++g) b[g] = *(const V*)(px[g] + k);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
#pragma unroll
        for (int h = 0; h < H; ++h) a[h][i] = i < left ? pw[h][k + i] : (T)0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) b[g][i] = i < left ? px[g][k + i] : (T)0.0f;
      }
    }
    multiply(a, b);
  }

  // Lane l has row l % 16 of each 16 and columns 4 (l / 16) .. + 4.
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][h][g][lane & 15][4 * (lane >> 4) + r] = acc[h][g][r];
  __syncthreads();
  for (int t = threadIdx.x; t < H * G * 256; t += blockDim.x) {
    float* const s = &sums[0][t / 256 / G][t / 256 % G][t / 16 % 16][t % 16];
    float v = s[0];
    for (int i = 1; i < waves; ++i) v += s[i * (H * G * 16 * 17)];
    s[0] = v;
  }
  __syncthreads();
  const int t = threadIdx.x;
  const int64_t m = t / 2, col = n0 + t % 2 * 8;
  if (m >= M || t >= 32 * G || col >= N) return;
  Drop drop = e.drop;
  load_key(drop);
  float v[8], g[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = sums[0][0][m / 16][m % 16][t % 2 * 8 + j];
    if constexpr (H == 2) g[j] = sums[0][1][m / 16][m % 16][t % 2 * 8 + j];
  }
  if (col + 8 <= N)
    finish<T, ACT, true>(e, drop, 1.0f, M, N, m, col, v, g);
  else
    finish<T, ACT, false>(e, drop, 1.0f, M, N, m, col, v, g);
}

// The products' parts, added in their order.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void k_join(Shape sh, Epilogue e) {
  constexpr bool kGated = ACT != GF_ACT_NONE;
  Drop drop = e.drop;
  load_key(drop);
  const float scale = scale_of(e);
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
    finish<T, ACT, false>(e, drop, scale, sh.M, sh.N, m, n, v, g);
  }
}

// ------------------------------------------------------------------------------------------
// Operands that the products cannot read in place: 32-bit matrices into three bfloat16 planes, and 16-bit ones whose
// rows are not whole, aligned groups of 16 bytes into rows that are.  Columns past the matrix become zero.  Bound by
// memory: 4096 x 640 and 5120 x 640 of 32 bits 12 us (59 MB, 4.9 TB/s).

// x = its 3 x 8 leading bits, by truncation: x - a0 and x - a0 - a1 are exact.  All have x's sign.  An infinity or a NaN
// stays in a0.  Planes that would be zero hold the smallest normal number instead, of x's sign, unless x is below 2^-100: an
// infinity times 0 would be a NaN where the product is infinite.  That adds 2^-25 of x at most.
__device__ inline void split(float x, bf16 out[3]) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, x), size = bits & 0x7fffffffu;
  const uint32_t least = size >= 0x0d800000u ? (bits & 0x80000000u) | 0x00800000u : 0u;
  const bool finite = size < 0x7f800000u;
  out[0] = __builtin_bit_cast(bf16, (uint16_t)((size > 0x7f800000u ? bits | 0x10000u : bits) >> 16));
  float left = finite ? x - __builtin_bit_cast(float, bits & 0xffff0000u) : 0.0f;
#pragma unroll
  for (int i = 1; i < 3; ++i) {
    const uint32_t top = __builtin_bit_cast(uint32_t, left) & 0xffff0000u;
    out[i] = __builtin_bit_cast(bf16, (uint16_t)((left == 0.0f ? least : top) >> 16));
    left -= __builtin_bit_cast(float, top);
  }
}

struct PackJob {
  int64_t rows, cols;
  const void* x;
  int64_t ldx;
  void* out;
  int64_t ld, plane;
};

// Up to two matrices in one launch: the first `blocks0` workgroups the first, the others the second.
template <typename T>
__global__ __launch_bounds__(256) void k_pack(PackJob job0, PackJob job1, unsigned blocks0) {
  const bool second = blockIdx.x >= blocks0;
  const PackJob a = second ? job1 : job0;
  const int64_t groups = a.ld / 8, block = second ? blockIdx.x - blocks0 : blockIdx.x, all = (second ? gridDim.x - blocks0 : blocks0) * 256ll;
  for (int64_t t = block * 256 + threadIdx.x; t < a.rows * groups; t += all) {
    const int64_t row = t / groups, c = t % groups * 8;
    const int n = a.cols - c < 8 ? (int)(a.cols - c) : 8;
    float v[8];
    load8(v, (const T*)a.x + row * a.ldx + c, n == 8, n);
    if constexpr (std::is_same_v<T, float>) {
      bf16x8 o[3];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bf16 s[3];
        split(v[j], s);
        o[0][j] = s[0], o[1][j] = s[1], o[2][j] = s[2];
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) *(bf16x8*)((bf16*)a.out + i * a.plane + row * a.ld + c) = o[i];
    } else {
      store8((T*)a.out + row * a.ld + c, v, true, 8);
    }
  }
}

// dz: the gradient of x W^T + b from dy.  Linear: the masked dy as it is; the scale of what is kept is left to the sums
// (`scale` for the bias's, Epilogue::scale for the products), so that nothing is rounded here and nothing can overflow.
// Gated: the value's columns, then the gate's; dv = d act(g), dg = d v act'(g), d the masked and scaled dy.  In 16 bits
// they are rounded to the tensors' type, because the matrix cores take it so: of the same size as dx's and dW's own
// rounding, which makes 1.4 of one; the bias's sums take them before.  A dropped place's are zero whatever its value and
// gate are: the output there is 0, not 0 times them.  The kept value and gate are asked for first, ahead of dy's branch and of
// the generator (16384 x 1280 in bfloat16: 46 us so, 54 us after them).
// 8 columns from c on, of which n are the matrix's; zero past those.
template <typename T, int ACT, int H>
__device__ inline void make_dz(const Drop& d, int64_t rows, const T* dy, int64_t lddy, void* saved, int64_t saved_ld, int64_t row, int64_t c,
                               int n, float (&g)[H][8]) {
  float value[8], gate[8];
  if constexpr (H == 2) Saved<T>{saved, rows, saved_ld}.get(row, c, value, gate);
  load8(g[0], dy + row * lddy + c, n == 8, n);
  uint32_t there = (1u << n) - 1;  // a bit for each that is the matrix's and kept: eight conditions would be branches
  if (d.threshold != 0) {
    uint32_t bits[4];
    random_block(d, (uint32_t)row, (uint32_t)(c >> 3), bits);
#pragma unroll
    for (int j = 0; j < 8; ++j) there &= ~((uint32_t)!kept(d, bits, j) << j);
  }
  if constexpr (H == 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[0][j] = there >> j & 1 ? g[0][j] * d.scale : 0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float slope;
      const float a = activation<ACT>(gate[j], &slope), v = g[0][j] * d.scale;
      const bool k = there >> j & 1;
      g[0][j] = k ? v * a : 0.0f;
      g[1][j] = k ? v * value[j] * slope : 0.0f;
    }
  }
}

// A product of a gradient, a value and a slope leaves float16's range at either end where dx and dW do not, so a gated dz
// in float16 is stored times a power of two that brings its largest finite element (k_peak) to [2^14, 2^15), which
// dx's and dW's sums take back (Epilogue::scale_at).  An element keeps its 11 bits down to 2^-29 of the largest, and lies within
// 2^-40 of that below.  That costs one pass over dy, value and gate more: 8192 x 5120 75 us (336 MB, 4.5 TB/s).
template <typename T, int ACT>
constexpr bool kScaledDz = std::is_same_v<T, f16> && ACT != GF_ACT_NONE;
constexpr int kPeaks = 1024;  // workgroups, and their maxima

template <typename T, int ACT>
__global__ __launch_bounds__(256) void k_peak(Drop d, int64_t rows, int64_t out, const T* dy, int64_t lddy, void* saved, int64_t saved_ld,
                                              float* peaks) {
  __shared__ float part[256];
  load_key(d);
  const uint32_t groups = (uint32_t)((out + 7) / 8);
  const int64_t first = blockIdx.x * 256ll + threadIdx.x, all = gridDim.x * 256ll;
  int64_t row = first / groups;
  uint32_t group = (uint32_t)(first % groups);
  const int64_t row_step = all / groups;
  const uint32_t group_step = (uint32_t)(all % groups);
  float peak = 0.0f;
  while (row < rows) {
    const int64_t c = 8ll * group;
    float g[2][8];
    make_dz<T, ACT>(d, rows, dy, lddy, saved, saved_ld, row, c, out - c < 8 ? (int)(out - c) : 8, g);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = fabsf(g[h][j]);
        peak = fmaxf(peak, a < INFINITY ? a : 0.0f);  // a NaN is not
      }
    row += row_step, group += group_step;
    if (group >= groups) group -= groups, ++row;
  }
  part[threadIdx.x] = peak;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  peak = fmaxf(fmaxf(part[threadIdx.x], part[threadIdx.x + 64]), fmaxf(part[threadIdx.x + 128], part[threadIdx.x + 192]));
#pragma unroll
  for (int i = 32; i > 0; i >>= 1) peak = fmaxf(peak, __shfl_xor(peak, i));
  if (threadIdx.x == 0) peaks[blockIdx.x] = peak;
}

// The power of two of k_peak's maxima, for the whole workgroup.
__device__ inline float dz_factor(const float* peaks, int count) {
  __shared__ float part[4];
  float peak = 0.0f;
  for (int i = threadIdx.x; i < count; i += 256) peak = fmaxf(peak, peaks[i]);
#pragma unroll
  for (int i = 32; i > 0; i >>= 1) peak = fmaxf(peak, __shfl_xor(peak, i));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = peak;
  __syncthreads();
  peak = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  if (peak == 0.0f) return 1.0f;
  const int e = (int)(__builtin_bit_cast(uint32_t, peak) >> 23);  // peak in [2^(e - 127), 2^(e - 126))
  return __builtin_bit_cast(float, (uint32_t)(127 + min(127 + 14 - e, 120)) << 23);
}

// dz, bound by memory: 8192 x 5120 gated in bfloat16 84 us (462 MB, 5.5 TB/s).  It is written as the products read it
// ([rows, ld], in planes for 32 bits, zero past its columns), and its columns' sums: a workgroup takes 256 columns of dy
// and `chunk` rows, 8 columns a thread in 8 interleaved rows, and leaves its sums in `sums` [row chunk][columns of dz],
// or, of one chunk, in dbias.  `peaks`: k_peak's, followed by the place for the power of two's inverse (NULL: no such).
// Four waves a SIMD, which float32's gelu_tanh would miss by a few registers (4096 x 2560: 47 us, 53 us with three).
template <typename T, int ACT>
__global__ __launch_bounds__(256, 4) void k_dz(Drop d, int64_t rows, int64_t out, int64_t chunk, const T* dy, int64_t lddy, void* saved,
                                            int64_t saved_ld, void* dz, int64_t ld, int64_t plane, float* sums, T* dbias, float scale,
                                            float* peaks, int peak_count) {
  constexpr bool kGated = ACT != GF_ACT_NONE;
  constexpr int H = kGated ? 2 : 1;
  __shared__ float part[H][8][256 + 8];
  load_key(d);
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int64_t c = (blockIdx.x * 32ll + lane) * 8, width = H * out;
  const int n = c >= out ? 0 : out - c < 8 ? (int)(out - c) : 8;
  float sum[H][8] = {}, factor = 1.0f;
  if constexpr (kScaledDz<T, ACT>) {
    if (peaks != nullptr) {
      factor = dz_factor(peaks, peak_count);
      if (blockIdx.x + blockIdx.y == 0 && threadIdx.x == 0) peaks[kPeaks] = 1.0f / factor;  // exact
    }
  }
  if (n > 0) {
    const int64_t end = (blockIdx.y + 1) * chunk < rows ? (blockIdx.y + 1) * chunk : rows;
    for (int64_t row = blockIdx.y * chunk + line; row < end; row += 8) {
      float g[H][8];
      make_dz<T, ACT>(d, rows, dy, lddy, saved, saved_ld, row, c, n, g);
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[h][j] += g[h][j];
        if (dz == nullptr) continue;
        if constexpr (kScaledDz<T, ACT>)
#pragma unroll
          for (int j = 0; j < 8; ++j) g[h][j] *= factor;
        // the last columns' store also clears what follows them, up to ld
        const int64_t at = row * ld + h * out + c;
        const bool last = h == H - 1 && c + 8 >= out;
        const int put = last ? (int)(ld - h * out - c) : n;
        if constexpr (std::is_same_v<T, float>) {
          float part[3][8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            bf16 o[3];
            split(g[h][j], o);
            part[0][j] = (float)o[0], part[1][j] = (float)o[1], part[2][j] = (float)o[2];
          }
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            bf16* to = (bf16*)dz + i * plane + at;
            store8(to, part[i], put == 8, put);
            for (int j = 8; j < put; ++j) to[j] = (bf16)0.0f;
          }
        } else {
          store8((T*)dz + at, g[h], put == 8, put);
          for (int j = 8; j < put; ++j) ((T*)dz)[at + j] = (T)0.0f;
        }
      }
    }
  }
  if (sums == nullptr && dbias == nullptr) return;
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
    s *= scale;
    if (dbias != nullptr)
      dbias[h * out + col] = (T)s;  // one chunk
    else
      sums[blockIdx.y * width + h * out + col] = s;
  }
}

// The chunks' sums of 32 columns a workgroup, added in a fixed order.
template <typename T>
__global__ __launch_bounds__(256) void k_join_sums(int64_t chunks, int64_t cols, const float* sums, T* out) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (int64_t i = line; i < chunks; i += 8) s += sums[i * cols + c];
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

int check_shape(const gf_ff_args* a) {
  if (a == nullptr) return fail(GF_E_INVALID_ARGUMENT, "args must not be NULL");
  GF_TRY(check_dtype(a->dtype));
  if (a->activation < GF_ACT_NONE || a->activation > GF_ACT_SILU)
    return fail(GF_E_INVALID_ARGUMENT, "unknown activation %d", (int)a->activation);
  if (a->rows < 0 || a->in_features <= 0 || a->out_features <= 0)
    return fail(GF_E_INVALID_ARGUMENT, "rows must not be negative and in_features and out_features must be positive");
  if (a->rows > kMaxSize || a->in_features > kMaxSize / 2 || a->out_features > kMaxSize / 4)
    return fail(GF_E_INVALID_ARGUMENT, "rows, in_features or out_features too large");
  const int64_t weight_rows = a->out_features * (a->activation == GF_ACT_NONE ? 1 : 2);
  if (std::max(a->rows, weight_rows) * a->in_features > kMaxElements || a->rows * weight_rows > kMaxElements)
    return fail(GF_E_INVALID_ARGUMENT, "rows, in_features or out_features too large");
  for (const int64_t ld : {a->ldx, a->ldw, a->ldr, a->lddy})
    if (ld > kMaxElements || ld < -kMaxElements) return fail(GF_E_INVALID_ARGUMENT, "row stride too large");
  return check_dropout(&a->dropout);
}

int64_t weight_rows(const gf_ff_args* a) { return a->out_features * (a->activation == GF_ACT_NONE ? 1 : 2); }
int64_t saved_ld(const gf_ff_args* a) { return round_up(a->out_features, 8); }

bool aligned(const void* p, int64_t ld, int size) { return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0; }

template <typename T>
bool reads_in_place(const void* x, int64_t cols, int64_t ld) {
  return !std::is_same_v<T, float> && aligned(x, ld, 2) && cols % 8 == 0;
}

// The matrices that have to be packed, and their launch.
struct Packs {
  PackJob job[2];
  int n = 0;
};

// x as a product reads it: itself where it can be, else what `packs` is given to make.
template <typename T>
Matrix operand(Arena& ws, Packs& packs, const void* x, int64_t rows, int64_t cols, int64_t ld) {
  if (reads_in_place<T>(x, cols, ld)) return {x, ld, 0, (int32_t)cols};
  constexpr int kBytes = 2 * kPlanes<T>;
  const int64_t width = round_up(cols, 8), plane = rows * width;
  void* const out = ws.take(plane * kBytes);
  packs.job[packs.n++] = {rows, cols, x, ld, out, width, plane};
  return {out, width, plane, (int32_t)width};
}

template <typename T>
int pack(bool run, const Packs& packs, hipStream_t s) {
  GF_RUN if (packs.n != 0) {
    unsigned blocks[2] = {};
    for (int i = 0; i < packs.n; ++i) blocks[i] = blocks_for(packs.job[i].rows * packs.job[i].ld / 8);
    k_pack<T><<<blocks[0] + blocks[1], 256, 0, s>>>(packs.job[0], packs.job[packs.n - 1], blocks[0]);
    GF_LAUNCH_CHECK("k_pack");
  }
  return GF_OK;
}

constexpr int kUnits = 256;  // compute units

// How a product is cut into workgroups: tiles, and `splits` parts along k that k_join adds.
enum class Tile { k256x256, k256x160, k256x128, k128x128 };
struct Cut {
  Tile tile;
  int32_t splits;
};

struct TileKind {
  Tile tile;
  int64_t m, n, slots;  // slots: workgroups at a time
  double step, round;   // us
};

// The cut whose estimated time is least, from what was measured.  In 16 bits a step of 64 takes 1.59 us with a
// 256 x 256 tile on each compute unit (4096 x 4096 x 8192: 203 us, 1.35 PFLOP/s), 1.18 us with 256 x 160
// (8192 x 1280 x 10240, one round: 191 us, against 208 us in 160 tiles of 256 x 256) and 0.98 us with two of 128 x 128
// (250 us for the first: twice the bytes from L2 for each operation).  Where not all units work, those that do run faster
// (160 tiles: 1.30 us a step): the chip is held by its power.  A round costs about 7, 7 and 3 us besides, and split
// parts are written and read back at about 4 TB/s, by one more launch.  What the epilogue writes is not in it, so a gated
// forward that keeps value and gate takes longer than it says, by whatever cut: 16384 x 320 -> 1280 72 us where it says 40,
// 8192 x 1280 -> 5120 241 where it says 194, 4096 x 640 -> 2560 in 32 bits 172 where it says 145.  In 32 bits a step of 32 takes 2.35 us with 256 x 128 and 1.25 us with
// 128 x 128 on each unit (4096 x 4096 x 2048: 284 to 329 us and 302 to 344 us, by the operands' layouts).
constexpr TileKind kTiles16[] = {{Tile::k256x256, 256, 256, kUnits, 1.59, 7.0}, {Tile::k256x160, 256, 160, kUnits, 1.18, 7.0}, {Tile::k128x128, 128, 128, 2 * kUnits, 0.98, 3.0}};
constexpr TileKind kTiles32[] = {{Tile::k256x128, 256, 128, kUnits, 2.35, 7.0}, {Tile::k128x128, 128, 128, kUnits, 1.25, 4.0}};

template <bool F32>
Cut choose_cut(int64_t M, int64_t columns, int64_t steps, bool gated) {
  constexpr const TileKind* kinds = F32 ? kTiles32 : kTiles16;
  Cut best{};
  double least = 1e300;
  for (int i = 0; i < (F32 ? 2 : 3); ++i) {
    const TileKind& k = kinds[i];
    if (gated && k.tile == Tile::k256x160) continue;  // its halves would not be whole matrix instructions
    const int64_t tiles = ((M + k.m - 1) / k.m) * ((columns + k.n - 1) / k.n);
    for (int64_t splits = 1; splits <= 32 && splits * 2 <= std::max<int64_t>(steps, 2); ++splits) {
      const double each = (double)((steps + splits - 1) / splits) * k.step;
      const int64_t full = tiles * splits / k.slots, rest = tiles * splits % k.slots;
      double us = full * (each + k.round);
      if (rest != 0) us += each * std::max(0.72, 0.5 + 0.5 * rest / k.slots) + k.round;
      if (splits > 1) us += M * columns * (8.0 * splits + (F32 ? 4 : 2)) / 4e6 + 8.0;
      if (us < least) least = us, best = {k.tile, (int32_t)splits};
    }
  }
  return best;
}

template <typename T, bool PKC, bool QKC, int ACT, int WM, int WN, int TM, int TN>
int product_tiled(Arena& ws, bool run, int64_t M, int64_t N, int64_t K, const Matrix& p, const Matrix& q, int64_t second, Epilogue e,
                  int64_t splits, hipStream_t s) {
  constexpr int BM = WM * TM, BO = WN * TN / (ACT == GF_ACT_NONE ? 1 : 2);
  Shape sh{M, N, K, 0, 0, 1, 0};
  const int64_t tm = (M + BM - 1) / BM, tn = (N + BO - 1) / BO, steps = (K + kStep<T> - 1) / kStep<T>;
  if (tm * tn > (int64_t(1) << 30)) return fail(GF_E_INVALID_ARGUMENT, "rows, in_features or out_features too large");
  sh.tiles_m = (int32_t)tm, sh.tiles_n = (int32_t)tn;
  sh.steps = (int32_t)((steps + splits - 1) / splits);
  sh.splits = (int32_t)((steps + sh.steps - 1) / sh.steps);
  const bool join = sh.splits > 1;
  e.partial = nullptr;
  if (join) e.partial = (float*)ws.take(sh.splits * M * round_up(N, 8) * (ACT == GF_ACT_NONE ? 1 : 2) * 4);
  GF_RUN {
    k_product<T, PKC, QKC, ACT, WM, WN, TM, TN><<<dim3((unsigned)(tm * tn), (unsigned)sh.splits), WM * WN * 64, 0, s>>>(sh, p, q, second, e);
    GF_LAUNCH_CHECK("k_product");
    if (join) {
      k_join<T, ACT><<<blocks_for(M * ((N + 7) / 8)), 256, 0, s>>>(sh, e);
      GF_LAUNCH_CHECK("k_join");
    }
  }
  return GF_OK;
}

template <typename T, bool PKC, bool QKC, int ACT>
int product(Arena& ws, bool run, int64_t M, int64_t N, int64_t K, const Matrix& p, const Matrix& q, int64_t second, const Epilogue& e,
            hipStream_t s) {
  // a load's 32-bit offset spans a tile's rows (K-contiguous) or a step's (row-contiguous)
  if (std::max(p.ld, q.ld) * 2 * 256 >= (int64_t(1) << 31)) return fail(GF_E_INVALID_ARGUMENT, "row stride too large");
  const Cut cut = choose_cut<std::is_same_v<T, float>>(M, ACT == GF_ACT_NONE ? N : 2 * N, (K + kStep<T> - 1) / kStep<T>, ACT != GF_ACT_NONE);
#define FF_TILED(...) return product_tiled<T, PKC, QKC, ACT, __VA_ARGS__>(ws, run, M, N, K, p, q, second, e, cut.splits, s)
  if constexpr (std::is_same_v<T, float>) {
    if (cut.tile == Tile::k256x128) FF_TILED(4, 2, 64, 64);
    FF_TILED(4, 2, 32, 64);
  } else {
    if constexpr (ACT == GF_ACT_NONE) {
      if (cut.tile == Tile::k256x160) FF_TILED(8, 1, 32, 160);
      if (cut.tile == Tile::k256x256) FF_TILED(2, 4, 128, 64);
      FF_TILED(2, 2, 64, 64);
    } else {  // waves of 128 columns: 64 of each half, whole lines of the output
      if (cut.tile == Tile::k256x256) FF_TILED(4, 2, 64, 128);
      FF_TILED(4, 1, 32, 128);
    }
  }
#undef FF_TILED
}

template <typename T, int ACT>
int few(const gf_ff_args& a, const Epilogue& e, hipStream_t s) {
  const dim3 grid((unsigned)((a.out_features + 15) / 16));
  // 16 waves where each still has 4 chunks of 64 bytes or more, 8 else
  const unsigned threads = a.in_features * (int64_t)sizeof(T) >= 16 * 4 * 64 ? 1024 : 512;
  auto* kernel = a.rows <= 16 ? k_few<T, ACT, 1> : a.rows <= 32 ? k_few<T, ACT, 2> : k_few<T, ACT, 4>;
  kernel<<<grid, threads, 0, s>>>(a.rows, a.out_features, a.in_features, (const T*)a.x, a.ldx, (const T*)a.weight, a.ldw, e);
  GF_LAUNCH_CHECK("k_few");
  return GF_OK;
}

// The forward's launches, or (run false) its workspace.
int forward(const gf_ff_args& a, Arena& ws, bool run, hipStream_t s) {
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_activation(a.activation, [&](auto act) {
      const Epilogue e{a.y, a.bias, a.residual, a.ldr, a.saved, saved_ld(&a), nullptr, make_drop(a.dropout)};
      if (a.rows <= 64) {
        GF_RUN return few<T, act.value>(a, e, s);
        return (int)GF_OK;
      }
      Packs packs;
      const Matrix x = operand<T>(ws, packs, a.x, a.rows, a.in_features, a.ldx);
      const Matrix w = operand<T>(ws, packs, a.weight, weight_rows(&a), a.in_features, a.ldw);
      GF_TRY(pack<T>(run, packs, s));
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
      Drop drop = make_drop(a.dropout);
      Epilogue e{};
      if (ACT == GF_ACT_NONE) std::swap(drop.scale, e.scale);
      const bool products = a.dx != nullptr || a.dweight != nullptr;
      Matrix dz{};
      Packs packs;
      // linear, nothing dropped: dz is dy, where the products can read it so
      const bool same = ACT == GF_ACT_NONE && drop.threshold == 0 && reads_in_place<T>(a.dy, out, a.lddy);
      if (same && products) dz = operand<T>(ws, packs, a.dy, a.rows, out, a.lddy);
      const bool make = products && !same;
      if (make) {
        dz.ld = round_up(wr, 8), dz.plane = a.rows * dz.ld, dz.width = (int32_t)dz.ld;
        dz.p = ws.take(dz.plane * 2 * kPlanes<T>);
      }
      if (make || a.dbias != nullptr) {
        // rows in chunks of at least 8 until there are about 4 workgroups a compute unit; up to 64 rows in one chunk, whose
        // sums are the bias's gradient (a launch less)
        const int64_t across = (out + 255) / 256;
        int64_t chunks = a.rows <= 64 ? 1 : std::max<int64_t>(std::min<int64_t>(4 * kUnits / across, a.rows / 8), 1);
        const int64_t chunk = (a.rows + chunks - 1) / chunks;
        chunks = (a.rows + chunk - 1) / chunk;
        float* peaks = nullptr;
        const int peak_blocks = (int)std::min<int64_t>((a.rows * ((out + 7) / 8) + 255) / 256, kPeaks);
        if (kScaledDz<T, ACT> && make) {
          peaks = (float*)ws.take((kPeaks + 1) * 4);
          GF_RUN e.scale_at = peaks + kPeaks;
        }
        float* sums = a.dbias != nullptr && chunks > 1 ? (float*)ws.take(chunks * wr * 4) : nullptr;
        GF_RUN {
          if constexpr (kScaledDz<T, ACT>) {
            if (make) {
              k_peak<T, ACT><<<peak_blocks, 256, 0, s>>>(drop, a.rows, out, (const T*)a.dy, a.lddy, a.saved, saved_ld(&a), peaks);
              GF_LAUNCH_CHECK("k_peak");
            }
          }
          k_dz<T, ACT><<<dim3((unsigned)across, (unsigned)chunks), 256, 0, s>>>(
              drop, a.rows, out, chunk, (const T*)a.dy, a.lddy, a.saved, saved_ld(&a), make ? (void*)dz.p : nullptr, dz.ld, dz.plane, sums,
              sums == nullptr ? (T*)a.dbias : nullptr, e.scale, peaks, peak_blocks);
          GF_LAUNCH_CHECK("k_dz");
          if (sums != nullptr) {
            k_join_sums<T><<<(unsigned)((wr + 31) / 32), 256, 0, s>>>(chunks, wr, sums, (T*)a.dbias);
            GF_LAUNCH_CHECK("k_join_sums");
          }
        }
      }
      Matrix w{}, x{};
      if (a.dx != nullptr) w = operand<T>(ws, packs, a.weight, wr, a.in_features, a.ldw);
      if (a.dweight != nullptr) x = operand<T>(ws, packs, a.x, a.rows, a.in_features, a.ldx);
      GF_TRY(pack<T>(run, packs, s));
      if (a.dx != nullptr) {
        e.out = a.dx;
        GF_TRY((product<T, true, false, GF_ACT_NONE>(ws, run, a.rows, a.in_features, wr, dz, w, 0, e, s)));
      }
      if (a.dweight != nullptr) {
        e.out = a.dweight;
        GF_TRY((product<T, false, false, GF_ACT_NONE>(ws, run, wr, a.in_features, a.rows, dz, x, 0, e, s)));
      }
      return (int)GF_OK;
    });
  });
}

}  // namespace

extern "C" {

int gf_dropout_add(int32_t dtype, const gf_dropout* dropout, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                   const void* residual, int64_t ldr, void* y, int64_t ldy, void* stream) {
  GF_TRY(check_dtype(dtype));
  GF_TRY(check_dropout(dropout));
  if (rows < 0 || cols < 0 || rows > kMaxSize || cols > kMaxSize) return fail(GF_E_INVALID_ARGUMENT, "rows or cols negative or too large");
  if (rows == 0 || cols == 0) return GF_OK;
  GF_TRY(check_matrix("x", x, rows, ldx, cols, size_of(dtype)));
  GF_TRY(check_matrix("y", y, rows, ldy, cols, size_of(dtype)));
  if (residual != nullptr) GF_TRY(check_matrix("residual", residual, rows, ldr, cols, size_of(dtype)));
  const Drop d = make_drop(*dropout);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto* kernel = residual != nullptr ? k_dropout<T, true> : k_dropout<T, false>;
    kernel<<<blocks_for(rows * ((cols + 7) / 8)), 256, 0, (hipStream_t)stream>>>(d, rows, cols, (const T*)x, ldx, (const T*)residual, ldr, (T*)y,
                                                                                 ldy);
    GF_LAUNCH_CHECK("k_dropout");
    return (int)GF_OK;
  });
}

size_t gf_ff_saved_bytes(const gf_ff_args* args) {
  if (check_shape(args) != GF_OK || args->activation == GF_ACT_NONE) return 0;
  const int64_t element = args->dtype == GF_DTYPE_F32 ? Saved<float>::kBytes : args->dtype == GF_DTYPE_BF16 ? Saved<bf16>::kBytes : Saved<f16>::kBytes;
  return (size_t)(args->rows * saved_ld(args) * element);
}

size_t gf_ff_workspace_bytes(const gf_ff_args* args, int32_t is_backward) {
  if (check_shape(args) != GF_OK || args->rows == 0) return 0;
  Arena count{nullptr};
  const int rc = is_backward ? backward(*args, count, false, nullptr) : forward(*args, count, false, nullptr);
  return rc == GF_OK ? count.used : 0;
}

int gf_ff_forward(const gf_ff_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  GF_TRY(check_shape(args));
  const gf_ff_args& a = *args;
  if (a.rows == 0) return GF_OK;
  const int size = size_of(a.dtype);
  GF_TRY(check_matrix("x", a.x, a.rows, a.ldx, a.in_features, size));
  GF_TRY(check_matrix("weight", a.weight, weight_rows(&a), a.ldw, a.in_features, size));
  GF_TRY(check_matrix("y", a.y, a.rows, a.out_features, a.out_features, size));
  if (a.residual != nullptr) {
    if (a.activation != GF_ACT_NONE) return fail(GF_E_INVALID_ARGUMENT, "a gated product takes no residual");
    GF_TRY(check_matrix("residual", a.residual, a.rows, a.ldr, a.out_features, size));
  }
  if (a.saved != nullptr) GF_TRY(check_matrix("saved", a.saved, 1, 1, 1, 16));
  Arena count{nullptr}, ws{(uint8_t*)workspace};
  GF_TRY(forward(a, count, false, nullptr));
  GF_TRY(check_workspace(count.used, workspace, workspace_bytes));
  return forward(a, ws, true, (hipStream_t)stream);
}

int gf_ff_backward(const gf_ff_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  GF_TRY(check_shape(args));
  const gf_ff_args& a = *args;
  const int size = size_of(a.dtype);
  GF_TRY(check_matrix("x", a.x, a.rows, a.ldx, a.in_features, size));
  GF_TRY(check_matrix("weight", a.weight, weight_rows(&a), a.ldw, a.in_features, size));
  GF_TRY(check_matrix("dy", a.dy, a.rows, a.lddy, a.out_features, size));
  if (a.activation != GF_ACT_NONE) GF_TRY(check_matrix("saved", a.saved, 1, 1, 1, 16));
  if (a.rows == 0) return fail(GF_E_INVALID_ARGUMENT, "a backward needs rows");
  Arena count{nullptr}, ws{(uint8_t*)workspace};
  GF_TRY(backward(a, count, false, nullptr));
  GF_TRY(check_workspace(count.used, workspace, workspace_bytes));
  return backward(a, ws, true, (hipStream_t)stream);
}

}  // extern "C"
