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
//
// Times at the kernels are medians within whole passes, forward and backward on two states in turn, under a profiler; times that compare two
// forms or numbers of workgroups are of one kernel repeated, whose inputs the caches may partly hold.
#include "elements.h"

namespace {

using f32x4 = float __attribute__((ext_vector_type(4)));

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

// Rows and lanes.  A lane holds G groups of 8 consecutive columns of a row.  A row takes 16 lanes (up to 128 columns), a wave (up to 1536),
// or all waves of a workgroup; else a workgroup takes several rows at a time.
//
// Sums go over a row's lanes by cross-lane instructions, no LDS; past a wave the waves' sums meet in LDS, two numbers at once, at one
// barrier: the places alternate, and whoever writes one again has passed the barrier behind which all have read it.
constexpr int kMaxWaves = 16;

template <int CTRL, int ROWS = 0xf>
__device__ __attribute__((always_inline)) inline float lanes_moved(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, ROWS == 0xf));
}

// The sum over 16 consecutive lanes (WIDE: over the wave), the same bits in each.
template <bool WIDE>
__device__ __attribute__((always_inline)) inline float lanes_sum(float v) {
  v += lanes_moved<0xB1>(v);   // lane ^ 1
  v += lanes_moved<0x4E>(v);   // lane ^ 2
  v += lanes_moved<0x141>(v);  // the other four of eight
  v += lanes_moved<0x140>(v);  // the other eight of sixteen
  if constexpr (WIDE) {
    v += lanes_moved<0x142, 0xa>(v);  // lane 15's to the second sixteen, lane 47's to the fourth
    v += lanes_moved<0x143, 0xc>(v);  // lane 31's to the upper half
    v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
  }
  return v;
}

enum class Row { kPart, kWave, kWaves };  // a row of 16 lanes, of a wave, of the workgroup's waves

template <Row R, int G>
struct Place {
  int cols, lane, wave, waves, sub;  // lane of the row's wave (or part of one); which of the row's waves; which of the workgroup's rows
  float2 (*meet)[kMaxWaves];
  float inverse_last;  // 1 / the columns of the row's last wave
  int slot = 0;

  __device__ Place(int cols, float2 (*meet)[kMaxWaves]) : cols(cols), waves(R == Row::kWaves ? blockDim.x >> 6 : 1), meet(meet) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (R == Row::kPart) {
      lane = threadIdx.x & 15, wave = 0, sub = threadIdx.x >> 4;
    } else {
      lane = threadIdx.x & 63, sub = R == Row::kWave ? w : 0, wave = R == Row::kWave ? 0 : w;
    }
    inverse_last = R == Row::kWaves ? 1.0f / (float)(cols - (waves - 1) * 512 * G) : 0.0f;
  }
  static __host__ __device__ int rows_at_once(int threads) { return R == Row::kPart ? threads / 16 : R == Row::kWave ? threads / 64 : 1; }

  __device__ int col(int g) const { return ((wave * G + g) * (R == Row::kPart ? 16 : 64) + lane) * 8; }
  __device__ int count(int g) const {
    const int n = cols - col(g);
    return n < 0 ? 0 : n < 8 ? n : 8;
  }

  // a and b summed over the row
  __device__ float2 sum2(float a, float b) {
    float2 v{lanes_sum<R != Row::kPart>(a), lanes_sum<R != Row::kPart>(b)};
    if constexpr (R == Row::kWaves) {
      v = exchange(v);
      v = {lanes_sum<false>(v.x), lanes_sum<false>(v.y)};
    }
    return v;
  }

  // Each wave's v to the lane of its number in every sixteen lanes of the row, zero to the others.
  __device__ float2 exchange(float2 v) {
    if (lane == 0) meet[slot][wave] = v;
    __syncthreads();
    const int i = threadIdx.x & 15;
    v = meet[slot][i];
    slot ^= 1;
    return i < waves ? v : float2{0.0f, 0.0f};
  }

  // s / n, one step from s times the rounded 1 / n: exact where the quotient is, so a row of one value has it for a mean.
  static __device__ float quotient(float s, float n, float inverse) {
    const float q = s * inverse;
    return __builtin_fmaf(__builtin_fmaf(-q, n, s), inverse, q);
  }

  // The mean and the sum of squares about it.  Each wave takes its own about its own mean, from registers, and the waves' are joined
  // (Chan, Golub, LeVeque: "Updating formulae and a pairwise algorithm for computing sample variances", 1979): nothing cancels, at
  // one barrier.
  __device__ float2 spread(const float x[G][8], float inverse) {
    float s = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += x[g][j];
    s = lanes_sum<R != Row::kPart>(s);
    constexpr int kWhole = 512 * G;
    const float mean = R != Row::kWaves ? quotient(s, (float)cols, inverse) : s * (wave + 1 < waves ? 1.0f / kWhole : inverse_last);
    float d[G][8], m = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) d[g][j] = x[g][j] - mean;
    clear(d);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = __builtin_fmaf(d[g][j], d[g][j], m);
    m = lanes_sum<R != Row::kPart>(m);
    if constexpr (R != Row::kWaves) return {mean, m};
    const float2 v = exchange({s, m});
    const float total = quotient(lanes_sum<false>(v.x), (float)cols, inverse);
    const int i = threadIdx.x & 15;
    const float size = i + 1 < waves ? (float)kWhole : i + 1 == waves ? (float)(cols - (waves - 1) * kWhole) : 0.0f;
    const float off = v.x * (i + 1 < waves ? 1.0f / kWhole : inverse_last) - total;
    return {total, lanes_sum<false>(__builtin_fmaf(size * off, off, v.y))};
  }

  // 8 elements a group, zero past the row.
  template <typename T>
  __device__ void load(Vec<T, 8> v[G], const T* row) const {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int n = count(g);
      v[g] = (T)0.0f;
      if (n == 8) {
        v[g] = *(const Vec<T, 8>*)(row + col(g));
      } else if (n > 0) {
#pragma unroll
        for (int j = 0; j < 7; ++j)
          if (j < n) v[g][j] = row[col(g) + j];
      }
    }
  }
  template <typename T>
  __device__ void store(T* row, const float v[G][8]) const {
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (count(g) > 0) store8(row + col(g), v[g], count(g) == 8, count(g));
  }
  // Past the row, zero.
  __device__ void clear(float v[G][8]) const {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int n = count(g);
      if (n < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j >= n) v[g][j] = 0.0f;
      }
    }
  }
};

template <typename T, int G>
__device__ __attribute__((always_inline)) inline void widen(float v[G][8], const Vec<T, 8> from[G]) {
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[g][j] = (float)from[g][j];
}

// A half's map n -> n times + plus for a group of rows.  The branch's: gate * weight, gate * bias.  The next norm's: (1 + scale) * weight,
// (1 + scale) * bias + shift.  It is in registers for a chunk of rows where a lane has one group of columns; where it has more, in LDS, a
// copy for all rows, so that registers are left for two rows on their way.
template <int G, bool SHARED>
struct Maps {
  float own[SHARED ? 1 : 4][SHARED ? 1 : G][8];
  f32x4 (*shared)[G][2][64];  // [4][group][half][lane]
  int lane;
  __device__ void put(int which, int g, const float v[8]) {
    if constexpr (!SHARED) {
#pragma unroll
      for (int j = 0; j < 8; ++j) own[which][g][j] = v[j];
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) shared[which][g][h][lane] = f32x4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
    }
  }
  __device__ void get(int which, int g, float v[8]) const {
    if constexpr (!SHARED) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = own[which][g][j];
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 q = shared[which][g][h][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * h + j] = q[j];
      }
    }
  }
};
enum { kBranchTimes, kBranchPlus, kNextTimes, kNextPlus };

// 8 of a row of parameters, or of what stands for it where there is none.
template <typename T, typename P>
__device__ __attribute__((always_inline)) inline Vec<T, 8> row8(const P& at, int g, const T* p, float without) {
  const int n = at.count(g);
  Vec<T, 8> v = (T)(p == nullptr ? without : 0.0f);
  if (p != nullptr && n == 8) {
    v = *(const Vec<T, 8>*)(p + at.col(g));
  } else if (n < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j >= n) v[j] = (T)0.0f;
      else if (p != nullptr) v[j] = p[at.col(g) + j];
  }
  return v;
}

// Everything is asked for before anything is used.  In LDS the waves share out the groups.
template <typename T, int G, bool BRANCH, bool NEXT, bool SHARED, typename P>
__device__ __attribute__((always_inline)) inline void make_maps(Maps<G, SHARED>& m, const Norms<T>& a, const P& at, int64_t group, int wave, int waves) {
  auto one = [&](int g) __attribute__((always_inline)) {
    Vec<T, 8> f, w, b, f2, w2, b2, s2;
    if constexpr (BRANCH) {
      f = row8(at, g, a.gate ? a.gate + group * a.ld_gate : nullptr, 1.0f);
      w = row8(at, g, a.weight, 1.0f);
      b = row8(at, g, a.bias, 0.0f);
    }
    if constexpr (NEXT) {
      f2 = row8(at, g, a.scale ? a.scale + group * a.ld_scale : nullptr, 0.0f);
      w2 = row8(at, g, a.next_weight, 1.0f);
      b2 = row8(at, g, a.next_bias, 0.0f);
      s2 = row8(at, g, a.shift ? a.shift + group * a.ld_shift : nullptr, 0.0f);
    }
    float times[8], plus[8];
    if constexpr (BRANCH) {
      const float value = a.gate ? 1.0f : a.gate_value;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float factor = value * (float)f[j];
        times[j] = factor * (float)w[j], plus[j] = a.bias ? factor * (float)b[j] : 0.0f;  // an infinite gate times no bias is no NaN
      }
      m.put(kBranchTimes, g, times), m.put(kBranchPlus, g, plus);
    }
    if constexpr (NEXT) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float factor = 1.0f + (float)f2[j];
        times[j] = factor * (float)w2[j], plus[j] = a.next_bias ? __builtin_fmaf(factor, (float)b2[j], (float)s2[j]) : (float)s2[j];
      }
      m.put(kNextTimes, g, times), m.put(kNextPlus, g, plus);
    }
  };
  if constexpr (SHARED) {
    for (int g = wave; g < G; g += waves) one(g);
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g) one(g);
  }
}

// Whether they are in LDS: where a wave has a row of several groups.
template <Row R, int G>
constexpr bool kMapsShared = R == Row::kWave && G > 1;

// 1 / sqrt(v) by the hardware's (1 unit in the last place), which takes a subnormal number for zero.
__device__ __attribute__((always_inline)) inline float inverse_root(float v) {
  const bool low = v < 0x1p-96f;
  const float r = __builtin_amdgcn_rsqf(low ? v * 0x1p64f : v);
  return low ? r * 0x1p32f : r;
}

// x becomes n(x), zero past the row; returns 1 / deviation (rms: 1 / root mean square).
template <int G, typename P>
__device__ __attribute__((always_inline)) inline float normalise(float x[G][8], int kind, float eps, float inverse, P& at) {
  float rstd;
  if (kind == GF_NORM_LAYER) {
    const float2 s = at.spread(x, inverse);
    rstd = inverse_root(__builtin_fmaf(s.y, inverse, eps));
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[g][j] = (x[g][j] - s.x) * rstd;
    at.clear(x);
  } else {
    float v = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) v = __builtin_fmaf(x[g][j], x[g][j], v);
    rstd = inverse_root(__builtin_fmaf(at.sum2(v, 0.0f).x, inverse, eps));
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[g][j] *= rstd;
  }
  return rstd;
}

// The gradient of x from that of n(x), in place: rstd (g - mean g - n(x) mean(g n(x))), without mean g for rms; zero past the row.
template <int G, typename P>
__device__ __attribute__((always_inline)) inline void through_norm(float g_[G][8], const float n_[G][8], int kind, float rstd, float inverse, P& at) {
  float a = 0.0f, b = 0.0f;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < 8; ++j) a += g_[g][j], b = __builtin_fmaf(g_[g][j], n_[g][j], b);
  const float2 s = at.sum2(a, b);
  a = kind == GF_NORM_LAYER ? s.x * inverse : 0.0f;
  b = s.y * inverse;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < 8; ++j) g_[g][j] = rstd * (g_[g][j] - __builtin_fmaf(n_[g][j], b, a));
  if (kind == GF_NORM_LAYER) at.clear(g_);
}

// Chunks of rows, each of one group: `chunks` a group of `rows` rows, `all` together.
struct Chunks {
  int64_t rows, chunks, all;
};

// The maps' LDS of a kernel, and a barrier around its filling.
#define GF_MAPS(BRANCH, NEXT)                                                                                            \
  constexpr bool kShared = kMapsShared<R, G>;                                                                            \
  __shared__ f32x4 map_words[kShared ? 4 : 1][kShared ? G : 1][2][64];                                                   \
  Maps<G, kShared> maps;                                                                                                 \
  maps.lane = at.lane, maps.shared = (f32x4(*)[G][2][64])map_words;                                                      \
  auto set_maps = [&](int64_t group) {                                                                                   \
    if (kShared) __syncthreads();                                                                                        \
    make_maps<T, G, BRANCH, NEXT, kShared>(maps, a, at, group, kShared ? at.sub : 0, kShared ? (int)blockDim.x >> 6 : 1); \
    if (kShared) __syncthreads();                                                                                        \
  }

// Forward.  BRANCH: s from x and the residual; NEXT: h from s (without BRANCH, from x).  The next row is on its way while one is worked on.
// In bfloat16: gate_add of 16384 x 2560 51 us (5.0 TB/s: memory), gate_add_norm of 8192 x 1280 22 us (3.9 TB/s: two statistics a row one after
// the other), norm of 16384 x 320 11 us (1.9 TB/s: 684 workgroups of four waves are 11 waves a unit, fewer than their registers let it hold, and
// 24 of their 64 lanes are idle); one row of 1280 3.9 us.
template <typename T, Row R, int G, int THREADS, bool BRANCH, bool NEXT>
__global__ __launch_bounds__(THREADS) void k_norm_forward(Norms<T> a, Chunks cut) {
  __shared__ float2 meet[2][kMaxWaves];
  Place<R, G> at(a.cols, meet);
  GF_MAPS(BRANCH, NEXT);
  const int at_once = at.rows_at_once(blockDim.x);
  for (int64_t chunk = blockIdx.x; chunk < cut.all; chunk += gridDim.x) {
    const int64_t group = chunk / cut.chunks, first = chunk % cut.chunks * cut.rows;
    const int64_t begin = group * a.group_rows + first, end = group * a.group_rows + (first + cut.rows < a.group_rows ? first + cut.rows : a.group_rows);
    Vec<T, 8> vx[G], vr[BRANCH ? G : 1];
    auto fetch = [&](int64_t row) {
      at.load(vx, a.x + row * a.ldx);
      if constexpr (BRANCH) at.load(vr, a.residual + row * a.ldr);
    };
    int64_t row = begin + at.sub;
    if (row < end) fetch(row);
    set_maps(group);
    for (; row < end; row += at_once) {
      asm volatile("" ::: "memory");  // what LDS holds of the maps stays there
      float v[G][8], r[BRANCH ? G : 1][8];
      widen<T, G>(v, vx);
      if constexpr (BRANCH) widen<T, G>(r, vr);
      if (row + at_once < end) fetch(row + at_once);
      if constexpr (BRANCH) {
        if (a.kind != GF_NORM_NONE) normalise<G>(v, a.kind, a.eps, a.inverse, at);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float w[8], b[8];
          maps.get(kBranchTimes, g, w), maps.get(kBranchPlus, g, b);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[g][j] = __builtin_fmaf(a.residual_scale, r[g][j], __builtin_fmaf(v[g][j], w[j], b[j]));
        }
        if (a.stream != nullptr) at.store(a.stream + row * a.cols, v);
      }
      if constexpr (NEXT) {
        normalise<G>(v, a.next_kind, a.next_eps, a.inverse, at);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float w[8], b[8];
          maps.get(kNextTimes, g, w), maps.get(kNextPlus, g, b);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[g][j] = __builtin_fmaf(v[g][j], w[j], b[j]);
        }
        at.store(a.normed + row * a.cols, v);
      }
    }
  }
}

// Column sums of a chunk of rows, per element: of ds, ds n(x), dh, dh n'(s).  A half that is not there has none in memory.
constexpr int kSums = 4;

// Backward, by chunks of rows.  SUMS: the column sums too, into parts [chunk][2 of each half][width].  In bfloat16: gate_add of 16384 x 2560
// 54 to 58 us (4.3 to 4.7 TB/s), gate_add_norm of 8192 x 1280 42 us (3.0 TB/s, nine waves a unit where the registers let it hold twelve;
// repeated without sums 31 us, 4.1 TB/s), norm of 16384 x 320 15 us (2.1 TB/s, eight waves a unit).
template <typename T, Row R, int G, int THREADS, bool BRANCH, bool NEXT, bool SUMS>
__global__ __launch_bounds__(THREADS) void k_norm_backward(Norms<T> a, Chunks cut, float* parts, int64_t width) {
  __shared__ float2 meet[2][kMaxWaves];
  constexpr int kSpan = (R == Row::kPart ? 128 : 512) * G, kRows = R == Row::kPart ? 16 : 8;  // columns that a row's lanes hold; rows at a time
  __shared__ f32x4 together[2][SUMS && R != Row::kWaves ? kRows : 1][SUMS && R != Row::kWaves ? kSpan / 4 : 1];
  Place<R, G> at(a.cols, meet);
  GF_MAPS(BRANCH, NEXT);
  const int at_once = at.rows_at_once(blockDim.x);
  for (int64_t chunk = blockIdx.x; chunk < cut.all; chunk += gridDim.x) {
    const int64_t group = chunk / cut.chunks, first = chunk % cut.chunks * cut.rows;
    const int64_t begin = group * a.group_rows + first, end = group * a.group_rows + (first + cut.rows < a.group_rows ? first + cut.rows : a.group_rows);
    const bool needs_x = NEXT || SUMS || a.kind != GF_NORM_NONE;
    // The next row is on its way while one is worked on: x and the residual, and the gradients too where registers are left (else those
    // come while the row's statistics are made).
    constexpr bool kAhead = G == 1 || !(BRANCH && NEXT);
    Vec<T, 8> vx[G] = {}, vr[BRANCH && NEXT ? G : 1], vs[BRANCH ? G : 1] = {}, vh[NEXT ? G : 1];
    auto fetch_gradients = [&](int64_t row) {
      if constexpr (BRANCH) {
        if (a.dstream != nullptr) at.load(vs, a.dstream + row * a.ld_dstream);
      }
      if constexpr (NEXT) at.load(vh, a.dnormed + row * a.ld_dnormed);
    };
    auto fetch = [&](int64_t row) {
      if (needs_x) at.load(vx, a.x + row * a.ldx);
      if constexpr (BRANCH && NEXT) at.load(vr, a.residual + row * a.ldr);
      if constexpr (kAhead) fetch_gradients(row);
    };
    int64_t row = begin + at.sub;
    if (row < end) fetch(row);
    set_maps(group);
    float sums[SUMS ? kSums : 1][G][8] = {};
    auto add = [&](int k, const float d[G][8], const float n[G][8]) {
      if constexpr (SUMS) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int j = 0; j < 8; ++j) sums[k][g][j] += d[g][j], sums[k + 1][g][j] = __builtin_fmaf(d[g][j], n[g][j], sums[k + 1][g][j]);
      }
    };
    for (; row < end; row += at_once) {
      asm volatile("" ::: "memory");  // what LDS holds of the maps stays there
      if constexpr (!kAhead) fetch_gradients(row);
      float x[G][8], r[BRANCH && NEXT ? G : 1][8], d[G][8];
      widen<T, G>(x, vx);
      if constexpr (BRANCH && NEXT) widen<T, G>(r, vr);
      Vec<T, 8> ws[BRANCH ? G : 1], wh[NEXT ? G : 1];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if constexpr (BRANCH) ws[g] = vs[g];
        if constexpr (NEXT) wh[g] = vh[g];
      }
      if (row + at_once < end) fetch(row + at_once);
      float rstd = 1.0f;
      if constexpr (BRANCH) {
        if (a.kind != GF_NORM_NONE) rstd = normalise<G>(x, a.kind, a.eps, a.inverse, at);
      }
      if constexpr (NEXT) {
        float s[G][8];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float w[8], b[8];
          if constexpr (BRANCH) maps.get(kBranchTimes, g, w), maps.get(kBranchPlus, g, b);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (BRANCH)
              s[g][j] = __builtin_fmaf(a.residual_scale, r[g][j], __builtin_fmaf(x[g][j], w[j], b[j]));
            else
              s[g][j] = x[g][j];
          }
        }
        const float next_rstd = normalise<G>(s, a.next_kind, a.next_eps, a.inverse, at);
        widen<T, G>(d, wh);
        add(2, d, s);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float w[8];
          maps.get(kNextTimes, g, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) d[g][j] *= w[j];
        }
        through_norm<G>(d, s, a.next_kind, next_rstd, a.inverse, at);
      }
      if constexpr (BRANCH) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int j = 0; j < 8; ++j) d[g][j] = NEXT ? d[g][j] + (float)ws[g][j] : (float)ws[g][j];
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
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float w[8];
            maps.get(kBranchTimes, g, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) d[g][j] *= w[j];
          }
          if (a.kind != GF_NORM_NONE) through_norm<G>(d, x, a.kind, rstd, a.inverse, at);
        }
      }
      if (a.dx != nullptr) at.store(a.dx + row * a.cols, d);
    }
    if constexpr (SUMS) {
#pragma unroll
      for (int k = BRANCH ? 0 : 2; k < (NEXT ? kSums : 2); k += 2) {
        float* const out = parts + (BRANCH && NEXT ? chunk * kSums + k : chunk * 2) * width;
        if (R == Row::kWaves || at_once == 1) {
#pragma unroll
          for (int g = 0; g < G; ++g)
            if (at.count(g) > 0) store8(out + at.col(g), sums[k][g], true, 8), store8(out + width + at.col(g), sums[k + 1][g], true, 8);
          continue;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float* const v = sums[k + i][g] + 4 * h;
              together[i][at.sub][at.col(g) / 4 + h] = f32x4{v[0], v[1], v[2], v[3]};
            }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * (kSpan / 4); c += blockDim.x) {
          const int i = c / (kSpan / 4), q = c % (kSpan / 4);
          if (q * 4 >= width) continue;
          f32x4 v = together[i][0][q];
#pragma unroll
          for (int n = 1; n < kRows; ++n)
            if (n < at_once) v += together[i][n][q];
          *(f32x4*)(out + i * width + q * 4) = v;
        }
      }
      __syncthreads();
    }
  }
}

// The chunks' sums into gradients: 16 columns a workgroup, the branch's (z = 0) or the next norm's.  With S0 = sum d, S1 = sum d n of a
// group, w, b the half's weight and bias and f its factor (the gate; 1 + scale):
//   of the factor  w S1 + b S0;   of the shift  S0;   of w  sum over groups of f S1;   of b  sum over groups of f S0.
// 4 lanes take 16 columns, 128 such members of a workgroup share out the groups, `team` of them (a power of two) one group: all chunks of
// it are asked for at once (sums of 16384 x 2560, repeated: 10.8 us; 32 columns a workgroup 12.8, 8, less than a line of memory, 18).  A slab (y) is
// a range of groups, and what is shared by all groups goes to `partial` [slab][half][4][width] (of the weight, the bias, the factor, the
// shift) where there are several slabs.  6 to 11 us: a launch and the trips to memory of sums that other dies have written.
template <typename T>
struct Half {
  const T *weight, *bias, *factor;
  int64_t ld_factor, ld_shift;
  float one, value;  // the factor is one + factor[], or `value`
  T *dweight, *dbias, *dfactor, *dshift;
};

// Asked for only: what needs it waits for it.
template <typename T>
__device__ __attribute__((always_inline)) inline Vec<T, 4> load4(const T* p, int64_t c, int n, float without) {
  Vec<T, 4> v = (T)without;
  if (p == nullptr) return v;
  if (n == 4) return *(const Vec<T, 4>*)(p + c);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < n) v[j] = p[c + j];
  return v;
}

template <typename T>
__device__ __attribute__((always_inline)) inline f32x4 widen4(Vec<T, 4> v) {
  return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}

template <typename T>
__device__ __attribute__((always_inline)) inline void store4(T* p, int64_t c, int n, f32x4 v) {
  if (n == 4) {
    *(Vec<T, 4>*)(p + c) = Vec<T, 4>{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < n) p[c + j] = (T)v[j];
  }
}

__device__ __attribute__((always_inline)) inline f32x4 from_lane(f32x4 v, int mask) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __shfl_xor(v[j], mask);
  return v;
}

constexpr int kFinishThreads = 512, kFinishLanes = 4, kFinishMembers = 64 / kFinishLanes;  // lanes of 4 columns each; members of a wave

template <typename T>
__global__ __launch_bounds__(kFinishThreads) void k_norm_finish(Half<T> branch, Half<T> next, int half0, int32_t cols, int64_t groups, int64_t chunks,
                                                      const float* parts, int64_t width, int team, float* partial) {
  __shared__ f32x4 meet[4][kFinishThreads / 64][kFinishLanes];
  const int lane = threadIdx.x % kFinishLanes, member = threadIdx.x / kFinishLanes, wave = threadIdx.x >> 6, half = half0 + blockIdx.z;
  const bool first_of_wave = (threadIdx.x & 63) < kFinishLanes;
  const Half<T>& h = half == 0 ? branch : next;
  const int64_t c = blockIdx.x * (4ll * kFinishLanes) + lane * 4;
  const int n = cols - c < 0 ? 0 : cols - c < 4 ? (int)(cols - c) : 4;
  const int64_t slab = (groups + gridDim.y - 1) / gridDim.y, g0 = blockIdx.y * slab, g1 = g0 + slab < groups ? g0 + slab : groups;
  const int teams = kFinishThreads / kFinishLanes / team, of = member & (team - 1);
  const Vec<T, 4> w = load4(h.weight, c, n, 1.0f), b = load4(h.bias, c, n, 0.0f);
  f32x4 shared[4] = {};
  for (int64_t base = g0; base < g1; base += teams) {
    const int64_t g = base + member / team;
    f32x4 s0 = 0.0f, s1 = 0.0f;
    const Vec<T, 4> factor = load4(h.factor != nullptr && g < g1 ? h.factor + g * h.ld_factor : nullptr, c, n, 0.0f);
    if (n > 0 && g < g1) {
#pragma unroll 8
      for (int64_t i = of; i < chunks; i += team) {
        const float* p = parts + ((g * chunks + i) * gridDim.z + blockIdx.z) * 2 * width + c;  // 4 of them: width is a multiple of 8
        s0 += *(const f32x4*)p, s1 += *(const f32x4*)(p + width);
      }
    }
    for (int i = 1; i < team && i < kFinishMembers; i *= 2) s0 += from_lane(s0, kFinishLanes * i), s1 += from_lane(s1, kFinishLanes * i);
    if (team > kFinishMembers) {
      __syncthreads();
      if (first_of_wave) meet[0][wave][lane] = s0, meet[1][wave][lane] = s1;
      __syncthreads();
      s0 = 0.0f, s1 = 0.0f;
      const int w0 = wave & ~(team / kFinishMembers - 1);
      for (int i = 0; i < team / kFinishMembers; ++i) s0 += meet[0][w0 + i][lane], s1 += meet[1][w0 + i][lane];
    }
    if (n > 0 && g < g1 && of == 0) {
      const f32x4 f = h.factor != nullptr ? h.one + widen4<T>(factor) : f32x4(h.value);
      shared[0] += f * s1, shared[1] += f * s0;
      const f32x4 own = widen4<T>(w) * s1 + (h.bias != nullptr ? widen4<T>(b) * s0 : f32x4(0.0f));
      if (h.dfactor != nullptr) {
        if (h.ld_factor != 0) store4(h.dfactor + g * cols, c, n, own);
        else shared[2] += own;
      }
      if (h.dshift != nullptr) {
        if (h.ld_shift != 0) store4(h.dshift + g * cols, c, n, s0);
        else shared[3] += s0;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int i = 1; i < kFinishMembers; i *= 2) shared[k] += from_lane(shared[k], kFinishLanes * i);
    if (first_of_wave) meet[k][wave][lane] = shared[k];
  }
  __syncthreads();
  if (member >= 4 || n == 0) return;
  f32x4 v = 0.0f;
#pragma unroll
  for (int i = 0; i < kFinishThreads / 64; ++i) v += meet[member][i][lane];
  if (partial != nullptr) {
    *(f32x4*)(partial + (((int64_t)blockIdx.y * gridDim.z + blockIdx.z) * 4 + member) * width + c) = v;
    return;
  }
  T* const out = member == 0 ? h.dweight : member == 1 ? h.dbias : member == 2 ? (h.ld_factor == 0 ? h.dfactor : nullptr) : h.ld_shift == 0 ? h.dshift : nullptr;
  if (out != nullptr) store4(out, c, n, v);
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
  for (int64_t i = 0; i < slabs; ++i) v += partial[((i * gridDim.z + blockIdx.z) * 4 + which) * width + c];
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

template <Row R, int G, int THREADS>
struct Form {
  static constexpr Row row = R;
  static constexpr int groups = G, threads = THREADS;
};

// How a row is held: 16 lanes up to 128 columns, a wave up to `wave_cols`, else a workgroup's waves, 512 columns each, past 6144 (12 waves,
// as many as have the registers) 1024.
template <typename F>
int with_form(int64_t cols, int64_t wave_cols, F f) {
  if (cols <= 128) return f(Form<Row::kPart, 1, 256>());
  if (cols <= 512) return f(Form<Row::kWave, 1, 512>());
  if (cols <= std::min<int64_t>(wave_cols, 1024)) return f(Form<Row::kWave, 2, 512>());
  if (cols <= std::min<int64_t>(wave_cols, 1536)) return f(Form<Row::kWave, 3, 512>());
  if (cols <= 6144) return f(Form<Row::kWaves, 1, 768>());
  if (cols <= 8192) return f(Form<Row::kWaves, 2, 512>());
  return f(Form<Row::kWaves, 2, 1024>());
}

// The widest row that a wave takes alone.  8192 x 1280 in bfloat16, gate_add_norm, repeated: 22 us forward (three waves a row: 26 to 29), 31 backward
// without sums (33).  The sums of both halves leave a wave with three groups a lane no registers: 54 us by three waves, 66 by one.
// With few rows a row's time counts: one of 1280 takes 3.2 us by three waves, 5.6 by one.  2048 rows give each of 256
// units eight waves; the border was not timed at other widths.
int64_t wave_cols(const gf_norm_args& a, bool sums) {
  if (a.rows < 2048) return 512;
  return sums && a.residual != nullptr && a.next_kind != GF_NORM_NONE ? 1024 : 1536;
}

// Threads of a workgroup: as many rows at a time as `most` waves hold, but no more than there are in a group.
template <Row R, int G>
int threads_of(int64_t cols, int64_t group_rows, int most) {
  if (R == Row::kWaves) return 64 * (int)((cols + 512 * G - 1) / (512 * G));
  if (R == Row::kPart) return (int)std::min<int64_t>(round_up(group_rows * 16, 64), most * 64);
  return 64 * (int)std::min<int64_t>(group_rows, most);
}

// Each group in chunks of whole turns of a workgroup, until there are about `want` chunks.
Chunks cut_rows(int64_t rows, int64_t group_rows, int at_once, int64_t want) {
  const int64_t groups = rows / group_rows, turns = (group_rows + at_once - 1) / at_once;
  const int64_t each = std::max<int64_t>((turns * groups + want - 1) / want, 1);
  Chunks c;
  c.rows = std::min(each, turns) * at_once;
  c.chunks = (group_rows + c.rows - 1) / c.rows;
  c.all = groups * c.chunks;
  return c;
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
  const bool sums = wants_sums(a);
  return with_dtype(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_form(a.cols, wave_cols(a, sums), [&](auto form) {
      constexpr Row R = form.row;
      constexpr int G = form.groups, kThreads = form.threads;
      return with_halves(a, [&](auto branch, auto next) {
        constexpr bool kBranch = branch.value, kNext = next.value, kSumless = R == Row::kWave && G == 3 && kBranch && kNext;
        // Workgroups for each of 256 compute units as their registers allow (12 waves for both halves' sums, 16 for one's), and each of them its
        // chunks' sums to write and k_norm_finish to read: gate_add of 16384 x 2560, repeated, in 512 workgroups 63 and 10 us, 768 56 and 11,
        // 1024 63 and 15.  Without sums two, which the barriers or loads of one do not keep waiting (8192 x 1280 gate_add_norm: 31 us; one of 8 waves 37).
        const int threads = threads_of<R, G>(a.cols, a.group_rows, R == Row::kPart || (!sums && G > 1) ? 4 : 8);
        const int fit = R == Row::kWaves ? std::min(std::max((kBranch && kNext ? 12 : 16) * 64 / threads, 1), 3) : 1;
        const Chunks cut = cut_rows(a.rows, a.group_rows, Place<R, G>::rows_at_once(threads), 256 * (sums ? fit : 2));
        const int64_t chunks = cut.chunks, all = cut.all;
        const int64_t slabs = groups <= 1024 ? 1 : std::min<int64_t>((groups + 511) / 512, 64);
        const int half0 = kBranch ? 0 : 1, halves = (kBranch ? 1 : 0) + (kNext ? 1 : 0);
        float* const parts = sums ? (float*)ws.take(all * 2 * halves * width * 4) : nullptr;
        float* const partial = sums && slabs > 1 ? (float*)ws.take(slabs * halves * 4 * width * 4) : nullptr;
        GF_RUN {
          const Norms<T> n = make_norms<T>(a);
          const unsigned grid = (unsigned)std::min<int64_t>(all, 1 << 20);
          if (!sums) {
            k_norm_backward<T, R, G, kThreads, kBranch, kNext, false><<<grid, threads, 0, s>>>(n, cut, nullptr, 0);
          } else if constexpr (!kSumless) {
            k_norm_backward<T, R, G, kThreads, kBranch, kNext, true><<<grid, threads, 0, s>>>(n, cut, parts, width);
          }
          GF_LAUNCH_CHECK("k_norm_backward");
          if (sums) {
            const Half<T> b{n.weight, n.bias, n.gate, n.ld_gate, 0, 0.0f, n.gate_value, n.dweight, n.dbias, n.dgate, nullptr};
            const Half<T> f{n.next_weight, n.next_bias, n.scale, n.ld_scale, n.ld_shift, 1.0f, 1.0f, n.dnext_weight, n.dnext_bias, n.dscale, n.dshift};
            int team = 1;
            while (team < kFinishThreads / kFinishLanes && team * 2 * groups <= kFinishThreads / kFinishLanes) team *= 2;
            const dim3 blocks((unsigned)((a.cols + 4 * kFinishLanes - 1) / (4 * kFinishLanes)), (unsigned)slabs, halves);
            k_norm_finish<T><<<blocks, kFinishThreads, 0, s>>>(b, f, half0, n.cols, groups, chunks, parts, width, team, partial);
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
    return with_form(a.cols, wave_cols(a, false), [&](auto form) {
      constexpr Row R = form.row;
      constexpr int G = form.groups, kThreads = form.threads;
      return with_halves(a, [&](auto branch, auto next) {
        // enough workgroups to fill the units, each with rows enough that its maps and first row count for little (16384 x 2560 gate_add,
        // repeated: 46 us, with 1024 workgroups 55)
        const int threads = threads_of<R, G>(a.cols, a.group_rows, 4);
        const Chunks cut = cut_rows(a.rows, a.group_rows, Place<R, G>::rows_at_once(threads), R == Row::kWaves ? 512 : 768);
        const unsigned grid = (unsigned)std::min<int64_t>(cut.all, 1 << 20);
        k_norm_forward<T, R, G, kThreads, branch.value, next.value><<<grid, threads, 0, (hipStream_t)stream>>>(make_norms<T>(a), cut);
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
