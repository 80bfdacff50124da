// Sampling of tokens from logits by temperature, top-k, top-p and min-p, from given uniforms, and the filtered
// distributions themselves.
//
// Of a row l of V logits with largest one m (NaN counts as -inf), temperature t, and the tokens ranked by falling
// logit, equal ones by index:
//   w_x = exp((l_x - m) / t);  K: the first k in rank (all without a k; t = 0: the first alone)
//   P: of K those whose predecessors in K weigh less than p of K's total, and the first one
//   kept: of P those with w_x >= min_p
// The distribution is w over the kept tokens; the token is the first x in index order with
// w_0 + ... + w_x > u (the kept tokens' total).
//
// What is kept is decided by a comparison of sums over up to 10^5 terms, and a draw lies next to a border once
// in a few thousand tokens if sums are off by 10^-7; so weights are float64 (2^f by its Taylor series, 2 10^-13), and
// sums are float64 in a fixed order or integers, which have none.
//
// Nothing is sorted.  A row is cut into chunks, one per block:
//   scan     the chunk's maximum, and what the row's filters need: with top-k a histogram of how many logits
//            lie in each bin of 1/16 below the maximum, with top-p of their mass, without both the mass alone
//   select   finds in the row's joined histograms the bins that hold the borders; of the chunk, lists the few tokens in
//            those bins, and adds up the mass of what is kept for certain (min-p alone: what is kept)
//   draw     one block per row: decides the border by a radix selection among the listed tokens (by rank, by
//            mass, by index among equal ones), draws the chunk by the chunks' masses, and the token in it
//   write    the probabilities, in place of the draw
#include "tq_common.h"

namespace tq {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kTileTokens = kThreads * 8;  // a thread takes 8 tokens in a row
constexpr int kBins = 512, kTail = kBins - 1;  // the last bin has everything below the others
constexpr int kMaxChunks = 512;
constexpr int kShort = 2048;  // listed tokens that fit the draw's shared memory
constexpr double kUnit = 0x1p48;  // of a chunk's masses: at most 2^15 tokens of weight <= 1 in 63 bits

struct SampleArgs {
  const void* logits;
  int64_t ld;  // elements between rows
  int N, V;
  // one setting for all rows, or one per row
  const float* t_rows;
  const int32_t* k_rows;
  const float* p_rows;
  const float* m_rows;
  double t, p, m;
  int k;
  const float* uniforms;  // [N], or null: probabilities
  int64_t* tokens;        // [N]
  float* probs;           // [N, V]
  int C, lg_chunk;        // chunks of a row, tokens of a chunk
  // workspace
  struct RowState* state;  // [N]
  float* top;              // [N, C] chunk's maximum
  double* mass;            // [N, C] certain mass, relative to the chunk's (scan) or the row's maximum (select)
  uint64_t* total;         // [N, C] of the histogram
  int32_t* listed;         // [N, C]
  uint64_t* hist;          // [N, C, kBins]
  uint16_t* list;          // [N, C << lg_chunk] places in the chunk
};

// What a row's borders are: written by select (goal, cut) and draw (the rest)
struct RowState {
  double goal;       // top-p: mass at which tokens are no longer kept
  int cut;           // 0: top-p's border is not needed (min-p is stricter)
  uint32_t key;      // kept: larger keys, and this key up to index `last`
  int last;
  float top;
  double inverse;    // 1 / kept mass
};

enum Mode { kAll, kMinP, kTopP, kTopK };

// A row's settings as the kernels use them
struct Settings {
  Mode mode;
  int k;
  double c;      // log2(e) / t
  double p, m;
  __device__ __forceinline__ Settings(const SampleArgs& a, int row) {
    const double t = a.t_rows ? static_cast<double>(a.t_rows[row]) : a.t;
    k = a.k_rows ? a.k_rows[row] : a.k;
    p = a.p_rows ? static_cast<double>(a.p_rows[row]) : a.p;
    m = a.m_rows ? static_cast<double>(a.m_rows[row]) : a.m;
    const bool greedy = !(t > 0.0);
    if (greedy) k = 1;
    c = fmin(1.4426950408889634 / (greedy ? 1.0 : t), 1e300);
    m = m > 0.0 ? fmin(m, 1.0) : 0.0;
    const bool by_rank = k > 0 && k < a.V, by_mass = p < 1.0;
    if (!by_mass) p = 1.0;
    mode = by_rank ? kTopK : by_mass ? kTopP : m > 0.0 ? kMinP : kAll;
  }
};

// 2^y, y <= 0: 2^n by the exponent, 2^f for |f| <= 1/2 by the series of exp(f ln 2) up to the 10th power
__device__ __forceinline__ double exp2_f64(double y) {
  constexpr double L = 0.6931471805599453;
  constexpr double A[11] = {1.0, L, L * L / 2, L * L * L / 6, L * L * L * L / 24, L * L * L * L * L / 120,
                            L * L * L * L * L * L / 720, L * L * L * L * L * L * L / 5040, L * L * L * L * L * L * L * L / 40320,
                            L * L * L * L * L * L * L * L * L / 362880, L * L * L * L * L * L * L * L * L * L / 3628800};
  y = fmax(y, -1200.0);
  const double r = rint(y), f = y - r;
  double s = A[10];
#pragma unroll
  for (int i = 9; i >= 0; --i) s = fma(s, f, A[i]);
  return ldexp(s, static_cast<int>(r));
}
// a logit's weight under maximum m (finite, or v = m)
__device__ __forceinline__ double weight(float v, float m, double c) {
  return exp2_f64((static_cast<double>(v) - static_cast<double>(m)) * c);
}

// Falling bins of 1/16 on an absolute grid, so that chunks with other maxima have the same ones.  Monotone
// in v; logits beyond 2^27 / 16 share their bins.
__device__ __forceinline__ int grid_of(float v) { return static_cast<int>(floorf(fminf(fmaxf(v * 16.f, -0x1p27f), 0x1p27f))); }
__device__ __forceinline__ int bin_of(float v, int grid_top) { return min(grid_top - grid_of(v), kTail); }
// larger for larger floats
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Eight logits from x on; what is not there is -inf, and so is a NaN.
template <int DT>
__device__ __forceinline__ void load_logits(const void* row, int x, int V, float (&v)[8]) {
  if (x + 8 <= V) {
    if constexpr (DT == TQ_F32) {
      __builtin_memcpy(v, static_cast<const float*>(row) + x, 32);
    } else {
      uint16_t r[8];
      __builtin_memcpy(r, static_cast<const uint16_t*>(row) + x, 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = DT == TQ_F16 ? h2f(r[j]) : bf16_to_f32(r[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x + j < V ? load_act<DT>(row, x + j) : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = v[j] == v[j] ? v[j] : -INFINITY;
}
template <int DT>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int row) {
  return static_cast<const uint8_t*>(a.logits) + row * a.ld * (DT == TQ_F32 ? 4 : 2);
}
// Under an infinite maximum only infinite logits have a weight: as 0 against -inf, maximum 0.
__device__ __forceinline__ float tame(float v, float m) { return m == INFINITY ? (v == INFINITY ? 0.f : -INFINITY) : v; }
__device__ __forceinline__ float tame(float m) { return m == INFINITY ? 0.f : m; }

// ---------------------------------------------------------------- over a wave, over a block
template <class T, class Op>
__device__ __forceinline__ T wave_all(T v, Op op) {
#pragma unroll
  for (int sh = 32; sh >= 1; sh >>= 1) v = op(v, static_cast<T>(__shfl_xor(v, sh, 64)));
  return v;
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int sh = 1; sh < 64; sh <<= 1) {
    const T t = __shfl_up(v, sh, 64);
    if (lane >= sh) v += t;
  }
  return v;
}
// of all threads, in a fixed order; s: kWaves values, free again behind the next barrier
template <class T, class Op>
__device__ __forceinline__ T block_all(T v, T* s, Op op) {
  v = wave_all(v, op);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  T r = s[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = op(r, s[w]);
  return r;
}
struct Sum {
  template <class T>
  __device__ __forceinline__ T operator()(T a, T b) const {
    return a + b;
  }
};
struct Max {
  template <class T>
  __device__ __forceinline__ T operator()(T a, T b) const {
    return a > b ? a : b;
  }
};

__device__ __forceinline__ float row_top(const SampleArgs& a, int row) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  for (int c = lane; c < a.C; c += 64) m = fmaxf(m, a.top[static_cast<int64_t>(row) * a.C + c]);
  return wave_all(m, Max{});
}

// ---------------------------------------------------------------- scan
template <int DT, int NV>
__global__ void __launch_bounds__(kThreads) sample_scan_kernel(SampleArgs a) {
  __shared__ uint64_t s_hist[kBins];
  __shared__ float s_max[kWaves];
  __shared__ double s_sum[kWaves];
  __shared__ uint64_t s_total[kWaves];
  const int row = blockIdx.x / a.C, c = blockIdx.x - row * a.C, tid = threadIdx.x;
  const void* const src = row_of<DT>(a, row);
  float v[NV / 8][8];
#pragma unroll
  for (int j = 0; j < NV / 8; ++j) load_logits<DT>(src, (c << a.lg_chunk) + j * kTileTokens + tid * 8, a.V, v[j]);
  const Settings set(a, row);
  if (tid < kBins) s_hist[tid] = 0;
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < NV / 8; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, v[j][e]);
  m = block_all(m, s_max, Max{});
  const int64_t at = static_cast<int64_t>(row) * a.C + c;
  if (tid == 0) a.top[at] = m;
  if (set.mode == kMinP) return;
  if (m == -INFINITY) {
    if (tid == 0) {
      a.mass[at] = 0.0;
      a.total[at] = 0;
    }
    if (set.mode != kAll && tid < kBins) a.hist[at * kBins + tid] = 0;
    return;
  }
  const float mt = tame(m);
  if (set.mode == kAll) {
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NV / 8; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += weight(tame(v[j][e], m), mt, set.c);
    sum = block_all(sum, s_sum, Sum{});
    if (tid == 0) a.mass[at] = sum;
    return;
  }
  const int top = grid_of(mt);
  uint64_t sum = 0;
#pragma unroll
  for (int j = 0; j < NV / 8; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = tame(v[j][e], m);
      if (x == -INFINITY) continue;
      uint64_t n = 1;
      // 16 + w has units of 2^-48 in its last place
      if (set.mode == kTopP) n = __double_as_longlong(weight(x, mt, set.c) + 16.0) & 0xFFFFFFFFFFFFFull;
      sum += n;
      atomicAdd(reinterpret_cast<unsigned long long*>(s_hist + bin_of(x, top)), static_cast<unsigned long long>(n));
    }
  sum = block_all(sum, s_total, Sum{});  // its barrier is behind the histogram, too
  if (tid == 0) a.total[at] = sum;
  if (tid < kBins) a.hist[at * kBins + tid] = s_hist[tid];
}

// ---------------------------------------------------------------- select
template <int DT, int NV>
__global__ void __launch_bounds__(kThreads) sample_select_kernel(SampleArgs a) {
  __shared__ double s_sum[kWaves];
  __shared__ uint64_t s_own[kWaves];
  __shared__ double s_factor[kMaxChunks];  // units of a chunk's masses
  __shared__ int s_off[kMaxChunks];        // its first bin among the row's
  __shared__ int s_lo, s_hi, s_listed;
  const int row = blockIdx.x / a.C, c = blockIdx.x - row * a.C, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Settings set(a, row);
  if (set.mode == kAll) return;  // block-uniform
  const void* const src = row_of<DT>(a, row);
  float v[NV / 8][8];
#pragma unroll
  for (int j = 0; j < NV / 8; ++j) load_logits<DT>(src, (c << a.lg_chunk) + j * kTileTokens + tid * 8, a.V, v[j]);
  const int64_t at0 = static_cast<int64_t>(row) * a.C, at = at0 + c;
  const float m = row_top(a, row), mt = tame(m);
  if (m == -INFINITY) {  // nothing to keep
    if (tid == 0) {
      a.mass[at] = 0.0;
      a.listed[at] = 0;
      if (c == 0) a.state[row] = RowState{0.0, 0, 0, 0, m, 0.0};
    }
    return;
  }
  if (set.mode == kMinP) {
    double sum = 0.0;
    // a logit this far below the maximum weighs less than min_p, by a margin for the rounding of both sides
    const float far = static_cast<float>((log2(set.m) - 0.001) / set.c * (1 + 1e-6) + static_cast<double>(mt) - 1e-6 * fabs(static_cast<double>(mt)));
#pragma unroll
    for (int j = 0; j < NV / 8; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = tame(v[j][e], m);
        if (x >= far) {
          const double w = weight(x, mt, set.c);
          sum += w >= set.m ? w : 0.0;
        }
      }
    sum = block_all(sum, s_sum, Sum{});
    if (tid == 0) {
      a.mass[at] = sum;
      a.listed[at] = 0;
      if (c == 0) a.state[row] = RowState{0.0, 0, 0, 0, m, 0.0};
    }
    return;
  }
  // ---- the row's histogram: bin `tid`
  const int top = grid_of(mt);
  for (int i = tid; i < a.C; i += kThreads) {
    const float ct = a.top[at0 + i];
    s_off[i] = ct == -INFINITY ? kBins : top - grid_of(tame(ct, m));
    s_factor[i] = ct == -INFINITY ? 0.0 : weight(tame(ct, m), mt, set.c) / (set.mode == kTopP ? kUnit : 1.0);
    if (set.mode == kTopK && ct != -INFINITY) s_factor[i] = 1.0;
  }
  if (tid == 0) {
    s_lo = kTail;
    s_hi = kTail;
    s_listed = 0;
  }
  __syncthreads();
  double mine = 0.0, all = 0.0;
  uint64_t own = 0;
  if (tid < kTail) {
    for (int i = 0; i < a.C; ++i) {
      const int b = tid - s_off[i];
      if (b >= 0) {
        const uint64_t h = a.hist[(at0 + i) * kBins + b];
        mine += static_cast<double>(h) * s_factor[i];
        if (i == c) own = h;
      }
    }
  }
  for (int i = 0; i < a.C; ++i) all += static_cast<double>(a.total[at0 + i]) * s_factor[i];
  double upto = wave_scan(mine);
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += s_sum[w];
  // the bins' masses are off by less than 2^-24 of the total
  const double margin = set.mode == kTopP ? all * 0x1p-20 : 0.5;
  const double goal = set.mode == kTopP ? set.p * all : static_cast<double>(set.k);
  if (tid < kTail) {
    if (upto >= goal - margin) atomicMin(&s_lo, tid);
    if (upto >= goal + (set.mode == kTopP ? margin : -margin)) atomicMin(&s_hi, tid);
  }
  __syncthreads();
  int lo = set.mode == kTopK ? 0 : s_lo;
  int hi = s_hi;
  bool cut = true;
  if (set.mode == kTopP && set.m > 0.0) {  // bins in which min-p's border can lie
    const double edge = log2(set.m) / set.c, slack = 1e-5 * (1.0 + fabs(edge) + fabs(static_cast<double>(mt)));
    const int near = bin_of(static_cast<float>(mt + edge + slack), top), far = bin_of(static_cast<float>(mt + edge - slack), top);
    if (far < lo) {  // stricter than top-p
      lo = near < 0 ? 0 : near;
      hi = far;
      cut = false;
    } else if (near < lo) {
      lo = near < 0 ? 0 : near;
    }
  }
  // ---- certain mass and listed tokens of this chunk
  own = tid < lo ? own : 0;
  own = block_all(own, s_own, Sum{});
#pragma unroll
  for (int j = 0; j < NV / 8; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = tame(v[j][e], m);
      const int b = bin_of(x, top);
      const bool on = x != -INFINITY && b >= lo && b <= hi;
      const uint64_t some = __ballot(on);
      if (!some) continue;
      int to = 0;
      if (lane == 0) to = atomicAdd(&s_listed, __popcll(some));
      to = __shfl(to, 0, 64) + __popcll(some & ((1ull << lane) - 1));
      if (on) a.list[(at << a.lg_chunk) + to] = static_cast<uint16_t>(j * kTileTokens + tid * 8 + e);
    }
  __syncthreads();
  if (tid == 0) {
    a.mass[at] = static_cast<double>(own) * s_factor[c];
    a.listed[at] = s_listed;
    if (c == 0) a.state[row] = RowState{goal, cut, 0, 0, m, 0.0};
  }
}

// ---------------------------------------------------------------- draw
struct DrawSmem {
  uint64_t hist[256];
  uint64_t part[kWaves];
  double sum[kWaves];
  float top[kWaves];
  uint32_t keys[kWaves];
  double mass[kMaxChunks];
  uint64_t extra[kMaxChunks];  // kept among the listed tokens
  int off[kMaxChunks];         // a chunk's first listed token
  float v[kShort];
  int x[kShort];
  uint64_t rest, tie;
  uint32_t digit;
  int chunk, pick;
  double bar;
};

// The listed tokens of a row: fn(logit, index), every thread some of them
template <int DT>
struct Listed {
  const SampleArgs& a;
  DrawSmem& s;
  const void* src;
  int row, n;
  float m;
  __device__ __forceinline__ Listed(const SampleArgs& a_, DrawSmem& s_, int row_, float m_) : a(a_), s(s_), src(row_of<DT>(a_, row_)), row(row_), m(m_) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (wave == 0) {
      int run = 0;
      for (int c0 = 0; c0 < a.C; c0 += 64) {
        const int k = c0 + lane < a.C ? a.listed[static_cast<int64_t>(row) * a.C + c0 + lane] : 0;
        const int upto = wave_scan(k);
        if (c0 + lane < a.C) s.off[c0 + lane] = run + upto - k;
        run += __shfl(upto, 63, 64);
      }
      if (lane == 0) s.pick = run;
    }
    __syncthreads();
    n = s.pick;
    if (n <= kShort) {
      far([&](float v, int x, int at) {
        s.v[at] = v;
        s.x[at] = x;
      });
      __syncthreads();
    }
  }
  template <class Fn>
  __device__ __forceinline__ void far(Fn fn) const {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int c = wave; c < a.C; c += kWaves) {
      const int64_t at = static_cast<int64_t>(row) * a.C + c;
      const int k = (c + 1 < a.C ? s.off[c + 1] : n) - s.off[c];
      for (int i = lane; i < k; i += 64) {
        const int x = (c << a.lg_chunk) + a.list[(at << a.lg_chunk) + i];
        fn(tame(load_act<DT>(src, x), m), x, s.off[c] + i);
      }
    }
  }
  template <class Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    if (n <= kShort) {
      for (int i = threadIdx.x; i < n; i += kThreads) fn(s.v[i], s.x[i]);
    } else {
      far([&](float v, int x, int) { fn(v, x); });
    }
  }
};

// Among listed tokens: the digit in which the running sum of their values, from the largest digit down (FALL) or
// from the smallest up, reaches goal; goal becomes what is left of it in front of that digit, and `in` the digit's sum.
// Where the sum never reaches it: the last digit that holds any.
template <bool FALL, class Each>
__device__ __forceinline__ uint32_t pick_digit(DrawSmem& s, uint64_t& goal, uint64_t& in, Each each) {
  const int tid = threadIdx.x;
  if (tid < 256) s.hist[tid] = 0;
  __syncthreads();
  each([&](uint32_t digit, uint64_t value) {
    atomicAdd(reinterpret_cast<unsigned long long*>(s.hist + digit), static_cast<unsigned long long>(value));
  });
  __syncthreads();
  if (tid < 64) {
    uint64_t h[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = s.hist[FALL ? 255 - (4 * tid + i) : 4 * tid + i];
      sum += h[i];
    }
    const uint64_t upto = wave_scan(sum);
    const uint64_t over = __ballot(sum != 0 && upto >= goal), some = __ballot(sum != 0);
    const int l = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 0;
    if (tid == l) {
      uint64_t before = upto - sum, at = before, held = 0;
      int d = 0;
      bool done = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!done && h[i] != 0) {
          d = i;
          before = at;
          held = h[i];
          done = at + h[i] >= goal;
        }
        at += h[i];
      }
      const int pos = 4 * l + d;
      s.digit = FALL ? 255 - pos : pos;
      s.rest = goal > before ? goal - before : 0;
      s.tie = held;
    }
  }
  __syncthreads();
  goal = s.rest;
  in = s.tie;
  return s.digit;
}

// The border in rank: of the listed tokens with key(...) below or at it.  value: 1 (by rank) or the token's mass; kept are
// the tokens whose predecessors' values sum to less than goal (>= 1).
template <int DT, class Value>
__device__ __forceinline__ void pick_border(const Listed<DT>& list, DrawSmem& s, uint64_t goal, Value value, uint32_t& key, int& last) {
  uint32_t prefix = 0, mask = 0;
  uint64_t in = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    const uint32_t d = pick_digit<true>(s, goal, in, [&](auto add) {
      list.each([&](float v, int x) {
        const uint32_t k = key_of(v);
        if ((k & mask) == prefix) {
          const uint64_t n = value(v, x);
          if (n) add((k >> shift) & 255, n);
        }
      });
    });
    prefix |= d << shift;
    mask |= 255u << shift;
  }
  key = prefix;
  // equal logits have equal values: how many of them are kept, the first in index order
  uint64_t one = 0, ties = 0;
  list.each([&](float v, int x) {
    if (key_of(v) == key) {
      const uint64_t n = value(v, x);
      one = n > one ? n : one;
      ties += n != 0;
    }
  });
  one = block_all(one, s.part, Max{});
  __syncthreads();
  ties = block_all(ties, s.part, Sum{});
  __syncthreads();
  uint64_t keep = one ? (goal + one - 1) / one : 1;
  if (keep < 1) keep = 1;
  last = 0x7FFFFFFF;
  if (keep >= ties) return;
  uint32_t at = 0;
  mask = 0;
  for (int shift = 16; shift >= 0; shift -= 8) {
    const uint32_t d = pick_digit<false>(s, keep, in, [&](auto add) {
      list.each([&](float v, int x) {
        if (key_of(v) == key && (static_cast<uint32_t>(x) & mask) == at && value(v, x)) add((x >> shift) & 255, 1);
      });
    });
    at |= d << shift;
    mask |= 255u << shift;
  }
  last = static_cast<int>(at);
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_draw_kernel(SampleArgs a) {
  __shared__ DrawSmem s;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Settings set(a, row);
  const int64_t at0 = static_cast<int64_t>(row) * a.C;
  const float m = row_top(a, row), mt = tame(m);
  if (m == -INFINITY) {  // no token has a weight
    if (tid == 0) {
      if (a.tokens) a.tokens[row] = -1;
      else a.state[row] = RowState{0.0, 0, 0xFFFFFFFFu, -1, m, 0.0};
    }
    return;
  }
  for (int c = tid; c < a.C; c += kThreads) {
    double f = a.mass[at0 + c];
    if (set.mode == kAll) {
      const float ct = a.top[at0 + c];
      f = ct == -INFINITY ? 0.0 : f * weight(tame(ct, m), mt, set.c);
    }
    s.mass[c] = set.mode == kTopK ? 0.0 : f;
    s.extra[c] = 0;
  }
  __syncthreads();

  // ---- the border
  uint32_t key = 0;
  int last = 0x7FFFFFFF;
  double unit = 1.0;
  if (set.mode >= kTopP) {
    const RowState st = a.state[row];
    const Listed<DT> list(a, s, row, m);
    float peak = -INFINITY;
    list.each([&](float v, int) { peak = fmaxf(peak, v); });
    peak = block_all(peak, s.top, Max{});
    // masses of listed tokens as integers: the heaviest is 2^(61 - bits of their number)
    const double big = peak == -INFINITY ? 1.0 : weight(peak, mt, set.c);
    unit = big > 0.0 ? ldexp(1.0, 30 + __builtin_clz(list.n | 1)) / big : 0.0;
    if (!(unit < INFINITY)) unit = 0.0;
    const auto integer = [&](float v) -> uint64_t {
      const double w = weight(v, mt, set.c);
      if (!(w > 0.0)) return 0;
      const uint64_t n = static_cast<uint64_t>(w * unit + 0.5);
      return n ? n : 1;
    };
    if (set.mode == kTopK) {
      pick_border(list, s, static_cast<uint64_t>(set.k), [](float, int) -> uint64_t { return 1; }, key, last);
      if (set.p < 1.0) {
        const uint32_t key_k = key;
        const int last_k = last;
        const auto value = [&](float v, int x) -> uint64_t {
          const uint32_t k = key_of(v);
          return k > key_k || (k == key_k && x <= last_k) ? integer(v) : 0;
        };
        uint64_t sum = 0;
        list.each([&](float v, int x) { sum += value(v, x); });
        __syncthreads();
        sum = block_all(sum, s.part, Sum{});
        __syncthreads();
        const double goal = ceil(set.p * static_cast<double>(sum));
        pick_border(list, s, goal >= 1.0 ? static_cast<uint64_t>(goal) : 1, value, key, last);
      }
    } else if (st.cut) {
      double certain = 0.0;
      for (int c = 0; c < a.C; ++c) certain += s.mass[c];
      const double goal = ceil((st.goal - certain) * unit);
      if (goal >= 1.0 || !(certain > 0.0)) {
        pick_border(list, s, goal >= 1.0 ? static_cast<uint64_t>(goal) : 1, [&](float v, int) { return integer(v); }, key, last);
      } else {  // what is certain reaches the goal
        key = key_of(peak);
        last = -1;
      }
    }
    list.each([&](float v, int x) {
      const uint32_t k = key_of(v);
      if ((k > key || (k == key && x <= last)) && weight(v, mt, set.c) >= set.m)
        atomicAdd(reinterpret_cast<unsigned long long*>(s.extra + (x >> a.lg_chunk)), static_cast<unsigned long long>(integer(v)));
    });
    __syncthreads();
  }

  // ---- the chunk: the first whose running sum passes u times the total
  const auto of_chunk = [&](int c) { return s.mass[c] + (unit > 0.0 ? static_cast<double>(s.extra[c]) / unit : 0.0); };
  if (wave == 0) {
    double sum = 0.0;
    for (int c = lane; c < a.C; c += 64) sum += of_chunk(c);
    const double total = wave_all(sum, Sum{});
    if (!a.tokens) {
      if (lane == 0) a.state[row] = RowState{0.0, 0, key, last, m, 1.0 / total};
    } else {
      const double goal = static_cast<double>(a.uniforms[row]) * total;
      double run = 0.0, bar = 0.0;
      int chunk = -1;
      for (int c0 = 0; c0 < a.C; c0 += 64) {
        const double v = c0 + lane < a.C ? of_chunk(c0 + lane) : 0.0;
        const double upto = wave_scan(v) + run;
        const uint64_t some = __ballot(v > 0.0), over = __ballot(v > 0.0 && upto > goal);
        if (some) {
          const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
          chunk = c0 + l;
          bar = goal - (__shfl(upto, l, 64) - __shfl(v, l, 64));
        }
        if (over) break;
        run = __shfl(upto, 63, 64);
      }
      if (lane == 0) {
        s.chunk = chunk;
        s.bar = bar;
        s.pick = -1;
      }
    }
  }
  if (!a.tokens) return;
  __syncthreads();
  // ---- the token in it
  const int chunk = s.chunk;
  if (chunk < 0) {
    if (tid == 0) a.tokens[row] = -1;
    return;
  }
  double run = s.bar;  // what is left to pass
  const int end = min(a.V, (chunk + 1) << a.lg_chunk);
  int fallback = -1;   // the last kept token, should rounding leave the bar beyond all of them
  for (int x0 = chunk << a.lg_chunk; x0 < end; x0 += kTileTokens) {
    float v[8];
    const int x = x0 + tid * 8;
    load_logits<DT>(row_of<DT>(a, row), x < end ? x : a.V, a.V, v);
    double w[8], sum = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = tame(v[e], m);
      const uint32_t k = key_of(y);
      w[e] = 0.0;
      if (y != -INFINITY && (k > key || (k == key && x + e <= last))) {
        const double ww = weight(y, mt, set.c);
        w[e] = ww >= set.m ? ww : 0.0;
      }
      sum += w[e];
    }
    double upto = wave_scan(sum);
    if (lane == 63) s.sum[wave] = upto;
    __syncthreads();
    double before = upto - sum, all = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) before += s.sum[i];
      all += s.sum[i];
    }
    double at = before;
    int found = -1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (w[e] > 0.0) {
        at += w[e];
        if (found < 0 && at > run) found = x + e;
        fallback = x + e;
      }
    }
    // the smallest index that passes: a key that atomicMax orders
    if (found >= 0) atomicMax(&s.pick, 0x7FFFFFFF - found);
    __syncthreads();
    if (s.pick >= 0) break;
    run -= all;
  }
  if (s.pick < 0) {  // block-uniform
    const uint32_t most = block_all(static_cast<uint32_t>(fallback + 1), s.keys, Max{});
    if (tid == 0) a.tokens[row] = static_cast<int64_t>(most) - 1;
  } else if (tid == 0) {
    a.tokens[row] = 0x7FFFFFFF - s.pick;
  }
}

// ---------------------------------------------------------------- write
template <int DT>
__global__ void __launch_bounds__(256) sample_write_kernel(SampleArgs a, int tiles) {
  const int row = blockIdx.x / tiles, x = ((blockIdx.x - row * tiles) * 256 + threadIdx.x) * 8;
  if (x >= a.V) return;
  const Settings set(a, row);
  const RowState st = a.state[row];
  float v[8], out[8];
  load_logits<DT>(row_of<DT>(a, row), x, a.V, v);
  const float mt = tame(st.top);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = tame(v[e], st.top);
    const uint32_t k = key_of(y);
    out[e] = 0.f;
    if (y != -INFINITY && (k > st.key || (k == st.key && x + e <= st.last))) {
      const double w = weight(y, mt, set.c);
      out[e] = w >= set.m ? static_cast<float>(w * st.inverse) : 0.f;
    }
  }
  float* const to = a.probs + static_cast<int64_t>(row) * a.V + x;
  if (x + 8 <= a.V) {
    __builtin_memcpy(to, out, 32);
  } else {
    for (int e = 0; x + e < a.V; ++e) to[e] = out[e];
  }
}

// ---------------------------------------------------------------- launch
struct SamplePlan {
  int nv, C, lg_chunk;
  int64_t state, top, mass, total, listed, hist, list, bytes;  // offsets
};

// Values a thread takes: as many as leave 512 blocks, two to a compute unit.
static SamplePlan plan_sample(int64_t N, int64_t V) {
  SamplePlan p{};
  p.nv = 32;
  const auto chunks = [&](int nv) { return (V + kThreads * nv - 1) / (kThreads * nv); };
  while (p.nv > 8 && N * chunks(p.nv) < 512 && chunks(p.nv / 2) <= kMaxChunks) p.nv /= 2;
  p.C = static_cast<int>(chunks(p.nv));
  p.lg_chunk = __builtin_ctz(kThreads * p.nv);
  const int64_t n = N * p.C;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 15) / 16 * 16;
    return here;
  };
  p.state = take(N * static_cast<int64_t>(sizeof(RowState)));
  p.top = take(n * 4);
  p.mass = take(n * 8);
  p.total = take(n * 8);
  p.listed = take(n * 4);
  p.hist = take(n * kBins * 8);
  p.list = take((n << p.lg_chunk) * 2);
  p.bytes = at;
  return p;
}
static bool sample_shape(int64_t N, int64_t V) {
  return N >= 1 && V >= 1 && V <= (int64_t(1) << 24) && N < (int64_t(1) << 31) && N * ((V + 2047) / 2048) < (int64_t(1) << 31);
}

template <int DT>
static void launch_sample(const SampleArgs& a, const SamplePlan& p, bool select, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.N * p.C));
  if (p.nv == 32) sample_scan_kernel<DT, 32><<<grid, kThreads, 0, s>>>(a);
  else if (p.nv == 16) sample_scan_kernel<DT, 16><<<grid, kThreads, 0, s>>>(a);
  else sample_scan_kernel<DT, 8><<<grid, kThreads, 0, s>>>(a);
  if (select) {
    if (p.nv == 32) sample_select_kernel<DT, 32><<<grid, kThreads, 0, s>>>(a);
    else if (p.nv == 16) sample_select_kernel<DT, 16><<<grid, kThreads, 0, s>>>(a);
    else sample_select_kernel<DT, 8><<<grid, kThreads, 0, s>>>(a);
  }
  sample_draw_kernel<DT><<<dim3(a.N), kThreads, 0, s>>>(a);
  if (!a.tokens) {
    const int tiles = (a.V + 2047) / 2048;
    sample_write_kernel<DT><<<dim3(static_cast<unsigned>(a.N) * tiles), 256, 0, s>>>(a, tiles);
  }
}

static int run_sample(const char* what, SampleArgs& a, int32_t dtype, double temperature, int32_t top_k, double top_p,
                      double min_p, void* workspace, int64_t bytes, void* stream) {
  TQ_REQUIRE(a.N >= 0 && a.V >= 1 && a.ld >= 0, "%s: bad shape", what);
  TQ_REQUIRE(dtype == TQ_F32 || dtype == TQ_F16 || dtype == TQ_BF16, "%s: unknown dtype %d", what, dtype);
  TQ_REQUIRE(temperature >= 0.0 && top_k >= 0 && top_p >= 0.0 && min_p >= 0.0,
             "%s: temperature, top_k, top_p and min_p must not be negative", what);
  if (a.N == 0) return TQ_OK;
  TQ_REQUIRE(sample_shape(a.N, a.V), "%s: at most 2^24 tokens and 2^31 tiles of 2048, got %d rows of %d", what, a.N, a.V);
  TQ_REQUIRE(a.logits && (a.probs || (a.tokens && a.uniforms)), "%s: null pointer", what);
  const SamplePlan p = plan_sample(a.N, a.V);
  TQ_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && bytes >= p.bytes,
             "%s: the workspace must be 16-byte aligned and hold %lld bytes", what, (long long)p.bytes);
  a.t = temperature;
  a.k = top_k;
  a.p = top_p;
  a.m = min_p;
  a.C = p.C;
  a.lg_chunk = p.lg_chunk;
  uint8_t* const w = static_cast<uint8_t*>(workspace);
  a.state = reinterpret_cast<RowState*>(w + p.state);
  a.top = reinterpret_cast<float*>(w + p.top);
  a.mass = reinterpret_cast<double*>(w + p.mass);
  a.total = reinterpret_cast<uint64_t*>(w + p.total);
  a.listed = reinterpret_cast<int32_t*>(w + p.listed);
  a.hist = reinterpret_cast<uint64_t*>(w + p.hist);
  a.list = reinterpret_cast<uint16_t*>(w + p.list);
  // without filters the masses of the first pass are all there is to know
  const bool select = a.t_rows || a.k_rows || a.p_rows || a.m_rows || !(temperature > 0.0) || (top_k > 0 && top_k < a.V) ||
                      top_p < 1.0 || min_p > 0.0;
  hipStream_t s = as_stream(stream);
  if (dtype == TQ_F32) launch_sample<TQ_F32>(a, p, select, s);
  else if (dtype == TQ_F16) launch_sample<TQ_F16>(a, p, select, s);
  else launch_sample<TQ_BF16>(a, p, select, s);
  return launch_status(what);
}

}  // namespace tq

using namespace tq;

extern "C" {

int64_t tq_sample_workspace_size(int32_t N, int32_t V) { return sample_shape(N, V) ? plan_sample(N, V).bytes : 0; }

int tq_sample_tokens(const void* logits, int32_t dtype, int64_t ld, int32_t N, int32_t V, const float* uniforms,
                     const float* temperatures, double temperature, const int32_t* top_ks, int32_t top_k,
                     const float* top_ps, double top_p, const float* min_ps, double min_p, int64_t* tokens,
                     void* workspace, int64_t workspace_bytes, void* stream) {
  SampleArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.N = N;
  a.V = V;
  a.uniforms = uniforms;
  a.t_rows = temperatures;
  a.k_rows = top_ks;
  a.p_rows = top_ps;
  a.m_rows = min_ps;
  a.tokens = tokens;
  return run_sample("tq_sample_tokens", a, dtype, temperature, top_k, top_p, min_p, workspace, workspace_bytes, stream);
}

int tq_filter_probs(const void* logits, int32_t dtype, int64_t ld, int32_t N, int32_t V, const float* temperatures,
                    double temperature, const int32_t* top_ks, int32_t top_k, const float* top_ps, double top_p,
                    const float* min_ps, double min_p, float* probs, void* workspace, int64_t workspace_bytes,
                    void* stream) {
  SampleArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.N = N;
  a.V = V;
  a.t_rows = temperatures;
  a.k_rows = top_ks;
  a.p_rows = top_ps;
  a.m_rows = min_ps;
  a.probs = probs;
  return run_sample("tq_filter_probs", a, dtype, temperature, top_k, top_p, min_p, workspace, workspace_bytes, stream);
}

}  // extern "C"
