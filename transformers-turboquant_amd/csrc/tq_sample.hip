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
// in a few thousand tokens if sums are off by 10^-7; so weights are float64 (2^f by its Taylor series, 3 10^-13, 2^-41.6), and
// sums are float64 in a fixed order or integers, which have none (of listed tokens in units of at most 2^-62 of the total, each
// off by less than a unit, so n of them by n 2^-62).  Both together: less than 2^-40 of the total for up to 2^20 tokens, 2^-37
// for 2^24.
//
// A row is never sorted.  It is cut into chunks, one per block, and then finished by one block:
//   scan     the chunk's maximum; without filters its mass; for top-p its mass, and a histogram of it over bins of
//            1/16 below the maximum, as far down as tokens can be kept (all those of weight below (1 - p) / V of the
//            largest together weigh less than (1 - p) of the total, so p of it stands before them); for
//            top-k a list of the tokens down to the bin that k threads' own maxima reach.  From k = 513 on, a block having 512
//            threads, and from about 460 on in chunks of 4096 that is every token: the list, of a quarter of the chunk, does not hold
//            them, and the finish reads the row again (64 rows of 128256: k 50 16.6 us, 400 30, 512 74, 1000 92, 20000
//            325; one row: 400 42, 500 100)
//   select   (top-p, min-p) finds the bins that hold the row's border in the joined histograms, and lists what is
//            kept (min-p), the tokens down to the border if they are few, or else those of its bins alone, with the
//            mass of what is kept for certain above them
//   finish   up to 64 listed tokens are ranked by one wave, 256 by the block; among more (5120 in shared memory) the border is
//            found in its bin, and there by rank or, of many equal ones, digit by digit; drawn from the list if it holds
//            all that is kept, else by the chunks' masses
//   write    the probabilities of rows that keep many; the others' are few, in a row that the scan has cleared
#include "tq_common.h"

namespace tq {

constexpr int kThreads = 1024, kWaves = kThreads / 64;  // of the finish
constexpr int kScan = 512, kScanWaves = kScan / 64;     // of scan and select: a thread takes runs of 8 tokens
constexpr int kBins = 512, kTail = kBins - 1;  // the last bin has everything below the others
constexpr int kMaxChunks = 1024;
constexpr int kShort = 5120;  // tokens that are taken into shared memory
constexpr int kRanked = 256;  // of them, tokens that are ranked one against the other
constexpr int kFew = 1024;    // tokens down to the border that are listed with it

enum Mode { kAll, kMinP, kTopP, kTopK };

// A row's settings as the kernels use them
struct Settings {
  int mode, k;
  double c;     // log2(e) / t
  double low;   // a logit this far below the maximum weighs nothing (2^-1200)
  double p, m;
  float far;    // kept tokens' logits are down to this far from the maximum (top-p, min-p)
  float tiny;   // what is further weighs less than 2^-46 of the maximum together (top-p)

  // t: NaN and what is not positive count as 0
  __host__ __device__ Settings(int V, double t, int k_, double p_, double m_) : k(k_), p(p_), m(m_) {
    const bool greedy = !(t > 0.0);
    if (greedy) k = 1;
    c = 1.4426950408889634 / (greedy ? 1.0 : t);
    c = !(c < 1e290) ? 1e290 : c < 1e-290 ? 1e-290 : c;
    low = -1200.0 / c;
    m = m > 0.0 ? (m < 1.0 ? m : 1.0) : 0.0;
    const bool by_rank = k > 0 && k < V, by_mass = p < 1.0;
    if (!by_mass) p = 1.0;
    mode = by_rank ? kTopK : by_mass ? kTopP : m > 0.0 ? kMinP : kAll;
    // log2 of the least weight, with room for its rounding
    double y = m > 0.0 ? log2(m) : -1100.0;
    if (mode == kTopP) y = fmax(y, log2((1.0 - p) / V) - 1.0);
    const double d = (0.001 - y) / c;
    far = d < 3e38 ? static_cast<float>(d * 1.000001) : INFINITY;
    const double z = (46.01 + log2(static_cast<double>(V))) / c;
    tiny = z < 3e38 ? static_cast<float>(z * 1.000001) : INFINITY;
  }
};

// Top-p: the row's mass and the bins that are listed
struct RowCut {
  double total;
  int lo, hi;
};

// A row's border, and whether its probabilities are written already
struct RowState {
  uint32_t key;  // kept: larger keys, and this key up to index `last`
  int last;
  float top;
  int done;
  double inverse;  // 1 / kept mass
};

struct SampleArgs {
  const void* logits;
  int64_t ld;  // elements between rows
  int N, V;
  // one setting for all rows, or (an array) one per row
  const float* t_rows;
  const int32_t* k_rows;
  const float* p_rows;
  const float* m_rows;
  double t, p, m;
  int k;
  Settings all;            // where no setting is the rows' own
  const float* uniforms;   // [N], or null: probabilities
  int64_t* tokens;         // [N]
  float* probs;            // [N, V]
  int C, lg_chunk, lg_room;  // chunks of a row, tokens of a chunk, places in its list
  // workspace
  Settings* rows;   // [N], or null: `all`
  RowState* state;  // [N]
  RowCut* cut;      // [N]
  float* top;       // [N, C] chunk's maximum
  double* mass;     // [N, C] of the chunk, relative to its maximum
  double* kept;     // [N, C] of what is kept for certain, relative to the row's
  int32_t* listed;  // [N, C] tokens in the list; more than fit: it is not used
  int32_t* depth;   // [N, C] bins of the histogram
  float* hist;      // [N, C, kBins]
  uint2* list;      // [N, C, 2^lg_room] logit, index

  __device__ __forceinline__ const Settings& of(int row) const { return rows ? rows[row] : all; }
};

// Weights under a maximum: exp((v - top) / t) = 2^y as 2^n 2^f, n = rint(y): 2^f, |f| <= 1/2, by the series of
// exp(f ln 2) up to the 10th power (3 10^-13).  Adding 1.5 2^52 leaves n in the low word.  -inf weighs 0.
struct Weigh {
  double top, c, low;  // top: of finite logits, or one that v is not above
  __device__ __forceinline__ Weigh(const Settings& set, float m) : top(m), c(set.c), low(set.low) {}
  __device__ __forceinline__ double operator()(float v) const {
    constexpr double L = 0.6931471805599453, M = 0x1.8p52;
    constexpr double A[11] = {1.0, L, L * L / 2, L * L * L / 6, L * L * L * L / 24, L * L * L * L * L / 120,
                              L * L * L * L * L * L / 720, L * L * L * L * L * L * L / 5040, L * L * L * L * L * L * L * L / 40320,
                              L * L * L * L * L * L * L * L * L / 362880, L * L * L * L * L * L * L * L * L * L / 3628800};
    double d = static_cast<double>(v) - top, s;
    asm("v_max_f64 %0, %1, %2" : "=v"(d) : "v"(d), "v"(low));  // fmax would quiet `low` first
    const double t = fma(d, c, M), f = fma(d, c, -(t - M));
    // the series with its constants as scalar operands; the compiler's own form copies each to vector registers
    // (9 of ~45 instructions a token)
    asm("v_fma_f64 %0, %1, %2, %3\n\t"
        "v_fma_f64 %0, %0, %2, %4\n\t"
        "v_fma_f64 %0, %0, %2, %5\n\t"
        "v_fma_f64 %0, %0, %2, %6\n\t"
        "v_fma_f64 %0, %0, %2, %7\n\t"
        "v_fma_f64 %0, %0, %2, %8\n\t"
        "v_fma_f64 %0, %0, %2, %9\n\t"
        "v_fma_f64 %0, %0, %2, %10\n\t"
        "v_fma_f64 %0, %0, %2, %11\n\t"
        "v_fma_f64 %0, %0, %2, 1.0"
        : "=&v"(s)
        : "v"(A[10]), "v"(f), "s"(A[9]), "s"(A[8]), "s"(A[7]), "s"(A[6]), "s"(A[5]), "s"(A[4]), "s"(A[3]), "s"(A[2]), "s"(A[1]));
    return ldexp(s, static_cast<int>(__double_as_longlong(t)));
  }
};

// Falling bins of 1/16 on an absolute grid, so that chunks with other maxima have the same ones.  Monotone
// in v; logits beyond 2^27 / 16 share their bins.
__device__ __forceinline__ int grid_of(float v) { return static_cast<int>(floorf(fminf(fmaxf(v * 16.f, -0x1p27f), 0x1p27f))); }
// the least float on the grid from g on (the last value has everything below it)
__device__ __forceinline__ float edge_of(int g) { return g > -(1 << 27) ? __double2float_ru(g * 0.0625) : -3.4028235e38f; }
__device__ __forceinline__ int bin_of(float v, int grid_top) { return min(grid_top - grid_of(v), kTail); }
// larger for larger floats
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Eight logits from x on, as they are in memory; what is not there is -inf.
template <int DT>
struct Run {
  uint32_t r[DT == TQ_F32 ? 8 : 4];
  __device__ __forceinline__ void load(const void* row, int x, int V) {
    if constexpr (DT == TQ_F32) {
      if (x + 8 <= V) {
        __builtin_memcpy(r, static_cast<const float*>(row) + x, 32);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = x + e < V ? static_cast<const uint32_t*>(row)[x + e] : 0xFF800000u;
      }
    } else {
      constexpr uint32_t kLow = DT == TQ_F16 ? 0xFC00u : 0xFF80u;
      if (x + 8 <= V) {
        __builtin_memcpy(r, static_cast<const uint16_t*>(row) + x, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const uint32_t lo = x + e < V ? static_cast<const uint16_t*>(row)[x + e] : kLow;
          const uint32_t hi = x + e + 1 < V ? static_cast<const uint16_t*>(row)[x + e + 1] : kLow;
          r[e / 2] = lo | hi << 16;
        }
      }
    }
  }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (DT == TQ_F32) return __uint_as_float(r[e]);
    else if constexpr (DT == TQ_F16) return h2f(static_cast<uint16_t>(e & 1 ? r[e / 2] >> 16 : r[e / 2] & 0xFFFF));
    else return __uint_as_float(e & 1 ? r[e / 2] & 0xFFFF0000u : r[e / 2] << 16);
  }
};
// eight logits, NaN as -inf
template <int DT>
__device__ __forceinline__ void load_logits(const void* row, int x, int V, float (&v)[8]) {
  Run<DT> run;
  run.load(row, x, V);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = fmaxf(run[e], -INFINITY);  // of a NaN the other operand
}
template <int DT>
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int row) {
  return static_cast<const uint8_t*>(a.logits) + row * a.ld * (DT == TQ_F32 ? 4 : 2);
}
// Under an infinite maximum only infinite logits have a weight: as 0 against -inf, maximum 0.
__device__ __forceinline__ float tame(float v, float m) { return m == INFINITY ? (v == INFINITY ? 0.f : -INFINITY) : v; }
__device__ __forceinline__ float tame(float m) { return m == INFINITY ? 0.f : m; }
// a chunk's or listed logit, tamed by its own chunk's maximum already, under the row's
__device__ __forceinline__ bool counts(float chunk_top, float m) { return m != INFINITY || chunk_top == INFINITY; }

// ---------------------------------------------------------------- over a wave, over a block
// Lane to lane through DPP (shifts within rows of 16 lanes, then lane 15 of row 0 into row 1 and of row 2 into
// row 3, then lane 31 into the upper half), no LDS round trips.  A lane without a source gets `none`.
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp_from(T none, T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
  } else {
    const uint64_t x = __builtin_bit_cast(uint64_t, v), o = __builtin_bit_cast(uint64_t, none);
    const uint32_t lo = __builtin_amdgcn_update_dpp(static_cast<int>(o), static_cast<int>(x), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(static_cast<int>(o >> 32), static_cast<int>(x >> 32), CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
  }
}
struct Sum {
  template <class T>
  static __device__ __forceinline__ T none() {
    return T(0);
  }
  template <class T>
  __device__ __forceinline__ T operator()(T a, T b) const {
    return a + b;
  }
};
struct Max {
  template <class T>
  static __device__ __forceinline__ T none() {
    if constexpr (__is_floating_point(T)) return -INFINITY;
    else return T(-1) < T(0) ? T(T(1) << (8 * sizeof(T) - 1)) : T(0);
  }
  template <class T>
  __device__ __forceinline__ T operator()(T a, T b) const {
    return a > b ? a : b;
  }
};
template <class T>
__device__ __forceinline__ T lane_value(T v, int l) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
  } else {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(x), l), hi = __builtin_amdgcn_readlane(static_cast<int>(x >> 32), l);
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
  }
}
// inclusive, over all lanes of a wave
template <class T, class Op = Sum>
__device__ __forceinline__ T wave_scan(T v, Op op = Op()) {
  const T none = Op::template none<T>();
  v = op(dpp_from<0x111, 0xF>(none, v), v);
  v = op(dpp_from<0x112, 0xF>(none, v), v);
  v = op(dpp_from<0x114, 0xF>(none, v), v);
  v = op(dpp_from<0x118, 0xF>(none, v), v);
  v = op(dpp_from<0x142, 0xA>(none, v), v);
  return op(dpp_from<0x143, 0xC>(none, v), v);
}
template <class T, class Op>
__device__ __forceinline__ T wave_all(T v, Op op) {
  return lane_value(wave_scan(v, op), 63);
}
// of all threads, in a fixed order; s: a value per wave, free again behind the next barrier
template <int W, class T, class Op>
__device__ __forceinline__ T block_all(T v, T* s, Op op) {
  v = wave_all(v, op);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  T r = s[0];
#pragma unroll
  for (int w = 1; w < W; ++w) r = op(r, s[w]);
  return r;
}
__device__ __forceinline__ void add_lds(uint64_t* p, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(p), static_cast<unsigned long long>(v));
}

// ---------------------------------------------------------------- scan
// A thread's tokens of a chunk: runs of 8 in a row, kScan * 8 apart, at most 64.  They are read anew in every pass
// (from the caches behind the first): held in registers, 64 of them leave one wave per SIMD.  NaN are NaN.
template <int DT, class Fn>
__device__ __forceinline__ void each_run(const SampleArgs& a, int row, int chunk, float m, Fn fn) {
  const void* const src = row_of<DT>(a, row);
  const int x0 = (chunk << a.lg_chunk) + static_cast<int>(threadIdx.x) * 8, runs = 1 << (a.lg_chunk - 12);
  static_assert(kScan * 8 == 1 << 12, "tokens of a block's run");
  Run<DT> next;
  next.load(src, x0, a.V);
#pragma unroll 1
  for (int r = 0; r < runs; ++r) {
    const int x = x0 + r * (kScan * 8);
    const Run<DT> run = next;
    if (r + 1 < runs) next.load(src, x + kScan * 8, a.V);  // flies meanwhile
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = run[e];
    if (m == INFINITY) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tame(v[e], m);
    }
    fn(v, r, x);
  }
}

// units of a weight: 16 + w has 2^-48 in its last place
__device__ __forceinline__ uint64_t units_of(double w) { return __double_as_longlong(w + 16.0) & 0xFFFFFFFFFFFFFull; }

// The block's listed tokens, bit 8 r + e of `on` for token e of the thread's run r: to the chunk's list, in any order
template <int DT>
__device__ __forceinline__ void list_tokens(const SampleArgs& a, int row, int chunk, float m, uint64_t on, int* s_listed) {
  const int mine = __popcll(on);
  int to = wave_scan(mine);
  const int all = __builtin_amdgcn_readlane(to, 63);
  if (!all) return;
  int base = 0;
  if ((threadIdx.x & 63) == 0) base = atomicAdd(s_listed, all);
  to += __builtin_amdgcn_readfirstlane(base) - mine;
  const int room = 1 << a.lg_room, x0 = (chunk << a.lg_chunk) + static_cast<int>(threadIdx.x) * 8;
  uint2* const list = a.list + ((static_cast<int64_t>(row) * a.C + chunk) << a.lg_room);
  const void* const src = row_of<DT>(a, row);
#pragma unroll 1
  for (; on && to < room; on &= on - 1, ++to) {
    const int i = __builtin_ctzll(on), x = x0 + (i >> 3) * (kScan * 8) + (i & 7);
    list[to] = uint2{__float_as_uint(tame(load_act<DT>(src, x), m)), static_cast<uint32_t>(x)};
  }
}

// The bin up to which the sum over 512 bins (8 to each lane of a wave) reaches `goal`: kTail if none does
template <class T>
__device__ __forceinline__ int reach_bin(const T (&h)[8], T goal) {
  const int lane = threadIdx.x & 63;
  T sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += h[i];
  const T upto = wave_scan(sum);
  const uint64_t over = __ballot(upto >= goal);
  if (!over) return kTail;
  T run = upto - sum;
  int bin = 8 * lane;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    run += h[i];
    bin += run < goal;
  }
  return min(__builtin_amdgcn_readlane(bin, __builtin_ctzll(over)), kTail);
}

struct ScanSmem {
  uint64_t hist[kBins];
  uint64_t part[kScanWaves];
  double sum[kScanWaves];
  float top[kScanWaves];
  int depth[kScanWaves];
  int listed, bin;
  Settings set;
  __device__ ScanSmem() = delete;
};

// Settings of a row, in shared memory where they are the row's own: made by one thread
__device__ __forceinline__ void make_settings(const SampleArgs& a, int row, Settings* to) {
  *to = Settings(a.V, a.t_rows ? a.t_rows[row] : a.t, a.k_rows ? a.k_rows[row] : a.k, a.p_rows ? a.p_rows[row] : a.p,
                 a.m_rows ? a.m_rows[row] : a.m);
}

// Top-p over 512 rows of 151936 in bf16, zeros written for the probabilities (0.47 GB, 91 us at a copy's rate): 123 us, bound by
// the weights' float64 series (18 float64 instructions of ~35 a token; the VALU issues in two thirds of the cycles).
// 64 rows of 128256 in f32 15 us (33 MB), 256 rows under min-p, the maxima alone, 10 us (66 MB): a read from
// memory.  A single row of 50257 4.4 us: two dependent round trips.
template <int DT>
__global__ void __launch_bounds__(kScan) sample_scan_kernel(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t s_raw[sizeof(ScanSmem)];
  ScanSmem& s = *reinterpret_cast<ScanSmem*>(s_raw);
  const int row = blockIdx.x / a.C, c = blockIdx.x - row * a.C, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float most = -INFINITY;
  each_run<DT>(a, row, c, 0.f, [&](const float (&v)[8], int, int) {
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, v[e]);
  });
  static_assert(kScan == kBins, "a bin per thread");
  s.hist[tid] = 0;
  if (tid == 0) {
    s.listed = 0;
    if (a.rows) {
      make_settings(a, row, &s.set);
      if (c == 0) a.rows[row] = s.set;
    }
  }
  const float m = block_all<kScanWaves>(most, s.top, Max{});
  const Settings& set = a.rows ? s.set : a.all;
  const int mode = set.mode;
  const int64_t at = static_cast<int64_t>(row) * a.C + c;
  if (tid == 0) a.top[at] = m;
  if (a.probs && mode != kAll) {  // kept tokens are filled in later
    float* const to = a.probs + static_cast<int64_t>(row) * a.V;
    const int end = min(a.V, (c + 1) << a.lg_chunk);
#pragma unroll 1
    for (int x = (c << a.lg_chunk) + tid * 8; x < end; x += kScan * 8) {
      const float zero[8] = {};
      if (x + 8 <= a.V) {
        __builtin_memcpy(to + x, zero, 32);
      } else {
        for (int e = 0; x + e < a.V; ++e) to[x + e] = 0.f;
      }
    }
  }
  if (mode == kMinP) return;
  if (m == -INFINITY) {
    if (tid == 0) {
      a.mass[at] = 0.0;
      a.listed[at] = 0;
      a.depth[at] = 0;
    }
    return;
  }
  const float mt = tame(m);
  const Weigh weigh(set, mt);
  const int top = grid_of(mt);
  if (mode == kAll) {
    double sum = 0.0;
    each_run<DT>(a, row, c, m, [&](const float (&v)[8], int, int) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += weigh(v[e]);
    });
    sum = block_all<kScanWaves>(sum, s.sum, Sum{});
    if (tid == 0) a.mass[at] = sum;
  } else if (mode == kTopK) {
    // k threads have a token in the bins down to this one: k tokens stand before all that is below
    most = tame(most, m);
    if (most != -INFINITY) add_lds(s.hist + bin_of(most, top), 1);
    __syncthreads();
    if (wave == 0) {
      int h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = 8 * lane + i < kTail ? static_cast<int>(s.hist[8 * lane + i]) : 0;
      const int bin = reach_bin(h, set.k);
      if (lane == 0) s.bin = bin;
    }
    __syncthreads();
    const float least = s.bin < kTail ? edge_of(top - s.bin) : -3.4028235e38f;
    uint64_t on = 0;
    if (most >= least)
      each_run<DT>(a, row, c, m, [&](const float (&v)[8], int r, int) {
#pragma unroll
        for (int e = 0; e < 8; ++e) on |= static_cast<uint64_t>(v[e] >= least) << (8 * r + e);
      });
    list_tokens<DT>(a, row, c, m, on, &s.listed);
    __syncthreads();
    if (tid == 0) a.listed[at] = s.listed;
  } else {
    const auto below = [&](float d) {  // a logit d below the maximum, rounded down
      const float x = mt - d;
      return x - 2e-7f * (fabsf(mt) + fabsf(x));
    };
    const float least = fmaxf(-3.4028235e38f, below(set.far)), tiny = below(set.tiny);
    double sum = 0.0;
    each_run<DT>(a, row, c, m, [&](const float (&v)[8], int, int) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = v[e];
        if (__any(x >= tiny)) {
          const double w = weigh(x);  // 0 of a NaN
          sum += w;
          if (x >= least) add_lds(s.hist + bin_of(x, top), units_of(w));
        }
      }
    });
    sum = block_all<kScanWaves>(sum, s.sum, Sum{});  // its barrier is behind the histogram, too
    const uint64_t h = s.hist[tid], some = __ballot(h != 0);
    if (lane == 0) s.depth[wave] = some ? 64 * wave + 64 - __builtin_clzll(some) : 0;
    __syncthreads();
    int deep = 0;
#pragma unroll
    for (int w = 0; w < kScanWaves; ++w) deep = max(deep, s.depth[w]);
    if (tid == 0) {
      a.mass[at] = sum;
      a.depth[at] = deep;
    }
    if (tid < deep) a.hist[at * kBins + tid] = static_cast<float>(h) * 0x1p-48f;
  }
}

// ---------------------------------------------------------------- select
struct SelectSmem {
  float bins[kBins];
  float factor[kMaxChunks];  // of a chunk's units: shares of the row's mass
  int off[kMaxChunks];       // its first bin among the row's
  int depth[kMaxChunks];
  double total[kScanWaves], sum[kScanWaves];
  int listed, lo, hi;
};

// Every block joins its row's histograms by itself (2 KB a chunk, from the L2; one launch less than with a join of its
// own), then reads its chunk again if its maximum reaches the border.  512 rows of 151936 43 us (156 MB), 64 of 128256
// 10 us, 16 of 151936 10 us.
template <int DT>
__global__ void __launch_bounds__(kScan) sample_select_kernel(SampleArgs a) {
  __shared__ SelectSmem s;
  const int row = blockIdx.x / a.C, c = blockIdx.x - row * a.C, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Settings& set = a.of(row);
  const int mode = set.mode;
  if (mode != kTopP && mode != kMinP) return;  // block-uniform
  const int64_t at0 = static_cast<int64_t>(row) * a.C, at = at0 + c;
  float m = -INFINITY;
  for (int i = lane; i < a.C; i += 64) m = fmaxf(m, a.top[at0 + i]);
  m = wave_all(m, Max{});
  if (tid == 0) s.listed = 0;
  if (m == -INFINITY) {
    if (tid == 0) {
      a.kept[at] = 0.0;
      a.listed[at] = 0;
    }
    return;
  }
  const float mt = tame(m);
  const Weigh weigh(set, mt);
  const double c2 = set.c, least = set.m;
  const int top = grid_of(mt);
  // Of what is kept for certain: in 64-bit floats, as rounded to 2^-48 of the maximum equal weights would all err to one
  // side, 150000 tokens of 2^-24 by 2^-32 of the total.
  double sum = 0.0;
  uint64_t on = 0;
  if (mode == kMinP) {
    __syncthreads();
    const float x1 = mt - set.far, far = fmaxf(-3.4028235e38f, x1 - 2e-7f * (fabsf(mt) + fabsf(x1)));
    each_run<DT>(a, row, c, m, [&](const float (&v)[8], int r, int) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        bool take = v[e] >= far;
        if (__any(take)) {
          const double w = weigh(v[e]);
          take = take && w >= least;
          sum += take ? w : 0.0;
          on |= static_cast<uint64_t>(take) << (8 * r + e);
        }
      }
    });
  } else {
    // ---- the row's histogram, as shares of its mass: bin `tid`
    double mine = 0.0;
    for (int i = tid; i < a.C; i += kScan) {
      const float ct = a.top[at0 + i];
      const bool in = ct != -INFINITY && counts(ct, m);
      const double f = in ? weigh(tame(ct)) : 0.0;
      mine += in ? f * a.mass[at0 + i] : 0.0;
      s.factor[i] = static_cast<float>(f);
      s.off[i] = in ? top - grid_of(tame(ct)) : kBins;
      s.depth[i] = in ? a.depth[at0 + i] : 0;
    }
    const double total = block_all<kScanWaves>(mine, s.total, Sum{});  // in a fixed order
    double share = 0.0;  // in float, equal shares of hundreds of chunks are all rounded to one side: 2^-16.8 at 598 of them
    for (int i0 = 0; i0 < a.C; i0 += 8) {
      float h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = min(i0 + i, a.C - 1);  // every load unconditional, so that they fly together
        h[i] = a.hist[(at0 + k) * kBins + min(max(tid - s.off[k], 0), kTail)];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = min(i0 + i, a.C - 1), b = tid - s.off[k];
        const bool in = i0 + i < a.C && b >= 0 && b < s.depth[k] && b < kTail;
        share += in ? static_cast<double>(h[i] * s.factor[k]) : 0.0;
      }
    }
    s.bins[tid] = tid < kTail ? static_cast<float>(share * (1.0 / total)) : 0.f;
    __syncthreads();
    if (wave == 0) {
      float h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = s.bins[8 * lane + i];
      // Off by less than 2^-19: a share by four roundings of 2^-24 of it (histogram, factor, their product, itself), the sum
      // up to a bin by some 20 of 2^-25.
      const float p = static_cast<float>(set.p);
      int lo = reach_bin(h, p - 0x1p-17f);
      int hi = reach_bin(h, p + 0x1p-17f);
      double edge = 0.0, slack = 0.0;  // min-p's border below the maximum
      if (least > 0.0) {  // nothing below it is kept, wherever top-p's may be
        edge = log2(least) / c2;
        slack = 1e-5 * (1.0 + fabs(edge) + fabs(static_cast<double>(mt)));
        hi = min(hi, max(0, bin_of(static_cast<float>(fmax(mt + edge - slack, -3e38)), top)));
      }
      // at most so many tokens down to there: a bin's mass over the least weight in it
      float few = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int b = 8 * lane + i;
        const float y = static_cast<float>((top - b) * 0.0625 - mt) * static_cast<float>(c2);
        if (b <= hi && h[i] > 0.f) few += h[i] * static_cast<float>(total) / fmaxf(__builtin_amdgcn_exp2f(fmaxf(y, -120.f)), 1e-30f);
      }
      few = wave_all(few, Sum{});
      if (hi < kTail && few < kFew) {
        lo = 0;
      } else if (least > 0.0) {  // what is certain is above min-p's border, too
        lo = min(lo, max(0, bin_of(static_cast<float>(fmin(mt + edge + slack, 3e38)), top)));
      }
      if (lane == 0) {
        s.lo = lo;
        s.hi = hi;
        if (c == 0) a.cut[row] = RowCut{total, lo, hi};
      }
    }
    __syncthreads();
    // as logits: certain from `sure` on, listed from `edge` on
    const float sure = s.lo > 0 ? edge_of(top - s.lo + 1) : INFINITY, edge = s.hi < kTail ? edge_of(top - s.hi) : -3.4028235e38f;
    if (a.top[at] >= edge)  // else the chunk has nothing to list
      each_run<DT>(a, row, c, m, [&](const float (&v)[8], int r, int) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool certain = v[e] >= sure;
          if (__any(certain)) {
            const double w = weigh(v[e]);
            sum += certain ? w : 0.0;
          }
          on |= static_cast<uint64_t>(v[e] >= edge && !certain) << (8 * r + e);
        }
      });
  }
  list_tokens<DT>(a, row, c, m, on, &s.listed);
  sum = block_all<kScanWaves>(sum, s.sum, Sum{});
  if (tid == 0) {
    a.kept[at] = sum;
    a.listed[at] = s.listed;
  }
}

// ---------------------------------------------------------------- finish
constexpr int kSegments = 2048;  // runs of 64 listed tokens that the table holds

struct FinishSmem {
  uint64_t token[kShort];  // key, then the complement of the index: larger ones rank first
  uint64_t value[kRanked];
  uint32_t segment[kSegments];  // chunk, run of 64
  union {
    uint64_t digits[512];
    uint32_t bins[kBins];
  };
  uint64_t part[kWaves];
  double sum[kWaves];
  double mass[kMaxChunks];     // of a row without filters, relative to its maximum
  uint64_t extra[kMaxChunks];  // kept tokens' mass as integers
  int listed[kMaxChunks];      // -1: its tokens are read from the row
  float top[kMaxChunks];
  uint64_t rest, one;
  uint32_t digit, ties;
  int segments, raw, lo, hi, n, chunk, pick;
  double bar;
};

// The tokens of a row that may be kept, fn(logit, index): the chunks' lists, 64 to a wave, and the chunks whose list
// does not hold them, by the whole block.
template <int DT>
struct Candidates {
  const SampleArgs& a;
  const FinishSmem& s;
  int row;
  float m;
  template <class Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const auto load = [&](int g, uint2& t) {
      if (g >= s.segments) return false;
      const uint32_t seg = s.segment[g];
      const int c = seg >> 16, i = (seg & 0xFFFF) * 64 + lane;
      const bool on = i < s.listed[c];
      if (on) t = a.list[((static_cast<int64_t>(row) * a.C + c) << a.lg_room) + i];
      return on;
    };
    uint2 next{};
    bool more = load(wave, next);
#pragma unroll 1
    for (int g = wave; g < s.segments; g += kWaves) {
      const uint2 t = next;
      const bool on = more;
      more = load(g + kWaves, next);  // flies meanwhile
      if (on) fn(__uint_as_float(t.x), static_cast<int>(t.y));
    }
    if (!s.raw) return;
#pragma unroll 1
    for (int c = 0; c < a.C; ++c) {
      if (s.listed[c] >= 0) continue;
      const int end = min(a.V, (c + 1) << a.lg_chunk);
#pragma unroll 1
      for (int x = (c << a.lg_chunk) + tid * 8; x < end; x += kThreads * 8) {
        float v[8];
        load_logits<DT>(row_of<DT>(a, row), x, a.V, v);
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const float y = tame(v[0], m);
          if (y != -INFINITY) fn(y, x + e);
#pragma unroll
          for (int i = 0; i < 7; ++i) v[i] = v[i + 1];
        }
      }
    }
  }
};

__device__ __forceinline__ uint64_t token_of(float v, int x) { return static_cast<uint64_t>(key_of(v)) << 32 | static_cast<uint32_t>(~x); }
__device__ __forceinline__ float logit_of(uint64_t token) {
  const uint32_t k = static_cast<uint32_t>(token >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ int index_of(uint64_t token) { return static_cast<int>(~static_cast<uint32_t>(token)); }

// The same for tokens in shared memory
struct Taken {
  const FinishSmem& s;
  int n;
  template <class Fn>
  __device__ __forceinline__ void each(Fn fn) const {
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kThreads) fn(logit_of(s.token[i]), index_of(s.token[i]));
  }
};

// Among some tokens: the digit (of 9 bits) in which the running sum of their values, from the largest digit down (FALL) or
// from the smallest up, reaches goal; goal becomes what is left of it in front of that digit.  Where the sum never
// reaches it: the last digit that holds any.
template <bool FALL, class Each>
__device__ __forceinline__ uint32_t pick_digit(FinishSmem& s, uint64_t& goal, Each each) {
  const int tid = threadIdx.x;
  if (tid < 512) s.digits[tid] = 0;
  __syncthreads();
  each([&](uint32_t digit, uint64_t value) { add_lds(s.digits + digit, value); });
  __syncthreads();
  if (tid < 64) {
    uint64_t h[8], sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[i] = s.digits[FALL ? 511 - (8 * tid + i) : 8 * tid + i];
      sum += h[i];
    }
    const uint64_t upto = wave_scan(sum);
    const uint64_t over = __ballot(sum != 0 && upto >= goal), some = __ballot(sum != 0);
    const int l = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 0;
    if (tid == l) {
      uint64_t before = upto - sum, at = before;
      int d = 0;
      bool done = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!done && h[i] != 0) {
          d = i;
          before = at;
          done = at + h[i] >= goal;
        }
        at += h[i];
      }
      const int pos = 8 * l + d;
      s.digit = FALL ? 511 - pos : pos;
      s.rest = goal > before ? goal - before : 0;
    }
  }
  __syncthreads();
  goal = s.rest;
  return s.digit;
}

// The index at which the running sum of some tokens' values, in index order, reaches goal.  top_digit: shift of the
// indices' highest digit.  each(fn(index, value)).
template <class Each>
__device__ __forceinline__ int pick_index(FinishSmem& s, uint64_t goal, int top_digit, Each each) {
  uint32_t at = 0;
#pragma unroll 1
  for (int shift = top_digit; shift >= 0; shift -= 9) {
    const uint32_t d = pick_digit<false>(s, goal, [&](auto add) {
      each([&](int x, uint64_t n) {
        if (static_cast<uint32_t>(x) >> shift >> 9 == at) add((x >> shift) & 511, n);
      });
    });
    at = at << 9 | d;
  }
  return static_cast<int>(at);
}

// The border in rank among some tokens.  value: 1 (by rank) or the token's mass, 0: not one of them; kept are the
// tokens whose predecessors' values sum to less than goal (>= 1).  First the bin that holds it, then (not of the last
// bin) 1/512 of that; as soon as no more than 64 tokens are left, a wave ranks them one against the other.  Among more,
// as equal ones are, the digits of their logits select it, and an index.
template <int DT, class Tokens, class Value>
__device__ __forceinline__ void pick_border(const Tokens& all, FinishSmem& s, int top, int top_digit, uint64_t goal, Value value,
                                            uint32_t& key, int& last) {
  const int tid = threadIdx.x;
  uint64_t rest = goal;
  int bin = 0;
#pragma unroll 1
  for (int level = 0; level < 2 && (level == 0 || bin < kTail); ++level) {
    const auto place = [&](float v) {
      const int b = bin_of(v, top);
      if (level == 0) return b;
      const float x = fminf(fmaxf(v * 16.f, -0x1p27f), 0x1p27f);
      // (of x from -2^-25 up to 0 the difference rounds to 1)
      return b == bin ? 511 - min(static_cast<int>((x - floorf(x)) * 512.f), 511) : -1;
    };
    if (tid == 0) s.ties = 0;
    const int at = pick_digit<false>(s, rest, [&](auto add) {
      all.each([&](float v, int x) {
        const int to = place(v);
        const uint64_t n = to >= 0 ? value(v, x) : 0;
        if (n) add(to, n);
      });
    });
    all.each([&](float v, int x) {
      if (place(v) != at) return;
      const uint64_t n = value(v, x);
      if (!n) return;
      const uint32_t i = atomicAdd(&s.ties, 1u);
      if (i < 64) {
        s.value[i] = token_of(v, x);
        s.value[64 + i] = n;
      }
    });
    __syncthreads();
    const int close = s.ties;
    if (close <= 64 && tid < 64) {
      const uint64_t t = tid < close ? s.value[tid] : 0;
      uint64_t before = 0;
      for (int j = 0; j < close; ++j) before += s.value[j] > t ? s.value[64 + j] : 0;
      const uint64_t border = ~wave_all(tid < close && before < rest ? ~t : 0, Max{});
      if (tid == 0) s.one = border;
    }
    __syncthreads();
    if (close <= 64) {
      key = close ? static_cast<uint32_t>(s.one >> 32) : 0;
      last = close ? index_of(s.one) : 0x7FFFFFFF;  // none at all: none ends what is kept
      __syncthreads();
      return;
    }
    bin = at;
  }
  // the bits in which floats of the type differ, from the top: 32, 19 (f16: sign, 8 of exponent, 10) or 16; those
  // below are all zero, or of a negative float all one
  constexpr int kBits = DT == TQ_F32 ? 32 : DT == TQ_F16 ? 19 : 16, kDigits = (kBits + 8) / 9, kLow = 32 - kBits;
  uint32_t prefix = 0;
#pragma unroll 1
  for (int shift = 9 * (kDigits - 1); shift >= 0; shift -= 9) {
    const uint32_t d = pick_digit<true>(s, goal, [&](auto add) {
      all.each([&](float v, int x) {
        const uint32_t k = key_of(v) >> kLow;
        if (static_cast<uint32_t>(static_cast<uint64_t>(k) >> (shift + 9)) == prefix) {
          const uint64_t n = value(v, x);
          if (n) add((k >> shift) & 511, n);
        }
      });
    });
    prefix = prefix << 9 | d;
  }
  key = prefix << kLow;
  if (kLow && !(key & 0x80000000u)) key |= (1u << kLow) - 1;
  // equal logits have equal values: how many of them are kept, the first in index order
  if (threadIdx.x == 0) {
    s.one = 0;
    s.ties = 0;
  }
  __syncthreads();
  all.each([&](float v, int x) {
    if (key_of(v) == key) {
      const uint64_t n = value(v, x);
      if (n) {
        s.one = n;
        atomicAdd(&s.ties, 1u);
      }
    }
  });
  __syncthreads();
  const uint64_t one = s.one;
  uint64_t keep = one ? goal / one + (goal % one != 0) : 1;  // (a goal that nothing reaches may be the largest integer)
  if (keep < 1) keep = 1;
  last = 0x7FFFFFFF;
  if (keep >= s.ties) return;
  last = pick_index(s, keep, top_digit, [&](auto fn) {
    all.each([&](float v, int x) {
      if (key_of(v) == key && value(v, x)) fn(x, 1);
    });
  });
}

__device__ __forceinline__ uint64_t ceiling(double g) {  // at least 1
  return g >= 0x1p63 ? ~0ull : g >= 1.0 ? static_cast<uint64_t>(ceil(g)) : 1;
}

// The border of a row: by rank, then by mass
template <int DT, class Tokens, class In, class Integer>
__device__ __forceinline__ void cut_row(const Tokens& all, FinishSmem& s, const Settings& set, int top, int top_digit, uint64_t mass_goal, In in,
                                        Integer integer, uint32_t& key, int& last) {
  if (set.mode == kTopK) pick_border<DT>(all, s, top, top_digit, static_cast<uint64_t>(set.k), [&](float, int) -> uint64_t { return 1; }, key, last);
  if (set.p >= 1.0) return;
  const uint32_t key_k = key;
  const int last_k = last;
  const auto value = [&](float v, int x) -> uint64_t {
    const uint32_t k = key_of(v);
    return in(v) && (k > key_k || (k == key_k && x <= last_k)) ? integer(v) : 0;
  };
  if (set.mode == kTopK) {
    uint64_t sum = 0;
    all.each([&](float v, int x) { sum += value(v, x); });
    sum = block_all<kWaves>(sum, s.part, Sum{});
    __syncthreads();
    mass_goal = ceiling(set.p * static_cast<double>(sum));
  }
  pick_border<DT>(all, s, top, top_digit, mass_goal, value, key, last);
  if (key < key_k || (key == key_k && last > last_k)) {  // all that the rank keeps
    key = key_k;
    last = last_k;
  }
}

// A row's whole list in s.token, n <= kRanked of them, or (ONE) at most 64 by one wave: a thread has a token, and meets
// every other.
template <bool ONE>
__device__ __forceinline__ void rank_tokens(const SampleArgs& a, FinishSmem& s, const Settings& set, int row, float m, int n, double goal) {
  const int tid = threadIdx.x;
  const auto sync = [] {
    if constexpr (ONE) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else __syncthreads();
  };
  const auto sum_of = [&](uint64_t v) {
    if constexpr (ONE) return wave_all(v, Sum{});
    else {
      __syncthreads();
      return block_all<kWaves>(v, s.part, Sum{});
    }
  };
  const Weigh weigh(set, tame(m));
  const uint64_t t = tid < n ? s.token[tid] : 0;
  const double w = tid < n ? weigh(logit_of(t)) : 0.0;
  constexpr double unit = ONE ? 0x1p55 : 0x1p53;  // the maximum is among them
  const uint64_t whole = static_cast<uint64_t>(w * unit + 0.5), val = w > 0.0 && !whole ? 1 : whole;
  const int x = index_of(t), padded = (n + 7) & ~7;
  if (tid < padded) {
    s.token[tid] = t;
    s.value[tid] = val;
  }
  sync();
  int rank = 0;
  uint64_t before = 0;
  if (ONE || tid < n) {
#pragma unroll 8
    for (int j = 0; j < padded; ++j) {
      const uint64_t v = s.value[j];
      const bool ahead = s.token[j] > t;
      rank += ahead;
      before += ahead ? v : 0;
    }
  }
  const bool in = tid < n && (set.mode != kTopK || rank < set.k);
  uint64_t bar = ~0ull;  // predecessors of a kept token sum to less
  if (set.mode == kTopP) bar = ceiling(goal * unit);
  else if (set.mode == kTopK && set.p < 1.0) bar = ceiling(set.p * static_cast<double>(sum_of(in ? val : 0)));
  const bool on = in && before < bar && w >= set.m;
  const uint64_t sum = sum_of(on ? val : 0);
  if (a.probs) {
    if (on) a.probs[static_cast<int64_t>(row) * a.V + x] = static_cast<float>(w * (unit / static_cast<double>(sum)));
    if (tid == 0) a.state[row] = RowState{0, 0, m, 1, 0.0};
    return;
  }
  const double pass = static_cast<double>(a.uniforms[row]) * static_cast<double>(sum);
  sync();
  if (tid < padded) s.value[tid] = on ? val : 0;
  sync();
  uint64_t upto = 0;  // of the kept tokens at or before it
  if (ONE || tid < n) {
#pragma unroll 8
    for (int j = 0; j < padded; ++j) {
      const uint64_t v = s.value[j];
      upto += index_of(s.token[j]) <= x ? v : 0;
    }
  }
  // the first index that passes; the last one, should u be 1 or more
  const bool over = on && static_cast<double>(upto) > pass;
  int first = over ? -x : -0x7FFFFFFF, end = on ? x : -1;
  if constexpr (ONE) {
    first = wave_all(first, Max{});
    end = wave_all(end, Max{});
  } else {
    first = block_all<kWaves>(first, reinterpret_cast<int*>(s.part), Max{});
    __syncthreads();
    end = block_all<kWaves>(end, reinterpret_cast<int*>(s.part), Max{});
  }
  if (tid == 0) a.tokens[row] = first > -0x7FFFFFFF ? -first : end;
}

// A block to a row, bound by its chain of steps: 7.5 us where one wave ranks the list, 12 to 15 where it is selected from
// hundreds (one pass over them to find the bin, one to gather it, a few to draw), 25 to 30 for a row that
// keeps tens of thousands.
template <int DT>
__global__ void __launch_bounds__(kThreads) sample_finish_kernel(SampleArgs a) {
  __shared__ FinishSmem s;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Settings& set = a.of(row);
  const int mode = set.mode;
  const int64_t at0 = static_cast<int64_t>(row) * a.C;
  const RowCut cut = mode == kTopP ? a.cut[row] : RowCut{0.0, 0, kTail};
  const int room = 1 << a.lg_room;
  for (int c = tid; c < a.C; c += kThreads) {
    s.top[c] = a.top[at0 + c];
    const int n = mode == kAll ? 0 : a.listed[at0 + c];
    s.listed[c] = n <= room ? n : -1;
    s.mass[c] = mode == kTopK ? 0.0 : mode == kAll ? a.mass[at0 + c] : a.kept[at0 + c];
    s.extra[c] = 0;
  }
  if (tid < kBins) s.bins[tid] = 0;
  if (tid == 0) {
    s.n = 0;
    s.raw = 0;
  }
  __syncthreads();
  float m = -INFINITY;
  for (int c = lane; c < a.C; c += 64) m = fmaxf(m, s.top[c]);
  m = wave_all(m, Max{});
  const float mt = tame(m);
  if (m == -INFINITY) {  // no token has a weight
    if (tid == 0) {
      if (a.tokens) a.tokens[row] = -1;
      else a.state[row] = RowState{0xFFFFFFFFu, -1, m, mode != kAll, 0.0};
    }
    return;
  }
  const int top = grid_of(mt);
  const Weigh weigh(set, mt);
  const double least = set.m;
  const Candidates<DT> all{a, s, row, m};
  uint32_t key = 0;  // the border
  int last = 0x7FFFFFFF;
  double unit = 1.0;  // listed tokens' masses as integers
  if (mode == kAll) {
    for (int c = tid; c < a.C; c += kThreads)
      s.mass[c] = s.top[c] == -INFINITY || !counts(s.top[c], m) ? 0.0 : s.mass[c] * weigh(tame(s.top[c]));
    __syncthreads();
  } else {
    // ---- a table of the lists' runs of 64, by the first wave
    if (wave == 0) {
      int run = 0, bad = 0, last_n = 0;
      for (int c0 = 0; c0 < a.C; c0 += 64) {
        const int c = c0 + lane;
        int n = c < a.C && counts(s.top[c], m) ? s.listed[c] : 0;
        if (c < a.C && !counts(s.top[c], m)) s.listed[c] = 0;
        int segs = n > 0 ? (n + 63) / 64 : 0;
        const int upto = wave_scan(segs), from = run + upto - segs;
        if (from + segs > kSegments) {  // no place in the table
          n = -1;
          s.listed[c] = -1;
          segs = 0;
        }
        for (int i = 0; i < segs; ++i) s.segment[from + i] = static_cast<uint32_t>(c) << 16 | static_cast<uint32_t>(i);
        bad |= n < 0;
        const uint64_t in = __ballot(segs > 0);
        if (in) last_n = __builtin_amdgcn_readlane(from + segs, 63 - __builtin_clzll(in));
        run += __builtin_amdgcn_readlane(upto, 63);
      }
      if (lane == 0) s.segments = min(last_n, kSegments);
      if (__any(bad) && lane == 0) s.raw = 1;
    }
    __syncthreads();
    int hi = cut.hi;
    const int lo = cut.lo;

    // ---- the listed tokens, as far as they can be sorted
    float peak = -INFINITY;
    const auto reach_rank = [&]() {  // the bin that k tokens in s.bins reach
      __syncthreads();
      if (wave == 0) {
        int h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = 8 * lane + i < kTail ? static_cast<int>(s.bins[8 * lane + i]) : 0;
        const int bin = reach_bin(h, set.k);
        if (lane == 0) {
          s.hi = bin;
          s.n = 0;
        }
      }
      __syncthreads();
      return s.hi;
    };
    // every chunk listed its own first k: of them all, those down to the bin that k reach
    const bool many = mode == kTopK && (s.raw || s.segments > 2 * kThreads / 64);
    if (many) {
      all.each([&](float v, int) { atomicAdd(s.bins + bin_of(v, top), 1u); });
      hi = reach_rank();
    }
    all.each([&](float v, int x) {
      const int b = bin_of(v, top);
      const bool on = b >= lo && b <= hi && (mode != kMinP || weigh(v) >= least);
      const uint64_t some = __ballot(on);
      if (!some) return;
      int to = 0;
      const int first = __builtin_ctzll(some);
      if (lane == first) to = atomicAdd(&s.n, __popcll(some));
      to = __builtin_amdgcn_readlane(to, first) + __popcll(some & ((1ull << lane) - 1));
      if (on) {
        peak = fmaxf(peak, v);
        if (to < kShort) s.token[to] = token_of(v, x);
      }
    });
    __syncthreads();
    int n = s.n;
    if (mode == kTopK && !many && n > 64) {  // n <= 2048
      uint64_t t[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        t[i] = tid + i * kThreads < n ? s.token[tid + i * kThreads] : 0;
        if (tid + i * kThreads < n) atomicAdd(s.bins + bin_of(logit_of(t[i]), top), 1u);
      }
      hi = reach_rank();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool on = tid + i * kThreads < n && bin_of(logit_of(t[i]), top) <= hi;
        const uint64_t some = __ballot(on);
        int to = 0;
        if (some && lane == 0) to = atomicAdd(&s.n, __popcll(some));
        to = __builtin_amdgcn_readfirstlane(to) + __popcll(some & ((1ull << lane) - 1));
        if (on) s.token[to] = t[i];
      }
      __syncthreads();
      n = s.n;
    }
    const bool alone = n <= kShort && lo == 0;  // the tokens in s.token are all that can be kept
    const double goal = set.p * cut.total;
    const auto integer = [&](double w) -> uint64_t {  // of listed tokens
      if (!(w > 0.0)) return 0;
      const uint64_t x = static_cast<uint64_t>(w * unit + 0.5);
      return x ? x : 1;
    };

    const int top_digit = 9 * ((31 - __builtin_clz(a.V - 1 | 1)) / 9);  // of an index
    if (alone && n <= kRanked) {
      if (n > 64) {
        rank_tokens<false>(a, s, set, row, m, n, goal);
      } else if (wave == 0) {
        rank_tokens<true>(a, s, set, row, m, n, goal);
      }
      return;
    }

    double certain = 0.0;  // stands above the listed tokens
    if (mode == kTopP && lo > 0)
      for (int c = 0; c < a.C; ++c) certain += s.mass[c];
    peak = block_all<kWaves>(peak, reinterpret_cast<float*>(s.part), Max{});
    __syncthreads();
    const auto in = [&](float v) {
      const int b = bin_of(v, top);
      return b >= lo && b <= hi;
    };
    const auto mass = [&](float v) { return integer(weigh(v)); };
    const Taken taken{s, n};
    // The unit has the total, the row's or the listed tokens', at 2^62 to 2^63 (of up to 2^24 integers, each less than one
    // off): next to n times the heaviest, equal light tokens' roundings would add up, to 2^-29 of the total at 150000.
    if (mode == kTopP) {
      int bits;
      frexp(cut.total, &bits);
      unit = ldexp(1.0, 63 - bits);
    } else if (mode == kTopK || alone) {  // the heaviest, of weight 1, is listed
      unit = ldexp(1.0, 30 + __builtin_clz(n));
      uint64_t sum = 0;
      const auto add = [&](float v, int) { sum += in(v) ? mass(v) : 0; };
      if (n <= kShort) taken.each(add);
      else all.each(add);
      sum = block_all<kWaves>(sum, s.part, Sum{});
      __syncthreads();
      unit = ldexp(unit, __builtin_clzll(sum + n) - 1);
    }
    const double g = (goal - certain) * unit;
    if (mode == kTopP && certain > 0.0 && !(g > 0.0)) {  // what is certain reaches the goal
      key = key_of(peak);
      last = -1;
    } else if (mode != kMinP) {
      if (n <= kShort) cut_row<DT>(taken, s, set, top, top_digit, ceiling(g), in, mass, key, last);
      else cut_row<DT>(all, s, set, top, top_digit, ceiling(g), in, mass, key, last);
    }
    const auto kept = [&](float v, int x) -> uint64_t {
      const uint32_t k = key_of(v);
      if (!(k > key || (k == key && x <= last))) return 0;
      const double w = weigh(v);
      return w >= least ? integer(w) : 0;
    };
    if (alone) {
      // ---- all that is kept stands in s.token
      uint64_t sum = 0;
      taken.each([&](float v, int x) { sum += kept(v, x); });
      sum = block_all<kWaves>(sum, s.part, Sum{});
      if (a.probs) {
        const double inverse = unit / static_cast<double>(sum);
        taken.each([&](float v, int x) {
          if (kept(v, x)) a.probs[static_cast<int64_t>(row) * a.V + x] = static_cast<float>(weigh(v) * inverse);
        });
        if (tid == 0) a.state[row] = RowState{0, 0, m, 1, 0.0};
        return;
      }
      // the first index at which the sum passes u times the total: digit by digit
      const uint64_t pass = static_cast<uint64_t>(fmin(fmax(static_cast<double>(a.uniforms[row]), 0.0), 1.0) * static_cast<double>(sum)) + 1;
      const int at = pick_index(s, pass, top_digit, [&](auto fn) {
        taken.each([&](float v, int x) {
          const uint64_t n = kept(v, x);
          if (n) fn(x, n);
        });
      });
      if (tid == 0) a.tokens[row] = at;
      return;
    }
    // ---- the chunks' kept masses: what is certain, and the listed tokens up to the border
    if (mode != kMinP) {
      all.each([&](float v, int x) {
        const uint32_t k = key_of(v);
        const int b = bin_of(v, top);
        if (b >= lo && b <= hi && (k > key || (k == key && x <= last))) {
          const double w = weigh(v);
          if (w >= least) add_lds(s.extra + (x >> a.lg_chunk), integer(w));
        }
      });
      __syncthreads();
      for (int c = tid; c < a.C; c += kThreads) s.mass[c] += static_cast<double>(s.extra[c]) / unit;
      __syncthreads();
    }
  }

  // ---- the chunk: the first whose running sum passes u times the total
  if (wave == 0) {
    double sum = 0.0;
    for (int c = lane; c < a.C; c += 64) sum += s.mass[c];
    const double total = wave_all(sum, Sum{});
    if (!a.tokens) {
      if (lane == 0) a.state[row] = RowState{key, last, m, 0, 1.0 / total};
    } else {
      const double goal = static_cast<double>(a.uniforms[row]) * total;
      double run = 0.0, bar = 0.0;
      int chunk = -1;
      for (int c0 = 0; c0 < a.C; c0 += 64) {
        const double v = c0 + lane < a.C ? s.mass[c0 + lane] : 0.0;
        const double upto = wave_scan(v) + run;
        const uint64_t some = __ballot(v > 0.0), over = __ballot(v > 0.0 && upto > goal);
        if (some) {
          const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
          chunk = c0 + l;
          bar = goal - (lane_value(upto, l) - lane_value(v, l));
        }
        if (over) break;
        run = lane_value(upto, 63);
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
#pragma unroll 1
  for (int x0 = chunk << a.lg_chunk; x0 < end; x0 += kThreads * 8) {
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
        const double ww = weigh(y);
        w[e] = ww >= least ? ww : 0.0;
      }
      sum += w[e];
    }
    double upto = wave_scan(sum);
    if (lane == 63) s.sum[wave] = upto;
    __syncthreads();
    double before = upto - sum, tile = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) before += s.sum[i];
      tile += s.sum[i];
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
    run -= tile;
  }
  if (s.pick < 0) {  // block-uniform
    const int most = block_all<kWaves>(fallback, reinterpret_cast<int*>(s.part), Max{});
    if (tid == 0) a.tokens[row] = most;
  } else if (tid == 0) {
    a.tokens[row] = 0x7FFFFFFF - s.pick;
  }
}

// ---------------------------------------------------------------- write
// Rows that are not written yet, in tiles of 2048 tokens.  Up to 2048 tiles have a block each.  Of more rows, most of
// which are written, the others' tiles are dealt to all blocks: every block finds them among the rows' states, 2048 at a time
// (3 of 512 rows of 151936 not written: 8 us; 17 with 8 blocks for every row.  5 rows of 50257: 1.8 and 3.9).
template <int DT>
__device__ __forceinline__ void write_tile(const SampleArgs& a, int row, const RowState& st, int tile) {
  const int x = (tile * 256 + static_cast<int>(threadIdx.x)) * 8;
  if (x >= a.V) return;
  const Settings& set = a.of(row);
  const Weigh weigh(set, tame(st.top));
  float v[8], out[8];
  load_logits<DT>(row_of<DT>(a, row), x, a.V, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = tame(v[e], st.top);
    const uint32_t k = key_of(y);
    out[e] = 0.f;
    if (y != -INFINITY && (k > st.key || (k == st.key && x + e <= st.last))) {
      const double w = weigh(y);
      out[e] = w >= set.m ? static_cast<float>(w * st.inverse) : 0.f;
    }
  }
  float* const to = a.probs + static_cast<int64_t>(row) * a.V + x;
  if (x + 8 <= a.V) {
    __builtin_memcpy(to, out, 32);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (x + e < a.V) to[e] = out[e];
  }
}
template <int DT>
__global__ void __launch_bounds__(256) sample_write_kernel(SampleArgs a, int tiles) {
  constexpr int kStep = 2048;
  __shared__ int s_row[kStep];
  __shared__ int s_count[kStep / 64];  // of 64 rows
  if (static_cast<int64_t>(a.N) * tiles <= gridDim.x) {
    const int row = blockIdx.x / tiles;
    const RowState st = a.state[row];
    if (!st.done) write_tile<DT>(a, row, st, blockIdx.x - row * tiles);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll 1
  for (int r0 = 0; r0 < a.N; r0 += kStep) {
    int done[kStep / 256];
#pragma unroll
    for (int i = 0; i < kStep / 256; ++i) done[i] = r0 + i * 256 + tid < a.N ? a.state[r0 + i * 256 + tid].done : 1;
    uint64_t todo[kStep / 256];
#pragma unroll
    for (int i = 0; i < kStep / 256; ++i) {
      todo[i] = __ballot(!done[i]);
      if (lane == 0) s_count[i * 4 + wave] = __popcll(todo[i]);
    }
    __syncthreads();
    // in rising order, which is the same in all blocks
    int rows = 0;
#pragma unroll
    for (int j = 0; j < kStep / 64; ++j) {
      if (wave == (j & 3) && !done[j / 4]) s_row[rows + __popcll(todo[j / 4] & ((1ull << lane) - 1))] = r0 + (j / 4) * 256 + tid;
      rows += s_count[j];
    }
    __syncthreads();
    const int64_t all = static_cast<int64_t>(rows) * tiles;
#pragma unroll 1
    for (int64_t t = blockIdx.x; t < all; t += gridDim.x) {
      const int i = static_cast<int>(static_cast<uint64_t>(t) / static_cast<unsigned>(tiles));
      write_tile<DT>(a, s_row[i], a.state[s_row[i]], static_cast<int>(t - static_cast<int64_t>(i) * tiles));
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- launch
struct SamplePlan {
  int C, lg_chunk;
  int64_t rows, state, cut, top, mass, kept, listed, depth, hist, list, bytes;  // offsets
};

// The chunks of a row, and the workspace: whatever the settings, which may be the rows' own, 2 bytes a token for lists and 2 KB
// a chunk for its histogram.
static SamplePlan plan_sample(int64_t N, int64_t V) {
  SamplePlan p{};
  p.lg_chunk = 15;
  const auto chunks = [&](int lg) { return (V + (int64_t(1) << lg) - 1) >> lg; };
  // More than a block to a compute unit, but not two of short chunks, as every block of a row joins the histograms of all
  // its chunks: 16 rows of 151936 in 304 blocks 34.0 us, in 608 36.3; 64 rows of 128256 in 512 39.6.
  while (p.lg_chunk > 12 && (chunks(p.lg_chunk - 1) == 1 || (N * chunks(p.lg_chunk) < 300 && chunks(p.lg_chunk - 1) <= kMaxChunks)))
    --p.lg_chunk;
  p.C = static_cast<int>(chunks(p.lg_chunk));
  const int64_t n = N * p.C;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 15) / 16 * 16;
    return here;
  };
  p.rows = take(N * static_cast<int64_t>(sizeof(Settings)));
  p.state = take(N * static_cast<int64_t>(sizeof(RowState)));
  p.cut = take(N * static_cast<int64_t>(sizeof(RowCut)));
  p.top = take(n * 4);
  p.mass = take(n * 8);
  p.kept = take(n * 8);
  p.listed = take(n * 4);
  p.depth = take(n * 4);
  p.hist = take(n * kBins * 4);
  p.list = take((n << (p.lg_chunk - 2)) * 8);  // a quarter of the tokens
  p.bytes = at;
  return p;
}
// A launch has fewer than 2^32 threads: kThreads to a row in the finish, kScan to a chunk in the scan
static bool sample_shape(int64_t N, int64_t V) {
  return N >= 1 && V >= 1 && V <= (int64_t(1) << 24) && N < (int64_t(1) << 32) / kThreads &&
         N * plan_sample(N, V).C < (int64_t(1) << 32) / kScan;
}

template <int DT>
static void launch_sample(const SampleArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.N * a.C));
  sample_scan_kernel<DT><<<grid, kScan, 0, s>>>(a);
  // rows' own settings may be any
  if (a.rows || a.all.mode == kTopP || a.all.mode == kMinP) sample_select_kernel<DT><<<grid, kScan, 0, s>>>(a);
  sample_finish_kernel<DT><<<dim3(a.N), kThreads, 0, s>>>(a);
  if (!a.tokens) {
    const int tiles = (a.V + 2047) / 2048;
    const int64_t all = static_cast<int64_t>(a.N) * tiles;
    sample_write_kernel<DT><<<dim3(static_cast<unsigned>(all < 2048 ? all : 2048)), 256, 0, s>>>(a, tiles);
  }
}

static int run_sample(const char* what, SampleArgs& a, int32_t dtype, double temperature, int32_t top_k, double top_p,
                      double min_p, void* workspace, int64_t bytes, void* stream) {
  TQ_REQUIRE(a.N >= 0 && a.V >= 1 && a.ld >= 0, "%s: bad shape", what);
  TQ_REQUIRE(dtype == TQ_F32 || dtype == TQ_F16 || dtype == TQ_BF16, "%s: unknown dtype %d", what, dtype);
  TQ_REQUIRE(temperature >= 0.0 && top_k >= 0 && top_p >= 0.0 && min_p >= 0.0,
             "%s: temperature, top_k, top_p and min_p must not be negative", what);
  if (a.N == 0) return TQ_OK;
  TQ_REQUIRE(sample_shape(a.N, a.V), "%s: at most 2^24 tokens, fewer than 2^22 rows and 2^23 chunks of 2^15 tokens, got %d rows of %d",
             what, a.N, a.V);
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
  a.lg_room = p.lg_chunk - 2;
  a.all = Settings(a.V, temperature, top_k, top_p, min_p);
  uint8_t* const w = static_cast<uint8_t*>(workspace);
  a.rows = a.t_rows || a.k_rows || a.p_rows || a.m_rows ? reinterpret_cast<Settings*>(w + p.rows) : nullptr;
  a.state = reinterpret_cast<RowState*>(w + p.state);
  a.top = reinterpret_cast<float*>(w + p.top);
  a.mass = reinterpret_cast<double*>(w + p.mass);
  a.kept = reinterpret_cast<double*>(w + p.kept);
  a.cut = reinterpret_cast<RowCut*>(w + p.cut);
  a.listed = reinterpret_cast<int32_t*>(w + p.listed);
  a.depth = reinterpret_cast<int32_t*>(w + p.depth);
  a.hist = reinterpret_cast<float*>(w + p.hist);
  a.list = reinterpret_cast<uint2*>(w + p.list);
  hipStream_t s = as_stream(stream);
  if (dtype == TQ_F32) launch_sample<TQ_F32>(a, s);
  else if (dtype == TQ_F16) launch_sample<TQ_F16>(a, s);
  else launch_sample<TQ_BF16>(a, s);
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
  SampleArgs a{.all = Settings(1, 1.0, 0, 1.0, 0.0)};
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
  SampleArgs a{.all = Settings(1, 1.0, 0, 1.0, 0.0)};
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
