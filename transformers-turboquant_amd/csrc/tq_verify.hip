// Verification of drafted tokens against the target model's probabilities, from given uniforms.
//
// Node 0 of a sequence is the last token already emitted; node i > 0 was drafted as a child of
// node parent(i) < i.  p_c is the target's distribution after node c.
//   tree (candidates chosen, no draft distribution): the children of a node are tried in index
//     order; child i is accepted iff u_i (1 - sum of p_c over the earlier children's tokens) < p_c(x_i),
//     which samples p_c exactly: what a rejected candidate leaves is p_c without it.
//   chain (x_i drawn from the draft's q_{i-1}): accepted iff u_i q_{i-1}(x_i) < p_{i-1}(x_i); a
//     rejection leaves (p_{i-1} - q_{i-1})+.
// The walk goes from the root to the first accepted child until a node has none; the next token is
// drawn from what is left at that node, w: the first x with w_0 + ... + w_x > u_0 sum(w).
//
// The walk needs a few probabilities per node (one lane each), the draw one row of the vocabulary
// (two for a chain), so the work is latency and one pass over that row: the row is cut into tiles of
// 2048 entries, summed over many blocks (every block repeats the walk: cheaper than a launch that only
// walks), then one block per sequence finds the tile and searches it.  Probabilities and sums are
// float64: the token is decided by a comparison of sums over up to ~10^5 terms, and in float32
// their rounding would move the border of a few tokens in a hundred thousand by more than the
// token's own probability.
//
// Measured: a chain of 5, V = 50257, one sequence 11.5 us (two launches of 4 us, each a few
// dependent round trips); chains of 8, V = 128256, 64 sequences 19.1 us (66 MB, 14.0 us for the sums: 4.7
// TB/s); trees of 32, V = 151936, 16 sequences in bf16 13.0 us (sums 8.6: 1.8 for the siblings' loop and 0.8 for
// striking the rejected tokens from the row, by timing copies without them; 6.1 for three dependent round
// trips, the walk and the row).
#include "tq_common.h"

namespace tq {

constexpr int kVerifyThreads = 256;
constexpr int kMaxNodes = 64;  // a node is a lane
constexpr int kTile = kVerifyThreads * 8;  // vocabulary entries summed together
constexpr int kLeftWords = 3 + kMaxNodes;

struct VerifyArgs {
  const int64_t* tokens;  // [B, T]
  const void* target;     // [B, T, V], strides tb, tt
  int64_t tb, tt;
  const void* draft;      // [B, T - 1, V], strides db, dt, or null
  int64_t db, dt;
  const float* uniforms;  // [B, T]
  const int32_t* parents; // [B, T] (ld_parents = T), [T] (0), or null: a chain
  int64_t ld_parents;
  int B, T, V;
  int ntile, per;         // tiles of a row, tiles per block
  double* sums;           // [B, 2, ntile]: of w, of p
  int64_t* left;          // [B, kLeftWords]: stop, nrej, residual, the rejected tokens
  int32_t* path;          // [B, T]
  int32_t* count;         // [B]
  int64_t* next;          // [B]
};

// lane l's value, l the same in every lane
__device__ __forceinline__ int lane_value(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ int64_t lane_value(int64_t v, int l) {
  const uint64_t u = static_cast<uint64_t>(v);
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(lane_value(static_cast<int>(u), l))) |
                              (static_cast<uint64_t>(static_cast<uint32_t>(lane_value(static_cast<int>(u >> 32), l))) << 32));
}
__device__ __forceinline__ double lane_value(double v, int l) {
  return __builtin_bit_cast(double, lane_value(__builtin_bit_cast(int64_t, v), l));
}

// what is left to draw from after the walk
struct Left {
  int stop;        // node whose distribution remains
  int nrej;        // tree: rejected tokens, in s_rej
  bool residual;   // chain: a rejected child, w = (p - q)+
};

// The walk, by the first wave of a block; the others get its outcome through LDS.
template <int DT>
__device__ __forceinline__ Left walk(const VerifyArgs& a, int b, int64_t* s_rej, int* s_left, bool write) {
  const int tid = threadIdx.x;
  if (tid < 64) {
    const int i = tid;
    const bool live = i < a.T;
    int par = -1;
    int64_t tok = -1;
    double u = 0.0;
    if (live) {
      par = a.parents ? a.parents[b * a.ld_parents + i] : i - 1;
      tok = a.tokens[static_cast<int64_t>(b) * a.T + i];
      u = static_cast<double>(a.uniforms[static_cast<int64_t>(b) * a.T + i]);
    }
    const bool inner = live && par >= 0 && par < i;
    double p = 0.0, bar = 0.0;
    if (inner && tok >= 0 && tok < a.V) p = static_cast<double>(load_act<DT>(a.target, b * a.tb + par * a.tt + tok));
    if (a.draft) {
      if (inner && tok >= 0 && tok < a.V) bar = u * static_cast<double>(load_act<DT>(a.draft, b * a.db + par * a.dt + tok));
    } else {
      // the earlier siblings in index order; a candidate that repeats one has nothing left to accept.
      // A node whose parent is not an earlier node has no place in the tree and is nobody's sibling.
      double rem = 1.0;
      const int T = a.parents ? a.T : 0;  // a chain has no siblings
      const int placed = inner ? par : -1;
      for (int j = 0; j < T; ++j) {
        const int pj = lane_value(placed, j);
        const int64_t tj = lane_value(tok, j);
        const double qj = lane_value(p, j);  // settled: every earlier sibling of j has had its turn
        if (j < i && pj == par) {
          rem -= qj;
          if (tj == tok) p = 0.0;
        }
      }
      bar = u * rem;
    }
    const bool good = inner && bar < p;
    uint64_t taken = 1;
    int cur = 0;
    for (int step = 1; step < a.T; ++step) {  // a child's index is above its parent's
      const uint64_t m = __ballot(good && par == cur);
      if (!m) break;
      cur = __builtin_ctzll(m);
      taken |= 1ull << cur;
    }
    const bool child = inner && par == cur;
    const uint64_t kids = __ballot(child);
    if (child && !a.draft) s_rej[__popcll(kids & ((1ull << i) - 1))] = tok;
    if (i == 0) {
      s_left[0] = cur;
      s_left[1] = a.draft ? 0 : __popcll(kids);
      s_left[2] = a.draft && kids != 0;
    }
    if (write && live) {
      const int n = __popcll(taken);
      if ((taken >> i) & 1) a.path[static_cast<int64_t>(b) * a.T + __popcll(taken & ((1ull << i) - 1))] = i;
      if (i >= n) a.path[static_cast<int64_t>(b) * a.T + i] = -1;
      if (i == 0) a.count[b] = n;
    }
  }
  __syncthreads();
  return Left{s_left[0], s_left[1], s_left[2] != 0};
}

// eight consecutive probabilities from x (fewer at the row's end: zeros)
template <int DT>
__device__ __forceinline__ void load_probs(const void* row, int x, int V, float (&v)[8]) {
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
    for (int j = 0; j < 8; ++j) v[j] = x + j < V ? load_act<DT>(row, x + j) : 0.f;
  }
}

// weights of eight entries from x on, and their plain probabilities; what is not a positive
// number weighs nothing
template <int DT>
__device__ __forceinline__ void weights8(const VerifyArgs& a, const void* prow, const void* qrow, const Left& l,
                                         const int64_t* s_rej, int x, double (&w)[8], double (&pl)[8]) {
  float p[8], q[8];
  load_probs<DT>(prow, x, a.V, p);
  if (l.residual) load_probs<DT>(qrow, x, a.V, q);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    pl[j] = p[j] > 0.f ? static_cast<double>(p[j]) : 0.0;
    const double r = l.residual ? static_cast<double>(p[j]) - static_cast<double>(q[j]) : static_cast<double>(p[j]);
    w[j] = r > 0.0 ? r : 0.0;
  }
  for (int k = 0; k < l.nrej; ++k) {
    const int64_t at = s_rej[k] - x;
    if (at >= 0 && at < 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at == j) w[j] = 0.0;
    }
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int sh = 32; sh >= 1; sh >>= 1) v += __shfl_xor(v, sh, 64);
  return v;
}

template <int DT>
__device__ __forceinline__ const void* row_at(const void* base, int64_t i) {
  return static_cast<const uint8_t*>(base) + i * (DT == TQ_F32 ? 4 : 2);
}

// inclusive sum over the wave
__device__ __forceinline__ double wave_scan(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int sh = 1; sh < 64; sh <<= 1) {
    const double t = __shfl_up(v, sh, 64);
    if (lane >= sh) v += t;
  }
  return v;
}

// The sums of w and of p over each tile of a row; a block takes a.per consecutive tiles.
template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) verify_sum_kernel(VerifyArgs a) {
  __shared__ int64_t s_rej[kMaxNodes];
  __shared__ int s_left[3];
  __shared__ double s_part[2][2][kVerifyThreads / 64];
  const int b = blockIdx.y, tid = threadIdx.x;
  const Left l = walk<DT>(a, b, s_rej, s_left, blockIdx.x == 0);
  if (blockIdx.x == 0) {  // the outcome, for the draw
    int64_t* const left = a.left + static_cast<int64_t>(b) * kLeftWords;
    if (tid < 3) left[tid] = s_left[tid];
    if (tid < l.nrej) left[3 + tid] = s_rej[tid];
  }
  const void* prow = row_at<DT>(a.target, b * a.tb + l.stop * a.tt);
  const void* qrow = l.residual ? row_at<DT>(a.draft, b * a.db + l.stop * a.dt) : nullptr;
  const int end = min(a.ntile, static_cast<int>(blockIdx.x + 1) * a.per);
  for (int t = blockIdx.x * a.per, odd = 0; t < end; ++t, odd ^= 1) {
    double sw = 0.0, sp = 0.0;
    const int x = t * kTile + tid * 8;
    if (x < a.V) {
      double w[8], p[8];
      weights8<DT>(a, prow, qrow, l, s_rej, x, w, p);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sw += w[j];
        sp += p[j];
      }
    }
    sw = wave_sum(sw);
    sp = wave_sum(sp);
    if ((tid & 63) == 0) {
      s_part[odd][0][tid >> 6] = sw;
      s_part[odd][1][tid >> 6] = sp;
    }
    __syncthreads();  // the next tile writes the other half: one barrier per tile suffices
    if (tid < 2) {
      double v = 0.0;
#pragma unroll
      for (int k = 0; k < kVerifyThreads / 64; ++k) v += s_part[odd][tid][k];
      a.sums[(static_cast<int64_t>(b) * 2 + tid) * a.ntile + t] = v;
    }
  }
}

// One block per sequence: the first wave scans the tiles' sums for the one in which the running sum
// passes u_0 sum(w), then the block scans that tile, 8 entries a thread.
template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) verify_pick_kernel(VerifyArgs a) {
  __shared__ int64_t s_rej[kMaxNodes];
  __shared__ double s_wave[kVerifyThreads / 64];
  __shared__ double s_bar;
  __shared__ int s_tile, s_mode, s_last;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t* const left = a.left + static_cast<int64_t>(b) * kLeftWords;
  Left l{static_cast<int>(left[0]), static_cast<int>(left[1]), left[2] != 0};
  if (tid < l.nrej) s_rej[tid] = left[3 + tid];
  if (wave == 0) {
    // nothing left (p and q equal to rounding, or every candidate's mass gone): draw from p itself
    double total = 0.0;
    int mode = 0;
    const double* s = a.sums + static_cast<int64_t>(b) * 2 * a.ntile;
    for (; mode < 2; ++mode, s += a.ntile) {
      double v = 0.0;
      for (int t = lane; t < a.ntile; t += 64) v += s[t];
      total = wave_sum(v);
      if (total > 0.0) break;
    }
    int tile = -1;
    double bar = 0.0;
    if (mode < 2) {
      const double goal = static_cast<double>(a.uniforms[static_cast<int64_t>(b) * a.T]) * total;
      double run = 0.0;  // of the steps before
      for (int t0 = 0; t0 < a.ntile; t0 += 64) {
        const double v = t0 + lane < a.ntile ? s[t0 + lane] : 0.0;
        const double upto = wave_scan(v) + run;
        const uint64_t some = __ballot(v > 0.0), over = __ballot(v > 0.0 && upto > goal);
        if (some) {  // the tile that passes the goal, or the last one with any weight
          const int at = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
          tile = t0 + at;
          bar = goal - (lane_value(upto, at) - lane_value(v, at));
        }
        if (over) break;
        run = lane_value(upto, 63);
      }
    }
    if (lane == 0) {
      s_tile = tile;
      s_mode = mode;
      s_bar = bar;
    }
  }
  if (tid == 0) s_last = -1;
  __syncthreads();
  const int tile = s_tile;
  if (tile < 0) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  if (s_mode == 1) {
    l.nrej = 0;
    l.residual = false;
  }
  const void* prow = row_at<DT>(a.target, b * a.tb + l.stop * a.tt);
  const void* qrow = l.residual ? row_at<DT>(a.draft, b * a.db + l.stop * a.dt) : nullptr;
  const int x = tile * kTile + tid * 8;
  double w[8], sum = 0.0;
  if (x < a.V) {
    double p[8];
    weights8<DT>(a, prow, qrow, l, s_rej, x, w, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += w[j];
  }
  const double upto = wave_scan(sum);
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  double before = 0.0;
  for (int k = 0; k < wave; ++k) before += s_wave[k];
  // the first thread whose entries pass the bar, or the last one with any weight
  const uint64_t some = __ballot(sum > 0.0), over = __ballot(sum > 0.0 && before + upto > s_bar);
  if (lane == 0 && some)
    atomicMax(&s_last, over ? (1 << 20) - (tid + __builtin_ctzll(over)) : tid + 63 - __builtin_clzll(some));
  __syncthreads();
  const int key = s_last, who = key >= (1 << 19) ? (1 << 20) - key : key;
  if (tid == who) {
    const double bar = s_bar - (before + (upto - sum));
    double run = 0.0;
    int pick = -1;
    bool done = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!done && w[j] > 0.0) {
        run += w[j];
        pick = x + j;
        done = run > bar;
      }
    }
    a.next[b] = pick;
  }
}

// A row's tiles go to blocks so that about 1024 blocks work in all (4 per compute unit); each block repeats
// the walk, so a block takes at least one tile and as many as that leaves.
static void plan_verify(int B, int V, int* ntile, int* per) {
  const int n = (V + kTile - 1) / kTile;
  int blocks = 1024 / (B > 0 ? B : 1);
  if (blocks < 1) blocks = 1;
  *ntile = n;
  *per = n > blocks ? (n + blocks - 1) / blocks : 1;
}

template <int DT>
static void launch_verify(const VerifyArgs& a, hipStream_t s) {
  verify_sum_kernel<DT><<<dim3((a.ntile + a.per - 1) / a.per, a.B), kVerifyThreads, 0, s>>>(a);
  verify_pick_kernel<DT><<<dim3(a.B), kVerifyThreads, 0, s>>>(a);
}

}  // namespace tq

using namespace tq;

extern "C" {

int64_t tq_verify_workspace_size(int32_t B, int32_t V) {
  if (B <= 0 || V <= 0) return 0;
  int ntile, per;
  plan_verify(B, V, &ntile, &per);
  return static_cast<int64_t>(B) * (2 * static_cast<int64_t>(ntile) + kLeftWords) * 8;
}

int tq_verify_drafts(const int64_t* tokens, const void* target_probs, int32_t dtype, int64_t stb, int64_t stt,
                     const void* draft_probs, int64_t sdb, int64_t sdt, const float* uniforms, const int32_t* parents,
                     int64_t ld_parents, int32_t B, int32_t T, int32_t V, int32_t* path, int32_t* count,
                     int64_t* next_token, void* workspace, int64_t workspace_bytes, void* stream) {
  TQ_REQUIRE(B >= 0 && T >= 1 && V >= 1, "tq_verify_drafts: bad shape");
  TQ_REQUIRE(T <= kMaxNodes, "tq_verify_drafts: at most %d nodes, got %d", kMaxNodes, T);
  TQ_REQUIRE(V < (1 << 30) && B <= 65535, "tq_verify_drafts: at most 65535 sequences and fewer than 2^30 tokens");
  TQ_REQUIRE(dtype == TQ_F32 || dtype == TQ_F16 || dtype == TQ_BF16, "tq_verify_drafts: unknown dtype %d", dtype);
  TQ_REQUIRE(!(parents && draft_probs),
             "tq_verify_drafts: tokens drawn from a draft distribution form a chain; a tree holds chosen candidates");
  if (B == 0) return TQ_OK;
  TQ_REQUIRE(tokens && target_probs && uniforms && path && count && next_token, "tq_verify_drafts: null pointer");
  TQ_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 8 == 0 &&
                 workspace_bytes >= tq_verify_workspace_size(B, V),
             "tq_verify_drafts: the workspace must be 8-byte aligned and hold %lld bytes",
             (long long)tq_verify_workspace_size(B, V));
  VerifyArgs a{};
  a.tokens = tokens;
  a.target = target_probs;
  a.tb = stb;
  a.tt = stt;
  a.draft = T > 1 ? draft_probs : nullptr;
  a.db = sdb;
  a.dt = sdt;
  a.uniforms = uniforms;
  a.parents = parents;
  a.ld_parents = ld_parents;
  a.B = B;
  a.T = T;
  a.V = V;
  plan_verify(B, V, &a.ntile, &a.per);
  a.sums = static_cast<double*>(workspace);
  a.left = static_cast<int64_t*>(workspace) + static_cast<int64_t>(B) * 2 * a.ntile;
  a.path = path;
  a.count = count;
  a.next = next_token;
  if (dtype == TQ_F32) launch_verify<TQ_F32>(a, as_stream(stream));
  else if (dtype == TQ_F16) launch_verify<TQ_F16>(a, as_stream(stream));
  else launch_verify<TQ_BF16>(a, as_stream(stream));
  return launch_status("tq_verify_drafts");
}

}  // extern "C"
