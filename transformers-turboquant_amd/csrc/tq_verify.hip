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
// (two for a chain), so the work is latency and one pass over that row: the row is cut into chunks
// summed by a block each (every block repeats the walk: cheaper than a launch that only walks),
// then one block per sequence finds the chunk and searches it.  Probabilities and sums are
// float64: the token is decided by a comparison of sums over up to ~10^5 terms, and in float32
// their rounding would move the border of a few tokens in a hundred thousand by more than the
// token's own probability.
#include "tq_common.h"

namespace tq {

constexpr int kVerifyThreads = 256;
constexpr int kMaxNodes = 64;  // a node is a lane

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
  int chunk, nchunk;      // vocabulary entries per block, chunks per row
  double* sums;           // [B, nchunk, 2]: of w, of p
  int32_t* path;          // [B, T]
  int32_t* count;         // [B]
  int64_t* next;          // [B]
};

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
      // a candidate that repeats an earlier sibling has nothing left to accept
      bool again = false;
      for (int j = 0; j < a.T; ++j) {
        const int pj = __shfl(par, j, 64);
        const int64_t tj = __shfl(tok, j, 64);
        again = again || (j < i && pj == par && tj == tok);
      }
      if (again) p = 0.0;
      double rem = 1.0;
      for (int j = 0; j < a.T; ++j) {
        const int pj = __shfl(par, j, 64);
        const double qj = __shfl(p, j, 64);
        if (j < i && pj == par) rem -= qj;
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

template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) verify_sum_kernel(VerifyArgs a) {
  __shared__ int64_t s_rej[kMaxNodes];
  __shared__ int s_left[3];
  __shared__ double s_part[2][kVerifyThreads / 64];
  const int b = blockIdx.y, c = blockIdx.x, tid = threadIdx.x;
  const Left l = walk<DT>(a, b, s_rej, s_left, c == 0);
  const void* prow = row_at<DT>(a.target, b * a.tb + l.stop * a.tt);
  const void* qrow = l.residual ? row_at<DT>(a.draft, b * a.db + l.stop * a.dt) : nullptr;
  const int end = min(a.V, (c + 1) * a.chunk);
  double sw = 0.0, sp = 0.0;
  for (int x = c * a.chunk + tid * 8; x < end; x += kVerifyThreads * 8) {
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
    s_part[0][tid >> 6] = sw;
    s_part[1][tid >> 6] = sp;
  }
  __syncthreads();
  if (tid < 2) {
    double t = 0.0;
#pragma unroll
    for (int k = 0; k < kVerifyThreads / 64; ++k) t += s_part[tid][k];
    a.sums[(static_cast<int64_t>(b) * a.nchunk + c) * 2 + tid] = t;
  }
}

template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) verify_pick_kernel(VerifyArgs a) {
  __shared__ int64_t s_rej[kMaxNodes];
  __shared__ int s_left[3];
  __shared__ double s_sum[kVerifyThreads];
  __shared__ double s_before;
  __shared__ int s_chunk, s_last, s_mode;
  const int b = blockIdx.x, tid = threadIdx.x;
  Left l = walk<DT>(a, b, s_rej, s_left, false);
  const double u = static_cast<double>(a.uniforms[static_cast<int64_t>(b) * a.T]);
  if (tid == 0) {
    const double* s = a.sums + static_cast<int64_t>(b) * a.nchunk * 2;
    // nothing left (p and q equal to rounding, or every candidate's mass gone): draw from p itself
    int which = 0;
    double total = 0.0;
    for (; which < 2; ++which) {
      total = 0.0;
      for (int c = 0; c < a.nchunk; ++c) total += s[2 * c + which];
      if (total > 0.0) break;
    }
    s_mode = which;
    s_chunk = -1;
    if (which < 2) {
      double run = 0.0;
      int last = 0;
      double last_run = 0.0;
      const double bar = u * total;
      for (int c = 0; c < a.nchunk; ++c) {
        const double v = s[2 * c + which];
        if (v > 0.0) {
          last = c;
          last_run = run;
          if (run + v > bar) break;
        }
        run += v;
      }
      s_chunk = last;
      s_before = bar - last_run;  // what the chunk's own running sum has to exceed
    }
  }
  __syncthreads();
  if (s_chunk < 0) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  if (s_mode == 1) {
    l.nrej = 0;
    l.residual = false;
  }
  const void* prow = row_at<DT>(a.target, b * a.tb + l.stop * a.tt);
  const void* qrow = l.residual ? row_at<DT>(a.draft, b * a.db + l.stop * a.dt) : nullptr;
  const int beg = s_chunk * a.chunk, end = min(a.V, beg + a.chunk);
  // each thread sums a run of `per` entries, one thread then searches the runs and its own entries
  const int per = ((end - beg + kVerifyThreads - 1) / kVerifyThreads + 7) / 8 * 8;
  const int mine = beg + tid * per, stop = min(end, mine + per);
  double sum = 0.0;
  for (int x = mine; x < stop; x += 8) {
    double w[8], p[8];
    weights8<DT>(a, prow, qrow, l, s_rej, x, w, p);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (x + j < stop) sum += w[j];
  }
  s_sum[tid] = sum;
  __syncthreads();
  if (tid == 0) {
    double run = 0.0, at = 0.0;
    int who = -1;
    for (int t = 0; t < kVerifyThreads; ++t) {
      if (s_sum[t] > 0.0) {
        who = t;
        at = run;
        if (run + s_sum[t] > s_before) break;
      }
      run += s_sum[t];
    }
    s_last = who;
    s_before -= at;
  }
  __syncthreads();
  if (tid == s_last) {
    double run = 0.0;
    int64_t pick = -1;
    bool done = false;
    for (int x = mine; x < stop && !done; x += 8) {
      double w[8], p[8];
      weights8<DT>(a, prow, qrow, l, s_rej, x, w, p);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!done && x + j < stop && w[j] > 0.0) {
          run += w[j];
          pick = x + j;
          done = run > s_before;
        }
      }
    }
    a.next[b] = pick;
  }
}

// chunks of a row: about 512 blocks in all, of at least 2048 entries (8 per thread)
static void plan_verify(int B, int V, int* chunk, int* nchunk) {
  int n = 512 / (B > 0 ? B : 1);
  if (n > 64) n = 64;
  if (n < 1) n = 1;
  int c = (V + n - 1) / n;
  if (c < 2048) c = 2048;
  c = (c + 7) / 8 * 8;
  *chunk = c;
  *nchunk = (V + c - 1) / c;
}

template <int DT>
static void launch_verify(const VerifyArgs& a, hipStream_t s) {
  verify_sum_kernel<DT><<<dim3(a.nchunk, a.B), kVerifyThreads, 0, s>>>(a);
  verify_pick_kernel<DT><<<dim3(a.B), kVerifyThreads, 0, s>>>(a);
}

}  // namespace tq

using namespace tq;

extern "C" {

int64_t tq_verify_workspace_size(int32_t B, int32_t V) {
  if (B <= 0 || V <= 0) return 0;
  int chunk, nchunk;
  plan_verify(B, V, &chunk, &nchunk);
  return static_cast<int64_t>(B) * nchunk * 2 * 8;
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
  plan_verify(B, V, &a.chunk, &a.nchunk);
  a.sums = static_cast<double*>(workspace);
  a.path = path;
  a.count = count;
  a.next = next_token;
  if (dtype == TQ_F32) launch_verify<TQ_F32>(a, as_stream(stream));
  else if (dtype == TQ_F16) launch_verify<TQ_F16>(a, as_stream(stream));
  else launch_verify<TQ_BF16>(a, as_stream(stream));
  return launch_status("tq_verify_drafts");
}

}  // extern "C"
