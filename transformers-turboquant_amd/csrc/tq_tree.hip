// Attention of drafted tokens over a paged compressed cache.
//
// Sequence b has n_b cached positions and T drafted tokens at positions n_b + i, all of them rows
// of its pages (position j: row j % P of page block_table[b, j / P]).  The drafted tokens form a
// tree: node i's parent is parents[i] < i, or -1 (it continues the cached text).  Node i sees the
// n_b cached positions, its ancestors and itself; T = 1 is a decoding step, parents[i] = i - 1
// the causal chain.  Per (node, query head) with the prepared queries of tq_query_prep:
//   s_j = scale (vn_j <q_rot, C[codes_j]> + coeff rn_j <q_proj, 2 sign_j - 1>)
//   p   = softmax over the visible j (f32, online)
//   o   = (sum_j p_j vnv_j Cv[vcodes_j]) Pi_v
//
// The columns of a kv head are its G query heads times the T nodes, c = i G + g.  A block takes up to
// 4 (tree_plane_kernel), 16 or 32 columns (tree_attn_kernel) of one kv head against a run of keys; each
// of its waves streams slabs of 32 keys of the packed planes into its own ring in LDS.  With few
// columns the stream of packed bytes bounds the work, from 32 on the matrix products do.
//
// Lengths live on the device (a captured graph replays with other lengths), so the split of the
// keys is made there: the rounds (32 keys per wave of a block) of all sequences, one after another,
// are dealt in equal stretches to `slots` blocks per column group and kv head, as many as the device
// holds at once.  A stretch may end inside a sequence and cover several; each (block,
// sequence) part leaves its (maximum, sum, O) in a record, and the merge joins a sequence's records,
// normalises and applies Pi_v.
#include "tq_tree.h"

namespace tq {

template <int D, int BITS, int NT, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))
tree_attn_kernel(TreeArgs a) {
  constexpr int RK = 32 * NW;
  __shared__ __attribute__((aligned(16))) TreeSmem<D, BITS, NT, NW> sm;
  const int tid = threadIdx.x, ct0 = blockIdx.y * (16 * NT), hkv = blockIdx.z;
  const int n0 = tree_length(a, tid & 63);
  const TreeTables<BITS> tables(a, tid);
  const TreeSplit<RK> split(a, n0);
  if (static_cast<int>(blockIdx.x) >= split.blocks) return;  // block-uniform
  int x = split.begin(blockIdx.x);
  const int x_end = split.begin(blockIdx.x + 1);
  tables.keys(sm.luts, tid);
  tables.values(sm.luts, tid);
  // one part after the other: the rounds of this block's stretch that belong to one sequence
  while (x < x_end) {
    int b, first, nkeys;
    split.sequence_at(a, x, b, first, nkeys);
    const int rec = static_cast<int>(blockIdx.x) + b, last = min(x_end, first + split.rounds(nkeys));
    const TreePart part{b, b, a.C, ct0, nkeys - a.T, (x - first) * RK, min(nkeys, (last - first) * RK),
                        (static_cast<int64_t>(rec) * a.Hkv + hkv) * a.C + ct0};
    x = last;
    tree_part<D, BITS, NT, NW, false>(a, part, hkv, sm);
  }
}

// ---------------------------------------------------------------- attention, scores from bit planes
// At most 4 columns (a decoding step of up to 4 query heads per kv head) and 1- or 2-bit key codes:
// both terms of a score are sums of query values over the set bits of the packed row, taken exactly
// from the integer matrix product (PlaneQuery: query values as base-256 digits in the rows, masked
// packed words as the columns, no lookups).  Keys stand on the N side, so that a lane has its own key
// against column lg: one exponential per (column, key) instead of one per key and column of a
// 16-wide tile.  P reaches the operand of O^T += V^T P^T through a small LDS tile of the wave; column n
// of O^T serves column n mod 4.
// 16 sequences of 8k to 32k, 32/8 heads, 3 bits, 267 MB: 75 us under a kernel trace, 3.5 TB/s (a copy reaches
// 4.9); a call in a row of calls takes 80 us with preparation and merge (6 us each in their trace), which leaves it
// 68 us, 3.9 TB/s.  Of 151k cycles the VALU issues in 76k and the LDS in 71k, 27k of them conflicts of the 64-entry
// value table.  Two waves per SIMD: at three or four, registers spill in the set-up (77 against 75 and 84 us in
// all, one sequence of 32k 24 against 29 and 41).
template <int D, int KB, int NW>
struct TreePlaneSmem {
  using L = SmallLuts<KB + 1>;
  using PQ = PlaneQuery<KB, 1, D>;
  static constexpr int R = D == 64 ? 3 : 2;  // slabs of a wave in flight
  using ST = TreeStream<D, KB, KB + 1, R>;
  static constexpr int NC = PQ::NC, LDM = D + 4;
  // slot r of the waves stands at r * STRIDE; the last NSTG slots first serve the queries' set-up
  static constexpr int STRIDE = NW * ST::SLOT;
  static constexpr int NSTG = (PQ::STAGE_BYTES + STRIDE - 1) / STRIDE;
  static_assert(NSTG < R, "a slot flies during the set-up");
  static constexpr int RING = R * STRIDE;
  static constexpr int MERGE = NW * NC * LDM * 4;
  static constexpr int AREA = RING > MERGE ? RING : MERGE;
  uint8_t luts[(L::BYTES + 15) / 16 * 16];
  __attribute__((aligned(16))) uint8_t area[AREA];
  __attribute__((aligned(16))) _Float16 p[NW][NC][32];  // P of a slab [column][key]
  uint64_t anc[64];
};

template <int D, int KB, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))
tree_plane_kernel(TreeArgs a) {
  using SM = TreePlaneSmem<D, KB, NW>;
  using L = typename SM::L;
  using PQ = typename SM::PQ;
  using ST = typename SM::ST;
  constexpr int BITS = KB + 1, VB = BITS, R = SM::R, NC = SM::NC, STRIDE = SM::STRIDE;
  constexpr int DB = D / 16, NPAIR = D / 32;
  constexpr int KLANE = ST::KC / 4, SLANE = ST::SC / 4, VFB = DB * VB, VW32 = VB == 3 ? 2 : 1;
  constexpr int NK = ST::NK, RK = NW * NK;
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr float TAU = kTau, PUP = kPup;

  __shared__ __attribute__((aligned(16))) SM sm;
  const uint8_t* const tV = sm.luts + L::VAL_OFF;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int hkv = blockIdx.z;
  const int n0 = tree_length(a, lane);
  const TreeTables<BITS> tables(a, tid);
  const TreeSplit<RK> split(a, n0);
  if (static_cast<int>(blockIdx.x) >= split.blocks) return;  // block-uniform
  int x = split.begin(blockIdx.x);
  const int x_end = split.begin(blockIdx.x + 1);

  DecodeArgs qa{};
  qa.q_rot = a.q_rot;
  qa.q_proj = a.q_proj;
  qa.kcent = a.kcent;
  qa.Hq = a.Hq;
  qa.Sq = a.T;
  qa.G = a.G;
  qa.C = a.C;
  tables.values(sm.luts, tid);
  const float fa = a.scale * LOG2E;
  const int vbit = l16 * VFB, vbase = (vbit >> 5) * 4, vshift = vbit & 31;
  uint8_t* const mine = sm.area + wave * ST::SLOT;
  const uint32_t mine_lds = lds_offset(mine);
  _Float16* const pt = &sm.p[wave][0][0];

  while (x < x_end) {
    int b, first, nkeys;
    split.sequence_at(a, x, b, first, nkeys);
    const int rec = static_cast<int>(blockIdx.x) + b;
    const int nctx = nkeys - a.T, last = min(x_end, first + split.rounds(nkeys));
    const int kbeg = (x - first) * RK, kend = min(nkeys, (last - first) * RK);
    x = last;

    // parents, the first slabs' pages and the queries come in one round trip
    const int par = tree_parent(a, b);
    const ST stream(a, b, hkv, kend);
    const int k0w = kbeg + wave * NK;
    int nrows[R], pages[R];
#pragma unroll
    for (int r = 0; r < R; ++r) pages[r] = k0w + r * RK < kend ? stream.page_of(k0w + r * RK) : -1;
    const uint64_t anc_lane = tree_ancestors(a, par);
    if (wave == 0) sm.anc[lane] = anc_lane;
    const uint64_t live = __ballot(anc_lane != 0);
    __syncthreads();  // tables and ancestors in place; the previous part is done with the LDS
    auto start = [&](int r) { nrows[r] = k0w + r * RK < kend ? stream.issue(k0w + r * RK, pages[r], mine_lds + r * STRIDE) : 0; };
#pragma unroll
    for (int r = 0; r < R - SM::NSTG; ++r) start(r);
    PQ pq;
    pq.setup(qa, b, hkv, sm.area + (R - SM::NSTG) * STRIDE, tid);
    __syncthreads();  // fragments held: the staging slots join the ring
#pragma unroll
    for (int r = R - SM::NSTG; r < R; ++r) start(r);
    const uint64_t anc = sm.anc[min(lg, a.C - 1) / a.G];  // of column lg

    // column state as in tree_attn_kernel, the same in the 16 lanes of a column
    float mref = 0.f, lim = -INFINITY, l_run = 0.f;
    float4v oacc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) oacc[db] = float4v{0.f, 0.f, 0.f, 0.f};

    auto slab = [&](auto edge_c, const uint8_t* src, int ks0, int rows) {
      constexpr bool EDGE = decltype(edge_c)::value;
      auto visible = [&](uint64_t tokens) { return tree_visible(tokens, nctx - ks0, rows) >> l16; };
      // ---- scores of keys ks0 + 16j + l16 for column lg
      float t1[2][1], t2[2][1];
      pq.dots2(src + ST::OFF_K + l16 * ST::KC + lg * KLANE, src + ST::OFF_S + l16 * ST::SC + lg * SLANE,
               src + ST::OFF_K + (16 + l16) * ST::KC + lg * KLANE, src + ST::OFF_S + (16 + l16) * ST::SC + lg * SLANE, t1, t2);
      uint32_t kn[2], rn[2], vn[2];  // norms, f16 in the low half
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint8_t* const nr = src + ST::OFF_N + (16 * j + l16) * 4;
        kn[j] = *reinterpret_cast<const uint32_t*>(nr);
        rn[j] = *reinterpret_cast<const uint32_t*>(nr + ST::NRM);
        vn[j] = *reinterpret_cast<const uint32_t*>(nr + 2 * ST::NRM);
      }
      if constexpr (EDGE) {  // keys that nobody sees weigh nothing, whatever their rows hold
        const uint32_t any = visible(live);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool on = any & (1u << (16 * j));
          kn[j] = on ? kn[j] : 0;
          rn[j] = on ? rn[j] : 0;
          vn[j] = on ? vn[j] : 0;
        }
      }
      // ---- log2-domain scores relative to mref, and the softmax step
      float sc[2];
      uint32_t see = 0;
      if constexpr (EDGE) see = visible(anc);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float s = fmaf(fma_f16(t1[j][0], kn[j], mul_f16(t2[j][0] * a.coeff, rn[j])), fa, -mref);
        sc[j] = !EDGE || (see & (1u << (16 * j))) ? s : -INFINITY;
      }
      const float lmax = max_raw(sc[0] + norm_exponent(vn[0]), sc[1] + norm_exponent(vn[1]));
      if (__any(lmax > lim)) {
        float m = lmax;
#pragma unroll
        for (int sh = 8; sh >= 1; sh >>= 1) m = fmaxf(m, __shfl_xor(m, sh, 64));
        const bool move = m > lim;
        const float shift = move ? m - PUP : 0.f;
        const float alpha = !move ? 1.f : lim == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-shift);
        sc[0] -= shift;
        sc[1] -= shift;
        mref += shift;
        lim = move ? TAU + PUP : lim;
        l_run *= alpha;
        const float ac = __shfl(alpha, 16 * (l16 & 3), 64);  // column l16 & 3 of O^T belongs to that lane group
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[db] *= ac;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float p = __builtin_amdgcn_exp2f(sc[j]);
        l_run += p;
        uint32_t v = vn[j];
        if constexpr (EDGE) v = sc[j] == -INFINITY ? 0 : v;  // a masked key's norm may be anything
        pt[lg * NK + 16 * j + l16] = static_cast<_Float16>(mul_f16(p, v));
      }
      // ---- O^T += V^T (P vn)^T, as in tree_attn_kernel; the 8 row reads go out as one batch
      uint32_t r0[2][4], r1[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint32_t* vp = reinterpret_cast<const uint32_t*>(src + ST::OFF_V + (16 * j + 4 * lg + kk) * ST::VC + vbase);
          r0[j][kk] = vp[0];
          if constexpr (VW32 == 2) r1[j][kk] = vp[1];
        }
      const _Float16* const pr = pt + (l16 & (NC - 1)) * NK + 4 * lg;
      const u32x2 p0 = *reinterpret_cast<const u32x2*>(pr);
      const u32x2 p1 = *reinterpret_cast<const u32x2*>(pr + 16);
      const half8 pb = __builtin_bit_cast(half8, u32x4{p0[0], p0[1], p1[0], p1[1]});
      __builtin_amdgcn_sched_barrier(0);
      constexpr uint32_t M = odd_fields<VB>();
      uint32_t w[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          if constexpr (VW32 == 2) w[j][kk] = __builtin_amdgcn_alignbit(r1[j][kk], r0[j][kk], vshift);
          else w[j][kk] = r0[j][kk] >> vshift;
        }
#pragma unroll
      for (int par = 0; par < 2; ++par) {
        uint32_t f[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t wa = w[j][2 * c], wb = w[j][2 * c + 1];
            f[j][c] = par ? bfi32(M, wb, wa >> VB) : bfi32(M, wb << VB, wa);
          }
        auto look = [&](auto ic) {  // a group is looked up while the one before it is multiplied
          constexpr int i = decltype(ic)::value;
          return __builtin_bit_cast(half8, u32x4{value_pair<VB, i>(tV, f[0][0]), value_pair<VB, i>(tV, f[0][1]),
                                                 value_pair<VB, i>(tV, f[1][0]), value_pair<VB, i>(tV, f[1][1])});
        };
        half8 va = look(std::integral_constant<int, 0>{});
        static_for<NPAIR>([&](auto ic) {
          constexpr int i = decltype(ic)::value;
          half8 next = va;
          if constexpr (i + 1 < NPAIR) next = look(std::integral_constant<int, i + 1>{});
          __builtin_amdgcn_sched_barrier(0);
          oacc[2 * i + par] = mfma16x16x32(va, pb, oacc[2 * i + par]);
          va = next;
        });
      }
    };

    int slot = 0, ks0 = k0w;
    auto slabs = [&](auto edge_c, int end) {
      stream.template run<RK, STRIDE>(ks0, end, nrows, slot, mine_lds,
                              [&](int at, int k0, int rows) { slab(edge_c, mine + at * STRIDE, k0, rows); });
    };
    slabs(std::false_type{}, min(kend, nctx) - (NK - 1));
    slabs(std::true_type{}, kend);

    // ---- the waves' states joined in LDS (the rings are done)
    constexpr int LDM = SM::LDM;
    float* const mrg = reinterpret_cast<float*>(sm.area);  // [wave][column][LDM]
    __syncthreads();
    if (l16 < NC) {
      float* const my = mrg + (wave * NC + l16) * LDM;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int db = 0; db < DB; db += 4)
          *reinterpret_cast<float4v*>(my + (lg * 4 + e) * DB + db) =
              float4v{oacc[db][e], oacc[db + 1][e], oacc[db + 2][e], oacc[db + 3][e]};
    }
    float l = l_run;
#pragma unroll
    for (int sh = 8; sh >= 1; sh >>= 1) l += __shfl_xor(l, sh, 64);
    if (l16 == 0) {
      float* const my = mrg + (wave * NC + lg) * LDM;
      my[D] = !anc || (lim == -INFINITY && l == l) ? -INFINITY : mref;
      my[D + 1] = l;
    }
    __syncthreads();
    tree_join<D, NW, NC>(a, mrg, (static_cast<int64_t>(rec) * a.Hkv + hkv) * a.C, a.C, tid);
  }
}

// ---------------------------------------------------------------- merge
// One block per (sequence, kv head, 4 CW columns): wave w joins columns w, w + 4, ... (the records'
// maxima and weights one per lane, then D / 64 dims per lane summed over the records, 16 / CW of them in
// flight per column), then out^T = Pi_v^T o^T on MFMA with both operands split into f16 hi + lo.
// Latency of three dependent round trips (lengths, records, output) bounds it: 4 to 8 us for a few
// records a column, 14 us for 8192 columns of 20 records (85 MB).  CW = 1 has the fewest of
// them in a row, CW = 4 reads Pi_v (64 KB) a quarter as often.
template <int D, int RK, int CW>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeArgs a) {
  using Finish = TreeFinish<D, CW>;
  using floatPL = typename Finish::floatPL;
  constexpr int PL = Finish::PL, NC = Finish::NC, NB = 16 / CW;
  __shared__ typename Finish::Smem sm;
  const int c0 = blockIdx.x * NC, hkv = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;

  const int n0 = tree_length(a, lane);  // before Pi_v: waited for first
  const Finish finish(a);
  const TreeSplit<RK> split(a, n0);
  int first = 0, n = 0;
  split.rounds_of(a, b, first, n);
  if (n > 0) {  // records k + b of the blocks k that hold the sequence's rounds
    const int k0 = split.block_of(first), k1 = split.block_of(first + n - 1);
    first = k0 + b;
    n = k1 - k0 + 1;
  }
  const int64_t step = static_cast<int64_t>(a.Hkv) * a.C;  // columns between records
  // one memory round trip for the first NB records of all the wave's columns: partial O, and a record's
  // maximum and sum per lane
  floatPL v0[CW][NB];
  float m0[CW], l0[CW];
#pragma unroll
  for (int k = 0; k < CW; ++k) {
    const int64_t at = (static_cast<int64_t>(first) * a.Hkv + hkv) * a.C + min(c0 + wave + 4 * k, a.C - 1);
#pragma unroll
    for (int q = 0; q < NB; ++q)
      v0[k][q] = q < n ? *reinterpret_cast<const floatPL*>(a.part_o + (at + q * step) * D + PL * lane) : floatPL{};
    m0[k] = lane < n ? a.part_ml[(at + lane * step) * 2] : -INFINITY;
    l0[k] = lane < n ? a.part_ml[(at + lane * step) * 2 + 1] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < CW; ++k) {
    const int cc = wave + 4 * k, c = c0 + cc;
    floatPL o = floatPL{};
    if (c < a.C) {
      const int64_t at = (static_cast<int64_t>(first) * a.Hkv + hkv) * a.C + c;
      const float* ml = a.part_ml + at * 2;
      const float* src = a.part_o + at * D + PL * lane;
      float mx = m0[k];
      for (int r = lane + 64; r < n; r += 64) mx = fmaxf(mx, ml[r * step * 2]);
#pragma unroll
      for (int sh = 32; sh >= 1; sh >>= 1) mx = fmaxf(mx, __shfl_xor(mx, sh, 64));
      float lsum = 0.f;
      for (int r0 = 0; r0 < n; r0 += 64) {
        float w = 0.f;
        if (r0 + lane < n) {
          const float m = r0 == 0 ? m0[k] : ml[(r0 + lane) * step * 2];
          if (m != -INFINITY) {
            w = __builtin_amdgcn_exp2f(m - mx);
            lsum += w * (r0 == 0 ? l0[k] : ml[(r0 + lane) * step * 2 + 1]);
          }
        }
        auto add = [&](const floatPL (&v)[NB], int u) {
#pragma unroll
          for (int q = 0; q < NB; ++q) {
            const float ww = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), u + q));
#pragma unroll
            for (int e = 0; e < PL; ++e) o[e] = fmaf(ww, v[q][e], o[e]);
          }
        };
        if (r0 == 0) add(v0[k], 0);
        const int nb = min(64, n - r0);
        for (int u = r0 == 0 ? NB : 0; u < nb; u += NB) {
          floatPL v[NB];
#pragma unroll
          for (int q = 0; q < NB; ++q)
            v[q] = u + q < nb ? *reinterpret_cast<const floatPL*>(src + (r0 + u + q) * step * D) : floatPL{};
          add(v, u);
        }
      }
#pragma unroll
      for (int sh = 32; sh >= 1; sh >>= 1) lsum += __shfl_xor(lsum, sh, 64);
      const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
      o *= inv;
    }
    Finish::put(sm, cc, o);
  }
  __syncthreads();
  finish.store(a, sm, b, hkv, c0);
}

// ---------------------------------------------------------------- launch
struct TreePlan {
  void (*kernel)(TreeArgs);
  int ncol;  // blocks along the columns
  int lg_least;
  int slots;
  int64_t bytes;
};

// What attends: scores from bit planes, or operands from tables for one or two tiles of 16 columns a block.
enum TreeKind { kPlanes, kOneTile, kTwoTiles };

using TreeKernel = void (*)(TreeArgs);
template <int D, int BITS>
static TreeKernel tree_kernel(TreeKind kind) {
  if constexpr (BITS <= 3) {
    if (kind == kPlanes) return &tree_plane_kernel<D, BITS - 1, 4>;
  }
  return kind == kOneTile ? &tree_attn_kernel<D, BITS, 1, 4> : &tree_attn_kernel<D, BITS, 2, 4>;
}
static TreeKernel tree_kernel(int d, int bits, TreeKind kind) {
  if (d == 64) return bits == 2 ? tree_kernel<64, 2>(kind) : bits == 3 ? tree_kernel<64, 3>(kind) : tree_kernel<64, 4>(kind);
  return bits == 2 ? tree_kernel<128, 2>(kind) : bits == 3 ? tree_kernel<128, 3>(kind) : tree_kernel<128, 4>(kind);
}

static TreePlan plan_tree(int B, int Hq, int Hkv, int T, int64_t maxpos, int d, int bits) {
  static int resident[2][3][3][16] = {};  // per kernel, per device
  const auto resident_of = [&](TreeKind kind) {
    return resident_blocks(reinterpret_cast<const void*>(tree_kernel(d, bits, kind)), 256, resident[d == 128][bits - 2][kind]);
  };
  TreePlan p{};
  const int C = Hq / Hkv * T;
  const int64_t most = static_cast<int64_t>(B) * ((maxpos + 127) / 128);  // rounds, at most
  // (Times below: attention and merge over prepared queries, calls in a row.)
  // Bit planes up to 4 columns: 16 x 32k, 32/8 heads 75.5 against 90 us with tables (2 bits 57 and 81, one
  // sequence of 4k 15.6 and 14.7); with two groups of 4 they lose (16/2 heads 41.8 and 37.2).
  // Two tiles share a slab's operands: 16 nodes of 16 x 32k 218 against 298 us.  While there are
  // few rounds to each resident block, the set-up of the queries and the records weigh more, and one tile is
  // faster: 16 nodes, one sequence of 4k 19.8 against 23.0 us, of 16k (4 rounds) 31.0 and 32.8.
  TreeKind kind = kTwoTiles;
  if (bits <= 3 && C <= 4) kind = kPlanes;
  else if (C <= 16 || most * Hkv * ((C + 31) / 32) <= 4 * static_cast<int64_t>(resident_of(kTwoTiles))) kind = kOneTile;
  p.kernel = tree_kernel(d, bits, kind);
  const int width = kind == kTwoTiles ? 32 : 16;
  p.ncol = (C + width - 1) / width;
  // One round is over soon and leaves a record for the merge.  With two tiles records are large and
  // two rounds to a stretch pay (64 columns, 4k keys: 22.9 against 25.3 us); else more blocks
  // do (planes, 1k keys: 12.1 against 12.8 us).
  p.lg_least = kind == kTwoTiles ? 1 : 0;
  const int res = resident_of(kind);
  p.slots = res / (Hkv * p.ncol);  // one round of resident blocks
  if (p.slots < 1) p.slots = 1;
  // With up to two rounds to each, half of them (a block to a compute unit, not two) leave half the set-ups
  // and records: 16 nodes, one sequence of 2k 14.7 against 16.8 us, of 4k 18.1 and 18.8; of 8k (four rounds)
  // 23.4 and 23.0.
  if (p.slots > 1 && most <= 2 * static_cast<int64_t>(p.slots)) p.slots /= 2;
  if (p.slots > most) p.slots = static_cast<int>(most);
  const int64_t nrec = static_cast<int64_t>(p.slots) + B;
  p.bytes = nrec * Hkv * C * static_cast<int64_t>(d + 2) * 4;
  return p;
}

static bool tree_shape(int B, int Hq, int Hkv, int T, int64_t maxpos, int d, int bits) {
  return B >= 1 && B <= 65535 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hkv <= 65535 && T >= 1 && T <= 64 && maxpos >= T &&
         maxpos <= (int64_t(1) << 24) && (d == 64 || d == 128) && bits >= 2 && bits <= 4 &&
         static_cast<int64_t>(B) * ((maxpos + 127) / 128) < (int64_t(1) << 31);
}

template <int D>
static void launch_tree(const TreeArgs& a, const TreePlan& p, hipStream_t s) {
  p.kernel<<<dim3(p.slots, p.ncol, a.Hkv), 256, 0, s>>>(a);
  // the widest blocks that still are two to a compute unit (16 columns) or one (8): 3904 columns of few
  // records 56 us in all with 8, 61 with 4, 57 with 16; 8192 columns of 20 records 215 with 16, 219 with 8
  const auto blocks = [&](int columns) { return static_cast<int64_t>((a.C + columns - 1) / columns) * a.Hkv * a.B; };
  const auto grid = [&](int columns) { return dim3((a.C + columns - 1) / columns, a.Hkv, a.B); };
  if (blocks(16) >= 512) tree_merge_kernel<D, 128, 4><<<grid(16), 256, 0, s>>>(a);
  else if (blocks(8) >= 256) tree_merge_kernel<D, 128, 2><<<grid(8), 256, 0, s>>>(a);
  else tree_merge_kernel<D, 128, 1><<<grid(4), 256, 0, s>>>(a);
}

int64_t tree_workspace(int B, int Hq, int Hkv, int T, int64_t maxpos, int d, int bits) {
  return plan_tree(B, Hq, Hkv, T, maxpos, d, bits).bytes;
}

void tree_attend(TreeArgs a, int d, int bits, void* workspace, hipStream_t s) {
  const TreePlan p = plan_tree(a.B, a.Hq, a.Hkv, a.T, a.maxpos, d, bits);
  a.slots = p.slots;
  a.lg_least = p.lg_least;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + (static_cast<int64_t>(p.slots) + a.B) * a.Hkv * a.C * d;
  if (d == 64) launch_tree<64>(a, p, s);
  else launch_tree<128>(a, p, s);
}

}  // namespace tq

using namespace tq;

extern "C" {

int64_t tq_tree_workspace_size(int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t table_width, int32_t page_size,
                               int32_t d, int32_t bits) {
  const int64_t maxpos = static_cast<int64_t>(table_width) * page_size;
  return tree_shape(B, Hq, Hkv, T, maxpos, d, bits) ? tree_workspace(B, Hq, Hkv, T, maxpos, d, bits) : 0;
}

int tq_tree_attention(const uint16_t* q_rot, const float* q_proj, const uint8_t* key_codes, const uint8_t* key_signs,
                      const uint16_t* key_rn, const uint16_t* key_vn, const uint16_t* key_centroids_f16, int32_t bits,
                      const uint8_t* val_codes, const uint16_t* val_vn, const float* val_centroids,
                      const uint16_t* val_pit_split, int64_t num_pages, int32_t page_size, const int32_t* block_table,
                      int64_t ld_table, int32_t table_width, const int32_t* lengths, const int32_t* parents,
                      int64_t ld_parents, int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t d, float coeff,
                      float scale, void* out, int32_t out_dtype, int64_t sob, int64_t soh, int64_t sos,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  if (d != 64 && d != 128) {
    set_error("tq_tree_attention: head_dim %d not supported (64 or 128)", d);
    return TQ_EUNSUPPORTED;
  }
  if (bits < 2 || bits > 4) {
    set_error("tq_tree_attention: bits %d not supported (2 to 4)", bits);
    return TQ_EUNSUPPORTED;
  }
  TQ_REQUIRE(B >= 0 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && T >= 1, "tq_tree_attention: bad shape");
  TQ_REQUIRE(T <= 64, "tq_tree_attention: at most 64 drafted tokens, got %d", T);
  TQ_REQUIRE(page_size >= 32 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0,
             "tq_tree_attention: page_size must be a power of two from 32 to 2^20, got %d", page_size);
  TQ_REQUIRE(num_pages >= 1 && num_pages < (int64_t(1) << 31) && ld_table >= table_width, "tq_tree_attention: bad pool");
  const int64_t maxpos = static_cast<int64_t>(table_width) * page_size;
  TQ_REQUIRE(maxpos >= T, "tq_tree_attention: a table of %d pages of %d does not hold %d drafted tokens", table_width, page_size, T);
  TQ_REQUIRE(out_dtype == TQ_F32 || out_dtype == TQ_F16 || out_dtype == TQ_BF16, "tq_tree_attention: unknown dtype %d", out_dtype);
  if (B == 0) return TQ_OK;
  TQ_REQUIRE(tree_shape(B, Hq, Hkv, T, maxpos, d, bits),
             "tq_tree_attention: at most 65535 sequences and kv heads, 2^24 positions a sequence, got %d, %d and %lld", B,
             Hkv, (long long)maxpos);
  TQ_REQUIRE(q_rot && q_proj && key_codes && key_signs && key_rn && key_vn && key_centroids_f16 && val_codes && val_vn &&
                 val_centroids && val_pit_split && block_table && lengths && out,
             "tq_tree_attention: null pointer");
  for (const void* p : {static_cast<const void*>(q_rot), static_cast<const void*>(q_proj), static_cast<const void*>(key_codes),
                        static_cast<const void*>(key_signs), static_cast<const void*>(val_codes), static_cast<const void*>(val_pit_split)})
    TQ_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "tq_tree_attention: queries, code planes and Pi_v must be 16-byte aligned");
  const int64_t bytes = tree_workspace(B, Hq, Hkv, T, maxpos, d, bits);
  TQ_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= bytes,
             "tq_tree_attention: the workspace must be 16-byte aligned and hold %lld bytes", (long long)bytes);
  TreeArgs a{};
  a.q_rot = q_rot;
  a.q_proj = q_proj;
  a.kcodes = key_codes;
  a.ksigns = key_signs;
  a.krn = key_rn;
  a.kvn = key_vn;
  a.kcent = key_centroids_f16;
  a.vcodes = val_codes;
  a.vvn = val_vn;
  a.vcent = val_centroids;
  a.table = block_table;
  a.ld_table = ld_table;
  a.lengths = lengths;
  a.parents = parents;
  a.ld_parents = ld_parents;
  a.num_pages = num_pages;
  a.lg_page = __builtin_ctz(static_cast<unsigned>(page_size));
  a.maxpos = static_cast<int>(maxpos);
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.T = T;
  a.G = Hq / Hkv;
  a.C = a.G * T;
  a.coeff = coeff;
  a.scale = scale;
  a.vpit = val_pit_split;
  a.out = out;
  a.out_dtype = out_dtype;
  a.sob = sob;
  a.soh = soh;
  a.sos = sos;
  tree_attend(a, d, bits, workspace, as_stream(stream));
  return launch_status("tq_tree_attention");
}

}  // extern "C"
