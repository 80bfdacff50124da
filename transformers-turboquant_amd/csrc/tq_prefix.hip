// Attention of sequences that share a long prefix, over a paged compressed cache.
//
// As tree attention (tq_tree.hip), of B sequences with T drafted tokens each; but consecutive sequences may
// have the same rows at their first positions: groups[b] = (id, shared), and sequences in a row with the same id and
// the same shared have positions [0, shared) in common.  The softmax over a sequence's keys is that over its parts,
// joined by their maxima and sums:
//   m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m), O = O1 2^(m1 - m) + O2 2^(m2 - m),
// so the shared rows are read and decoded for 16 or 32 columns of the group at a time (it has rows x T x G of a kv head;
// another tile of them decodes them again), and each sequence's own rows for its T x G.
//
// The work is a list of segments: a group's shared keys against a tile of 16 NTP of its columns, a
// sequence's own keys against a tile of 16 NTO of its own.  As in tree attention their rounds (32 keys per wave of
// a block) are dealt in stretches to as many blocks per kv head as the device holds at once, from the
// lengths and groups that stand on the device; each (block, segment) part leaves a record, and the merge joins those
// of the sequence's own segment and of the group's.  The stretches are equal in time, not in rounds: a round weighs
// what it takes, and a segment has a weight in front of its rounds for what a part takes besides them.
#include "tq_tree.h"

namespace tq {

struct PrefixArgs : TreeArgs {
  int older;              // blocks of a kv head that come first on their compute unit, of two (0: more or fewer fit)
};

// A group ends with a lane's step of 64 sequences (behind it the same group begins anew): every sequence is in one
// group, whatever the entries are, and what a lane has to know of a group stands in its own wave.
// The shared positions that are read together: whole slabs.  The rest of them is read with the own ones,
// through each sequence's own table row.
constexpr int kSlab = 32;

// Segments and rounds, dealt to the blocks as by TreeSplit: one sequence per lane, 64 per step.
// A sequence's segments are those of the group it is the first of (pt tiles of pr rounds), then its
// own (ot tiles of rounds(keys - start)).  The parts of block k in segment s have record k + s: walking
// along the rounds, every step to the next part moves to the next block, to a later segment or both.
//
// Positions on the way along all segments count units of about 2000 cycles: kPart for a part (queries, first
// slabs, join of the waves: 8 to 10 thousand cycles, as long as 2 rounds), then its rounds of 2 (one tile of columns, 4100
// cycles) or 3 (two tiles, 5800).  A block does the rounds that begin in its stretch.  Without the weights a
// block of four short sequences ends at 76 us where the others end at 51 (8 trees of 8 nodes on 16k keys of their
// group).
template <int RK, int WP, int WO>
struct PrefixSplit {
  static constexpr int kPart = WO > 16 ? 7 : 5;
  static constexpr int UP = WP > 16 ? 3 : 2, UO = WO > 16 ? 3 : 2;  // units of a round
  static constexpr int kLead = 9;
  static constexpr int LEAST = WP > 16 ? 6 : 2;                     // of a block, no fewer than of a round
  struct Row {
    int start, keys;   // own positions [start, keys), keys = 0: none
    int pr, pt, cols;  // of the group it is the first of: rounds of a tile, tiles, columns
    int first;         // of the sequence's group, -1 without one
    int pages;         // the first sequence of the group that has a place: its table row is read
  };
  Row r0;           // sequence `lane`
  int upto0, seg0;  // sums of units and segments up to it
  int ot;           // tiles of a sequence's own columns
  int total, blocks;
  int older, most;  // blocks in front, and their units
  int each, extra;  // units of the others, how many of them have one more

  __device__ __forceinline__ static int rounds(int keys) { return static_cast<int>(static_cast<unsigned>(keys + RK - 1) / RK); }
  __device__ __forceinline__ int own_rounds(const Row& r) const { return r.keys ? rounds(r.keys - r.start) : 0; }
  // units of a tile of shared and of own keys (a sequence without a place has none), and of all of a sequence's
  __device__ __forceinline__ static int shared_units(const Row& r) { return kPart + r.pr * UP; }
  __device__ __forceinline__ int own_units(const Row& r) const { return r.keys ? kPart + own_rounds(r) * UO : 0; }
  __device__ __forceinline__ int row_units(const Row& r) const { return shared_units(r) * r.pt + own_units(r) * ot; }
  __device__ __forceinline__ int row_segments(const Row& r) const { return r.pt + ot; }

  // sequence b0 + lane, by all lanes of a wave
  __device__ __forceinline__ static Row load(const PrefixArgs& a, int b0) {
    const int lane = threadIdx.x & 63, b = b0 + lane;
    int n = -1, id = -1, shared = 0;
    if (b < a.B) {
      n = a.lengths[b];
      id = a.groups[static_cast<int64_t>(b) * 2];
      shared = a.groups[static_cast<int64_t>(b) * 2 + 1];
    }
    const bool grouped = id >= 0 && shared >= kSlab && shared <= a.maxpos;
    const int id1 = __shfl_up(id, 1, 64), shared1 = __shfl_up(shared, 1, 64);
    const bool on = grouped && lane > 0 && id1 == id && shared1 == shared;  // goes on with the group before it
    const uint64_t heads = __ballot(grouped && !on), ons = __ballot(on);
    Row r{0, 0, 0, 0, 0, -1, b};
    const int least = id >= 0 && shared > 0 ? shared : 0;
    r.keys = n >= least && n <= a.maxpos - a.T ? n + a.T : 0;
    const uint64_t runs = __ballot(r.keys != 0);
    if (grouped) {
      r.first = b0 + 63 - __builtin_clzll(heads & (~0ull >> (63 - lane)));
      r.start = shared & ~(kSlab - 1);
      if (!on) {
        const uint64_t behind = lane < 63 ? ons >> (lane + 1) : 0;
        const int more = __builtin_ctzll(~behind);  // 63 at most
        const uint64_t mine = (runs >> lane) & (~0ull >> (63 - more));
        r.cols = (1 + more) * a.C;
        r.pt = mine ? (r.cols + WP - 1) / WP : 0;
        r.pr = rounds(r.start);
        r.pages = mine ? b + __builtin_ctzll(mine) : b;
      }
    }
    return r;
  }
  __device__ __forceinline__ PrefixSplit(const PrefixArgs& a, const Row& r) : r0(r) {
    ot = (a.C + WO - 1) / WO;
    upto0 = scan64(row_units(r0));
    seg0 = scan64(row_segments(r0));
    total = __builtin_amdgcn_readlane(upto0, 63);
    for (int b0 = 64; b0 < a.B; b0 += 64)
      total += __builtin_amdgcn_readlane(scan64(row_units(load(a, b0))), 63);
    blocks = min(a.slots, static_cast<int>(static_cast<unsigned>(total) / LEAST));  // (total is 0, or more than LEAST)
    each = blocks ? static_cast<unsigned>(total) / static_cast<unsigned>(blocks) : 0;
    older = blocks == a.slots ? a.older : 0;
    most = each + static_cast<int>(static_cast<uint64_t>(each) * kLead >> 6);
    const int others = blocks - older, left = total - older * most;
    each = others ? static_cast<unsigned>(left) / static_cast<unsigned>(others) : 0;
    extra = left - each * others;
  }
  __device__ __forceinline__ int begin(int k) const {
    const int behind = max(k - older, 0);
    return min(k, older) * most + behind * each + min(behind, extra);
  }
  __device__ __forceinline__ int block_of(int unit) const {
    if (unit < older * most) return static_cast<unsigned>(unit) / static_cast<unsigned>(most);
    const unsigned x = unit - older * most, big = extra * (each + 1);
    return older + (x < big ? x / static_cast<unsigned>(each + 1) : extra + (x - big) / static_cast<unsigned>(each));
  }
  // a sequence as all lanes see it: its first unit and segment, and its row
  struct At {
    int first, segment;
    Row r;
  };
  __device__ __forceinline__ At pick(const Row& r, int upto, int seg, int l) const {
    At at;
    at.r.start = __builtin_amdgcn_readlane(r.start, l);
    at.r.keys = __builtin_amdgcn_readlane(r.keys, l);
    at.r.pr = __builtin_amdgcn_readlane(r.pr, l);
    at.r.pt = __builtin_amdgcn_readlane(r.pt, l);
    at.r.cols = __builtin_amdgcn_readlane(r.cols, l);
    at.r.first = __builtin_amdgcn_readlane(r.first, l);
    at.r.pages = __builtin_amdgcn_readlane(r.pages, l);
    at.first = __builtin_amdgcn_readlane(upto, l) - row_units(at.r);
    at.segment = __builtin_amdgcn_readlane(seg, l) - row_segments(at.r);
    return at;
  }
  // the sequence of unit x < total
  __device__ __forceinline__ At sequence_at(const PrefixArgs& a, int x, int& b) const {
    Row r = r0;
    int upto = upto0, seg = seg0;
    for (int b0 = 0;; b0 += 64) {
      const uint64_t m = __ballot(x < upto);
      if (m) {
        const int l = __builtin_ctzll(m);
        b = b0 + l;
        return pick(r, upto, seg, l);
      }
      next(a, b0 + 64, r, upto, seg);
    }
  }
  __device__ __forceinline__ At sequence(const PrefixArgs& a, int b) const {
    Row r = r0;
    int upto = upto0, seg = seg0, b0 = 0;
    for (; b >= b0 + 64; b0 += 64) next(a, b0 + 64, r, upto, seg);
    return pick(r, upto, seg, b - b0);
  }

 private:
  __device__ __forceinline__ void next(const PrefixArgs& a, int b0, Row& r, int& upto, int& seg) const {
    const int run = __builtin_amdgcn_readlane(upto, 63), runs = __builtin_amdgcn_readlane(seg, 63);
    r = load(a, b0);
    upto = scan64(row_units(r)) + run;
    seg = scan64(row_segments(r)) + runs;
  }
};

// ---------------------------------------------------------------- attention
// A part is worked on as by tree attention (tree_part): a wave builds the matrix operands of 32 keys once and uses them for
// 16 NTP columns, which here belong to several sequences.  As there, weights times value norms and the value centroids (scaled
// so that they lose least) are f16 and sums f32: 1.0 to 1.6e-4 of an output's norm from float64, before its own rounding.
// 16 sequences of 32000 shared positions and 700 of their own, 32/8 heads, 3 bits (32 MB; 12.8 GFLOP, 11 us at a large library
// product's rate): 38 us under a kernel trace, 49 the call with preparation (6) and merge (8).  Neither memory nor the matrix
// unit ends it: of 76k cycles the VALU issues in 33k and the matrix unit is busy in 17k, over the two waves per
// SIMD that two tiles' registers leave, and about 10k pass before the first of a block's nine rounds is done.
// The blocks of a kv head are neighbours on one XCD (head along x), as they read the same rows at about the same time: 16
// trees of 16 nodes on 16k positions miss the L2 in 0.35 million lines, with the head along y, where all XCDs
// read all rows, in 3.5 million.
// Of the two blocks on a compute unit the first has its instructions taken first: it ends at 30 us where the second ends at
// 35, so that it is dealt 14% more (attention and merge 43 against 46 us, 64 sequences of 8k, 16/2 heads, 35 against 38).
// NTP and NTO tiles of 16 columns to a segment of shared and of own keys (NTO <= NTP).  Records have 16 NTP columns.
template <int D, int BITS, int NTP, int NW>
struct PrefixSmem : TreeSmem<D, BITS, NTP, NW> {
  float fs[16 * NTP];
};

template <int D, int BITS, int NTP, int NTO, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))
prefix_attn_kernel(PrefixArgs a) {
  constexpr int RK = 32 * NW, WP = 16 * NTP, WO = 16 * NTO;
  using Split = PrefixSplit<RK, WP, WO>;
  __shared__ __attribute__((aligned(16))) PrefixSmem<D, BITS, NTP, NW> sm;
  const int tid = threadIdx.x, hkv = blockIdx.x, block = blockIdx.y;
  const TreeTables<BITS> tables(a, tid);
  const Split split(a, Split::load(a, 0));
  if (block >= split.blocks) return;  // block-uniform
  int x = split.begin(block);
  const int x_end = split.begin(block + 1);
  tables.keys(sm.luts, tid);
  tables.values(sm.luts, tid);
  while (x < x_end) {
    int b;
    const typename Split::At at = split.sequence_at(a, x, b);
    const int before = Split::shared_units(at.r) * at.r.pt;  // the shared keys' tiles, in front of the own ones'
    const bool own = x - at.first >= before;
    const int units = own ? split.own_units(at.r) : Split::shared_units(at.r), from = at.first + (own ? before : 0);
    const int tile = static_cast<int>(static_cast<unsigned>(x - from) / static_cast<unsigned>(units));
    const int u0 = x - from - tile * units, u1 = min(u0 + x_end - x, units);
    const auto rounds_before = [&](int u) {  // rounds that begin in front of the segment's unit u
      const unsigned v = max(u - Split::kPart, 0);
      return static_cast<int>(own ? (v + Split::UO - 1) / Split::UO : (v + Split::UP - 1) / Split::UP);
    };
    const int r0 = rounds_before(u0), r1 = rounds_before(u1);
    const int64_t rec = ((static_cast<int64_t>(block) + at.segment + tile + (own ? at.r.pt : 0)) * a.Hkv + hkv) * WP;
    x += u1 - u0;
    if (r0 == r1) continue;
    if (own) {
      const TreePart part{b, b, a.C, tile * WO, at.r.keys - a.T, at.r.start + r0 * RK, min(at.r.keys, at.r.start + r1 * RK), rec};
      tree_part<D, BITS, NTO, NW, false>(a, part, hkv, sm);
    } else {
      const int end = min(at.r.start, r1 * RK);
      const TreePart part{b, at.r.pages, at.r.cols, tile * WP, end, r0 * RK, end, rec};
      tree_part<D, BITS, NTP, NW, true>(a, part, hkv, sm);
    }
  }
}

// ---------------------------------------------------------------- merge
// One block per (sequence, kv head, 4 CW columns), as tree_merge_kernel: a column's records are those of its
// tile of the group's shared keys, then those of its tile of the own ones.  8 us for 512 columns of 34 records (9 MB), 7 for 4096
// of a few: three dependent round trips (lengths and groups, records, output).
template <int D, int RK, int WP, int WO, int CW>
__global__ void __launch_bounds__(256) prefix_merge_kernel(PrefixArgs a) {
  using Split = PrefixSplit<RK, WP, WO>;
  using Finish = TreeFinish<D, CW>;
  using floatPL = typename Finish::floatPL;
  constexpr int PL = Finish::PL, NC = Finish::NC, NB = 16 / CW;
  __shared__ typename Finish::Smem sm;
  const int c0 = blockIdx.x * NC, hkv = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;

  const typename Split::Row r0 = Split::load(a, 0);  // before Pi_v: waited for first
  const Finish finish(a);
  const Split split(a, r0);
  const typename Split::At own = split.sequence(a, b);
  const typename Split::At head = own.r.first >= 0 && own.r.first != b ? split.sequence(a, own.r.first) : own;
  const int64_t step = static_cast<int64_t>(a.Hkv) * WP;  // columns between records
  // a column's records: n1 of the group's tile from column at1 on, those of its own tile from at2 on, n in all
  struct Records {
    int64_t at1, at2;
    int n1, n;
  };
  const auto records_of = [&](int c) {
    Records rs{0, 0, 0, 0};
    if (!own.r.keys) return rs;
    const auto list = [&](int first, int units, int rounds, int segment, int col, int64_t& at) {
      const int k0 = split.block_of(first + Split::kPart), k1 = split.block_of(first + Split::kPart + (rounds - 1) * units);
      at = ((static_cast<int64_t>(k0) + segment) * a.Hkv + hkv) * WP + col;
      return k1 - k0 + 1;
    };
    if (own.r.first >= 0) {
      const int pc = (b - own.r.first) * a.C + c, tile = pc / WP;
      rs.n1 = list(head.first + tile * Split::shared_units(head.r), Split::UP, head.r.pr, head.segment + tile, pc - tile * WP,
                   rs.at1);
    }
    const int tile = c / WO;
    rs.n = rs.n1 + list(own.first + Split::shared_units(own.r) * own.r.pt + tile * split.own_units(own.r), Split::UO,
                        split.own_rounds(own.r), own.segment + own.r.pt + tile, c - tile * WO, rs.at2);
    return rs;
  };
  const auto column = [&](const Records& rs, int q) { return q < rs.n1 ? rs.at1 + q * step : rs.at2 + (q - rs.n1) * step; };
  // one memory round trip for the first NB records of all the wave's columns: partial O, and a record's
  // maximum and sum per lane
  Records rs[CW];
  floatPL v0[CW][NB];
  float m0[CW], l0[CW];
#pragma unroll
  for (int k = 0; k < CW; ++k) {
    rs[k] = records_of(min(c0 + wave + 4 * k, a.C - 1));
#pragma unroll
    for (int q = 0; q < NB; ++q)
      v0[k][q] = q < rs[k].n ? *reinterpret_cast<const floatPL*>(a.part_o + column(rs[k], q) * D + PL * lane) : floatPL{};
    m0[k] = lane < rs[k].n ? a.part_ml[column(rs[k], lane) * 2] : -INFINITY;
    l0[k] = lane < rs[k].n ? a.part_ml[column(rs[k], lane) * 2 + 1] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < CW; ++k) {
    const int cc = wave + 4 * k, c = c0 + cc, n = rs[k].n;
    floatPL o = floatPL{};
    if (c < a.C) {
      const auto ml = [&](int q) { return a.part_ml + column(rs[k], q) * 2; };
      float mx = m0[k];
      for (int q = lane + 64; q < n; q += 64) mx = fmaxf(mx, ml(q)[0]);
#pragma unroll
      for (int sh = 32; sh >= 1; sh >>= 1) mx = fmaxf(mx, __shfl_xor(mx, sh, 64));
      float lsum = 0.f;
      for (int q0 = 0; q0 < n; q0 += 64) {
        float w = 0.f;
        if (q0 + lane < n) {
          const float m = q0 == 0 ? m0[k] : ml(q0 + lane)[0];
          if (m != -INFINITY) {
            w = __builtin_amdgcn_exp2f(m - mx);
            lsum += w * (q0 == 0 ? l0[k] : ml(q0 + lane)[1]);
          }
        }
        const auto add = [&](const floatPL (&v)[NB], int u) {
#pragma unroll
          for (int q = 0; q < NB; ++q) {
            const float ww = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), u + q));
#pragma unroll
            for (int e = 0; e < PL; ++e) o[e] = fmaf(ww, v[q][e], o[e]);
          }
        };
        if (q0 == 0) add(v0[k], 0);
        const int nb = min(64, n - q0);
        for (int u = q0 == 0 ? NB : 0; u < nb; u += NB) {
          floatPL v[NB];
#pragma unroll
          for (int q = 0; q < NB; ++q)
            v[q] = u + q < nb ? *reinterpret_cast<const floatPL*>(a.part_o + column(rs[k], q0 + u + q) * D + PL * lane) : floatPL{};
          add(v, u);
        }
      }
#pragma unroll
      for (int sh = 32; sh >= 1; sh >>= 1) lsum += __shfl_xor(lsum, sh, 64);
      o *= lsum == 0.f ? 0.f : 1.f / lsum;
    }
    Finish::put(sm, cc, o);
  }
  __syncthreads();
  finish.store(a, sm, b, hkv, c0);
}

// ---------------------------------------------------------------- launch
using PrefixKernel = void (*)(PrefixArgs);

struct PrefixPlan {
  PrefixKernel attend;
  int tiles, own_tiles;  // NTP, NTO
  int slots, older;
  bool apart;  // every sequence by itself, by tree attention
  int64_t records, bytes;
};

template <int D, int BITS>
static PrefixKernel prefix_kernel(int tiles, int own_tiles) {
  if (tiles == 1) return &prefix_attn_kernel<D, BITS, 1, 1, 4>;
  return own_tiles == 1 ? &prefix_attn_kernel<D, BITS, 2, 1, 4> : &prefix_attn_kernel<D, BITS, 2, 2, 4>;
}
static PrefixKernel prefix_kernel(int d, int bits, int tiles, int own_tiles) {
  if (d == 64)
    return bits == 2 ? prefix_kernel<64, 2>(tiles, own_tiles) : bits == 3 ? prefix_kernel<64, 3>(tiles, own_tiles)
                                                                          : prefix_kernel<64, 4>(tiles, own_tiles);
  return bits == 2 ? prefix_kernel<128, 2>(tiles, own_tiles) : bits == 3 ? prefix_kernel<128, 3>(tiles, own_tiles)
                                                                         : prefix_kernel<128, 4>(tiles, own_tiles);
}

static PrefixPlan plan_prefix(int B, int Hq, int Hkv, int T, int64_t maxpos, int d, int bits) {
  static int resident[2][3][3][16] = {};  // per kernel, per device
  PrefixPlan p{};
  const int C = Hq / Hkv * T;
  const auto rounds_of = [&](int columns) { return static_cast<int64_t>(B) * ((maxpos + 127) / 128) * Hkv * ((C + columns - 1) / columns); };
  p.tiles = static_cast<int64_t>(B) * C > 16 ? 2 : 1;
  p.own_tiles = C > 16 ? 2 : 1;
  p.attend = prefix_kernel(d, bits, p.tiles, p.own_tiles);
  const int res = resident_blocks(reinterpret_cast<const void*>(p.attend), 256,
                                  resident[d == 128][bits - 2][p.tiles + p.own_tiles - 2]);
  // Sharing saves the reading of keys and columns that are idle in tree attention's tiles.  Where neither counts it
  // is left out: a sequence's columns fill its two tiles, which decode the keys for themselves either way (8 trees of 8 nodes on
  // 16k shared keys, 32/8 heads, 79 us with tree attention against 80, no difference; 16 trees of 16 nodes 190 against 220; 7
  // nodes, 28 columns, 120 against 115; other numbers of full tiles are not measured), or a block of the device has no more
  // than one round to do (4 sequences of 1k, 12 heads of 64, 16.9 against 20.8 us; 16 of 128, 32/8 heads, 20.0 against 24.3;
  // 4 of 2k, 544 rounds to 512 blocks, 24.6 against 23.7).  The rounds are those of full tables, as lengths are the device's: short
  // sequences over tables of many more entries take the slower form.
  p.apart = C % 32 == 0 || rounds_of(32) <= res;
  if (p.apart) {
    p.bytes = tree_workspace(B, Hq, Hkv, T, maxpos, d, bits);
    return p;
  }
  p.slots = res / Hkv > 1 ? res / Hkv : 1;
  p.older = res == 2 * compute_units() ? p.slots / 2 : 0;
  // a sequence's own tiles, and as many of its group's at most
  const int own = (C + 16 * p.own_tiles - 1) / (16 * p.own_tiles);
  const int64_t segments = 2 * static_cast<int64_t>(B) * own;
  const int64_t most = segments * (7 + (maxpos + 127) / 128 * 3);  // units, of which a block has 2 or more
  if (p.slots > most / 2) p.slots = static_cast<int>(most / 2), p.older = 0;
  p.records = p.slots + segments;
  p.bytes = p.records * Hkv * (16 * p.tiles) * static_cast<int64_t>(d + 2) * 4;
  return p;
}

static bool prefix_shape(int B, int Hq, int Hkv, int T, int64_t maxpos, int d, int bits) {
  return B >= 1 && B <= 65535 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hkv <= 65535 && T >= 1 && T <= 64 && maxpos >= T &&
         maxpos <= (int64_t(1) << 24) && (d == 64 || d == 128) && bits >= 2 && bits <= 4 &&
         2 * static_cast<int64_t>(B) * ((static_cast<int64_t>(Hq / Hkv) * T + 15) / 16) * ((maxpos + 127) / 128) < (int64_t(1) << 28);
}

template <int D, int WP, int WO>
static void launch_prefix_merge(const PrefixArgs& a, hipStream_t s) {
  // as tree attention's merge: the widest blocks that still are two to a compute unit (16 columns) or one (8)
  const auto blocks = [&](int columns) { return static_cast<int64_t>((a.C + columns - 1) / columns) * a.Hkv * a.B; };
  const auto grid = [&](int columns) { return dim3((a.C + columns - 1) / columns, a.Hkv, a.B); };
  if (blocks(16) >= 512) prefix_merge_kernel<D, 128, WP, WO, 4><<<grid(16), 256, 0, s>>>(a);
  else if (blocks(8) >= 256) prefix_merge_kernel<D, 128, WP, WO, 2><<<grid(8), 256, 0, s>>>(a);
  else prefix_merge_kernel<D, 128, WP, WO, 1><<<grid(4), 256, 0, s>>>(a);
}

template <int D>
static void launch_prefix(const PrefixArgs& a, const PrefixPlan& p, hipStream_t s) {
  p.attend<<<dim3(a.Hkv, p.slots), 256, 0, s>>>(a);
  if (p.tiles == 1) launch_prefix_merge<D, 16, 16>(a, s);
  else if (p.own_tiles == 1) launch_prefix_merge<D, 32, 16>(a, s);
  else launch_prefix_merge<D, 32, 32>(a, s);
}

}  // namespace tq

using namespace tq;

extern "C" {

int64_t tq_prefix_workspace_size(int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t table_width, int32_t page_size,
                                 int32_t d, int32_t bits) {
  const int64_t maxpos = static_cast<int64_t>(table_width) * page_size;
  return prefix_shape(B, Hq, Hkv, T, maxpos, d, bits) ? plan_prefix(B, Hq, Hkv, T, maxpos, d, bits).bytes : 0;
}

int tq_prefix_attention(const uint16_t* q_rot, const float* q_proj, const uint8_t* key_codes, const uint8_t* key_signs,
                        const uint16_t* key_rn, const uint16_t* key_vn, const uint16_t* key_centroids_f16, int32_t bits,
                        const uint8_t* val_codes, const uint16_t* val_vn, const float* val_centroids,
                        const uint16_t* val_pit_split, int64_t num_pages, int32_t page_size, const int32_t* block_table,
                        int64_t ld_table, int32_t table_width, const int32_t* lengths, const int32_t* groups,
                        const int32_t* parents, int64_t ld_parents, int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t d,
                        float coeff, float scale, void* out, int32_t out_dtype, int64_t sob, int64_t soh, int64_t sos,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  if (d != 64 && d != 128) {
    set_error("tq_prefix_attention: head_dim %d not supported (64 or 128)", d);
    return TQ_EUNSUPPORTED;
  }
  if (bits < 2 || bits > 4) {
    set_error("tq_prefix_attention: bits %d not supported (2 to 4)", bits);
    return TQ_EUNSUPPORTED;
  }
  TQ_REQUIRE(B >= 0 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && T >= 1, "tq_prefix_attention: bad shape");
  TQ_REQUIRE(T <= 64, "tq_prefix_attention: at most 64 drafted tokens, got %d", T);
  TQ_REQUIRE(page_size >= 32 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0,
             "tq_prefix_attention: page_size must be a power of two from 32 to 2^20, got %d", page_size);
  TQ_REQUIRE(num_pages >= 1 && num_pages < (int64_t(1) << 31) && ld_table >= table_width, "tq_prefix_attention: bad pool");
  const int64_t maxpos = static_cast<int64_t>(table_width) * page_size;
  TQ_REQUIRE(maxpos >= T, "tq_prefix_attention: a table of %d pages of %d does not hold %d drafted tokens", table_width, page_size, T);
  TQ_REQUIRE(out_dtype == TQ_F32 || out_dtype == TQ_F16 || out_dtype == TQ_BF16, "tq_prefix_attention: unknown dtype %d", out_dtype);
  if (B == 0) return TQ_OK;
  TQ_REQUIRE(prefix_shape(B, Hq, Hkv, T, maxpos, d, bits),
             "tq_prefix_attention: at most 65535 sequences and kv heads, 2^24 positions a sequence and 2^31 / 8 (128 keys, 16 "
             "columns) blocks of work, got %d, %d and %lld", B, Hkv, (long long)maxpos);
  TQ_REQUIRE(q_rot && q_proj && key_codes && key_signs && key_rn && key_vn && key_centroids_f16 && val_codes && val_vn &&
                 val_centroids && val_pit_split && block_table && lengths && groups && out,
             "tq_prefix_attention: null pointer");
  for (const void* p : {static_cast<const void*>(q_rot), static_cast<const void*>(q_proj), static_cast<const void*>(key_codes),
                        static_cast<const void*>(key_signs), static_cast<const void*>(val_codes), static_cast<const void*>(val_pit_split)})
    TQ_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "tq_prefix_attention: queries, code planes and Pi_v must be 16-byte aligned");
  const PrefixPlan p = plan_prefix(B, Hq, Hkv, T, maxpos, d, bits);
  TQ_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= p.bytes,
             "tq_prefix_attention: the workspace must be 16-byte aligned and hold %lld bytes", (long long)p.bytes);
  PrefixArgs a{};
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
  a.groups = groups;
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
  hipStream_t s = as_stream(stream);
  if (p.apart) {
    tree_attend(a, d, bits, workspace, s);
    return launch_status("tq_prefix_attention");
  }
  a.slots = p.slots;
  a.older = p.older;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + p.records * Hkv * (16 * p.tiles) * d;
  if (d == 64) launch_prefix<64>(a, p, s);
  else launch_prefix<128>(a, p, s);
  return launch_status("tq_prefix_attention");
}

}  // extern "C"
