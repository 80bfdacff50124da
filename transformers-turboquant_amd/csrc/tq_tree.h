// What the kernels that attend over pages of a compressed cache share (tq_tree.hip, tq_prefix.hip): the split of
// the keys over blocks, the stream of packed rows, the work on one part, and the end of the merge.
#pragma once

#include "tq_decode.h"

namespace tq {

struct TreeArgs {
  const uint16_t* q_rot;  // [B, Hq, T, D]
  const float* q_proj;
  const uint8_t *kcodes, *ksigns;
  const uint16_t *krn, *kvn, *kcent;
  const uint8_t* vcodes;
  const uint16_t* vvn;
  const float* vcent;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  const int32_t* groups;  // null, or [B, 2]: what a sequence shares with others, and is no shorter than (tq_prefix.hip)
  const int32_t* parents;
  int64_t ld_parents;
  int64_t num_pages;
  int lg_page, maxpos;  // maxpos: positions a table row can hold
  int B, Hq, Hkv, T, G, C;
  int slots;            // blocks along x: stretches of the rounds of all sequences
  int lg_least;         // a stretch has 2^lg_least rounds or more, where there are as many
  float coeff, scale;
  float *part_o, *part_ml;  // records [slots + B, Hkv, C, D], [slots + B, Hkv, C, 2]
  const uint16_t* vpit;
  void* out;
  int out_dtype;
  int64_t sob, soh, sos;
};

// ---------------------------------------------------------------- the split of the keys
// length of sequence b, -1 behind the last and of one that is shorter than what it shares
__device__ __forceinline__ int tree_length(const TreeArgs& a, int b) {
  if (b >= a.B) return -1;
  const int n = a.lengths[b];
  if (!a.groups) return n;
  const int32_t* const g = a.groups + static_cast<int64_t>(b) * 2;
  return g[0] >= 0 && n < g[1] ? -1 : n;
}
// keys of a sequence of length n (cached and drafted), 0 where it does not fit its table
__device__ __forceinline__ int tree_keys(const TreeArgs& a, int n) { return n >= 0 && n <= a.maxpos - a.T ? n + a.T : 0; }
// Inclusive sum over the wave through DPP (shifts within rows of 16 lanes, then row 0's sum into
// row 1 and row 2's into row 3, then lane 31's into the upper half): no LDS round trips.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int scan64(int v) {
  v = dpp_add<0x111, 0xF>(v);
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);
  return dpp_add<0x143, 0xC>(v);
}

// Every wave of a block computes the same, 64 sequences per step (one per lane).  Block k of
// n = min(slots, R / 2^lg_least) has the rounds [begin(k), begin(k + 1)) of the R in all: R / n of them, the first
// R % n blocks one more.  Walking along the rounds, every step to the next part moves to the next
// block, the next sequence or both, so k + b is a different number for every part, and the
// parts of one sequence have consecutive ones: the record.
template <int RK>
struct TreeSplit {
  int k0, upto0;    // of sequence `lane`: its keys, and the sum of rounds up to it
  int total;        // rounds of all sequences
  int blocks;       // that have any: every one of them at least a round, so that no record is left unwritten
  int each, extra;  // rounds of a block, blocks with one more
  __device__ __forceinline__ static int rounds(int keys) { return static_cast<int>(static_cast<unsigned>(keys + RK - 1) / RK); }
  // n0: tree_length of sequence `lane`, loaded early by the caller
  __device__ __forceinline__ TreeSplit(const TreeArgs& a, int n0) {
    const int lane = threadIdx.x & 63;
    k0 = tree_keys(a, n0);
    upto0 = scan64(rounds(k0));
    total = __builtin_amdgcn_readlane(upto0, 63);
    for (int b0 = 64; b0 < a.B; b0 += 64)
      total += __builtin_amdgcn_readlane(scan64(rounds(tree_keys(a, tree_length(a, b0 + lane)))), 63);
    blocks = min(a.slots, static_cast<int>((static_cast<unsigned>(total) + (1u << a.lg_least) - 1) >> a.lg_least));
    each = blocks ? static_cast<unsigned>(total) / static_cast<unsigned>(blocks) : 0;
    extra = total - each * blocks;
  }
  __device__ __forceinline__ int begin(int k) const { return k * each + min(k, extra); }
  __device__ __forceinline__ int block_of(int round) const {
    const unsigned big = extra * (each + 1), x = round;
    return x < big ? x / static_cast<unsigned>(each + 1) : extra + (x - big) / static_cast<unsigned>(each);
  }
  // the sequence of round x < total, its first round and its keys
  __device__ __forceinline__ void sequence_at(const TreeArgs& a, int x, int& b, int& first, int& keys) const {
    int k = k0, upto = upto0;
    for (int b0 = 0;; b0 += 64) {
      const uint64_t m = __ballot(x < upto);
      if (m) {
        const int l = __builtin_ctzll(m);
        b = b0 + l;
        keys = __builtin_amdgcn_readlane(k, l);
        first = __builtin_amdgcn_readlane(upto, l) - rounds(keys);
        return;
      }
      next(a, b0 + 64, k, upto);
    }
  }
  // first round and number of rounds of sequence b
  __device__ __forceinline__ void rounds_of(const TreeArgs& a, int b, int& first, int& n) const {
    int k = k0, upto = upto0;
    int b0 = 0;
    for (; b >= b0 + 64; b0 += 64) next(a, b0 + 64, k, upto);
    n = rounds(__builtin_amdgcn_readlane(k, b - b0));
    first = __builtin_amdgcn_readlane(upto, b - b0) - n;
  }

 private:
  // on to the 64 sequences from b0 on
  __device__ __forceinline__ static void next(const TreeArgs& a, int b0, int& k, int& upto) {
    const int run = __builtin_amdgcn_readlane(upto, 63);
    k = tree_keys(a, tree_length(a, b0 + static_cast<int>(threadIdx.x & 63)));
    upto = scan64(rounds(k)) + run;
  }
};

// What a block works on at a time: some columns of a kv head against a run of keys.
struct TreePart {
  int row;         // the sequence of column 0
  int pages;       // the one whose table row gives the pages
  int cols, ct0;   // the part's columns are those of [ct0, cols) that fit its tiles
  int nctx;        // key positions below nctx are cached, drafted tokens behind
  int kbeg, kend;  // positions
  int64_t rec;     // record of column ct0
};

// Bit t of the result: node `lane` sees drafted token t (its ancestors and itself).  A parent that
// is neither -1 nor an earlier node leaves the node without a place: it sees nothing and nothing
// sees it.  Pointer doubling: after k steps a lane has its next 2^k ancestors.
__device__ __forceinline__ int tree_parent(const TreeArgs& a, int b) {
  const int i = threadIdx.x & 63;
  return i >= a.T ? -2 : a.parents ? a.parents[b * a.ld_parents + i] : i - 1;
}
__device__ __forceinline__ uint64_t tree_ancestors(const TreeArgs& a, int par) {
  const int i = threadIdx.x & 63;
  const bool placed = par >= -1 && par < i;
  uint64_t seen = placed ? 1ull << i : 0;
  int up = placed ? par : -1;
  for (int reach = 1; reach < a.T; reach <<= 1) {
    const int src = up < 0 ? i : up;
    const uint64_t s = __shfl(seen, src, 64);
    const int u = __shfl(up, src, 64);
    if (up >= 0) {
      seen |= s;
      up = u;
    }
  }
  return placed ? seen : 0;
}

// Bit k: key ks0 + k of a slab of `rows` rows is cached, or a drafted token in `tokens`; the slab's first
// drafted token has bit d = n_b - ks0.
__device__ __forceinline__ uint32_t tree_visible(uint64_t tokens, int d, int rows) {
  const uint64_t cached = d <= 0 ? 0 : d >= 32 ? ~0ull : (1ull << d) - 1;
  const uint64_t drafted = d <= -64 || d >= 32 ? 0 : d >= 0 ? tokens << d : tokens >> -d;
  return static_cast<uint32_t>((cached | drafted) & ((1ull << rows) - 1));
}

// A thread's entries of the lookup tables (SmallLuts): everything that a block loads before it
// knows its sequence is loaded at once, the tables are written when it has arrived.
template <int BITS>
struct TreeTables {
  using L = SmallLuts<BITS>;
  static constexpr int KB = L::KB, VB = L::VB, KM = (1 << KB) - 1, VM = (1 << VB) - 1;
  uint16_t k0, k1;
  float v0, v1;
  __device__ __forceinline__ TreeTables(const TreeArgs& a, int tid)
      : k0(a.kcent[KB == 1 ? 0 : tid & KM]), k1(a.kcent[KB == 1 ? 1 : (tid >> KB) & KM]), v0(a.vcent[tid & VM]),
        v1(a.vcent[(tid >> VB) & VM]) {}
  __device__ __forceinline__ void keys(uint8_t* t, int tid) const {
    if (tid < 16) {
      half4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = static_cast<_Float16>((tid >> j) & 1 ? 1.f : -1.f);
      *reinterpret_cast<half4*>(t + L::SGN_OFF + tid * 8) = v;
    }
    if constexpr (KB == 1) {
      typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
      if (tid < 16)
        *reinterpret_cast<u16x4*>(t + L::KEY_OFF + tid * 8) =
            u16x4{tid & 1 ? k1 : k0, tid & 2 ? k1 : k0, tid & 4 ? k1 : k0, tid & 8 ? k1 : k0};
    } else {
      if (tid < L::KEY_BYTES / 4) *reinterpret_cast<uint32_t*>(t + L::KEY_OFF + tid * 4) = k0 | static_cast<uint32_t>(k1) << 16;
    }
  }
  __device__ __forceinline__ void values(uint8_t* t, int tid) const {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    if (tid < L::VAL_BYTES / 4)
      *reinterpret_cast<half2v*>(t + L::VAL_OFF + tid * 4) = half2v{static_cast<_Float16>(v0), static_cast<_Float16>(v1)};
  }
};

// ---------------------------------------------------------------- the stream of packed rows
// A wave's ring of slabs of 32 keys, filled by direct copies to LDS.
template <int D, int KB, int VB, int R>
struct TreeStream {
  static constexpr int KC = D * KB / 8, SC = D / 8, VC = D * VB / 8;
  static constexpr int NK = 32;  // keys of a slab
  static constexpr int OFF_K = 0, OFF_S = NK * KC, OFF_V = OFF_S + NK * SC, OFF_N = OFF_V + NK * VC;
  static constexpr int NRM = NK * 4;
  static constexpr int SLOT = OFF_N + 3 * NRM;
  static constexpr int NKD = (NK * KC + 1023) / 1024, NSD = (NK * SC + 1023) / 1024, NVD = (NK * VC + 1023) / 1024;
  static constexpr int NDMA = NKD + NSD + NVD + 3;
  // (read by scalar loads, through the constant address space: a vector load's wait would reach
  // back past the copies in flight)
  typedef const __attribute__((address_space(4))) int32_t* const_i32;

  const TreeArgs& a;
  const int hkv, lane, kend;
  const_i32 pages;

  __device__ __forceinline__ TreeStream(const TreeArgs& a_, int b, int hkv_, int kend_)
      : a(a_), hkv(hkv_), lane(threadIdx.x & 63), kend(kend_),
        pages((const_i32)reinterpret_cast<uintptr_t>(a_.table + b * a_.ld_table)) {}
  // A slab's 32 keys lie in one page (pages hold 32 or more, slabs start at multiples of 32)
  __device__ __forceinline__ int page_of(int kb) const { return pages[kb >> a.lg_page]; }
  __device__ __forceinline__ void copy_plane(const i32x4& r, uint32_t dst, int bytes, int nrounds) const {
    const uint32_t lo = lane * 16;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c >= nrounds) break;
      if ((c + 1) * 1024 <= bytes || lane * 16 < bytes - c * 1024) dma16(r, dst + c * 1024, lo + c * 1024);
    }
  }
  // copy the slab of keys [kb, kb + 32) to LDS offset dst; returns how many of its rows exist: up to
  // the part's last key, none where its page is not in the pool
  __device__ __forceinline__ int issue(int kb, int page, uint32_t dst) const {
    const bool in = page >= 0 && page < a.num_pages;
    const int64_t row = in ? ((static_cast<int64_t>(page) * a.Hkv + hkv) << a.lg_page) + (kb & ((1 << a.lg_page) - 1)) : 0;
    const int rows = in ? min(NK, kend - kb) : 0;
    wait_lds();  // earlier reads of this slot have landed
    copy_plane(rows_desc(a.kcodes + row * KC, KC, 0, rows), dst + OFF_K, NK * KC, NKD);
    copy_plane(rows_desc(a.ksigns + row * SC, SC, 0, rows), dst + OFF_S, NK * SC, NSD);
    copy_plane(rows_desc(a.vcodes + row * VC, VC, 0, rows), dst + OFF_V, NK * VC, NVD);
    if (lane < 32) {
      dma_u16(rows_desc(a.kvn + row, 2, 0, rows), dst + OFF_N, lane * 2);
      dma_u16(rows_desc(a.krn + row, 2, 0, rows), dst + OFF_N + NRM, lane * 2);
      dma_u16(rows_desc(a.vvn + row, 2, 0, rows), dst + OFF_N + 2 * NRM, lane * 2);
    }
    return rows;
  }
  // until the slab issued `later` slabs ago has landed
  __device__ __forceinline__ static void wait_slab(int later) {
    static_assert((R == 2 || R == 3) && 2 * NDMA < 64, "ring of 2 or 3 slots");
    if (R == 3 && later >= 2) wait_vm<2 * NDMA>();
    else if (later >= 1) wait_vm<NDMA>();
    else wait_vm<0>();
  }
  // the wave's slabs from ks0 on up to `end`, every RK keys, in ring slots STRIDE bytes apart; work(ring
  // slot, first key, rows)
  template <int RK, int STRIDE, class Work>
  __device__ __forceinline__ void run(int& ks0, int end, int (&nrows)[R], int& slot, uint32_t ring, Work work) const {
    for (; ks0 < end; ks0 += RK) {
      // the next R - 1 slabs, as far as they exist, were issued after this one
      const int later = (kend - 1 - ks0) / RK;
      const bool more = later >= R;
      const int page = more ? page_of(ks0 + R * RK) : -1;  // read ahead of the slab's work
      wait_slab(later);
      if (nrows[0]) work(slot, ks0, nrows[0]);
#pragma unroll
      for (int r = 1; r < R; ++r) nrows[r - 1] = nrows[r];
      if (more) nrows[R - 1] = issue(ks0 + R * RK, page, ring + slot * STRIDE);
      slot = slot + 1 == R ? 0 : slot + 1;
    }
  }
};

// The waves' states of up to TC columns joined into a record: thread (column tid / 16, dims
// D / 16 (tid % 16) ..); mrg [wave][column][D + 4] holds O, the maximum (log2) and the sum.
template <int D, int NW, int TC>
__device__ __forceinline__ void tree_join(const TreeArgs& a, const float* mrg, int64_t at, int ncols, int tid) {
  constexpr int LDM = D + 4, DB = D / 16;
  const int c = tid >> 4, d0 = (tid & 15) * DB;
  if (tid >= 16 * TC || c >= ncols) return;
  float m[NW], mx = -INFINITY, ls = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    m[w] = mrg[(w * TC + c) * LDM + D];
    mx = fmaxf(mx, m[w]);
  }
  float4v o[DB / 4];
#pragma unroll
  for (int i = 0; i < DB / 4; ++i) o[i] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float* s = mrg + (w * TC + c) * LDM;
    const float f = m[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[w] - mx);
    const float lw = s[D + 1];
    ls += f == 0.f ? 0.f : f * lw;
#pragma unroll
    for (int i = 0; i < DB / 4; ++i) {
      const float4v x4 = *reinterpret_cast<const float4v*>(s + d0 + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] += f == 0.f ? 0.f : f * x4[e];
    }
  }
  at += c;
#pragma unroll
  for (int i = 0; i < DB / 4; ++i) *reinterpret_cast<float4v*>(a.part_o + at * D + d0 + 4 * i) = o[i];
  if ((tid & 15) == 0) {
    a.part_ml[at * 2] = mx;
    a.part_ml[at * 2 + 1] = ls;
  }
}

// ---------------------------------------------------------------- attention, operands from tables
// NT tiles of 16 columns.  A wave builds the MFMA operands of a slab once through small lookup tables and
// uses them for every column tile: keys on the M side, so that the scores a lane ends with (4 keys x
// its column) are its own part of P^T, the operand of O^T += V^T P^T.  q_proj (f32) takes two f16
// parts, so that there are three passes of scores and one of values to a key and column.
// P is rounded to f16 (relative 2^-11 of each weight, a hundredth of what the codes lose), sums and
// maxima are f32.
// 16 nodes, 16 sequences of 8k to 32k, 32/8 heads, 3 bits, 0.17 TFLOP of matrix work: 224 us for a call in a row of
// calls, preparation and merge included (11 and 13 us in their trace), so at most 200 us and 0.86 PFLOP/s (a large
// library product reaches 1.16); under a kernel trace, where the clock is lower, 237 us at least and 270 in the
// median.  Of 462k cycles the matrix unit is busy in 164k, the VALU in 231k, the LDS in 239k, over the two waves
// per SIMD that the registers of two tiles leave.  Measured against it and dropped: four tiles at one wave per
// SIMD (236 against 275 us in all), three waves with spills (226 and 309), operands looked up a step ahead at
// two tiles (216 and 224).
//
// The shared memory is one object, so that the lookup tables lie at LDS address 0: a lookup's byte
// offset then is its address (elsewhere every lookup pays an addition, 86 of ~330 VALU instructions
// a slab).
template <int D, int BITS, int NT, int NW>
struct TreeSmem {
  using L = SmallLuts<BITS>;
  static constexpr int R = 3;  // slabs of a wave in flight
  using ST = TreeStream<D, L::KB, L::VB, R>;
  static constexpr int RING = NW * R * ST::SLOT;
  static constexpr int LDM = D + 4;  // floats of a column in the merge of the waves: O, maximum, sum
  static constexpr int MERGE = NW * 16 * LDM * 4;
  static constexpr int QKIND = NT * (D / 32) * 1024;  // fragments of one kind: q_rot, q_proj hi, q_proj lo
  uint8_t luts[(L::BYTES + 15) / 16 * 16];
  __attribute__((aligned(16))) uint8_t area[RING > MERGE ? RING : MERGE];
  __attribute__((aligned(16))) uint8_t q[3 * QKIND];
  uint64_t anc[64];
  float qmax[NW];
};

// Products with an f16 factor in the low half of y, which v_fma_mix takes as it is (a fused multiply-add
// with +0, so that the compiler does not split it into a conversion and a product; and not inline asm, whose
// operands the compiler does not keep apart from the matrix and transcendental instructions that
// write them):
//   mul_f16 = x y, fma_f16 = x y + z in f32; mul2_f16 = (f16(x0 y0), f16(x1 y1)), one rounding each
__device__ __forceinline__ float low_f16(uint32_t y) {
  typedef _Float16 half2v __attribute__((ext_vector_type(2)));
  return static_cast<float>(__builtin_bit_cast(half2v, y)[0]);
}
__device__ __forceinline__ float fma_f16(float x, uint32_t y, float z) { return fmaf(x, low_f16(y), z); }
__device__ __forceinline__ float mul_f16(float x, uint32_t y) { return fmaf(x, low_f16(y), 0.f); }
__device__ __forceinline__ uint32_t mul2_f16(float x0, uint32_t y0, float x1, uint32_t y1) {
  typedef _Float16 half2v __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, half2v{static_cast<_Float16>(mul_f16(x0, y0)), static_cast<_Float16>(mul_f16(x1, y1))});
}

// The f16 operand is P vn, so a column's reference is that of s + E (log2 units), E being a key's
// f16 exponent field: vn < 2^(E - 14).  Weights are p = 2^(s - mref) with mref = max(s + E) - PUP at the
// last move, the maximum over the keys that the column sees, and the reference moves when s + E exceeds
// it by more than TAU: p vn < 2^(PUP + TAU - 14) = 2^14 within f16's range, and the largest was 2^5 or
// more when the reference moved.  A contribution p vn that is 2^-30 of the column's largest still
// reaches the operand, whose subnormals end at 2^-24, whatever norms the other keys have.  (A norm below
// 2^-14 counts as 2^-14.)  p itself stays below 2^28, in f32.
constexpr float kTau = 8.0f, kPup = 20.0f;
__device__ __forceinline__ float norm_exponent(uint32_t vn) { return static_cast<float>(vn >> 10); }

// One part by a block, NT tiles of 16 columns.
// SHARED: the columns are those of several sequences, column c being column c % C of sequence row + c / C,
// against cached keys that all of them have; nothing of a sequence may reach another's columns, so each column has a
// scale of its own.
template <int D, int BITS, int NT, int NW, bool SHARED, class SM>
__device__ __forceinline__ void tree_part(const TreeArgs& a, const TreePart& p, int hkv, SM& sm) {
  using L = typename SM::L;
  constexpr int KB = L::KB, VB = L::VB;
  constexpr int KS = D / 32;           // score k-steps
  constexpr int DB = D / 16;           // value row blocks: lane l16 holds dims DB l16 .. DB l16 + DB - 1
  constexpr int NPAIR = D / 32;        // pair-table groups per parity
  using ST = typename SM::ST;
  constexpr int KC = ST::KC, SC = ST::SC, VC = ST::VC;
  constexpr int KLANE = KC / 4, KW32 = (KLANE + 3) / 4, SLANE = SC / 4;
  constexpr int VFB = DB * VB;
  constexpr int VW32 = (VB == 3) ? 2 : 1;
  constexpr int NK = ST::NK, RK = NW * NK;
  constexpr int OFF_K = ST::OFF_K, OFF_S = ST::OFF_S, OFF_V = ST::OFF_V, OFF_N = ST::OFF_N, NRM = ST::NRM;
  constexpr int SLOT = ST::SLOT, R = SM::R;
  constexpr int QKIND = NT * KS * 1024;  // bytes of a kind of query fragments
  static_assert(QKIND <= SM::QKIND, "query fragments fit");
  constexpr bool HOLD_HI = NT == 1 || D == 64;  // q_proj hi fragments in registers
  constexpr bool AHEAD = NT == 1;  // score operands looked up a step ahead, where registers allow
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr float TAU = kTau, PUP = kPup;

  uint8_t* const area = sm.area;
  const uint8_t* const tS = sm.luts + L::SGN_OFF;
  const uint8_t* const tK = sm.luts + L::KEY_OFF;
  const uint8_t* const tV = sm.luts + L::VAL_OFF;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int b = p.row, ct0 = p.ct0, nctx = p.nctx, kbeg = p.kbeg, kend = p.kend;
  const float fa = a.scale * LOG2E;
  float qs;
  const int vbit = l16 * VFB, vbase = (vbit >> 5) * 4, vshift = vbit & 31;
  uint8_t* const mine = area + wave * (R * SLOT);
  const uint32_t mine_lds = lds_offset(mine);

  // parents, the first slabs' pages and the queries come in one round trip
  int par = -1;
  if constexpr (!SHARED) par = tree_parent(a, b);
  const ST stream(a, p.pages, hkv, kend);
  const int k0w = kbeg + wave * NK;
  int nrows[R], pages[R];
#pragma unroll
  for (int r = 0; r < R; ++r) pages[r] = k0w + r * RK < kend ? stream.page_of(k0w + r * RK) : -1;
  constexpr int TPC = 64 * NW / (16 * NT), DPT = D / TPC;  // threads per column, dims per thread
  static_assert(DPT == 4 || DPT == 8 || DPT == 16, "whole fragments or halves of one");
  const int qcol = tid / TPC, d0 = (tid % TPC) * DPT;
  float4v pj4[DPT / 4];
  half4 rt4[DPT / 4];
  {
    int c = min(ct0 + qcol, p.cols - 1), r = 0;
    if constexpr (SHARED) {
      r = c / a.C;
      c -= r * a.C;
    }
    const int node = c / a.G;
    const int64_t row = ((static_cast<int64_t>(b + r) * a.Hq + hkv * a.G + (c - node * a.G)) * a.T + node) * D + d0;
#pragma unroll
    for (int i = 0; i < DPT / 4; ++i) {
      pj4[i] = *reinterpret_cast<const float4v*>(a.q_proj + row + 4 * i);
      rt4[i] = *reinterpret_cast<const half4*>(a.q_rot + row + 4 * i);
    }
  }
  uint64_t live = 0;  // tokens with a place: some node sees them
  if constexpr (!SHARED) {
    const uint64_t anc_lane = tree_ancestors(a, par);
    if (wave == 0) sm.anc[lane] = anc_lane;
    live = __ballot(anc_lane != 0);
  }
  __syncthreads();  // tables and ancestors in place; the previous part is done with the LDS

  // the first slabs fly while the queries are set up
#pragma unroll
  for (int r = 0; r < R; ++r) nrows[r] = k0w + r * RK < kend ? stream.issue(k0w + r * RK, pages[r], mine_lds + r * SLOT) : 0;

  // ---- the block's queries, laid out by all its threads as B fragments (lane (column l16, group lg)
  // of k-step ks holds dims lg D / 4 + 8 ks ..): q_rot, and coeff q_proj (f32) as f16 hi + lo
  // parts.  All are scaled by one power of two qs that puts the largest q_rot or coeff q_proj in
  // [2^13, 2^14): q_rot stays exact, and the lo parts stay normal f16 down to 2^-17 of it.
  // Columns behind the last repeat it; they are not stored.
  {
    const int col = qcol;
    float pj[DPT], rt[DPT];
#pragma unroll
    for (int i = 0; i < DPT; i += 4) {
      const float4v x4 = pj4[i / 4];
      const half4 h4 = rt4[i / 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pj[i + e] = x4[e] * a.coeff;
        rt[i + e] = static_cast<float>(h4[e]);
      }
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < DPT; ++i) {  // of the finite ones: a column with others spoils itself only
      if (fabsf(pj[i]) < INFINITY) m = fmaxf(m, fabsf(pj[i]));
      if (fabsf(rt[i]) < INFINITY) m = fmaxf(m, fabsf(rt[i]));
    }
    if constexpr (SHARED) {
#pragma unroll
      for (int sh = TPC / 2; sh >= 1; sh >>= 1) m = fmaxf(m, __shfl_xor(m, sh, 64));
      int ex;
      frexpf(m, &ex);  // as qproj_split_scale, of a column
      qs = m > 0.f && m <= 3.0e38f ? ldexpf(1.f, min(14 - ex, 100)) : 1.f;
      if (tid % TPC == 0) sm.fs[col] = fa / qs;
    } else {
      m = wave_max(m);
      if (lane == 0) sm.qmax[wave] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, sm.qmax[w]);
      qs = fminf(qproj_split_scale(m), 0x1p100f);
    }
    constexpr int PER = DPT < 8 ? DPT : 8;
#pragma unroll
    for (int i = 0; i < DPT; i += PER) {
      const int d = d0 + i, lgd = d / (D / 4), ks = (d % (D / 4)) / 8;
      _Float16* const dst =
          reinterpret_cast<_Float16*>(sm.q + (((col / 16) * KS + ks) * 64 + lgd * 16 + col % 16) * 16) + d % 8;
      typedef _Float16 halfP __attribute__((ext_vector_type(PER)));
      halfP r, hi, lo;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        _Float16 h, l;
        split_f16(pj[i + e] * qs, h, l);
        r[e] = static_cast<_Float16>(rt[i + e] * qs);
        hi[e] = h;
        lo[e] = l;
      }
      *reinterpret_cast<halfP*>(dst) = r;
      *reinterpret_cast<halfP*>(dst + QKIND / 2) = hi;
      *reinterpret_cast<halfP*>(dst + QKIND) = lo;
    }
    __syncthreads();
  }
  auto qfrag = [&](int kind, int t, int ks) -> half8 {
    return *reinterpret_cast<const half8*>(sm.q + kind * QKIND + ((t * KS + ks) * 64 + lane) * 16);
  };
  uint64_t anc[NT];  // of the lane's column in each tile
  float fs[NT];
  half8 qr[NT][KS], qh[HOLD_HI ? NT : 1][KS];  // held; the others are read from LDS at their use
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = min(ct0 + 16 * t + l16, p.cols - 1);
    if constexpr (SHARED) {  // every node with a place sees every key
      const int r = c / a.C, node = (c - r * a.C) / a.G;
      const int up = a.parents ? a.parents[(b + r) * a.ld_parents + node] : node - 1;
      anc[t] = up >= -1 && up < node ? ~0ull : 0;
      fs[t] = sm.fs[16 * t + l16];
    } else {
      anc[t] = sm.anc[c / a.G];
      fs[t] = fa / qs;
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qr[t][ks] = qfrag(0, t, ks);
      if constexpr (HOLD_HI) qh[t][ks] = qfrag(1, t, ks);
    }
  }

  // Column state: the reference mref, O and l relative to it, and lim, the largest s + E - mref that
  // does not move it (-inf while the column has none; mref is 0 then).
  float mref[NT], lim[NT], l_run[NT];
  float4v oacc[NT][DB];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    mref[t] = 0.f;
    lim[t] = -INFINITY;
    l_run[t] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) oacc[t][db] = float4v{0.f, 0.f, 0.f, 0.f};
  }

  // EDGE: some of the slab's rows do not exist, or hold drafted tokens
  auto slab = [&](auto edge_c, const uint8_t* src, int ks0, int rows) {
    constexpr bool EDGE = decltype(edge_c)::value;
    auto visible = [&](uint64_t tokens) { return tree_visible(tokens, nctx - ks0, rows); };
    // ---- everything the slab needs from its raw rows; the lane's keys are ks0 + 16j + 4lg + e
    uint32_t kw[2][KW32], sw[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      load_key_field<KLANE>(src + OFF_K + (16 * j + l16) * KC + lg * KLANE, kw[j]);
      sw[j] = load_sign_field<D>(src + OFF_S + (16 * j + l16) * SC + lg * SLANE);
    }
    // ---- scores S^T = K^ Q^T (term 1) and Sign Q_proj^T (term 2); a key operand feeds every tile.
    float4v s1[NT][2], s2[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s1[t][j] = float4v{0.f, 0.f, 0.f, 0.f};
        s2[t][j] = float4v{0.f, 0.f, 0.f, 0.f};
      }
    constexpr int NB = AHEAD ? 2 : 1;
    half8 sg[NB][2], kc[NB][2], hi[NB][NT], lo[NB][NT];
    auto look = [&](auto cc) {
      constexpr int ks = decltype(cc)::value, h = ks % NB;
#pragma unroll
      for (int j = 0; j < 2; ++j) sg[h][j] = nib2x4<ks>(tS, sw[j]);
#pragma unroll
      for (int j = 0; j < 2; ++j) kc[h][j] = key_operand<KB, KW32, ks>(tK, kw[j]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (HOLD_HI) hi[h][t] = qh[t][ks];
        else hi[h][t] = qfrag(1, t, ks);
        lo[h][t] = qfrag(2, t, ks);
      }
    };
    if constexpr (AHEAD) look(std::integral_constant<int, 0>{});
    static_for<KS>([&](auto cc) {
      constexpr int ks = decltype(cc)::value, h = ks % NB, next = ks + NB - 1;
      if constexpr (next < KS) look(std::integral_constant<int, next>{});
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) s2[t][j] = mfma16x16x32(sg[h][j], hi[h][t], s2[t][j]);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) s1[t][j] = mfma16x16x32(kc[h][j], qr[t][ks], s1[t][j]);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) s2[t][j] = mfma16x16x32(sg[h][j], lo[h][t], s2[t][j]);
      if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
    });
    // ---- norms
    u32x4 kn[2], rn[2], vn[2];  // norms, f16 in the low half
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* const n = src + OFF_N + (16 * j + 4 * lg) * 4;
      kn[j] = *reinterpret_cast<const u32x4*>(n);
      rn[j] = *reinterpret_cast<const u32x4*>(n + NRM);
      vn[j] = *reinterpret_cast<const u32x4*>(n + 2 * NRM);
    }
    if constexpr (EDGE) {  // keys that nobody sees weigh nothing, whatever their rows hold
      const uint32_t any = visible(live) >> (4 * lg);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool on = any & (1u << (16 * j + e));
          kn[j][e] = on ? kn[j][e] : 0;
          rn[j][e] = on ? rn[j][e] : 0;
          vn[j][e] = on ? vn[j][e] : 0;
        }
    }
    // ---- log2-domain scores relative to mref, and the softmax step
    float sc[NT][2][4];
    bool hit = false;
    // the lane's largest score and largest exponent bound its s + E
    const float top = norm_exponent(max(max(max(vn[0][0], vn[0][1]), max(vn[0][2], vn[0][3])),
                                        max(max(vn[1][0], vn[1][1]), max(vn[1][2], vn[1][3]))));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      uint32_t see = 0;
      if constexpr (EDGE) see = visible(anc[t]) >> (4 * lg);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = fmaf(fma_f16(s1[t][j][e], kn[j][e], mul_f16(s2[t][j][e], rn[j][e])), fs[t], -mref[t]);
          sc[t][j][e] = !EDGE || (see & (1u << (16 * j + e))) ? x : -INFINITY;
        }
      const float lmax = max8_raw(sc[t][0][0], sc[t][0][1], sc[t][0][2], sc[t][0][3], sc[t][1][0], sc[t][1][1],
                                  sc[t][1][2], sc[t][1][3]);
      hit = hit || lmax + top > lim[t];
    }
    if (__any(hit)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) m = fmaxf(m, sc[t][j][e] + norm_exponent(vn[j][e]));
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const bool move = m > lim[t];
        const float shift = move ? m - PUP : 0.f;
        const float alpha = !move ? 1.f : lim[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-shift);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[t][j][e] -= shift;
        mref[t] += shift;
        lim[t] = move ? TAU + PUP : lim[t];
        l_run[t] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[t][db] *= alpha;
      }
    }
    // ---- value words: the lane's field of each of its keys, key pairs interleaved: f[par][j][c] holds
    // the even (0) or odd (1) dims of keys 16j + 4lg + 2c, + 1
    constexpr uint32_t M = odd_fields<VB>();
    uint32_t f[2][2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(src + OFF_V + (16 * j + 4 * lg + kk) * VC + vbase);
        if constexpr (VW32 == 2) w[kk] = __builtin_amdgcn_alignbit(vp[1], vp[0], vshift);
        else w[kk] = vp[0] >> vshift;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        f[0][j][c] = bfi32(M, w[2 * c + 1] << VB, w[2 * c]);
        f[1][j][c] = bfi32(M, w[2 * c + 1], w[2 * c] >> VB);
      }
    }
    // ---- P vn as the f16 operand
    half8 pb[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float p[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) p[j][e] = __builtin_amdgcn_exp2f(sc[t][j][e]);
      l_run[t] += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = i >> 1, e = 2 * (i & 1);
        uint32_t v0 = vn[j][e], v1 = vn[j][e + 1];
        if constexpr (EDGE) {  // a masked key's norm may be anything: it takes no part in the product
          v0 = sc[t][j][e] == -INFINITY ? 0 : v0;
          v1 = sc[t][j][e + 1] == -INFINITY ? 0 : v1;
        }
        w[i] = mul2_f16(p[j][e], v0, p[j][e + 1], v1);
      }
      pb[t] = __builtin_bit_cast(half8, w);
    }
    // ---- O^T += V^T (P vn)^T over the slab's 32 keys: K slot 8lg + 4j + e is key 16j + 4lg + e; an A
    // dword is one dim of a key pair, read from the pair table
#pragma unroll
    for (int par = 0; par < 2; ++par)
      static_for<NPAIR>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const half8 va = __builtin_bit_cast(
            half8, u32x4{value_pair<VB, i>(tV, f[par][0][0]), value_pair<VB, i>(tV, f[par][0][1]),
                         value_pair<VB, i>(tV, f[par][1][0]), value_pair<VB, i>(tV, f[par][1][1])});
#pragma unroll
        for (int t = 0; t < NT; ++t) oacc[t][2 * i + par] = mfma16x16x32(va, pb[t], oacc[t][2 * i + par]);
      });
  };

  // first the slabs of cached keys only, then those that hold drafted tokens or end the part
  int slot = 0, ks0 = k0w;
  auto slabs = [&](auto edge_c, int end) {
    stream.template run<RK, SLOT>(ks0, end, nrows, slot, mine_lds,
                            [&](int at, int k0, int rows) { slab(edge_c, mine + at * SLOT, k0, rows); });
  };
  slabs(std::false_type{}, min(kend, nctx) - (NK - 1));
  if constexpr (!SHARED) slabs(std::true_type{}, kend);

  // ---- the waves' states joined in LDS, one column tile at a time (the rings are done)
  constexpr int LDM = SM::LDM;
  float* const mrg = reinterpret_cast<float*>(area);  // [wave][column][LDM]
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    __syncthreads();
    float l = l_run[t];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    float* const my = mrg + (wave * 16 + l16) * LDM;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int db = 0; db < DB; db += 4)
        *reinterpret_cast<float4v*>(my + (lg * 4 + e) * DB + db) =
            float4v{oacc[t][db][e], oacc[t][db + 1][e], oacc[t][db + 2][e], oacc[t][db + 3][e]};
    if (lg == 0) {
      // a node without a place leaves an empty record; a column of NaN scores, whose maximum never
      // moved, a NaN one
      my[D] = !anc[t] || (lim[t] == -INFINITY && l == l) ? -INFINITY : mref[t];
      my[D + 1] = l;
    }
    __syncthreads();
    tree_join<D, NW, 16>(a, mrg, p.rec + 16 * t, p.cols - ct0 - 16 * t, tid);
  }
}

// ---------------------------------------------------------------- the end of a merge
// out^T = Pi_v^T o^T for 4 CW normalised columns of a kv head, on MFMA with both operands split into
// f16 hi + lo.  A block of 4 waves; Pi_v's fragments are loaded when it is made.
template <int D, int CW>
struct TreeFinish {
  static constexpr int PL = D / 64, RB = D / 64, NC = 4 * CW;
  typedef float floatPL __attribute__((ext_vector_type(PL)));  // a lane's dims of a column
  struct Smem {
    __attribute__((aligned(16))) float o[NC][D + 4];
    float up[NC];
  };
  half8 ah[RB][D / 32], al[RB][D / 32];
  __device__ __forceinline__ explicit TreeFinish(const TreeArgs& a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, lg = lane >> 4;
    const _Float16* Ph = reinterpret_cast<const _Float16*>(a.vpit);
    const _Float16* Pl = Ph + D * D;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int i = wave * (D / 4) + rb * 16 + l16;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        ah[rb][ks] = *reinterpret_cast<const half8*>(Ph + i * D + ks * 32 + lg * 8);
        al[rb][ks] = *reinterpret_cast<const half8*>(Pl + i * D + ks * 32 + lg * 8);
      }
    }
  }
  // column cc of the block, by one wave
  __device__ __forceinline__ static void put(Smem& s, int cc, floatPL o) {
    const int lane = threadIdx.x & 63;
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < PL; ++e) {
      s.o[cc][PL * lane + e] = o[e];
      m = fmaxf(m, fabsf(o[e]));
    }
#pragma unroll
    for (int sh = 32; sh >= 1; sh >>= 1) m = fmaxf(m, __shfl_xor(m, sh, 64));
    if (lane == 0) {
      int ex;
      frexpf(fminf(m, 3.0e38f), &ex);
      s.up[cc] = m > 0.f ? ldexpf(kSplit, -ex) : 1.f;  // scaled |o| < kSplit
    }
  }
  // columns [c0, c0 + NC) of sequence b's C, put() and a barrier behind them
  __device__ __forceinline__ void store(const TreeArgs& a, const Smem& s, int b, int hkv, int c0) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, lg = lane >> 4;
    const int lc = l16 & (NC - 1);  // with fewer than 16 columns the others repeat them and are not stored
    const float up = s.up[lc];
    half8 bh[D / 32], bl[D / 32];
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        _Float16 h, lo;
        split_f16(s.o[lc][ks * 32 + lg * 8 + e] * up, h, lo);
        bh[ks][e] = h;
        bl[ks][e] = lo;
      }
    const int c = c0 + l16;
    const bool mine = l16 < NC && c < a.C;
    const int qi = mine ? c / a.G : 0, h = hkv * a.G + (mine ? c % a.G : 0);
    const float down = kUnsplit2 / up * kSplit;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float4v f = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        f = mfma16x16x32(ah[rb][ks], bh[ks], f);
        f = mfma16x16x32(al[rb][ks], bh[ks], f);
        f = mfma16x16x32(ah[rb][ks], bl[ks], f);
      }
      if (mine) {
        const int64_t off = static_cast<int64_t>(b) * a.sob + static_cast<int64_t>(h) * a.soh +
                            static_cast<int64_t>(qi) * a.sos + wave * (D / 4) + rb * 16 + lg * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = f[e] * down;
          if (a.out_dtype == TQ_BF16) store_act<TQ_BF16>(a.out, off + e, v);
          else if (a.out_dtype == TQ_F16) store_act<TQ_F16>(a.out, off + e, v);
          else store_act<TQ_F32>(a.out, off + e, v);
        }
      }
    }
  }
};

// Tree attention's workspace and launch; `a` holds what the caller gave (shapes, operands, output).
int64_t tree_workspace(int B, int Hq, int Hkv, int T, int64_t maxpos, int d, int bits);
void tree_attend(TreeArgs a, int d, int bits, void* workspace, hipStream_t s);

}  // namespace tq
