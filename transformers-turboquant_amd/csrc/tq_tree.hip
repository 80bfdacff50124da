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
// length of sequence b, -1 behind the last
__device__ __forceinline__ int tree_length(const TreeArgs& a, int b) { return b < a.B ? a.lengths[b] : -1; }
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

template <int D, int BITS, int NT, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))
tree_attn_kernel(TreeArgs a) {
  using SM = TreeSmem<D, BITS, NT, NW>;
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
  constexpr int QKIND = SM::QKIND;
  constexpr bool HOLD_HI = NT == 1 || D == 64;  // q_proj hi fragments in registers
  constexpr bool AHEAD = NT == 1;  // score operands looked up a step ahead, where registers allow
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr float TAU = kTau, PUP = kPup;

  __shared__ __attribute__((aligned(16))) SM sm;
  uint8_t* const luts = sm.luts;
  uint8_t* const area = sm.area;
  const uint8_t* tS = luts + L::SGN_OFF;
  const uint8_t* tK = luts + L::KEY_OFF;
  const uint8_t* tV = luts + L::VAL_OFF;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int ct0 = blockIdx.y * (16 * NT), hkv = blockIdx.z;
  const int n0 = tree_length(a, lane);
  const TreeTables<BITS> tables(a, tid);
  const TreeSplit<RK> split(a, n0);
  if (static_cast<int>(blockIdx.x) >= split.blocks) return;  // block-uniform
  int x = split.begin(blockIdx.x);
  const int x_end = split.begin(blockIdx.x + 1);

  tables.keys(luts, tid);
  tables.values(luts, tid);
  const float fa = a.scale * LOG2E;
  float qs;
  const int vbit = l16 * VFB, vbase = (vbit >> 5) * 4, vshift = vbit & 31;
  uint8_t* const mine = area + wave * (R * SLOT);
  const uint32_t mine_lds = lds_offset(mine);

  // ---- one part after the other: the rounds of this block's stretch that belong to one sequence
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
    constexpr int TPC = 64 * NW / (16 * NT), DPT = D / TPC;  // threads per column, dims per thread
    static_assert(DPT == 4 || DPT == 8 || DPT == 16, "whole fragments or halves of one");
    const int qcol = tid / TPC, d0 = (tid % TPC) * DPT;
    float4v pj4[DPT / 4];
    half4 rt4[DPT / 4];
    {
      const int c = min(ct0 + qcol, a.C - 1), node = c / a.G;
      const int64_t row = ((static_cast<int64_t>(b) * a.Hq + hkv * a.G + (c - node * a.G)) * a.T + node) * D + d0;
#pragma unroll
      for (int i = 0; i < DPT / 4; ++i) {
        pj4[i] = *reinterpret_cast<const float4v*>(a.q_proj + row + 4 * i);
        rt4[i] = *reinterpret_cast<const half4*>(a.q_rot + row + 4 * i);
      }
    }
    const uint64_t anc_lane = tree_ancestors(a, par);
    if (wave == 0) sm.anc[lane] = anc_lane;
    const uint64_t live = __ballot(anc_lane != 0);  // tokens with a place: some node sees them
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
      m = wave_max(m);
      if (lane == 0) sm.qmax[wave] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, sm.qmax[w]);
      qs = fminf(qproj_split_scale(m), 0x1p100f);
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
    const float fs = fa / qs;
    auto qfrag = [&](int kind, int t, int ks) -> half8 {
      return *reinterpret_cast<const half8*>(sm.q + kind * QKIND + ((t * KS + ks) * 64 + lane) * 16);
    };
    uint64_t anc[NT];  // of the lane's column in each tile
    half8 qr[NT][KS], qh[HOLD_HI ? NT : 1][KS];  // held; the others are read from LDS at their use
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      anc[t] = sm.anc[min(ct0 + 16 * t + l16, a.C - 1) / a.G];
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
            const float x = fmaf(fma_f16(s1[t][j][e], kn[j][e], mul_f16(s2[t][j][e], rn[j][e])), fs, -mref[t]);
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
    slabs(std::true_type{}, kend);

    // ---- the waves' states joined in LDS, one column tile at a time (the rings are done)
    constexpr int LDM = SM::LDM;
    float* const mrg = reinterpret_cast<float*>(area);  // [wave][column][LDM]
    const int64_t base = (static_cast<int64_t>(rec) * a.Hkv + hkv) * a.C + ct0;
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
      tree_join<D, NW, 16>(a, mrg, base + 16 * t, a.C - ct0 - 16 * t, tid);
    }
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
  constexpr int PL = D / 64, RB = D / 64, NC = 4 * CW, NB = 16 / CW;
  typedef float floatPL __attribute__((ext_vector_type(PL)));
  __shared__ __attribute__((aligned(16))) float o_s[NC][D + 4];
  __shared__ float s_up[NC];
  const int c0 = blockIdx.x * NC, hkv = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, l16 = lane & 15, lg = lane >> 4;

  const int n0 = tree_length(a, lane);  // before Pi_v: waited for first
  const _Float16* Ph = reinterpret_cast<const _Float16*>(a.vpit);
  const _Float16* Pl = Ph + D * D;
  half8 ah[RB][D / 32], al[RB][D / 32];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int i = wave * (D / 4) + rb * 16 + l16;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) {
      ah[rb][ks] = *reinterpret_cast<const half8*>(Ph + i * D + ks * 32 + lg * 8);
      al[rb][ks] = *reinterpret_cast<const half8*>(Pl + i * D + ks * 32 + lg * 8);
    }
  }
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
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < PL; ++e) {
      o_s[cc][PL * lane + e] = o[e];
      m = fmaxf(m, fabsf(o[e]));
    }
#pragma unroll
    for (int sh = 32; sh >= 1; sh >>= 1) m = fmaxf(m, __shfl_xor(m, sh, 64));
    if (lane == 0) {
      int ex;
      frexpf(fminf(m, 3.0e38f), &ex);
      s_up[cc] = m > 0.f ? ldexpf(kSplit, -ex) : 1.f;  // scaled |o| < kSplit
    }
  }
  __syncthreads();

  const int lc = l16 & (NC - 1);  // with fewer than 16 columns the others repeat them and are not stored
  const float up = s_up[lc];
  half8 bh[D / 32], bl[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      _Float16 h, lo;
      split_f16(o_s[lc][ks * 32 + lg * 8 + e] * up, h, lo);
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

}  // namespace tq

using namespace tq;

extern "C" {

int64_t tq_tree_workspace_size(int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t table_width, int32_t page_size,
                               int32_t d, int32_t bits) {
  const int64_t maxpos = static_cast<int64_t>(table_width) * page_size;
  return tree_shape(B, Hq, Hkv, T, maxpos, d, bits) ? plan_tree(B, Hq, Hkv, T, maxpos, d, bits).bytes : 0;
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
  const TreePlan p = plan_tree(B, Hq, Hkv, T, maxpos, d, bits);
  TQ_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= p.bytes,
             "tq_tree_attention: the workspace must be 16-byte aligned and hold %lld bytes", (long long)p.bytes);
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
  a.slots = p.slots;
  a.lg_least = p.lg_least;
  a.coeff = coeff;
  a.scale = scale;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + (static_cast<int64_t>(p.slots) + B) * Hkv * a.C * d;
  a.vpit = val_pit_split;
  a.out = out;
  a.out_dtype = out_dtype;
  a.sob = sob;
  a.soh = soh;
  a.sos = sos;
  hipStream_t s = as_stream(stream);
  if (d == 64) launch_tree<64>(a, p, s);
  else launch_tree<128>(a, p, s);
  return launch_status("tq_tree_attention");
}

}  // extern "C"
