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
// The columns of a kv head are its G query heads times the T nodes, c = i G + g.  A block takes NT
// tiles of 16 columns of one kv head against a run of keys; each of its waves streams slabs of 32
// keys of the packed planes into its own LDS ring, builds the MFMA operands of a slab once
// through small lookup tables and uses them for every column tile: keys on the M side, so that
// the scores a lane ends with (4 keys x its column) are its own part of P^T, the operand of
// O^T += V^T P^T.  With 16 columns the stream of packed bytes bounds the work, from 32 on
// the matrix products do, which is why the decoded operands are shared by the column tiles.
//
// Lengths live on the device (a captured graph replays with other lengths), so the split of the
// keys is made there: all sequences are cut into chunks of one common number of rounds (a
// round: 32 keys per wave), chosen so that about `slots` chunks exist in all; long
// sequences get many, short ones few.  A chunk leaves its (maximum, sum, O) in a record; the
// merge joins a sequence's records, normalises and applies Pi_v.
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
  int slots;            // chunks aimed at, over all sequences
  int nrec;             // records (blocks along x)
  float coeff, scale;
  float *part_o, *part_ml;  // records [nrec, Hkv, C, D], [nrec, Hkv, C, 2]
  const uint16_t* vpit;
  void* out;
  int out_dtype;
  int64_t sob, soh, sos;
};

// ---------------------------------------------------------------- the split of the keys
// keys of sequence b (cached and drafted), 0 where its length does not fit its table
__device__ __forceinline__ int tree_keys(const TreeArgs& a, int b) {
  const int n = a.lengths[b];
  return n >= 0 && n <= a.maxpos - a.T ? n + a.T : 0;
}
// Every wave of a block computes the same, 64 sequences per step (one per lane).
template <int RK>
struct TreeSplit {
  int chunk;  // rounds per chunk
  __device__ __forceinline__ static int rounds(const TreeArgs& a, int b) {
    return b < a.B ? (tree_keys(a, b) + RK - 1) / RK : 0;
  }
  __device__ __forceinline__ explicit TreeSplit(const TreeArgs& a) {
    const int lane = threadIdx.x & 63;
    int total = 0;
    for (int b = lane; b < a.B; b += 64) total += rounds(a, b);
#pragma unroll
    for (int sh = 32; sh >= 1; sh >>= 1) total += __shfl_xor(total, sh, 64);
    chunk = __builtin_amdgcn_readfirstlane(max(1, (total + a.slots - 1) / a.slots));
  }
  __device__ __forceinline__ static int scan(int v) {  // inclusive sum over the wave
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int sh = 1; sh < 64; sh <<= 1) {
      const int t = __shfl_up(v, sh, 64);
      if (lane >= sh) v += t;
    }
    return v;
  }
  // the sequence of record `rec` and its chunk within the sequence; false behind the last record
  __device__ __forceinline__ bool find(const TreeArgs& a, int rec, int& b, int& k) const {
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int c = (rounds(a, b0 + lane) + chunk - 1) / chunk;
      const int upto = scan(c);
      const uint64_t m = __ballot(rec < upto);
      if (m) {
        const int l = __builtin_ctzll(m);
        b = __builtin_amdgcn_readfirstlane(b0 + l);
        k = __builtin_amdgcn_readfirstlane(rec - __shfl(upto - c, l, 64));
        return true;
      }
      rec -= __builtin_amdgcn_readfirstlane(__shfl(upto, 63, 64));
    }
    return false;
  }
  // first record of sequence b and how many it has
  __device__ __forceinline__ void records(const TreeArgs& a, int b, int& first, int& n) const {
    const int lane = threadIdx.x & 63;
    first = 0;
    for (int b0 = 0;; b0 += 64) {
      const int c = (rounds(a, b0 + lane) + chunk - 1) / chunk;
      const int upto = scan(c);
      if (b < b0 + 64) {
        first = __builtin_amdgcn_readfirstlane(first + __shfl(upto - c, b - b0, 64));
        n = __builtin_amdgcn_readfirstlane(__shfl(c, b - b0, 64));
        return;
      }
      first += __shfl(upto, 63, 64);
    }
  }
};

// Bit t of the result: node `lane` sees drafted token t (its ancestors and itself).  A parent that
// is neither -1 nor an earlier node leaves the node without a place: it sees nothing and nothing
// sees it.  Pointer doubling: after k steps a lane has its next 2^k ancestors.
__device__ __forceinline__ uint64_t tree_ancestors(const TreeArgs& a, int b) {
  const int i = threadIdx.x & 63;
  int par = -2;
  if (i < a.T) par = a.parents ? a.parents[b * a.ld_parents + i] : i - 1;
  const bool placed = par >= -1 && par < i;
  uint64_t seen = placed ? 1ull << i : 0;
  int up = placed ? par : -1;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
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

// ---------------------------------------------------------------- attention
template <int D, int BITS, int NT, int NW>
struct TreeSmem {
  using L = SmallLuts<BITS>;
  static constexpr int KC = D * L::KB / 8, SC = D / 8, VC = D * L::VB / 8;
  static constexpr int NK = 32;  // keys of a wave's slab
  static constexpr int OFF_K = 0, OFF_S = NK * KC, OFF_V = OFF_S + NK * SC, OFF_N = OFF_V + NK * VC;
  static constexpr int NRM = NK * 4;
  static constexpr int SLOT = OFF_N + 3 * NRM;
  static constexpr int R = 2;
  static constexpr int QF = 3 * (D / 32);  // query fragments of a column tile: q_rot, q_proj hi, lo
  static constexpr int QBYTES = NT > 1 ? NT * QF * 1024 : 0;
  static constexpr int RING = NW * R * SLOT;
  static constexpr int MERGE = NW * 16 * (D + 2) * 4;
  static constexpr int MAIN = RING + QBYTES > MERGE ? RING + QBYTES : MERGE;
};

template <int D, int BITS, int NT, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NT == 1 ? 3 : 2)))
tree_attn_kernel(TreeArgs a) {
  using SM = TreeSmem<D, BITS, NT, NW>;
  using L = typename SM::L;
  constexpr int KB = L::KB, VB = L::VB;
  constexpr int KS = D / 32;           // score k-steps
  constexpr int DB = D / 16;           // value row blocks: lane l16 holds dims DB l16 .. DB l16 + DB - 1
  constexpr int NPAIR = D / 32;        // pair-table groups per parity
  constexpr int KC = SM::KC, SC = SM::SC, VC = SM::VC;
  constexpr int KLANE = KC / 4, KW32 = (KLANE + 3) / 4, SLANE = SC / 4;
  constexpr int VFB = DB * VB;
  constexpr int VW32 = (VB == 3) ? 2 : 1;
  constexpr int NK = SM::NK, RK = NW * NK;
  constexpr int OFF_K = SM::OFF_K, OFF_S = SM::OFF_S, OFF_V = SM::OFF_V, OFF_N = SM::OFF_N, NRM = SM::NRM;
  constexpr int SLOT = SM::SLOT, R = SM::R, QF = SM::QF;
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr float TAU = 8.0f;  // a column's reference moves when a score exceeds it by more (log2 units)
  // weights are 2^(s - m + PUP) <= 2^(TAU + PUP): keys down to ~2^-31 of the heaviest still reach
  // the f16 operand P, whose subnormals end at 2^-24, and p vn / vcap stays below the f16 maximum
  constexpr float PUP = 6.0f;

  __shared__ __attribute__((aligned(16))) uint8_t luts[L::BYTES];
  __shared__ __attribute__((aligned(16))) uint8_t area[SM::MAIN];
  __shared__ __attribute__((aligned(16))) float fac[NW][3][NK];  // a slab's fa vn_k, fb rn_k, vn_v / vcap
  __shared__ uint64_t s_anc[64];
  __shared__ float s_max[NW];
  const uint8_t* tS = luts + L::SGN_OFF;
  const uint8_t* tK = luts + L::KEY_OFF;
  const uint8_t* tV = luts + L::VAL_OFF;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int rec = blockIdx.x, ct0 = blockIdx.y * (16 * NT), hkv = blockIdx.z;
  const TreeSplit<RK> split(a);
  int b = 0, part = 0;
  if (!split.find(a, rec, b, part)) return;  // block-uniform
  const int nkeys = tree_keys(a, b), nctx = nkeys - a.T;
  const int kbeg = part * split.chunk * RK, kend = min(nkeys, kbeg + split.chunk * RK);

  {
    DecodeArgs t{};
    t.kcent = a.kcent;
    t.vcent = a.vcent;
    for (int i = tid; i < 256; i += 64 * NW) build_small_luts<BITS, true>(t, luts, i);
  }
  const uint64_t anc_lane = tree_ancestors(a, b);
  if (wave == 0) s_anc[lane] = anc_lane;
  // drafted tokens that some node sees; the rows of the others count as empty
  uint64_t live = anc_lane;
#pragma unroll
  for (int sh = 32; sh >= 1; sh >>= 1) live |= __shfl_xor(live, sh, 64);

  // ---- the block's queries as B fragments.  q_proj (f32) enters as f16 hi + lo parts, scaled
  // together by a power of two that keeps both in range (qproj_split_scale)
  auto qrow_of = [&](int c) {
    return ((static_cast<int64_t>(b) * a.Hq + hkv * a.G + c % a.G) * a.T + c / a.G) * D;
  };
  float qmax = 0.f;
  for (int c = wave; c < 16 * NT; c += NW) {
    if (ct0 + c < a.C) {
      const float* q = a.q_proj + qrow_of(ct0 + c);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) qmax = fmaxf(qmax, fabsf(q[e * 64 + lane]));
    }
  }
  qmax = wave_max(qmax);
  if (lane == 0) s_max[wave] = qmax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) qmax = fmaxf(qmax, s_max[w]);
  const float qs = qproj_split_scale(qmax);
  const float fa = a.scale * LOG2E;
  const float fb = a.coeff * fa / qs;

  uint64_t anc[NT];  // of the lane's column in each tile
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = ct0 + 16 * t + l16;
    anc[t] = c < a.C ? s_anc[c / a.G] : 0;
  }
  half8 qreg[NT == 1 ? QF : 1];
  uint8_t* const qlds = area + SM::RING;
  auto fragments = [&](int t, half8 (&f)[QF]) {
    const int c = ct0 + 16 * t + l16;
    const int64_t row = c < a.C ? qrow_of(c) : 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = lg * (D / 4) + ks * 8;
      half8 hi = half8{}, lo = half8{}, r = half8{};
      if (c < a.C) {
        split8s(a.q_proj + row + d0, qs, hi, lo);
        r = *reinterpret_cast<const half8*>(a.q_rot + row + d0);
      }
      f[ks] = r;
      f[KS + ks] = hi;
      f[2 * KS + ks] = lo;
    }
  };
  if constexpr (NT == 1) {
    fragments(0, qreg);
  } else {
    for (int t = wave; t < NT; t += NW) {
      half8 f[QF];
      fragments(t, f);
#pragma unroll
      for (int i = 0; i < QF; ++i) *reinterpret_cast<half8*>(qlds + ((t * QF + i) * 64 + lane) * 16) = f[i];
    }
  }
  auto qfrag = [&](int t, int f) -> half8 {
    if constexpr (NT == 1) return qreg[f];
    else return *reinterpret_cast<const half8*>(qlds + ((t * QF + f) * 64 + lane) * 16);
  };

  // ---- the stream
  const int vbit = l16 * VFB, vbase = (vbit >> 5) * 4, vshift = vbit & 31;
  uint8_t* const mine = area + wave * (R * SLOT);
  const uint32_t mine_lds = lds_offset(mine);
  constexpr int NKD = (NK * KC + 1023) / 1024, NSD = (NK * SC + 1023) / 1024, NVD = (NK * VC + 1023) / 1024;
  constexpr int NDMA = NKD + NSD + NVD + 3;
  auto copy_plane = [&](const i32x4& r, uint32_t dst, int bytes, int nrounds) {
    const uint32_t lo = lane * 16;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c >= nrounds) break;
      if ((c + 1) * 1024 <= bytes || lane * 16 < bytes - c * 1024) dma16(r, dst + c * 1024, lo + c * 1024);
    }
  };
  // rows of a slab that exist: up to the chunk's last key, none where its page is not in the pool.
  // A slab's 32 keys lie in one page (pages hold 32 or more, slabs start at multiples of 32).
  auto page_of = [&](int kb) -> int {
    const int p = a.table[b * a.ld_table + (kb >> a.lg_page)];
    return __builtin_amdgcn_readfirstlane(p);
  };
  auto issue = [&](int kb, int slot) {
    const int page = page_of(kb);
    const bool in = page >= 0 && page < a.num_pages;
    const int64_t row = in ? ((static_cast<int64_t>(page) * a.Hkv + hkv) << a.lg_page) + (kb & ((1 << a.lg_page) - 1)) : 0;
    const int rows = in ? min(NK, kend - kb) : 0;
    const uint32_t dst = mine_lds + slot * SLOT;
    wait_lds();  // earlier reads of this slot have landed
    copy_plane(rows_desc(a.kcodes + row * KC, KC, 0, rows), dst + OFF_K, NK * KC, NKD);
    copy_plane(rows_desc(a.ksigns + row * SC, SC, 0, rows), dst + OFF_S, NK * SC, NSD);
    copy_plane(rows_desc(a.vcodes + row * VC, VC, 0, rows), dst + OFF_V, NK * VC, NVD);
    if (lane < 32) {
      dma_u16(rows_desc(a.kvn + row, 2, 0, rows), dst + OFF_N, lane * 2);
      dma_u16(rows_desc(a.krn + row, 2, 0, rows), dst + OFF_N + NRM, lane * 2);
      dma_u16(rows_desc(a.vvn + row, 2, 0, rows), dst + OFF_N + 2 * NRM, lane * 2);
    }
  };
  auto wait_slot = [&](int later) {
    if (later >= 1) wait_vm<NDMA>();
    else wait_vm<0>();
  };

  float m_run[NT], l_run[NT];
  // value norms enter P as vn / vcap <= 1; vcap is a power of two that only grows (O is rescaled
  // when it does) and multiplies O back at the end
  float vcap = 0x1p-24f, inv_vcap = 0x1p24f;
  float4v oacc[NT][DB];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m_run[t] = -INFINITY;
    l_run[t] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) oacc[t][db] = float4v{0.f, 0.f, 0.f, 0.f};
  }
  float (*fw)[NK] = fac[wave];

  auto slab = [&](const uint8_t* src, int ks0) {
    const int page = page_of(ks0);
    const int rows = page >= 0 && page < a.num_pages ? min(NK, kend - ks0) : 0;
    const bool edge = rows < NK || ks0 + NK > nctx;  // wave-uniform: a visibility to look up
    // ---- per-key factors, one value per lane and pass; keys that nobody sees get zeros
#pragma unroll
    for (int i0 = 0; i0 < 3 * NK; i0 += 64) {
      const int i = i0 + lane, which = i / NK, k = i % NK;
      float v = (i < 3 * NK)
          ? h2f(static_cast<uint16_t>(*reinterpret_cast<const uint32_t*>(src + OFF_N + which * NRM + k * 4)))
          : 0.f;
      if (edge) {
        const int t = ks0 + k - nctx;
        if (k >= rows || (t >= 0 && !((live >> (t & 63)) & 1))) v = 0.f;
      }
      if (i0 + 63 >= 2 * NK) {  // this pass holds value norms: keep them <= vcap
        const float vv = (which == 2) ? v : 0.f;
        if (__any(vv > vcap)) {
          float t = fminf(vv, 65504.f);
#pragma unroll
          for (int sh = 32; sh >= 1; sh >>= 1) t = fmaxf(t, __shfl_xor(t, sh, 64));
          int ex;
          frexpf(t, &ex);  // t < 2^ex; every lane holds the same t
          ex = __builtin_amdgcn_readfirstlane(ex);
          const float cap = ldexpf(1.f, ex);
          if (cap > vcap) {
            const float shrink = vcap / cap;
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
              for (int db = 0; db < DB; ++db) oacc[c][db] *= shrink;
            vcap = cap;
            inv_vcap = ldexpf(1.f, -ex);
          }
        }
      }
      if (i < 3 * NK) fw[which][k] = (which == 0) ? fa * v : (which == 1 ? fb * v : v * inv_vcap);
    }
    // ---- the slab's key operands, shared by the column tiles
    half8 kc[2][KS], sg[2][KS];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t kw[KW32];
      load_key_field<KLANE>(src + OFF_K + (16 * j + l16) * KC + lg * KLANE, kw);
      const uint32_t sw = load_sign_field<D>(src + OFF_S + (16 * j + l16) * SC + lg * SLANE);
      static_for<KS>([&](auto cc) {
        constexpr int ks = decltype(cc)::value;
        kc[j][ks] = key_operand<KB, KW32, ks>(tK, kw);
        sg[j][ks] = nib2x4<ks>(tS, sw);
      });
    }
    // ---- scores, softmax step and P of one column tile after the other
    half8 pb[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float4v s1[2], s2[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s1[j] = float4v{0.f, 0.f, 0.f, 0.f};
        s2[j] = float4v{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const half8 qr = qfrag(t, ks), qh = qfrag(t, KS + ks), ql = qfrag(t, 2 * KS + ks);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s1[j] = mfma16x16x32(kc[j][ks], qr, s1[j]);
          s2[j] = mfma16x16x32(sg[j][ks], qh, s2[j]);
          s2[j] = mfma16x16x32(sg[j][ks], ql, s2[j]);
        }
      }
      float sc[2][4];  // log2-domain scores of keys ks0 + 16j + 4lg + e for this lane's column
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4v ka = *reinterpret_cast<const float4v*>(&fw[0][16 * j + 4 * lg]);
        const float4v kb2 = *reinterpret_cast<const float4v*>(&fw[1][16 * j + 4 * lg]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j][e] = fmaf(s2[j][e], kb2[e], s1[j][e] * ka[e]);
      }
      if (edge) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = 16 * j + 4 * lg + e, d = ks0 + k - nctx;
            const bool sees = k < rows && (d < 0 || ((anc[t] >> (d & 63)) & 1));
            if (!sees) sc[j][e] = -INFINITY;
          }
      }
      const float lmax = max8_raw(sc[0][0], sc[0][1], sc[0][2], sc[0][3], sc[1][0], sc[1][1], sc[1][2], sc[1][3]);
      if (__any(lmax > m_run[t] + TAU)) {
        float x = lmax;
        x = fmaxf(x, __shfl_xor(x, 16, 64));
        x = fmaxf(x, __shfl_xor(x, 32, 64));
        if (x > m_run[t] + TAU) {
          const float alpha = (m_run[t] == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(m_run[t] - x);
          m_run[t] = x;
          l_run[t] *= alpha;
#pragma unroll
          for (int db = 0; db < DB; ++db) oacc[t][db] *= alpha;
        }
      }
      const float m_use = (m_run[t] == -INFINITY) ? 0.f : m_run[t] - PUP;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4v nv = *reinterpret_cast<const float4v*>(&fw[2][16 * j + 4 * lg]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(sc[j][e] - m_use);
          l_run[t] += p;
          // a masked key's norm may be anything: it takes no part in the product
          const float pv = edge && sc[j][e] == -INFINITY ? 0.f : p * nv[e];
          pb[t][4 * j + e] = static_cast<_Float16>(pv);
        }
      }
    }
    // ---- O^T += V^T (P vn)^T over the slab's 32 keys: K slot 8lg + 4j + e is key 16j + 4lg + e;
    // an A dword is one dim of a key pair, read from the pair table after interleaving the two
    // keys' code fields (parity 0: even dims, 1: odd dims)
    constexpr uint32_t M = odd_fields<VB>();
    uint32_t w[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(src + OFF_V + (16 * j + 4 * lg + kk) * VC + vbase);
        if constexpr (VW32 == 2) w[j][kk] = __builtin_amdgcn_alignbit(vp[1], vp[0], vshift);
        else w[j][kk] = vp[0] >> vshift;
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
      static_for<NPAIR>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const half8 va = __builtin_bit_cast(half8, u32x4{value_pair<VB, i>(tV, f[0][0]), value_pair<VB, i>(tV, f[0][1]),
                                                         value_pair<VB, i>(tV, f[1][0]), value_pair<VB, i>(tV, f[1][1])});
#pragma unroll
        for (int t = 0; t < NT; ++t) oacc[t][2 * i + par] = mfma16x16x32(va, pb[t], oacc[t][2 * i + par]);
      });
    }
  };

  __builtin_amdgcn_s_waitcnt(0);  // no load of the compiler's own reaches back past a copy
  const int k0w = kbeg + wave * NK;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (k0w + r * RK < kend) issue(k0w + r * RK, r);
  __syncthreads();  // tables and queries in place
  for (int k0 = k0w; k0 < kend; k0 += R * RK) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int ks0 = k0 + r * RK;
      if (ks0 < kend) {
        wait_slot(ks0 + RK < kend ? 1 : 0);
        slab(mine + r * SLOT, ks0);
        if (ks0 + R * RK < kend) issue(ks0 + R * RK, r);
      }
    }
  }

  // ---- the waves' states joined in LDS, one column tile at a time (rings and queries are done)
  float* const mrg = reinterpret_cast<float*>(area);  // [wave][column][D + 2]
  const int64_t base = (static_cast<int64_t>(rec) * a.Hkv + hkv) * a.C + ct0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    __syncthreads();
    float l = l_run[t];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    float* my = mrg + (wave * 16 + l16) * (D + 2);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e) my[(lg * 4 + e) * DB + db] = oacc[t][db][e] * vcap;
    if (lg == 0) {
      // a node without a place leaves an empty record; a column of NaN scores, whose maximum never
      // moved, a NaN one
      my[D] = !anc[t] ? -INFINITY : (m_run[t] == -INFINITY && l != l) ? 0.f : m_run[t];
      my[D + 1] = l;
    }
    __syncthreads();
    const int ncol = min(16, a.C - ct0 - 16 * t);
    for (int it = tid; it < ncol * D; it += 64 * NW) {
      const int c = it / D, d = it % D;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) mx = fmaxf(mx, mrg[(w * 16 + c) * (D + 2) + D]);
      float o = 0.f, ls = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float* s = mrg + (w * 16 + c) * (D + 2);
        if (s[D] != -INFINITY) {
          const float f = __builtin_amdgcn_exp2f(s[D] - mx);
          o += f * s[d];
          ls += f * s[D + 1];
        }
      }
      a.part_o[(base + 16 * t + c) * D + d] = o;
      if (d == 0) {
        a.part_ml[(base + 16 * t + c) * 2] = mx;
        a.part_ml[(base + 16 * t + c) * 2 + 1] = ls;
      }
    }
  }
}

// ---------------------------------------------------------------- merge
// One block per (sequence, kv head, 16 columns): wave w joins columns w, w + 4, ... (the records'
// maxima and weights one per lane, then D / 64 dims per lane summed over the records), then
// out^T = Pi_v^T o^T on MFMA with both operands split into f16 hi + lo.
template <int D, int RK>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeArgs a) {
  constexpr int PL = D / 64, RB = D / 64;
  typedef float floatPL __attribute__((ext_vector_type(PL)));
  __shared__ __attribute__((aligned(16))) float o_s[16][D + 4];
  __shared__ float s_up[16];
  const int c0 = blockIdx.x * 16, hkv = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, l16 = lane & 15, lg = lane >> 4;
  const TreeSplit<RK> split(a);
  int first = 0, n = 0;
  split.records(a, b, first, n);

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
  const int64_t step = static_cast<int64_t>(a.Hkv) * a.C;  // columns between records
  for (int k = 0; k < 4; ++k) {
    const int cc = wave + 4 * k, c = c0 + cc;
    floatPL o = floatPL{};
    if (c < a.C) {
      const int64_t at = (static_cast<int64_t>(first) * a.Hkv + hkv) * a.C + c;
      const float* ml = a.part_ml + at * 2;
      const float* src = a.part_o + at * D + PL * lane;
      float mx = -INFINITY;
      for (int r = lane; r < n; r += 64) mx = fmaxf(mx, ml[r * step * 2]);
#pragma unroll
      for (int sh = 32; sh >= 1; sh >>= 1) mx = fmaxf(mx, __shfl_xor(mx, sh, 64));
      float lsum = 0.f;
      for (int r0 = 0; r0 < n; r0 += 64) {
        float w = 0.f;
        if (r0 + lane < n) {
          const float m = ml[(r0 + lane) * step * 2];
          if (m != -INFINITY) {
            w = __builtin_amdgcn_exp2f(m - mx);
            lsum += w * ml[(r0 + lane) * step * 2 + 1];
          }
        }
        const int nb = min(64, n - r0);
        for (int u = 0; u < nb; u += 8) {
          floatPL v[8];
#pragma unroll
          for (int q = 0; q < 8; ++q)
            v[q] = u + q < nb ? *reinterpret_cast<const floatPL*>(src + (r0 + u + q) * step * D) : floatPL{};
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float ww = __shfl(w, (u + q) & 63, 64);
#pragma unroll
            for (int e = 0; e < PL; ++e) o[e] = fmaf(ww, v[q][e], o[e]);
          }
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

  const float up = s_up[l16];
  half8 bh[D / 32], bl[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      _Float16 h, lo;
      split_f16(o_s[l16][ks * 32 + lg * 8 + e] * up, h, lo);
      bh[ks][e] = h;
      bl[ks][e] = lo;
    }
  const int c = c0 + l16;
  if (c >= a.C) return;
  const int qi = c / a.G, h = hkv * a.G + c % a.G;
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

// ---------------------------------------------------------------- launch
struct TreePlan {
  int nt, nw;   // column tiles of a block, waves of a block
  int ncol;     // blocks along the columns
  int slots, nrec;
  int64_t bytes;
};

template <int D, int BITS, int NT, int NW>
static int tree_resident() {
  static int cache[16] = {};
  return resident_blocks(reinterpret_cast<const void*>(&tree_attn_kernel<D, BITS, NT, NW>), 64 * NW, cache);
}
template <int D, int BITS>
static int tree_resident_nt(int nt) {
  return nt == 1 ? tree_resident<D, BITS, 1, 4>() : tree_resident<D, BITS, 2, 4>();
}

static TreePlan plan_tree(int B, int Hq, int Hkv, int T, int64_t maxpos, int d, int bits) {
  TreePlan p{};
  const int C = Hq / Hkv * T;
  p.nt = C <= 16 ? 1 : 2;
  p.nw = 4;
  p.ncol = (C + 16 * p.nt - 1) / (16 * p.nt);
  int res;
  if (d == 64) res = bits == 2 ? tree_resident_nt<64, 2>(p.nt) : bits == 3 ? tree_resident_nt<64, 3>(p.nt) : tree_resident_nt<64, 4>(p.nt);
  else res = bits == 2 ? tree_resident_nt<128, 2>(p.nt) : bits == 3 ? tree_resident_nt<128, 3>(p.nt) : tree_resident_nt<128, 4>(p.nt);
  const int rk = 32 * p.nw;
  p.slots = res / (Hkv * p.ncol);
  if (p.slots < 1) p.slots = 1;
  // sum of ceil(rounds / chunk) <= slots + B, and at most every round
  const int64_t most = static_cast<int64_t>(B) * ((maxpos + rk - 1) / rk);
  const int64_t nrec = static_cast<int64_t>(p.slots) + B < most ? static_cast<int64_t>(p.slots) + B : most;
  p.nrec = static_cast<int>(nrec);
  p.bytes = nrec * Hkv * C * static_cast<int64_t>(d + 2) * 4;
  return p;
}

static bool tree_shape(int B, int Hq, int Hkv, int T, int64_t maxpos, int d, int bits) {
  return B >= 1 && B <= 65535 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hkv <= 65535 && T >= 1 && T <= 64 && maxpos >= T &&
         maxpos <= (int64_t(1) << 24) && (d == 64 || d == 128) && bits >= 2 && bits <= 4 &&
         static_cast<int64_t>(B) * ((maxpos + 127) / 128) < (int64_t(1) << 31);
}

template <int D, int BITS>
static void launch_tree(const TreeArgs& a, const TreePlan& p, hipStream_t s) {
  const dim3 grid(p.nrec, p.ncol, a.Hkv);
  if (p.nt == 1) tree_attn_kernel<D, BITS, 1, 4><<<grid, 256, 0, s>>>(a);
  else tree_attn_kernel<D, BITS, 2, 4><<<grid, 256, 0, s>>>(a);
  tree_merge_kernel<D, 128><<<dim3((a.C + 15) / 16, a.Hkv, a.B), 256, 0, s>>>(a);
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
  a.nrec = p.nrec;
  a.coeff = coeff;
  a.scale = scale;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + static_cast<int64_t>(p.nrec) * Hkv * a.C * d;
  a.vpit = val_pit_split;
  a.out = out;
  a.out_dtype = out_dtype;
  a.sob = sob;
  a.soh = soh;
  a.sos = sos;
  hipStream_t s = as_stream(stream);
  if (d == 64) {
    if (bits == 2) launch_tree<64, 2>(a, p, s);
    else if (bits == 3) launch_tree<64, 3>(a, p, s);
    else launch_tree<64, 4>(a, p, s);
  } else {
    if (bits == 2) launch_tree<128, 2>(a, p, s);
    else if (bits == 3) launch_tree<128, 3>(a, p, s);
    else launch_tree<128, 4>(a, p, s);
  }
  return launch_status("tq_tree_attention");
}

}  // extern "C"
