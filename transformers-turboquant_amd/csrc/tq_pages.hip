// Pages of a compressed cache: rows written into pages, gathered out of them, pages copied, and
// the rows of an accepted path of drafted tokens moved down behind the cached ones.
//
// A pool holds `num_pages` pages of `page_size` positions; every plane of a layer is
// [num_pages, H, page_size, width] bytes, so the positions of one kv head in a page are
// contiguous rows and a page of a plane is one contiguous piece.  A sequence's position j is row
// j % page_size of page block_table[b, j / page_size].  Indices live on the device, so every
// kernel checks them against the pool and the table before it uses them: a row whose page is
// outside the pool (-1 in the table: no page) is neither read nor written.
//
// All of it is bytes that move once in and once out; nothing is computed.  A large copy moves 4.9 TB/s on
// MI355X (in and out together).  Measured, 3 bits, head_dim 128, 8 kv heads, pages of 64:
//   write 4 x 2000 rows (13 MB)       6.0 us, 2.2 TB/s   launch and one round trip
//   read 4 x 9000 positions (37 MB)  11.7 us, 3.1 TB/s   the table's lookup before each piece's load
//   copy 16 pages in 32 layers (53 MB) 9.8 us, 5.4 TB/s  memory
//   keep 16 paths of 16, 32 layers (3 MB) 6.0 us         three dependent round trips
#include "tq_common.h"

namespace tq {

constexpr int kPlanes = 6;  // key codes, signs, rn, vn; value codes, vn

struct PagePlanes {
  uint8_t* pool[kPlanes];
  uint8_t* rows[kPlanes];     // contiguous rows [B, H, S, width] (write: source, read: target)
  uint32_t width[kPlanes];    // bytes per row
  uint32_t unit[kPlanes];     // bytes per copied piece: the largest of 16, 8, 4, 2, 1 that divides the width
  int64_t layer[kPlanes];     // bytes between layers of the pool
  const int32_t* table;
  int64_t ld_table;
  int table_width;
  int64_t num_pages;
  int lg_page;
  int H;
};

template <typename U>
__device__ __forceinline__ void copy_unit(uint8_t* dst, const uint8_t* src) {
  *reinterpret_cast<U*>(dst) = *reinterpret_cast<const U*>(src);
}
__device__ __forceinline__ void copy_piece(uint8_t* dst, const uint8_t* src, uint32_t unit) {
  switch (unit) {
    case 16: copy_unit<uint4>(dst, src); break;
    case 8: copy_unit<uint2>(dst, src); break;
    case 4: copy_unit<uint32_t>(dst, src); break;
    case 2: copy_unit<uint16_t>(dst, src); break;
    default: *dst = *src; break;
  }
}
__device__ __forceinline__ void zero_piece(uint8_t* dst, uint32_t unit) {
  switch (unit) {
    case 16: *reinterpret_cast<uint4*>(dst) = uint4{0, 0, 0, 0}; break;
    case 8: *reinterpret_cast<uint2*>(dst) = uint2{0, 0}; break;
    case 4: *reinterpret_cast<uint32_t*>(dst) = 0; break;
    case 2: *reinterpret_cast<uint16_t*>(dst) = 0; break;
    default: *dst = 0; break;
  }
}

// row of position `pos` of sequence b and head h in any plane of the pool, or -1
__device__ __forceinline__ int64_t page_row(const PagePlanes& a, int b, int h, int64_t pos) {
  if (pos < 0) return -1;
  const int64_t slot = pos >> a.lg_page;
  if (slot >= a.table_width) return -1;
  const int64_t page = a.table[b * a.ld_table + slot];
  if (page < 0 || page >= a.num_pages) return -1;
  return ((page * a.H + h) << a.lg_page) + (pos & ((int64_t(1) << a.lg_page) - 1));
}

// ---------------------------------------------------------------- rows in and out
// WRITE: rows [B, H, S] of the source planes to positions at[b] + s; otherwise positions s < at[b]
// to rows [B, H, S] of the target planes, zeros behind.  A block takes a stretch of one (sequence,
// head, plane).  Code planes move in pieces of a row; the rows of a page are contiguous, so both sides
// run through in order.  Norm planes (2 bytes a row) move in groups of 8 rows that lie together in
// a page; the flat side of a group starts anywhere, so it is accessed as unaligned 16 bytes.  (One piece a
// thread and one norm at a time took 14.6 us for the read above, four pieces in flight and groups 11.7.)
constexpr int kRowSteps = 4;  // pieces of a thread, loaded together (the read above: 11.6 us; with 2 or 8 of them 12.8)
template <bool WRITE>
__device__ __forceinline__ void code_pieces(const PagePlanes& a, int p, int b, int h, int64_t flat_row, int from, int S) {
  const uint32_t unit = a.unit[p], per = a.width[p] / unit;
  const uint32_t n = static_cast<uint32_t>(S) * per, i0 = blockIdx.x * (256 * kRowSteps) + threadIdx.x;
  uint8_t* const flat = a.rows[p] + flat_row * a.width[p];
  uint8_t* pool[kRowSteps];
#pragma unroll
  for (int k = 0; k < kRowSteps; ++k) {
    const uint32_t i = i0 + k * 256, s = i / per;
    pool[k] = nullptr;
    if (i < n && (WRITE || static_cast<int>(s) < from)) {
      const int64_t row = page_row(a, b, h, static_cast<int64_t>(WRITE ? from : 0) + s);
      if (row >= 0) pool[k] = a.pool[p] + row * a.width[p] + (i - s * per) * unit;
    }
  }
  if (unit == 16) {  // the usual widths: every load in flight before the first store
    uint4 v[kRowSteps];
#pragma unroll
    for (int k = 0; k < kRowSteps; ++k) {
      const int64_t i = i0 + k * 256;
      v[k] = uint4{0, 0, 0, 0};
      if (pool[k]) v[k] = *reinterpret_cast<const uint4*>(WRITE ? flat + i * 16 : pool[k]);
    }
#pragma unroll
    for (int k = 0; k < kRowSteps; ++k) {
      const int64_t i = i0 + k * 256;
      if (WRITE && pool[k]) *reinterpret_cast<uint4*>(pool[k]) = v[k];
      if (!WRITE && i < n) *reinterpret_cast<uint4*>(flat + i * 16) = v[k];
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < kRowSteps; ++k) {
    const int64_t i = i0 + k * 256;
    if (WRITE && pool[k]) copy_piece(pool[k], flat + i * unit, unit);
    if (!WRITE && i < n) {
      if (pool[k]) copy_piece(flat + i * unit, pool[k], unit);
      else zero_piece(flat + i * unit, unit);
    }
  }
}

template <bool WRITE>
__device__ __forceinline__ void norm_groups(const PagePlanes& a, int p, int b, int h, int64_t flat_row, int from, int S) {
  const int64_t first = WRITE ? from : 0;  // position of flat row 0
  const int64_t pos = ((first >> 3) + blockIdx.x * 256 + threadIdx.x) << 3;
  if (pos >= first + S) return;
  const int64_t row = page_row(a, b, h, pos);  // a page holds whole groups
  uint16_t* const flat = reinterpret_cast<uint16_t*>(a.rows[p]) + flat_row + (pos - first);
  uint16_t* const pool = reinterpret_cast<uint16_t*>(a.pool[p]) + (row >= 0 ? row : 0);
  const int64_t live = WRITE ? first + S : min(static_cast<int64_t>(from), first + S);
  if (row >= 0 && pos >= first && pos + 8 <= live) {
    uint4 v;
    __builtin_memcpy(&v, WRITE ? flat : pool, 16);
    __builtin_memcpy(WRITE ? pool : flat, &v, 16);
    return;
  }
  for (int j = 0; j < 8; ++j) {
    if (pos + j < first || pos + j >= first + S) continue;
    if constexpr (WRITE) {
      if (row >= 0) pool[j] = flat[j];
    } else {
      flat[j] = row >= 0 && pos + j < live ? pool[j] : 0;
    }
  }
}

template <bool WRITE>
__global__ void __launch_bounds__(256) page_rows_kernel(PagePlanes a, const int32_t* at, int64_t BH, int S) {
  const int p = blockIdx.y;
  for (int64_t bh = blockIdx.z; bh < BH; bh += gridDim.z) {
    const int b = static_cast<int>(bh / a.H), h = static_cast<int>(bh - static_cast<int64_t>(b) * a.H);
    const int from = at[b];
    if (WRITE && from < 0) continue;
    if (p == 2 || p == 3 || p == 5) norm_groups<WRITE>(a, p, b, h, bh * S, from, S);
    else code_pieces<WRITE>(a, p, b, h, bh * S, from, S);
  }
}

// ---------------------------------------------------------------- whole pages
// page dst[i] of every layer := page src[i]; 16-byte pieces of the six planes one after another
__global__ void __launch_bounds__(256) page_copy_kernel(PagePlanes a, const int32_t* src, const int32_t* dst) {
  const int64_t s = src[blockIdx.y], d = dst[blockIdx.y];
  if (s < 0 || s >= a.num_pages || d < 0 || d >= a.num_pages) return;
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
#pragma unroll
  for (int p = 0; p < kPlanes; ++p) {
    const int64_t bytes = (static_cast<int64_t>(a.H) * a.width[p]) << a.lg_page;
    if (i < bytes / 16) {
      uint8_t* const base = a.pool[p] + blockIdx.z * a.layer[p] + i * 16;
      copy_unit<uint4>(base + d * bytes, base + s * bytes);
      return;
    }
    i -= bytes / 16;
  }
}

// ---------------------------------------------------------------- an accepted path
// Position lengths[b] + path[b, i] moves to lengths[b] + i for i < count[b].  Source and target
// rows overlap, so a block (one wave: one sequence, head and layer) has every row in registers
// before it writes the first.  A piece of a row only meets the same piece of other rows, so rows too
// many for the registers go in several passes over stretches of pieces.  Rows that stay where
// they are (path[i] == i, the root always) are not touched.
// U: bytes of a code piece (8 where every code width is a multiple, else 1); the three norms are
// pieces of their own.
constexpr int kKeepPieces = 4;  // of a lane
template <int U>
__global__ void __launch_bounds__(64) page_keep_kernel(PagePlanes a, const int32_t* lengths, const int32_t* path,
                                                       const int32_t* count, int T, int32_t* new_lengths) {
  __shared__ int64_t s_from[64], s_to[64];
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, i = threadIdx.x;
  const int n = min(max(count[b], 0), T);
  const int64_t at = lengths[b];
  if (i == 0 && h == 0 && layer == 0) new_lengths[b] = static_cast<int32_t>(at) + (at >= 0 ? n : 0);
  int64_t from = -1, to = -1;
  if (i < n && at >= 0) {
    const int k = path[static_cast<int64_t>(b) * T + i];
    if (k >= 0 && k < T && k != i) {
      from = page_row(a, b, h, at + k);
      to = page_row(a, b, h, at + i);
      if (to < 0) from = -1;
    }
  }
  const uint64_t moved = __ballot(from >= 0);
  const uint32_t m = __popcll(moved);
  if (m == 0) return;
  if (from >= 0) {
    const int k = __popcll(moved & ((1ull << i) - 1));
    s_from[k] = from;
    s_to[k] = to;
  }
  __syncthreads();
  const uint32_t c0 = a.width[0] / U, c1 = c0 + a.width[1] / U, c2 = c1 + a.width[4] / U;  // pieces of the code planes
  const uint32_t per = c2 + 3, span = 64 * kKeepPieces / m < per ? 64 * kKeepPieces / m : per;
  for (uint32_t q0 = 0; q0 < per; q0 += span) {
    const uint32_t width = per - q0 < span ? per - q0 : span;
    uint8_t* dst[kKeepPieces];
    uint2 v[kKeepPieces];
    bool norm[kKeepPieces];
#pragma unroll
    for (int k = 0; k < kKeepPieces; ++k) {
      const uint32_t x = i + 64 * k, r = x / width, q = q0 + (x - r * width);
      dst[k] = nullptr;
      norm[k] = q >= c2;
      if (r < m) {
        const int p = q < c0 ? 0 : q < c1 ? 1 : q < c2 ? 4 : q == c2 ? 2 : q == c2 + 1 ? 3 : 5;
        const uint32_t w = a.width[p], off = norm[k] ? 0 : (q - (p == 0 ? 0 : p == 1 ? c0 : c1)) * U;
        uint8_t* const base = a.pool[p] + layer * a.layer[p] + off;
        const uint8_t* const src = base + s_from[r] * w;
        dst[k] = base + s_to[r] * w;
        if (norm[k]) v[k].x = *reinterpret_cast<const uint16_t*>(src);
        else if constexpr (U == 8) v[k] = *reinterpret_cast<const uint2*>(src);
        else v[k].x = *src;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kKeepPieces; ++k) {
      if (!dst[k]) continue;
      if (norm[k]) *reinterpret_cast<uint16_t*>(dst[k]) = static_cast<uint16_t>(v[k].x);
      else if constexpr (U == 8) *reinterpret_cast<uint2*>(dst[k]) = v[k];
      else *dst[k] = static_cast<uint8_t>(v[k].x);
    }
  }
}

static uint32_t unit_of(uint32_t w) { return w % 16 == 0 ? 16 : w % 8 == 0 ? 8 : w % 4 == 0 ? 4 : w % 2 == 0 ? 2 : 1; }

static int fill(const char* what, PagePlanes& a, void* const* pool, void* const* rows, int32_t H, int64_t num_pages,
                int32_t page_size, int32_t d, int32_t key_code_bits, int32_t val_bits, const int32_t* table,
                int64_t ld_table, int32_t table_width) {
  TQ_REQUIRE(supported_dim(d), "%s: head_dim %d not supported (multiples of 8 from 8 to 256)", what, d);
  TQ_REQUIRE(key_code_bits >= 1 && key_code_bits <= 8 && val_bits >= 1 && val_bits <= 8, "%s: bits must be in [1, 8]", what);
  TQ_REQUIRE(page_size >= 32 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0,
             "%s: page_size must be a power of two from 32 to 2^20, got %d", what, page_size);
  TQ_REQUIRE(H >= 1 && num_pages >= 1 && num_pages < (int64_t(1) << 31) && table_width >= 0 && ld_table >= table_width,
             "%s: bad shape", what);
  const int64_t w[kPlanes] = {out_cols(d, key_code_bits), d / 8, 2, 2, out_cols(d, val_bits), 2};
  for (int p = 0; p < kPlanes; ++p) {
    TQ_REQUIRE(pool[p] && reinterpret_cast<uintptr_t>(pool[p]) % 16 == 0, "%s: pool planes must be 16-byte aligned", what);
    a.pool[p] = static_cast<uint8_t*>(pool[p]);
    a.width[p] = static_cast<uint32_t>(w[p]);
    a.unit[p] = unit_of(a.width[p]);
    a.layer[p] = num_pages * H * static_cast<int64_t>(page_size) * w[p];
    a.rows[p] = nullptr;
    if (rows) {
      TQ_REQUIRE(rows[p] && reinterpret_cast<uintptr_t>(rows[p]) % a.unit[p] == 0,
                 "%s: row planes must be aligned to their pieces of %u bytes", what, a.unit[p]);
      a.rows[p] = static_cast<uint8_t*>(rows[p]);
    }
  }
  a.table = table;
  a.ld_table = ld_table;
  a.table_width = table_width;
  a.num_pages = num_pages;
  a.lg_page = __builtin_ctz(static_cast<unsigned>(page_size));
  a.H = H;
  return TQ_OK;
}

template <bool WRITE>
static int rows_call(const char* what, void* const* pool, void* const* rows, int32_t B, int32_t H, int32_t S, int32_t d,
                     int32_t key_code_bits, int32_t val_bits, int64_t num_pages, int32_t page_size,
                     const int32_t* table, int64_t ld_table, int32_t table_width, const int32_t* at, hipStream_t s) {
  TQ_REQUIRE(B >= 0 && S >= 0 && H >= 1, "%s: bad shape", what);
  if (B == 0 || S == 0) return TQ_OK;
  TQ_REQUIRE(pool && rows && (table || table_width == 0) && at, "%s: null pointer", what);
  PagePlanes a{};
  const int st = fill(what, a, pool, rows, H, num_pages, page_size, d, key_code_bits, val_bits, table, ld_table, table_width);
  if (st != TQ_OK) return st;
  TQ_REQUIRE(static_cast<int64_t>(S) * 256 < (int64_t(1) << 31), "%s: at most 2^23 rows per head in one call, got %d", what, S);
  uint32_t most = 0;  // pieces of the widest plane
  for (int p = 0; p < kPlanes; ++p) {
    const uint32_t n = static_cast<uint32_t>(S) * (a.width[p] / a.unit[p]);
    most = n > most ? n : most;
  }
  const int64_t BH = static_cast<int64_t>(B) * H;
  // enough blocks for the norm groups too: S / 8 groups and one more where the first begins inside
  const uint32_t nx = (most + 256 * kRowSteps - 1) / (256 * kRowSteps), ng = (static_cast<uint32_t>(S) / 8 + 2 + 255) / 256;
  const dim3 grid(nx > ng ? nx : ng, kPlanes, static_cast<unsigned>(BH < 65535 ? BH : 65535));
  page_rows_kernel<WRITE><<<grid, 256, 0, s>>>(a, at, BH, S);
  return launch_status(what);
}

}  // namespace tq

using namespace tq;

extern "C" {

int tq_page_write(void* const* pool, void* const* rows, int32_t B, int32_t H, int32_t S, int32_t d,
                  int32_t key_code_bits, int32_t val_bits, int64_t num_pages, int32_t page_size,
                  const int32_t* block_table, int64_t ld_table, int32_t table_width, const int32_t* start,
                  void* stream) {
  return rows_call<true>("tq_page_write", pool, rows, B, H, S, d, key_code_bits, val_bits, num_pages, page_size,
                         block_table, ld_table, table_width, start, as_stream(stream));
}

int tq_page_read(void* const* pool, void* const* rows, int32_t B, int32_t H, int32_t S, int32_t d,
                 int32_t key_code_bits, int32_t val_bits, int64_t num_pages, int32_t page_size,
                 const int32_t* block_table, int64_t ld_table, int32_t table_width, const int32_t* lengths,
                 void* stream) {
  return rows_call<false>("tq_page_read", pool, rows, B, H, S, d, key_code_bits, val_bits, num_pages, page_size,
                          block_table, ld_table, table_width, lengths, as_stream(stream));
}

int tq_page_copy(void* const* pool, int32_t layers, int32_t H, int32_t d, int32_t key_code_bits, int32_t val_bits,
                 int64_t num_pages, int32_t page_size, const int32_t* src, const int32_t* dst, int32_t n,
                 void* stream) {
  TQ_REQUIRE(layers >= 0 && n >= 0, "tq_page_copy: bad shape");
  if (layers == 0 || n == 0) return TQ_OK;
  TQ_REQUIRE(pool && src && dst, "tq_page_copy: null pointer");
  TQ_REQUIRE(layers <= 65535 && n <= 65535, "tq_page_copy: at most 65535 layers and copies, got %d and %d", layers, n);
  PagePlanes a{};
  const int st = fill("tq_page_copy", a, pool, nullptr, H, num_pages, page_size, d, key_code_bits, val_bits, nullptr, 0, 0);
  if (st != TQ_OK) return st;
  int64_t units = 0;
  for (int p = 0; p < kPlanes; ++p) units += static_cast<int64_t>(H) * page_size * a.width[p] / 16;
  const dim3 grid(static_cast<unsigned>((units + 255) / 256), n, layers);
  page_copy_kernel<<<grid, 256, 0, as_stream(stream)>>>(a, src, dst);
  return launch_status("tq_page_copy");
}

int tq_page_keep(void* const* pool, int32_t layers, int32_t B, int32_t H, int32_t T, int32_t d, int32_t key_code_bits,
                 int32_t val_bits, int64_t num_pages, int32_t page_size, const int32_t* block_table, int64_t ld_table,
                 int32_t table_width, const int32_t* lengths, const int32_t* path, const int32_t* count,
                 int32_t* new_lengths, void* stream) {
  TQ_REQUIRE(layers >= 1 && B >= 0 && T >= 1, "tq_page_keep: bad shape");
  TQ_REQUIRE(T <= 64, "tq_page_keep: at most 64 drafted tokens, got %d", T);
  if (B == 0) return TQ_OK;
  TQ_REQUIRE(pool && (block_table || table_width == 0) && lengths && path && count && new_lengths, "tq_page_keep: null pointer");
  TQ_REQUIRE(layers <= 65535 && B <= 65535, "tq_page_keep: at most 65535 layers and sequences, got %d and %d", layers, B);
  PagePlanes a{};
  const int st = fill("tq_page_keep", a, pool, nullptr, H, num_pages, page_size, d, key_code_bits, val_bits, block_table,
                      ld_table, table_width);
  if (st != TQ_OK) return st;
  const dim3 grid(H, B, layers);
  if (a.width[0] % 8 == 0 && a.width[1] % 8 == 0 && a.width[4] % 8 == 0)
    page_keep_kernel<8><<<grid, 64, 0, as_stream(stream)>>>(a, lengths, path, count, T, new_lengths);
  else
    page_keep_kernel<1><<<grid, 64, 0, as_stream(stream)>>>(a, lengths, path, count, T, new_lengths);
  return launch_status("tq_page_keep");
}

}  // extern "C"
