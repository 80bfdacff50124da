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
// All of it is bytes that move once in and once out; nothing is computed.
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
// WRITE: rows [B, H, S] of the source planes to positions start[b] + s; otherwise positions
// s < length[b] to rows [B, H, S] of the target planes, zeros behind.  A thread moves one piece; a
// plane's pieces are taken in row order, so both sides are read and written in runs.
template <bool WRITE>
__global__ void __launch_bounds__(256) page_rows_kernel(PagePlanes a, const int32_t* at, int B, int S) {
  const int p = blockIdx.y;
  const uint32_t unit = a.unit[p], per = a.width[p] / unit;
  const int64_t n = static_cast<int64_t>(B) * a.H * S * per;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / per;
    const uint32_t piece = static_cast<uint32_t>(i - r * per);
    const int64_t bh = r / S;
    const int s = static_cast<int>(r - bh * S), b = static_cast<int>(bh / a.H), h = static_cast<int>(bh - static_cast<int64_t>(b) * a.H);
    uint8_t* const flat = a.rows[p] + i * unit;
    if constexpr (WRITE) {
      const int64_t row = page_row(a, b, h, static_cast<int64_t>(at[b]) + s);
      if (at[b] >= 0 && row >= 0) copy_piece(a.pool[p] + row * a.width[p] + piece * unit, flat, unit);
    } else {
      const int64_t row = s < at[b] ? page_row(a, b, h, s) : -1;
      if (row >= 0) copy_piece(flat, a.pool[p] + row * a.width[p] + piece * unit, unit);
      else zero_piece(flat, unit);
    }
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
// rows overlap, so a block takes one (sequence, head, layer) and holds every moved row in LDS
// before it writes the first.  Rows that stay where they are (path[i] == i, the root always)
// are not touched.
constexpr int kKeepThreads = 128;
__global__ void __launch_bounds__(kKeepThreads) page_keep_kernel(PagePlanes a, const int32_t* lengths, const int32_t* path,
                                                                 const int32_t* count, int T, int32_t* new_lengths) {
  extern __shared__ __attribute__((aligned(16))) uint8_t held[];
  __shared__ int64_t s_from[64], s_to[64];
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
  const int n = min(max(count[b], 0), T);
  const int64_t at = lengths[b];
  if (tid == 0 && h == 0 && layer == 0) new_lengths[b] = static_cast<int32_t>(at) + (at >= 0 ? n : 0);
  int64_t from = -1, to = -1;
  if (tid < n && at >= 0) {
    const int k = path[static_cast<int64_t>(b) * T + tid];
    if (k >= 0 && k < T && k != tid) {
      from = page_row(a, b, h, at + k);
      to = page_row(a, b, h, at + tid);
      if (from < 0 || to < 0) from = -1;
    }
  }
  const uint64_t moved = __ballot(from >= 0);  // n <= 64: the rows are the first wave's lanes
  __shared__ int s_n;
  if (tid < 64) {
    if (from >= 0) {
      const int k = __popcll(moved & ((1ull << tid) - 1));
      s_from[k] = from;
      s_to[k] = to;
    }
    if (tid == 0) s_n = __popcll(moved);
  }
  __syncthreads();
  const int m = s_n;
  if (m == 0) return;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    uint32_t off = 0;
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
      const uint32_t w = a.width[p], unit = a.unit[p], per = w / unit;
      uint8_t* const base = a.pool[p] + layer * a.layer[p];
      for (uint32_t i = tid; i < m * per; i += kKeepThreads) {
        const uint32_t r = i / per, piece = (i - r * per) * unit;
        if (pass == 0) copy_piece(held + off + r * w + piece, base + s_from[r] * w + piece, unit);
        else copy_piece(base + s_to[r] * w + piece, held + off + r * w + piece, unit);
      }
      off += (m * w + 15) / 16 * 16;
    }
    __syncthreads();
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
  TQ_REQUIRE(pool && rows && table && at, "%s: null pointer", what);
  PagePlanes a{};
  const int st = fill(what, a, pool, rows, H, num_pages, page_size, d, key_code_bits, val_bits, table, ld_table, table_width);
  if (st != TQ_OK) return st;
  int64_t most = 0;
  for (int p = 0; p < kPlanes; ++p) {
    const int64_t n = static_cast<int64_t>(B) * H * S * (a.width[p] / a.unit[p]);
    most = n > most ? n : most;
  }
  const int64_t blocks = (most + 255) / 256;
  const dim3 grid(static_cast<unsigned>(blocks < 65536 ? blocks : 65536), kPlanes);
  page_rows_kernel<WRITE><<<grid, 256, 0, s>>>(a, at, B, S);
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
  TQ_REQUIRE(pool && block_table && lengths && path && count && new_lengths, "tq_page_keep: null pointer");
  TQ_REQUIRE(layers <= 65535 && B <= 65535, "tq_page_keep: at most 65535 layers and sequences, got %d and %d", layers, B);
  PagePlanes a{};
  const int st = fill("tq_page_keep", a, pool, nullptr, H, num_pages, page_size, d, key_code_bits, val_bits, block_table,
                      ld_table, table_width);
  if (st != TQ_OK) return st;
  uint32_t lds = 0;  // every row but the root can move: at most 34 KB (head_dim 256, 8 bits)
  for (int p = 0; p < kPlanes; ++p) lds += (T * a.width[p] + 15) / 16 * 16;
  page_keep_kernel<<<dim3(H, B, layers), kKeepThreads, lds, as_stream(stream)>>>(a, lengths, path, count, T, new_lengths);
  return launch_status("tq_page_keep");
}

}  // extern "C"
