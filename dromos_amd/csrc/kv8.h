// What the kernels of the 8-bit paged cache (lx_kv8) share: the host's checks, the device's view of a cache and of a call's
// rows, and the bounds that keep every access inside them whatever the numbers in device memory are.
#pragma once

#include "common.h"

namespace dro {

// Tokens of the cache are addressed by runs of 16: a block of one scale and a page are whole runs.
constexpr int kRun = 16;

struct Kv8Cache {
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  int pages, heads, page, dim;
  int block_shift;  // log2(block)
};

struct Kv8Batch {
  const int32_t* rows;
  const int32_t* lengths;
  const int32_t* table;
  int seqs, ld_table, max_rows, max_length, T;
};

// One sequence of a call: its first row, its rows, its tokens.
struct Kv8Span {
  int row0, rows, length;
};

__host__ __device__ __forceinline__ int clamp_int(int v, int low, int high) { return v < low ? low : v > high ? high : v; }

// Where a sequence's tokens end at most: by the caller's bound and by its line of the page table.
__host__ __device__ __forceinline__ int kv8_capacity(const Kv8Batch& b, int page) {
  const int64_t held = static_cast<int64_t>(b.ld_table) * page;
  return held < b.max_length ? static_cast<int>(held) : b.max_length;
}

__host__ __device__ __forceinline__ Kv8Span kv8_span_of(const Kv8Batch& b, int page, int from, int to, int length) {
  Kv8Span p;
  p.row0 = clamp_int(from, 0, b.T);
  const int end = clamp_int(to, 0, b.T);
  p.rows = end > p.row0 ? end - p.row0 : 0;
  p.length = clamp_int(length, 0, kv8_capacity(b, page));
  return p;
}

// The three numbers are asked for at once: no address depends on a branch.
__host__ __device__ __forceinline__ Kv8Span kv8_span(const Kv8Batch& b, int page, int s) {
  const int32_t* const rows = b.rows ? b.rows : b.lengths;
  const int from = rows[s], to = rows[b.rows ? s + 1 : s], length = b.lengths[s];
  return kv8_span_of(b, page, b.rows ? from : s, b.rows ? to : s + 1, length);
}

// The part of a block that row r of a call brings to the cache: tokens position .. end - 1 of the block that begins at
// `begin`, and the row behind them. A row has a part of its own where it is its sequence's first one with a place in the
// cache, or the first of its block; the others go with one in front of them, and rows beyond the caller's max_rows have none.
struct Kv8Piece {
  int position, begin, end, next;
  bool own;
};

__host__ __device__ __forceinline__ Kv8Piece kv8_piece(const Kv8Span& span, int max_rows, int block_shift, int r) {
  const int lead = span.length - span.rows;  // the position of the sequence's first row; negative: rows in front of any token
  const int stop = lead + (span.rows < max_rows ? span.rows : max_rows);
  Kv8Piece p;
  p.position = lead + (r - span.row0);
  if (p.position < 0 || p.position >= stop) {
    p.begin = p.end = 0;
    p.next = span.row0 + (p.position < 0 && span.length > 0 ? -lead : span.rows);
    p.own = false;
    return p;
  }
  p.begin = p.position >> block_shift << block_shift;
  p.end = p.begin + (1 << block_shift) < stop ? p.begin + (1 << block_shift) : stop;
  p.next = span.row0 + (p.end - lead);
  p.own = p.position == p.begin || p.position == (lead > 0 ? lead : 0);
  return p;
}

// The page that holds token t of sequence s, or -1 where the table names none of the cache's. t lies inside the sequence's
// line of the table (kv8_span's length does).
__host__ __device__ __forceinline__ int kv8_page(const Kv8Cache& c, const Kv8Batch& b, int s, int t) {
  const int page = b.table[static_cast<int64_t>(s) * b.ld_table + t / c.page];
  return page >= 0 && page < c.pages ? page : -1;
}

// First token row of (page, head) in k and v, in rows of dim codes; the scale of a token row r is number r >> block_shift.
__host__ __device__ __forceinline__ int64_t kv8_row(const Kv8Cache& c, int page, int head) {
  return (static_cast<int64_t>(page) * c.heads + head) * c.page;
}

// Host side: 0 or the status to refuse with.
inline int kv8_check_cache(const lx_kv8* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return kInvalid;
  if (c->type != LX_W_INT8 && c->type != LX_W_FP8)
    return c->type == LX_W_BF16 || c->type == LX_W_NVFP4 || c->type == LX_W_BF16X ? kNotSupported : kInvalid;
  if (c->dim != 64 && c->dim != 128 && c->dim != 192 && c->dim != 256) return kInvalid;
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return kInvalid;
  if (c->page < c->block || c->page > 4096 || c->page % c->block != 0) return kInvalid;
  if (c->pages < 1 || c->heads < 1 || c->heads > 1024) return kInvalid;
  if (static_cast<int64_t>(c->pages) * c->heads * c->page >= (int64_t{1} << 34)) return kInvalid;
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 != 0) return kInvalid;
  return kOk;
}

// Positions, and what is added to them on the way, stay below 2^31: no sequence has room for more than 2^30 tokens.
inline int kv8_check_batch(const lx_kv8_batch* b, int T, const lx_kv8& c) {
  if (!b || T < 0 || T >= (1 << 30) || b->seqs < 0 || b->seqs > (1 << 30) || b->max_rows < 0 || b->max_length < 0 || b->ld_table < 0) return kInvalid;
  if (T == 0 || b->seqs == 0) return kOk;
  if (!b->lengths || (b->ld_table > 0 && !b->table)) return kInvalid;
  if (b->max_length > (1 << 30) && static_cast<int64_t>(b->ld_table) * c.page > (1 << 30)) return kInvalid;
  return kOk;
}

inline Kv8Cache kv8_cache(const lx_kv8& c) {
  int shift = 4;
  while ((1 << shift) < c.block) ++shift;
  return {static_cast<const uint8_t*>(c.k), static_cast<const uint8_t*>(c.v), c.k_scale, c.v_scale, c.pages, c.heads, c.page, c.dim, shift};
}

inline Kv8Batch kv8_batch(const lx_kv8_batch& b, int T) {
  return {b.rows, b.lengths, b.table, b.seqs, b.ld_table, b.max_rows < T ? b.max_rows : T, b.max_length, T};
}

}  // namespace dro
