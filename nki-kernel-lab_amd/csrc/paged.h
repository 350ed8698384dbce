// Shared device helpers of the paged cache's kernels: which rows a sequence
// has, and where they are.
#pragma once

#include "common.h"
#include "flash_sched.h"

namespace nkl {

// Positions are held in 32 bits; lengths are cut off here (the entry points
// refuse tables of more rows), so that no sum of a position and a tile wraps.
constexpr int kMaxRows = 1 << 30;

struct CacheArgs {
  unsigned char* k;
  unsigned char* v;
  long k_page, k_head, k_row, v_page, v_head, v_row;  // element strides
  const int* table;                                   // null: row j of every sequence is row j of page 0
  long table_row;
  const int* lens;     // null: `len` rows each
  const int* q_start;  // null: `max_new` new rows each
  int pages, kv_heads, page_size, d, table_cols, batch, rows, max_new, len;
  int capacity;  // rows a table addresses
  fsched::Div32 dv_page;
};

// A sequence's new rows: rows [t0, t0 + n) of the packed tensors, at positions
// pos0 .. pos0 + n - 1 (pos0 < 0 where a sequence is shorter than its new
// rows); only the first `use` of them are worked on.
struct Seq {
  int t0, n, use, len, pos0;
};

__device__ __forceinline__ Seq seq_of(const CacheArgs& c, int b) {
  Seq s;
  if (c.q_start) {
    s.t0 = c.q_start[b];
    s.n = c.q_start[b + 1] - s.t0;
    // (offsets out of order or out of the packed rows hold no rows)
    if (s.t0 < 0 || s.t0 > c.rows || s.n < 0) s.n = 0;
    s.use = min(min(s.n, c.max_new), c.rows - s.t0);
    if (s.n == 0) s.use = 0;
  } else {
    s.t0 = b * c.max_new;
    s.n = s.use = c.max_new;
  }
  s.len = c.lens ? max(0, min(c.lens[b], kMaxRows)) : c.len;
  s.pos0 = s.len - s.n;
  return s;
}

// The page of row j of sequence b, or -1: no such row, or a table entry that
// names no page.
__device__ __forceinline__ int page_of(const CacheArgs& c, int b, int j, int& within) {
  within = 0;
  if (j < 0 || j >= c.capacity) return -1;
  const int pi = (int)fsched::div32(c.dv_page, (unsigned)j);
  within = j - pi * c.page_size;
  const int pid = c.table ? c.table[(long)b * c.table_row + pi] : 0;
  return (unsigned)pid < (unsigned)c.pages ? pid : -1;
}

// Host side: checks a cache description and fills CacheArgs (NKL_OK or a
// status with the error set).  e4m3: a cache of 8 bits is taken too.
int cache_args(const char* fn, const nkl_paged_cache* c, bool needs_seqs, CacheArgs& a, bool e4m3 = false);

inline int elem_bytes(int dtype) { return dtype == NKL_F32 ? 4 : dtype == NKL_E4M3 ? 1 : 2; }

}  // namespace nkl
