// What the paged-cache kernels share: the batch as the device sees it, and
// the cache's addressing.
//
// A sequence b has n = q_start[b + 1] - q_start[b] new rows (one, row b, when
// q_start is NULL), which are the last n of its kv_len[b] tokens.  Token t of
// it sits in slot t % page_size of page page_table[b][t / page_size].  The
// lengths, starts and page ids are device values that the host never sees:
// everything read through them is clamped or checked here, so that no value
// of theirs makes a kernel leave its buffers.
#pragma once

#include "common.h"

namespace fvx {

struct PagedBatch {
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* kv_len;
  const int32_t* q_start;  // NULL: one row per sequence
  int32_t n_rows, n_seqs, max_pages, n_pages;
  int32_t lg_page;  // log2 of the page size
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) {
  return v < lo ? lo : (v > hi ? hi : v);
}

// First new row and number of new rows of sequence b.
__device__ __forceinline__ void paged_rows(const PagedBatch& p, int b, int& q0, int& n) {
  if (!p.q_start) {
    q0 = b < p.n_rows ? b : p.n_rows;
    n = b < p.n_rows ? 1 : 0;
    return;
  }
  q0 = clampi(p.q_start[b], 0, p.n_rows);
  n = clampi(p.q_start[b + 1], q0, p.n_rows) - q0;
}

// The page of page index i of sequence b, -1 where the table has none or
// names a page that does not exist.
__device__ __forceinline__ int paged_page(const PagedBatch& p, int b, int i) {
  if (i < 0 || i >= p.max_pages) return -1;
  const int id = p.page_table[(int64_t)b * p.table_stride + i];
  return id >= 0 && id < p.n_pages ? id : -1;
}

}  // namespace fvx
