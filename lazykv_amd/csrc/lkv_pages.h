// Rows that lie one after the other or in pages of a pool: where a sequence's row is.
//
// A pool is a lkv_kv_rows whose "sequences" are its pages, of `tokens` rows each, a multiple of 16: sixteen rows that start at a
// multiple of 16 lie together, and a kernel looks a page up once for them. A table's entry that is no page of the
// pool stands for rows that are not there: they are not read, not attended and not written.
#pragma once

#include "lkv_mx.h"

namespace lkv {

constexpr int kPageShift = 36;

struct PagedRows {
  lkv_kv_rows rows;
  const int32_t* table;  // NULL: rows one after the other, `rows.seqs` sequences
  int64_t table_stride;
  uint64_t magic;     // ceil(2^36 / sixteens)
  int32_t sixteens;   // of a page
  int32_t capacity;   // rows of a sequence
};

// Sixteen rows of one head: where they start, in elements, and whether they are there.
struct Sixteen {
  int64_t at;
  bool there;
};

// Rows 16 * group .. of sequence b. group < 2^26 and sixteens <= 2^10: group * magic stays below 2^63 and the quotient is exact.
// UNIFORM: all lanes of a wave ask for the same, and the answer is kept in scalar registers.
template <int D, bool UNIFORM = true>
__device__ __forceinline__ Sixteen sixteen_of(const PagedRows& p, int b, int h, int group) {
  int64_t at = (int64_t)h * p.rows.head_stride;
  if (!p.table) return {at + (int64_t)b * p.rows.seq_stride + (int64_t)group * (16 * D), true};
  const int index = (int)(((uint64_t)(uint32_t)group * p.magic) >> kPageShift);
  int page = p.table[(int64_t)b * p.table_stride + index];
  if constexpr (UNIFORM) page = __builtin_amdgcn_readfirstlane(page);
  const bool there = (uint32_t)page < (uint32_t)p.rows.seqs;
  at += (int64_t)(there ? page : 0) * p.rows.seq_stride + (int64_t)((group - index * p.sixteens) * (16 * D));
  return {at, there};
}

// Element offset of row `row` of sequence b, or -1 where it is not there.
template <int D>
__device__ __forceinline__ int64_t row_of(const PagedRows& p, int b, int h, int64_t row) {
  if (row < 0 || row >= p.capacity) return -1;
  const Sixteen s = sixteen_of<D, false>(p, b, h, (int)(row >> 4));
  return s.there ? s.at + (row & 15) * D : -1;
}

}  // namespace lkv

// The checks of rows and their pages, and the kernels' view of them.
static inline int lkv_paged_rows(const lkv_kv_rows* r, const lkv_pages* pages, int n_seqs, int dtype, int head_dim, lkv::PagedRows& p) {
  LKV_CHECK_ARG(r, "NULL rows");
  if (int rc = lkv_check_rows(r, pages ? "pool" : "rows", pages ? r->seqs : n_seqs, dtype, head_dim)) return rc;
  p = {};
  p.rows = *r;
  if (!pages) {
    LKV_CHECK_ARG(r->tokens <= (1 << 30), "at most %d rows of a sequence, got %lld", 1 << 30, (long long)r->tokens);
    p.capacity = (int32_t)r->tokens;
    return LKV_OK;
  }
  LKV_CHECK_ARG(r->tokens > 0 && r->tokens % 16 == 0 && r->tokens <= 16384, "pages of %lld tokens: a multiple of 16, at most 16384", (long long)r->tokens);
  LKV_CHECK_ARG(pages->n_pages >= 0 && pages->seq_stride >= 0 && (pages->table || pages->n_pages == 0), "bad page table");
  LKV_CHECK_ARG(r->seqs > 0 || pages->n_pages == 0, "a pool without pages");
  LKV_CHECK_ARG(pages->n_pages * r->tokens <= (1 << 30), "at most %d rows of a sequence, got %lld", 1 << 30, (long long)(pages->n_pages * r->tokens));
  p.capacity = (int32_t)(pages->n_pages * r->tokens);
  p.sixteens = (int32_t)(r->tokens / 16);
  p.magic = ((1ull << lkv::kPageShift) + p.sixteens - 1) / p.sixteens;
  p.table = pages->table ? pages->table : (const int32_t*)r->k;  // without pages no row is below the capacity, and none is looked up
  p.table_stride = pages->seq_stride;
  return LKV_OK;
}
