// A KV cache in pages, shared by the kernels that read and write it.
//
// A pool [pages, 2, G, P, D] holds P rows of K and V of every KV head in one
// block (a page): within it a head's K rows are consecutive, then, G * P rows
// on, its V rows.  Row n of sequence b lies in page tables[b, n / P], row
// n % P; P is a power of two of at least 16, so that 16 aligned rows never
// part.  A table entry outside [0, pages) names no page: its rows are not
// there.
#pragma once
#include "common.cuh"

namespace sva {

struct Pages {
  unsigned char* pool;
  int64_t page_bytes;  // between the pages of one layer
  int64_t pages;
  const int32_t* tables;
  int64_t table_stride;
  int max_pages;  // entries of a row
  int bits;       // P = 1 << bits
};

// The page of a row's table entry `at`, or -1.
SVA_DEV int page_of(const Pages& p, int64_t seq, int at) {
  if (at < 0 || at >= p.max_pages) return -1;
  const int id = p.tables[seq * p.table_stride + at];
  return id >= 0 && id < p.pages ? id : -1;
}

inline bool page_rows_ok(int64_t rows) { return rows >= 16 && rows <= 1024 && (rows & (rows - 1)) == 0; }
inline int page_bits(int64_t rows) {
  int b = 0;
  while ((1ll << b) < rows) ++b;
  return b;
}

}  // namespace sva
