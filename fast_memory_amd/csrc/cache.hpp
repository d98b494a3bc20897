// The bookkeeping of a paged cache: one int32 array
//   meta [16] | length [R] | refs [n_pages] | table [R][M]
// R rows (sequences), row r holds length[r] tokens; token j of it lies in slot j % P of page table[r][j / P];
// refs[p] = rows that hold page p (0: free); table entries behind a row's last page are -1.
#pragma once
#include "common.hpp"

namespace fm {

// words of meta
constexpr int kMetaRefused = 0;  // calls refused since the caller last cleared it
constexpr int kMetaReason = 1;   // why the first of them was (fm_cache_reason)
constexpr int kMetaGo = 2;       // whether the call under way was accepted (its first launch tells its second)
constexpr int kMetaHint = 3;     // no page below this one is free

struct Book {
  int32_t* meta;
  int32_t* length;
  int32_t* refs;
  int32_t* table;
};

__host__ __device__ __forceinline__ Book book_of(int32_t* b, int n_pages, int R) {
  Book k;
  k.meta = b;
  k.length = b + FM_CACHE_META_INTS;
  k.refs = k.length + R;
  k.table = k.refs + n_pages;
  return k;
}

// P is a power of two; a row may hold up to 2^31 - 1 tokens
__host__ __device__ __forceinline__ int pages_of(int tokens, int log2p) {
  return (tokens >> log2p) + ((tokens & ((1 << log2p) - 1)) != 0);
}

static inline int log2_exact(int x) {  // -1: no power of two
  if (x < 1 || (x & (x - 1))) return -1;
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

}  // namespace fm
