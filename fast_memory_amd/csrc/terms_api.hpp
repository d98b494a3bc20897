// Arguments of the attention operators with score terms, as the entry points hand them to the kernels' launchers.
#pragma once
#include "cache.hpp"
#include "terms.hpp"

namespace fm {

struct FwdArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  Terms t;
  int H, G, S, L, d, dtype;
  float sm_scale;
};

struct BwdArgs {
  FwdArgs f;  // out and lse are inputs here
  const void* dout;
  const float* dlse;
  void *dq, *dk, *dv;
};

// A batch of new tokens over the pages of a cache; strides in elements.
struct PagedArgs {
  const void* q;
  int64_t q_token, q_head;
  const void *k, *v;
  const int32_t* book;
  int n_pages, R, M, page, log2p;
  const int32_t* cu;
  void* out;
  int64_t o_token, o_head;
  float* lse;
  int64_t l_token, l_head;
  int T, H, G, d;
  float sm_scale, softcap;
  const float* slopes;
  const int32_t* prefix;
  int dtype;
};

struct PagedRow {
  int row, len, q0, q1;  // row -1: a token behind the last row's, which belongs to nobody and sees nothing
  const int32_t* table;
};

// The row that holds token t: the first one that ends behind it.
__device__ __forceinline__ PagedRow paged_row(const PagedArgs& a, int row) {
  PagedRow p;
  const int32_t* len = a.book + FM_CACHE_META_INTS;
  const int64_t cap = int64_t(a.M) << a.log2p;
  p.row = row;
  p.len = int(min(int64_t(max(len[row], 0)), cap));
  p.q0 = min(max(a.cu[row], 0), a.T);
  p.q1 = min(max(a.cu[row + 1], p.q0), a.T);
  p.table = len + a.R + a.n_pages + int64_t(row) * a.M;
  return p;
}
__device__ __forceinline__ PagedRow paged_row_of_token(const PagedArgs& a, int t) {
  int lo = 0, hi = a.R - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid + 1] > t)
      hi = mid;
    else
      lo = mid + 1;
  }
  PagedRow p = paged_row(a, lo);
  if (t >= p.q1 || t < p.q0) p.row = -1;
  return p;
}

}  // namespace fm
