// Pages of a cache of local keys and values: appending, forking, dropping, compacting.
//
// The reference keeps its local keys as dense [k_heads, seq_len, d] tensors that live for one forward
// (memory.py:302-304); a server keeps them from step to step, for many sequences.  Here the pool is
// k, v [n_pages][H][P][d] (a page of one head is one contiguous block, which is what the attention reads) and all
// bookkeeping is one int32 array on the device (cache.hpp), so that no call reads anything back and all of them
// record into a graph.
//
// append and fork are two launches: one workgroup decides (checks the request, finds the free pages, writes tables
// and counts, or refuses the call as a whole and leaves everything as it was), then as many workgroups as there is
// data move the rows.  drop is one launch, compact again two.  Pages are handed out in one order whatever the
// schedule: the requests in row order, each from the lowest free page up.  All counts change by integer atomics
// whose order does not show in the result.
//
// Bound: HBM for the rows that move (each read once and written once, 16 bytes per lane).  For a decode step
// (some hundred kilobytes) the two launches and the search for free pages are all of it; the search starts at a
// page number below which nothing is free, kept with the bookkeeping, and ends with the last page it needs.
// Measured (16-bit, 8 heads, d = 128): compact of 1.07 GB 217 us = 4.9 TB/s, what a copy of 2 GiB reaches here, behind 13 us of
// bookkeeping; 96 MB of prompts 17 us = 5.8 TB/s behind 10; a token for each of 64 rows 4 us behind 7; a fork 6 behind 8: the
// deciding workgroup's chain of scans and dependent loads (a launch alone is 2).
#include <algorithm>
#include <initializer_list>

#include "cache.hpp"

namespace fm {

constexpr int kBookThreads = 1024;
constexpr int kBookPerThread = 8;                               // consecutive counts a thread looks at in a round
constexpr int kBookRound = kBookThreads * kBookPerThread;

// The call is refused: nothing changes but the two words that tell.
__device__ __forceinline__ void refuse(int32_t* meta, int reason) {
  if (threadIdx.x == 0) {
    meta[kMetaGo] = 0;
    if (meta[kMetaRefused] == 0) meta[kMetaReason] = reason;
    meta[kMetaRefused] += 1;
  }
}

// The first `want` free pages, ascending, into `out`; returns how many there are (>= want: all found).
// All threads of the workgroup call it; `hint` = a page below which none is free.
__device__ int find_free(const int32_t* __restrict__ refs, int n_pages, int hint, int want, int32_t* __restrict__ out,
                         int* smem) {
  int have = 0;
  for (int p0 = max(hint, 0); p0 < n_pages && have < want; p0 += kBookRound) {
    const int p = p0 + int(threadIdx.x) * kBookPerThread;
    unsigned free_ = 0;
#pragma unroll
    for (int u = 0; u < kBookPerThread; ++u)
      if (p + u < n_pages && refs[p + u] == 0) free_ |= 1u << u;
    int total;
    int at = have + block_excl_scan(__popc(free_), smem, &total);
    while (free_ && at < want) {
      out[at++] = p + __ffs(free_) - 1;
      free_ &= free_ - 1;
    }
    have += total;
  }
  return have;
}

__device__ __forceinline__ bool block_any(bool x, int* flag) {
  if (threadIdx.x == 0) *flag = 0;
  __syncthreads();
  if (x) *flag = 1;  // (every writer writes the same)
  __syncthreads();
  const bool r = *flag != 0;
  __syncthreads();
  return r;
}

// ---- append -----------------------------------------------------------------------------------------
__global__ __launch_bounds__(kBookThreads) void cache_append_book_kernel(int32_t* __restrict__ book, int n_pages, int R,
                                                                         int M, int log2p, const int32_t* __restrict__ cu,
                                                                         int T, int32_t* __restrict__ fresh) {
  __shared__ int smem[17], flag;
  const Book b = book_of(book, n_pages, R);
  const int tid = threadIdx.x;
  const int hint = b.meta[kMetaHint];
  const int64_t cap = min(int64_t(M) << log2p, int64_t(0x7fffffff));
  // what the rows need, and whether they may have it
  long long need = 0;
  bool bad_cu = (tid == 0) && (cu[0] != 0 || cu[R] > T), bad_len = false;
  for (int r = tid; r < R; r += kBookThreads) {
    const int n = cu[r + 1] - cu[r], old = b.length[r];
    bad_cu |= n < 0 || cu[r] < 0 || cu[r + 1] > T;
    if (n > 0) {
      bad_len |= old < 0 || int64_t(old) + n > cap;
      if (!bad_len && !bad_cu) need += pages_of(old + n, log2p) - pages_of(old, log2p);
    }
  }
  if (block_any(bad_cu, &flag)) return refuse(b.meta, FM_CACHE_BAD_REQUEST);
  if (block_any(bad_len, &flag)) return refuse(b.meta, FM_CACHE_ROW_FULL);
  __shared__ long long smem_ll[17];
  long long total_ll;
  block_excl_scan_ll(need, smem_ll, &total_ll);
  if (total_ll > n_pages) return refuse(b.meta, FM_CACHE_NO_PAGES);
  const int total = int(total_ll);
  if (total > 0 && find_free(b.refs, n_pages, hint, total, fresh, smem) < total) return refuse(b.meta, FM_CACHE_NO_PAGES);
  __syncthreads();  // fresh[] is read by other threads below
  // the rows in order, a thread a row: its new pages are the next ones of the list
  int base = 0;
  for (int r0 = 0; r0 < R; r0 += kBookThreads) {
    const int r = r0 + tid;
    int n = 0, old = 0, p0 = 0, k = 0;
    if (r < R) {
      n = cu[r + 1] - cu[r];
      old = b.length[r];
      p0 = pages_of(old, log2p);
      k = n > 0 ? pages_of(old + n, log2p) - p0 : 0;
    }
    int round;
    const int at = base + block_excl_scan(k, smem, &round);
    for (int i = 0; i < k; ++i) {
      const int page = fresh[at + i];
      b.table[int64_t(r) * M + p0 + i] = page;
      b.refs[page] = 1;
    }
    if (n > 0) b.length[r] = old + n;
    base += round;
  }
  if (tid == 0) {
    b.meta[kMetaGo] = 1;
    if (total > 0) b.meta[kMetaHint] = fresh[total - 1] + 1;
  }
}

// One token's rows after the other: H blocks of `row` units (U = 16, 4 or 2 bytes) from k_new / v_new into the page
// the token belongs to.
template <typename U>
__global__ __launch_bounds__(256) void cache_append_rows_kernel(
    U* __restrict__ kp, U* __restrict__ vp, int32_t* __restrict__ book, int n_pages, int R, int M, int log2p, int H, int row,
    const U* __restrict__ kn, const U* __restrict__ vn, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
    const int32_t* __restrict__ cu, int T) {
  const Book b = book_of(book, n_pages, R);
  if (!b.meta[kMetaGo]) return;
  const int last = cu[R];  // tokens behind the last row's belong to nobody
  for (int t = blockIdx.x; t < last; t += gridDim.x) {
    int lo = 0, hi = R - 1;  // the row: the first one that ends behind t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid + 1] > t)
        hi = mid;
      else
        lo = mid + 1;
    }
    const int at = b.length[lo] - (cu[lo + 1] - t);
    const int page = min(max(b.table[int64_t(lo) * M + (at >> log2p)], 0), n_pages - 1);
    const int64_t dst = ((int64_t(page) * H << log2p) + (at & ((1 << log2p) - 1))) * row;
    for (int e = threadIdx.x; e < H * row; e += 256) {
      const int h = e / row, c = e - h * row;
      const int64_t to = dst + ((int64_t(h) * row) << log2p) + c;
      kp[to] = kn[t * k_st + h * k_sh + c];
      vp[to] = vn[t * v_st + h * v_sh + c];
    }
  }
}

// ---- fork ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kBookThreads) void cache_fork_book_kernel(int32_t* __restrict__ book, int n_pages, int R,
                                                                       int M, int log2p, const int32_t* __restrict__ src,
                                                                       int32_t* __restrict__ fresh, int32_t* __restrict__ to) {
  __shared__ int smem[17], flag;
  const Book b = book_of(book, n_pages, R);
  const int tid = threadIdx.x, mask = (1 << log2p) - 1;
  const int hint = b.meta[kMetaHint];
  const int64_t cap = min(int64_t(M) << log2p, int64_t(0x7fffffff));
  bool bad = false;
  int want = 0;
  for (int r = tid; r < R; r += kBookThreads) {
    const int s = src[r];
    if (s < 0) continue;
    // a row that is forked into is empty and is nobody's source
    if (s >= R || s == r || b.length[r] != 0 || src[s] >= 0 || b.length[s] < 0 || b.length[s] > cap) {
      bad = true;
      continue;
    }
    want += (b.length[s] & mask) != 0;
  }
  if (block_any(bad, &flag)) return refuse(b.meta, FM_CACHE_BAD_REQUEST);
  int total;
  block_excl_scan(want, smem, &total);
  if (total > 0 && find_free(b.refs, n_pages, hint, total, fresh, smem) < total) return refuse(b.meta, FM_CACHE_NO_PAGES);
  __syncthreads();
  int base = 0;
  for (int r0 = 0; r0 < R; r0 += kBookThreads) {
    const int r = r0 + tid;
    const int s = r < R ? src[r] : -1;
    const bool part = s >= 0 && (b.length[s] & mask) != 0;
    int round;
    const int at = base + block_excl_scan(part ? 1 : 0, smem, &round);
    if (r < R) to[r] = part ? fresh[at] : -1;
    if (part) b.refs[fresh[at]] = 1;
    base += round;
  }
  if (tid == 0) {
    b.meta[kMetaGo] = 1;
    if (total > 0) b.meta[kMetaHint] = fresh[total - 1] + 1;
  }
}

// blockIdx.x = row; blockIdx.y = 0: its table and counts; 1 + h: head h of its last, partial page
template <typename U>
__global__ __launch_bounds__(256) void cache_fork_rows_kernel(U* __restrict__ kp, U* __restrict__ vp,
                                                              int32_t* __restrict__ book, int n_pages, int R, int M,
                                                              int log2p, int H, int row, const int32_t* __restrict__ src,
                                                              const int32_t* __restrict__ to) {
  const Book b = book_of(book, n_pages, R);
  if (!b.meta[kMetaGo]) return;
  const int r = blockIdx.x, s = src[r];
  if (s < 0) return;
  const int len = b.length[s], whole = len >> log2p, part = len & ((1 << log2p) - 1);  // (the source keeps its length)
  const int32_t* from = b.table + int64_t(s) * M;
  if (blockIdx.y == 0) {
    int32_t* mine = b.table + int64_t(r) * M;
    for (int i = threadIdx.x; i < whole; i += 256) {
      const int page = from[i];
      mine[i] = page;
      if (unsigned(page) < unsigned(n_pages)) atomicAdd(&b.refs[page], 1);
    }
    if (threadIdx.x == 0) {
      if (part) mine[whole] = to[r];
      b.length[r] = len;
    }
    return;
  }
  if (!part) return;
  const int h = int(blockIdx.y) - 1;
  const int64_t block = int64_t(row) << log2p;
  const int64_t a = (int64_t(min(max(from[whole], 0), n_pages - 1)) * H + h) * block;
  const int64_t z = (int64_t(min(max(to[r], 0), n_pages - 1)) * H + h) * block;
  for (int e = threadIdx.x; e < part * row; e += 256) {
    kp[z + e] = kp[a + e];
    vp[z + e] = vp[a + e];
  }
}

// ---- drop: one workgroup a row ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void cache_drop_kernel(int32_t* __restrict__ book, int n_pages, int R, int M, int log2p,
                                                         const int32_t* __restrict__ drop) {
  const Book b = book_of(book, n_pages, R);
  const int r = blockIdx.x, tid = threadIdx.x;
  const int len = min(int64_t(max(b.length[r], 0)), int64_t(M) << log2p);
  const int have = pages_of(len, log2p), n = min(max(drop[r], 0), have);
  if (n == 0) return;
  int32_t* mine = b.table + int64_t(r) * M;
  for (int i = tid; i < n; i += 256) {
    const int page = mine[i];
    if (unsigned(page) >= unsigned(n_pages)) continue;
    if (atomicSub(&b.refs[page], 1) == 1) atomicMin(&b.meta[kMetaHint], page);  // its last row
  }
  __syncthreads();
  for (int i0 = 0; i0 < have; i0 += 256) {  // what is left moves to the front, 256 entries at a time
    const int i = i0 + tid;
    int page = -1;
    if (i + n < have) page = mine[i + n];
    __syncthreads();
    if (i < have) mine[i] = page;
    __syncthreads();
  }
  if (tid == 0) b.length[r] = max(0, len - (n << log2p));
}

// ---- compact --------------------------------------------------------------------------------------------
// work: {number of moves, used pages} | from [n_pages] | to [n_pages] | new number of a page [n_pages]
__global__ __launch_bounds__(kBookThreads) void cache_compact_book_kernel(int32_t* __restrict__ book, int n_pages, int R,
                                                                          int32_t* __restrict__ work) {
  __shared__ int smem[17];
  const Book b = book_of(book, n_pages, R);
  int32_t* from = work + 4;
  int32_t* to = from + n_pages;
  int32_t* number = to + n_pages;
  const int tid = threadIdx.x;
  int mine = 0;
  for (int64_t p0 = 0; p0 < n_pages; p0 += kBookRound)
#pragma unroll
    for (int u = 0; u < kBookPerThread; ++u) {
      const int64_t p = p0 + tid + u * kBookThreads;
      mine += p < n_pages && b.refs[p] > 0;
    }
  int used;
  block_excl_scan(mine, smem, &used);
  // the free pages in front of `used` take the used pages behind it, both ascending; there are as many of each
  int holes = 0, movers = 0;
  for (int64_t p0 = 0; p0 < n_pages; p0 += kBookRound) {
    const int64_t p = p0 + int64_t(tid) * kBookPerThread;
    unsigned hole = 0, mover = 0;
#pragma unroll
    for (int u = 0; u < kBookPerThread; ++u) {
      if (p + u >= n_pages) continue;
      const bool is = b.refs[p + u] > 0;
      if (!is && p + u < used) hole |= 1u << u;
      if (is && p + u >= used) mover |= 1u << u;
      if (!is && p + u >= used) number[p + u] = int(p) + u;  // (no table names a free page; if one does, it still does)
    }
    int total;
    int at = holes + block_excl_scan(__popc(hole), smem, &total);
    holes += total;
    for (; hole; hole &= hole - 1) to[at++] = int(p) + __ffs(hole) - 1;
    at = movers + block_excl_scan(__popc(mover), smem, &total);
    movers += total;
    for (; mover; mover &= mover - 1) from[at++] = int(p) + __ffs(mover) - 1;
  }
  __syncthreads();
  for (int i = tid; i < movers; i += kBookThreads) {
    const int f = from[i], t = to[i];
    number[f] = t;
    b.refs[t] = b.refs[f];
    b.refs[f] = 0;
  }
  if (tid == 0) {
    work[0] = movers;
    work[1] = used;
    b.meta[kMetaHint] = used;
  }
}

// workgroups 0 .. n_table-1 renumber the tables, the others move pages
template <typename U>
__global__ __launch_bounds__(256) void cache_compact_pages_kernel(U* __restrict__ kp, U* __restrict__ vp,
                                                                  int32_t* __restrict__ book, int n_pages, int R, int M,
                                                                  int64_t page_units, const int32_t* __restrict__ work,
                                                                  int n_table) {
  const Book b = book_of(book, n_pages, R);
  const int32_t* from = work + 4;
  const int32_t* to = from + n_pages;
  const int32_t* number = to + n_pages;
  const int moves = work[0], used = work[1];
  if (moves == 0) return;
  if (int(blockIdx.x) < n_table) {
    const int64_t all = int64_t(R) * M;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += int64_t(n_table) * 256) {
      const int page = b.table[i];
      if (page >= used && page < n_pages) b.table[i] = number[page];
    }
    return;
  }
  // a piece = 1024 units of the keys' or the values' page: four independent loads a thread
  const int64_t pieces = (page_units + 1023) >> 10;
  const int64_t all = pieces * moves * 2;
  for (int64_t i = int64_t(blockIdx.x) - n_table; i < all; i += int64_t(gridDim.x) - n_table) {
    const int64_t move = i / (2 * pieces), rest = i - move * 2 * pieces;
    U* pool = rest < pieces ? kp : vp;
    const int64_t c = ((rest < pieces ? rest : rest - pieces) << 10) + threadIdx.x;
    const U* s = pool + int64_t(from[move]) * page_units;
    U* t = pool + int64_t(to[move]) * page_units;
    U x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c + 256 * u < page_units) x[u] = s[c + 256 * u];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c + 256 * u < page_units) t[c + 256 * u] = x[u];
  }
}

// The widest unit rows of `bytes` bytes can be moved in: every pointer and stride is a multiple of it.
static int unit_of(int64_t bytes, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
  for (int u : {16, 4}) {
    bool ok = bytes % u == 0;
    for (const void* p : ptrs) ok = ok && reinterpret_cast<uintptr_t>(p) % u == 0;
    for (int64_t s : strides) ok = ok && s % u == 0;
    if (ok) return u;
  }
  return 2;
}

static int cache_check(const char* name, const void* k, const void* v, const void* book, int n_pages, int R, int M, int P,
                       int H, int d, int dtype) {
  FM_REQUIRE(n_pages >= 1 && R >= 1 && M >= 1 && H >= 1 && d >= 1 && d <= FM_MAX_D, FM_ERR_ARG,
             "%s: n_pages=%d rows=%d width=%d H=%d d=%d", name, n_pages, R, M, H, d);
  FM_REQUIRE(P <= FM_CACHE_MAX_PAGE && log2_exact(P) >= 0, FM_ERR_ARG, "%s: page size %d is no power of two up to %d", name, P,
             FM_CACHE_MAX_PAGE);
  FM_REQUIRE(dtype_ok(dtype), FM_ERR_ARG, "%s: dtype=%d", name, dtype);
  FM_REQUIRE(k && v && book, FM_ERR_ARG, "%s: null pointer", name);
  FM_REQUIRE(H <= 65534 && n_pages <= (1 << 30), FM_ERR_UNSUPPORTED, "%s: H=%d n_pages=%d", name, H, n_pages);
  return FM_OK;
}

}  // namespace fm

#define FM_BY_UNIT(u, CALL) \
  do {                      \
    if ((u) == 16) {        \
      typedef uint4 U;      \
      CALL;                 \
    } else if ((u) == 4) {  \
      typedef uint32_t U;   \
      CALL;                 \
    } else {                \
      typedef uint16_t U;   \
      CALL;                 \
    }                       \
  } while (0)

extern "C" size_t fm_cache_book_ints(int n_pages, int rows, int width) {
  if (n_pages < 1 || rows < 1 || width < 1) return 0;
  return size_t(FM_CACHE_META_INTS) + rows + n_pages + size_t(rows) * width;
}

extern "C" size_t fm_cache_workspace(int n_pages, int rows) {
  if (n_pages < 1 || rows < 1) return 0;
  return (size_t(3) * n_pages + rows + 8) * 4;
}

extern "C" int fm_cache_append(void* k_pages, void* v_pages, int32_t* book, int n_pages, int rows, int width, int page,
                               int H, int d, const void* k_new, const void* v_new, int64_t k_token, int64_t k_head,
                               int64_t v_token, int64_t v_head, const int32_t* cu, int T, int dtype, void* ws,
                               size_t ws_bytes, void* stream) {
  using namespace fm;
  int rc = cache_check("fm_cache_append", k_pages, v_pages, book, n_pages, rows, width, page, H, d, dtype);
  if (rc) return rc;
  FM_REQUIRE(T >= 0 && cu && ws, FM_ERR_ARG, "fm_cache_append: T=%d or null pointer", T);
  FM_REQUIRE(T == 0 || (k_new && v_new), FM_ERR_ARG, "fm_cache_append: null pointer");
  FM_REQUIRE(ws_bytes >= fm_cache_workspace(n_pages, rows), FM_ERR_WORKSPACE, "fm_cache_append: workspace %zu < %zu", ws_bytes,
             fm_cache_workspace(n_pages, rows));
  const int e = dtype_bytes(dtype), lp = log2_exact(page);
  int32_t* fresh = static_cast<int32_t*>(ws);
  hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(cache_append_book_kernel, dim3(1), dim3(kBookThreads), 0, st, book, n_pages, rows, width, lp, cu, T, fresh);
  if (T > 0) {
    const int u = unit_of(int64_t(d) * e, {k_pages, v_pages, k_new, v_new}, {k_token * e, k_head * e, v_token * e, v_head * e});
    const unsigned grid = unsigned(std::min(T, 8192));
    FM_BY_UNIT(u, hipLaunchKernelGGL((cache_append_rows_kernel<U>), dim3(grid), dim3(256), 0, st, (U*)k_pages, (U*)v_pages, book,
                                     n_pages, rows, width, lp, H, d * e / u, (const U*)k_new, (const U*)v_new, k_token * e / u,
                                     k_head * e / u, v_token * e / u, v_head * e / u, cu, T));
  }
  return launch_status("fm_cache_append");
}

extern "C" int fm_cache_fork(void* k_pages, void* v_pages, int32_t* book, int n_pages, int rows, int width, int page, int H,
                             int d, const int32_t* src, int dtype, void* ws, size_t ws_bytes, void* stream) {
  using namespace fm;
  int rc = cache_check("fm_cache_fork", k_pages, v_pages, book, n_pages, rows, width, page, H, d, dtype);
  if (rc) return rc;
  FM_REQUIRE(src && ws, FM_ERR_ARG, "fm_cache_fork: null pointer");
  FM_REQUIRE(ws_bytes >= fm_cache_workspace(n_pages, rows), FM_ERR_WORKSPACE, "fm_cache_fork: workspace %zu < %zu", ws_bytes,
             fm_cache_workspace(n_pages, rows));
  const int e = dtype_bytes(dtype), lp = log2_exact(page);
  int32_t* fresh = static_cast<int32_t*>(ws);
  int32_t* to = fresh + n_pages;
  hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(cache_fork_book_kernel, dim3(1), dim3(kBookThreads), 0, st, book, n_pages, rows, width, lp, src, fresh, to);
  const int u = unit_of(int64_t(d) * e, {k_pages, v_pages}, {});
  FM_BY_UNIT(u, hipLaunchKernelGGL((cache_fork_rows_kernel<U>), dim3(unsigned(rows), unsigned(H + 1)), dim3(256), 0, st,
                                   (U*)k_pages, (U*)v_pages, book, n_pages, rows, width, lp, H, d * e / u, src, to));
  return launch_status("fm_cache_fork");
}

extern "C" int fm_cache_drop(int32_t* book, int n_pages, int rows, int width, int page, const int32_t* n_drop, void* stream) {
  using namespace fm;
  int rc = cache_check("fm_cache_drop", book, book, book, n_pages, rows, width, page, 1, 1, FM_F32);
  if (rc) return rc;
  FM_REQUIRE(n_drop, FM_ERR_ARG, "fm_cache_drop: null pointer");
  hipLaunchKernelGGL(cache_drop_kernel, dim3(unsigned(rows)), dim3(256), 0, as_stream(stream), book, n_pages, rows, width,
                     log2_exact(page), n_drop);
  return launch_status("fm_cache_drop");
}

extern "C" int fm_cache_compact(void* k_pages, void* v_pages, int32_t* book, int n_pages, int rows, int width, int page,
                                int H, int d, int dtype, void* ws, size_t ws_bytes, void* stream) {
  using namespace fm;
  int rc = cache_check("fm_cache_compact", k_pages, v_pages, book, n_pages, rows, width, page, H, d, dtype);
  if (rc) return rc;
  FM_REQUIRE(ws, FM_ERR_ARG, "fm_cache_compact: null pointer");
  FM_REQUIRE(ws_bytes >= fm_cache_workspace(n_pages, rows), FM_ERR_WORKSPACE, "fm_cache_compact: workspace %zu < %zu", ws_bytes,
             fm_cache_workspace(n_pages, rows));
  const int64_t bytes = int64_t(H) * page * d * dtype_bytes(dtype);
  int32_t* work = static_cast<int32_t*>(ws);
  hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(cache_compact_book_kernel, dim3(1), dim3(kBookThreads), 0, st, book, n_pages, rows, work);
  const int u = unit_of(bytes, {k_pages, v_pages}, {});
  const int n_table = int(std::min<int64_t>(64, ceil_div(int64_t(rows) * width, 256)));
  FM_BY_UNIT(u, hipLaunchKernelGGL((cache_compact_pages_kernel<U>), dim3(unsigned(n_table + 4096)), dim3(256), 0, st, (U*)k_pages,
                                   (U*)v_pages, book, n_pages, rows, width, bytes / u, work, n_table));
  return launch_status("fm_cache_compact");
}
