// Attention of new tokens over a paged cache, bf16 / fp16 at head dimensions 64, 128 and 256, pages of 16 keys or more.
//
// A row of the batch brings n new tokens, n G query rows for each KV head.  Two kernels share the batch, each leaving the
// other's rows alone (kFewRows): rows of few queries are bound by the bytes of their keys, rows of many by the products.
//
//   few    (paged_few_kernel) a workgroup per (row, KV head, piece of the keys).  Its four waves take tiles of 32 keys in
//          turn, straight from global memory into registers (every byte is used once, LDS would only add a hop), 16 KiB a
//          wave and tile; the other waves of a SIMD have theirs in flight meanwhile.  S^T = K.Q^T and O^T += V^T.P^T
//          by v_mfma_f32_16x16x32, 16 query rows at a time; V is read in 8-byte pieces whose 16-bit elements 32 byte
//          permutes put in the operand's order.  The waves' states meet in LDS at the end.
//   many   (paged_many_kernel) the tiled sweep of terms_tile.hpp over 128 query rows; a tile's rows are found through the
//          table, one page number per 16 keys, fetched a tile ahead.
//
// Where there are too few workgroups to fill the card the keys are cut into pieces (workgroups of one row and head), each
// of which leaves (m, l, O) in fp32, and a last launch joins them in order.  The number of pieces follows from the
// extents alone (what a captured graph may replay with other lengths), a piece's keys from the row's length.
#pragma once
#include <type_traits>

#include "terms_tile.hpp"

namespace fm {

// Query rows of a KV head up to which a row is `few`.  Measured, 8 KV heads, d = 128, bf16, few and many at 32 query rows: one row
// of 4096 keys 21.8 and 22.5 us, of 32 768 53.1 and 49.9, 16 rows of 4096 59.1 and 62.1, 64 of 512 28.6 and 29.4; at 40 query
// rows 16 of 4096 138 and 64.
constexpr int kFewRows = 32;
constexpr int kFewKeys = 32;   // keys of a tile of a wave

struct PagedTileArgs {
  PagedArgs p;
  TileScore score;
  int few_rows;              // rows with at most that many query rows are the few-kernel's, the others the other's
  int few_pieces, many_pieces;
  float* part_o;             // [units][D]
  float2* part_ml;           // [units] {m, l}, m in base 2
  int64_t many_base;         // the first unit of the many-kernel's
  int many_slots;
};

// ---- rows by the tokens there are ------------------------------------------------------------------------------------
// A cache may have many more rows than a call has tokens.  Workgroups and workspace are handed out over slots, of which there are
// min(R, T) a head (and piece) and one more for every full block of query rows: which rows have tokens is only known on the device.
// One token for one row of 32 768 keys, 8 KV heads, d = 128, bf16: 50 us in a cache of 1 to 512 rows (387 with a workgroup for every
// row of 128 or more, whose number leaves each a single piece), fp32 137 (340 to 1109).

// The last row i with first(i) <= s, first ascending: 64 candidates at a time, one load a lane and round.  All lanes call it.
template <class First>
__device__ __forceinline__ int last_row(int R, int s, const First& first) {
  int lo = 0, n = R;  // it is among rows lo .. lo + n - 1
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave, at = lane_id() * step;
    const unsigned long long m = __ballot(at < n && first(lo + at) <= s);
    const int k = m ? 63 - __clzll((long long)m) : 0;
    lo += k * step;
    n = min(step, n - k * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The slot of a row with tokens, its first at q0, among min(R, T): no two rows have the same.  With a token for each row and more
// it is the row itself, and no search is needed.
__device__ __forceinline__ int few_slot(const PagedArgs& p, int row, int q0) { return p.T >= p.R ? row : min(row, q0); }
__device__ __forceinline__ int few_row(const PagedArgs& p, int slot) {
  return p.T >= p.R ? slot : last_row(p.R, slot, [&](int i) { return min(i, max(p.cu[i], 0)); });
}

// Where a query row's pieces lie.  Beside a many-kernel the few-kernel's rows are counted within their row's slot, of which
// each has kFewRows at most: by token there would be units for all the others' too, gigabytes where a long prompt comes along.
__device__ __forceinline__ int64_t few_index(const PagedTileArgs& a, int slot, int r, int hk, int t, int hq) {
  const int64_t u = a.few_rows == kFewRows ? (int64_t(slot) * kFewRows + r) * a.p.H + hk : int64_t(t) * a.p.H * a.p.G + hq;
  return u * a.few_pieces;
}
__device__ __forceinline__ int64_t many_index(const PagedTileArgs& a, int t, int hq) {
  return a.many_base + (int64_t(t) * a.p.H * a.p.G + hq) * a.many_pieces;
}

// Where a page number leads: clamped into the pool.
__device__ __forceinline__ int64_t page_offset(const PagedArgs& p, int page, int d) {
  return int64_t(min(max(page, 0), p.n_pages - 1)) * p.H * p.page * d;
}

// Tokens in front of the first row's and behind the last row's: nothing to see.  As many lanes a query row as it has groups of four
// dimensions (a power of two, a wave at most); `first` of `step` workgroups.
template <typename E>
__device__ void paged_nobody(const PagedTileArgs& a, int first, int step) {
  const PagedArgs& p = a.p;
  const int HG = p.H * p.G, c0 = min(max(p.cu[0], 0), p.T), c1 = min(max(p.cu[p.R], c0), p.T);
  const unsigned n = unsigned(c0 + p.T - c1) * unsigned(HG);  // (T H G fits 31 bits)
  const bool fours = ((p.d | p.o_token | p.o_head) & 3) == 0 && reinterpret_cast<uintptr_t>(p.out) % (4 * sizeof(E)) == 0;
  int log2l = 0;
  while (log2l < 6 && (4 << log2l) < p.d) ++log2l;
  const int lane = int(threadIdx.x) & ((1 << log2l) - 1), rows = 256 >> log2l;
  for (unsigned i = unsigned(first * rows) + (threadIdx.x >> log2l); i < n; i += unsigned(step * rows)) {
    int t = int(i / unsigned(HG));
    const int hq = int(i - unsigned(t) * unsigned(HG));
    if (t >= c0) t += c1 - c0;
    E* out = (E*)p.out + t * p.o_token + hq * p.o_head;
    for (int c = 4 * lane; c < p.d; c += 4 << log2l) {
      if (fours) {
        typename std::conditional<sizeof(E) == 4, uint4, uint2>::type zero{};
        *reinterpret_cast<decltype(zero)*>(out + c) = zero;
      } else {
        for (int e = c; e < min(c + 4, p.d); ++e) Elem<E>::store(out + e, 0.f);
      }
    }
    if (lane == 0) p.lse[t * p.l_token + hq * p.l_head] = -FLT_MAX;
  }
}
// Workgroups for them, behind the others': one per 64 query rows of the call, 1024 at most.  They leave at once where every token
// is some row's.  A batch padded to 8192 tokens x 64 heads, d = 128, bf16, of which 4 are real: 62 us (7.8 ms with four workgroups).
inline int nobody_groups(const PagedArgs& p) {
  return int(std::min<int64_t>(1024, ceil_div(int64_t(p.T) * p.H * p.G, 64)));
}

// One query row's result: final where the keys are in one piece, else its piece's.  `o`: 64 lanes, dimensions l + 64 r.
template <typename E>
__device__ __forceinline__ void paged_row_result(const PagedTileArgs& a, const RowState& st, int t, int hq, int64_t at, int pieces) {
  if (pieces == 1) {
    row_write(st, a.p.d, (E*)a.p.out + t * a.p.o_token + hq * a.p.o_head, a.p.lse + t * a.p.l_token + hq * a.p.l_head);
    return;
  }
  const int lane = lane_id();
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (lane + 64 * r < a.p.d) a.part_o[at * a.p.d + lane + 64 * r] = st.acc[r];
  if (lane == 0) a.part_ml[at] = make_float2(st.m, st.l);
}

template <typename E>
__device__ __forceinline__ void paged_row_again(const PagedTileArgs& a, const PagedRow& pr, int t, int hq, int j0, int j1, int64_t at,
                                                int pieces) {
  QueryView qv;
  qv.pos = pr.len - (pr.q1 - t);
  qv.lim = seen_limit(qv.pos, pr.len, 1, a.p.prefix ? a.p.prefix[pr.row] : 0);
  qv.use_doc = false;
  qv.doc = -1;
  qv.slope2 = a.p.slopes ? a.p.slopes[hq] * kLog2e : 0.f;
  const int64_t head = int64_t(hq / a.p.G) * a.p.page * a.p.d, stride = int64_t(a.p.H) * a.p.page * a.p.d;
  const KeyRows<E> K{(const E*)a.p.k + head, pr.table, stride, a.p.log2p, a.p.n_pages, a.p.d};
  const KeyRows<E> V{(const E*)a.p.v + head, pr.table, stride, a.p.log2p, a.p.n_pages, a.p.d};
  const E* q = (const E*)a.p.q + t * a.p.q_token + hq * a.p.q_head;
  const RowState st = a.p.softcap > 0.f
                          ? row_forward<E, true>(q, K, V, qv, nullptr, j0, j1, Score<true>(a.p.sm_scale, a.p.softcap))
                          : row_forward<E, false>(q, K, V, qv, nullptr, j0, j1, Score<false>(a.p.sm_scale, 0.f));
  paged_row_result<E>(a, st, t, hq, at, pieces);
}

// the keys of piece i of n, in whole tiles of `tile`; a piece behind the last tile has j0 >= j1 and no tile j0 / tile .. either
__device__ __forceinline__ void piece_keys(int keys, int tile, int i, int n, int& j0, int& j1) {
  const int tiles = (keys + tile - 1) / tile, each = (tiles + n - 1) / n;
  j0 = min(i * each, tiles) * tile;
  j1 = min(j0 + each * tile, keys);
}

// The row and its first query row that slot s of ROWS query rows stands for: row i owns slots first(i) .. first(i + 1) - 1,
// first(i) = cu[i] G / ROWS + min(i, cu[i]): at least as many as it has blocks, and none before the first token.
template <int ROWS>
__device__ __forceinline__ void paged_slot(const PagedArgs& p, int s, int& row, int& r0) {
  auto first = [&](int i) {
    const int c = max(p.cu[i], 0);
    return int(int64_t(c) * p.G / ROWS) + min(i, c);
  };
  row = last_row(p.R, s, first);
  r0 = (s - first(row)) * ROWS;
}

// ---- few query rows ----------------------------------------------------------------------------------------------
template <int D>
struct FewTile {  // a wave's 32 keys in registers
  uint4 k[2][D / 32];   // key 16 b + l % 16, dimensions 32 s + 8 (l / 16) ..
  uint2 v[8][D / 64];   // keys 4 (l / 16) + r, then 16 + those; dimensions 64 j + 4 (l % 16) ..
};

template <int D>
constexpr size_t few_lds_bytes() {
  return 256 + 4 * 16 * (D + 4) * 4 + 4 * 16 * 8;
}

// waves of a SIMD: other waves' loads hide a wave's, so that none needs a second tile in registers
template <int D, int NQ>
constexpr int few_waves() {
  return D == 64 ? (NQ == 1 ? 4 : 3) : D == 128 ? (NQ == 1 ? 3 : 2) : (NQ == 1 ? 2 : 1);
}

template <bool F16, int D, int NQ>
__global__ __launch_bounds__(256, (few_waves<D, NQ>())) void paged_few_kernel(PagedTileArgs a) {
  using M = Mma<F16>;
  typedef typename M::f4 f4;
  typedef typename std::conditional<F16, f16_t, bf16_t>::type E;
  constexpr int NS = D / 32, NJ = D / 64, NM = D / 16;
  constexpr int LD = D + 4;  // a query's row of fp32 in LDS (the padding spreads the 16 queries over the banks)
  extern __shared__ __attribute__((aligned(256))) bf16_t lds_all[];
  int* flag = reinterpret_cast<int*>(lds_all);
  float* lds_o = reinterpret_cast<float*>(lds_all + 128);             // [4][16][LD]
  float2* lds_ml = reinterpret_cast<float2*>(lds_o + 4 * 16 * LD);     // [4][16]
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, c = l & 15, g = l >> 4;
  const int units = min(a.p.R, a.p.T) * a.p.H * a.few_pieces;
  if (int(blockIdx.x) >= units) return paged_nobody<E>(a, int(blockIdx.x) - units, int(gridDim.x) - units);
  // pieces of a row side by side, then its heads: the pages of a row are read at one time
  const int piece = int(blockIdx.x) % a.few_pieces, rh = int(blockIdx.x) / a.few_pieces;
  const int hk = rh % a.p.H, slot = rh / a.p.H, row = few_row(a.p, slot);
  const PagedRow pr = paged_row(a.p, row);
  const int n = pr.q1 - pr.q0, n_rows = n * a.p.G;
  if (n <= 0 || n_rows > a.few_rows || slot != few_slot(a.p, row, pr.q0)) return;
  const int prefix = a.p.prefix ? a.p.prefix[row] : 0;
  const int64_t head = int64_t(hk) * a.p.page * D;
  const bf16_t* K = (const bf16_t*)a.p.k + head;
  const bf16_t* V = (const bf16_t*)a.p.v + head;
  const int lp = a.p.log2p, slot_mask = a.p.page - 1;

  for (int r0 = 0; r0 < n_rows; r0 += 16 * NQ) {  // (one round, unless the caller's max_new was too small)
    if (tid == 0) *flag = 0;
    __syncthreads();
    // this lane's query rows: 16 i + c behind r0; row = token * G + head of the group
    int lim[NQ], pos[NQ];
    float slope2[NQ];
    uint4 qf[NQ][NS];
    int lim_hi = 0, lim_lo = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int r = r0 + 16 * i + c;
      const bool ok = r < n_rows;
      const int tok = ok ? r / a.p.G : 0, hq = hk * a.p.G + (ok ? r - tok * a.p.G : 0);
      pos[i] = pr.len - n + tok;
      lim[i] = ok ? seen_limit(pos[i], pr.len, 1, prefix) : 0;
      slope2[i] = a.p.slopes ? a.p.slopes[hq] * kLog2e : 0.f;
      const uint4* pq = reinterpret_cast<const uint4*>((const bf16_t*)a.p.q + (pr.q0 + tok) * a.p.q_token + hq * a.p.q_head + 8 * g);
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[i][s] = ok ? pq[4 * s] : make_uint4(0, 0, 0, 0);
    }
    {
      const int last_tok = (min(r0 + 16 * NQ, n_rows) - 1) / a.p.G, first_tok = r0 / a.p.G;
      lim_hi = seen_limit(pr.len - n + last_tok, pr.len, 1, prefix);
      lim_lo = seen_limit(pr.len - n + first_tok, pr.len, 1, prefix);
    }
    int j0, j1;
    piece_keys(lim_hi, kFewKeys, piece, a.few_pieces, j0, j1);

    f4 O[NQ][NM];
    float m[NQ], sum[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      m[i] = -INFINITY, sum[i] = 0.f;
#pragma unroll
      for (int x = 0; x < NM; ++x) O[i][x] = f4{0.f, 0.f, 0.f, 0.f};
    }
    bool dirty = false;
    // Tiles of 32 keys, w, w + 4, ..; keys behind the row's end repeat its last (their scores are masked).  A run of 16
    // keys lies in one page: two page numbers a tile, fetched a tile ahead of its rows.
    auto page_of = [&](int key) { return pr.table[min(key, pr.len - 1) >> lp]; };
    auto load = [&](FewTile<D>& x, int key0, int page0, int page1) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int64_t po = page_offset(a.p, b ? page1 : page0, D);
        const int kk = min(key0 + 16 * b + c, pr.len - 1) & slot_mask;
        const uint4* pk = reinterpret_cast<const uint4*>(K + po + int64_t(kk) * D + 8 * g);
#pragma unroll
        for (int s = 0; s < NS; ++s) x.k[b][s] = pk[4 * s];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kv = min(key0 + 16 * b + 4 * g + r, pr.len - 1) & slot_mask;
          const uint2* pv = reinterpret_cast<const uint2*>(V + po + int64_t(kv) * D + 4 * c);
#pragma unroll
          for (int j = 0; j < NJ; ++j) x.v[4 * b + r][j] = pv[16 * j];
        }
      }
    };
    auto compute = [&](const FewTile<D>& x, int key0) {
      const bool masked = key0 + 32 > lim_lo;
      uint4 pf[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        f4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          s[b] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < NS; ++k) s[b] = M::m16(x.k[b][k], qf[i][k], s[b]);
        }
        float y[8];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float z = s[b][r] * a.score.in;
            const int key = key0 + 16 * b + 4 * g + r;
            if (a.p.softcap > 0.f) z = a.score.out * (fabsf(z) <= kTanhSmall ? tanh_small(z) : tanh_large(z));
            z = fmaf(-slope2[i], fabsf(float(pos[i] - key)), z);
            if (masked && key >= lim[i]) z = -INFINITY;
            y[4 * b + r] = z;
          }
        float mx = y[0];
#pragma unroll
        for (int r = 1; r < 8; ++r) mx = fmaxf(mx, y[r]);
        mx = st_max_lane_groups(mx);
        if (__any(mx > m[i] + (kPUp<F16> + kPLazy<F16>))) {  // (m is held kPUp below the maximum)
          const float m_new = fmaxf(m[i], mx - kPUp<F16>), m_to = m_new == -INFINITY ? 0.f : m_new;
          const float alpha = __builtin_amdgcn_exp2f(m[i] - m_to);
          sum[i] *= alpha;
#pragma unroll
          for (int k = 0; k < NM; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) O[i][k][r] *= alpha;
          m[i] = m_new;
        }
        const float base = m[i] == -INFINITY ? 0.f : m[i];
        float s_tile = 0.f;  // (by itself first, see tile_sweep)
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          y[r] = __builtin_amdgcn_exp2f(y[r] - base);
          s_tile += y[r];
        }
        sum[i] += s_tile;
        pf[i] = make_uint4(M::pack2(y[0], y[1]), M::pack2(y[2], y[3]), M::pack2(y[4], y[5]), M::pack2(y[6], y[7]));
      }
      // values that 0 x would not erase, where some query does not see some key (the row's last key, repeated behind its end, is such
      // a place too: an infinite value of it is not NaN)
      if (masked) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
          for (int j = 0; j < NJ; ++j) dirty |= any_nonfinite<F16>(make_uint4(x.v[r][j].x, x.v[r][j].y, 0, 0));
      }
      // V^T operands: dimension 64 j + 4 c + e of the 8 keys, e = 0 .. 3, out of 8 pieces of 4 dimensions
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t lo = e < 2 ? x.v[2 * k][j].x : x.v[2 * k][j].y, hi = e < 2 ? x.v[2 * k + 1][j].x : x.v[2 * k + 1][j].y;
            o[k] = __builtin_amdgcn_perm(hi, lo, (e & 1) ? 0x07060302u : 0x05040100u);
          }
          const uint4 av = make_uint4(o[0], o[1], o[2], o[3]);
#pragma unroll
          for (int i = 0; i < NQ; ++i) O[i][4 * j + e] = M::m16(av, pf[i], O[i][4 * j + e]);
        }
    };
    {
      const int step = 4 * kFewKeys;
      int key = j0 + kFewKeys * w;
      int pa = 0, pb = 0;
      if (key < j1) pa = page_of(key), pb = page_of(key + 16);
      for (; key < j1; key += step) {
        FewTile<D> x;
        load(x, key, pa, pb);
        if (key + step < j1) pa = page_of(key + step), pb = page_of(key + step + 16);
        compute(x, key);
      }
    }
    if (dirty) *flag = 1;
    __syncthreads();
    const bool again = *flag != 0;
    if (again) {
      for (int r = r0 + w; r < min(r0 + 16 * NQ, n_rows); r += 4)
        paged_row_again<E>(a, pr, pr.q0 + r / a.p.G, hk * a.p.G + r % a.p.G, j0, j1,
                           few_index(a, slot, r, hk, pr.q0 + r / a.p.G, hk * a.p.G + r % a.p.G) + piece, a.few_pieces);
      __syncthreads();
      continue;
    }
    // the four waves' states of 16 queries at a time; lane (g, c) holds dimensions 64 (k / 4) + 16 g + 4 r + k % 4 of query c
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      float ls = sum[i] + __shfl_xor(sum[i], 16);
      ls += __shfl_xor(ls, 32);
      float* mine = lds_o + (w * 16 + c) * LD;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *reinterpret_cast<float4*>(mine + 64 * j + 16 * g + 4 * r) =
              make_float4(O[i][4 * j][r], O[i][4 * j + 1][r], O[i][4 * j + 2][r], O[i][4 * j + 3][r]);
      if (g == 0) lds_ml[w * 16 + c] = make_float2(m[i], ls);
      __syncthreads();
      // 16 threads a query, each D / 16 dimensions
      const int q = tid >> 4, r = r0 + 16 * i + q, part = tid & 15;
      if (r < n_rows) {
        float2 ml[4];
        float mt = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          ml[k] = lds_ml[k * 16 + q];
          mt = fmaxf(mt, ml[k].x);
        }
        const float base = mt == -INFINITY ? 0.f : mt;
        float f[4], lt = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f[k] = __builtin_amdgcn_exp2f(ml[k].x - base);
          lt = fmaf(ml[k].y, f[k], lt);
        }
        const int tok = r / a.p.G, hq = hk * a.p.G + (r - tok * a.p.G), t = pr.q0 + tok;
        const bool none = lt == 0.f;
        const float inv = a.few_pieces > 1 ? 1.f : none ? 0.f : 1.f / lt;
        const int64_t at = a.few_pieces > 1 ? few_index(a, slot, r, hk, t, hq) + piece : 0;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          const int d0 = 64 * u + 4 * part;
          float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 x = *reinterpret_cast<const float4*>(lds_o + (k * 16 + q) * LD + d0);
            // (a wave that had no tile holds zeros and weighs nothing: not even NaN comes of it)
            o[0] = fmaf(x.x, f[k], o[0]), o[1] = fmaf(x.y, f[k], o[1]), o[2] = fmaf(x.z, f[k], o[2]), o[3] = fmaf(x.w, f[k], o[3]);
          }
          if (a.few_pieces > 1)
            *reinterpret_cast<float4*>(a.part_o + at * D + d0) = make_float4(o[0], o[1], o[2], o[3]);
          else
            *reinterpret_cast<uint2*>((bf16_t*)a.p.out + t * a.p.o_token + hq * a.p.o_head + d0) =
                make_uint2(M::pack2(o[0] * inv, o[1] * inv), M::pack2(o[2] * inv, o[3] * inv));
        }
        if (part == 0) {
          if (a.few_pieces > 1)
            a.part_ml[at] = make_float2(mt, lt);
          else
            a.p.lse[t * a.p.l_token + hq * a.p.l_head] = none ? -FLT_MAX : tile_lse<F16>(mt, lt);
        }
      }
      __syncthreads();
    }
  }
}

// ---- many query rows ---------------------------------------------------------------------------------------------
template <int D, int KT>
struct PagedSource {
  const bf16_t *k, *v;   // this head's block of page 0
  PagedArgs p;
  const int32_t* table;
  int len;
  int ids;               // lane b: the page of keys 16 b .. of the tile to be issued next
  __device__ __forceinline__ void prefetch(int t) {
    const int key = min(t * KT + 16 * (lane_id() & (KT / 16 - 1)), len - 1);
    ids = table[key >> p.log2p];
  }
  __device__ __forceinline__ void issue(int t, uint32_t lds_k, uint32_t lds_v, int w, int lane) const {
    typedef TileLds<D, KT> T;
#pragma unroll
    for (int u = 0; u < T::kLoadsPerWave; ++u) {
      const int load = w + 4 * u;
      const int row = T::load_row(load, lane);
      // (a load's rows, 8 at most, lie in one run of 16 keys and so in one page)
      const int page = __builtin_amdgcn_readlane(ids, load * T::kRowsPerLoad / 16);
      const int64_t po = page_offset(p, page, D);
      const int slot = min(t * KT + row, len - 1) & (p.page - 1);
      const uint32_t voff = uint32_t(slot) * T::kRowBytes + T::load_chunk(row, lane);
      tile_load(lds_k + uint32_t(load) * 1024u, voff, ring_uniform_ptr(k + po));
      tile_load(lds_v + uint32_t(load) * 1024u, voff, ring_uniform_ptr(v + po));
    }
  }
};

template <int D>
constexpr size_t many_lds_bytes() {
  return 256 + 4 * size_t(TileLds<D, fwd_tile_keys<D>()>::kBytes);
}

template <bool F16, int D, int MODE>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_many_kernel(PagedTileArgs a) {
  using M = Mma<F16>;
  typedef typename std::conditional<F16, f16_t, bf16_t>::type E;
  constexpr int KT = fwd_tile_keys<D>();
  extern __shared__ __attribute__((aligned(256))) bf16_t lds_all[];
  int* flag = reinterpret_cast<int*>(lds_all);
  lds_char_t* lds = (lds_char_t*)(lds_all + 128);
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5;
  const int units = a.p.H * a.many_slots * a.many_pieces;
  if (int(blockIdx.x) >= units) return paged_nobody<E>(a, int(blockIdx.x) - units, int(gridDim.x) - units);
  // KV head first: the query blocks of a head run on one XCD and share its pages there
  const int hk = int(blockIdx.x) % a.p.H, rest = int(blockIdx.x) / a.p.H;
  const int piece = rest % a.many_pieces, slot = a.many_slots - 1 - rest / a.many_pieces;  // (a row's last tokens, which see most, first)
  int row, r0;
  paged_slot<kTQ>(a.p, slot, row, r0);
  const PagedRow pr = paged_row(a.p, row);
  const int n = pr.q1 - pr.q0, n_rows = n * a.p.G;
  if (n <= 0 || n_rows <= a.few_rows || r0 < 0 || r0 >= n_rows) return;
  if (tid == 0) *flag = 0;
  __syncthreads();
  const int prefix = a.p.prefix ? a.p.prefix[row] : 0;
  const int wr0 = r0 + 32 * w, r = wr0 + col;
  const bool ok = r < n_rows;
  const int tok = ok ? r / a.p.G : 0, hq = hk * a.p.G + (ok ? r - tok * a.p.G : 0), t = pr.q0 + tok;
  auto lim_of = [&](int rr) { return seen_limit(pr.len - n + rr / a.p.G, pr.len, 1, prefix); };
  TileQuery qy;
  qy.pos = pr.len - n + tok;
  qy.lim = ok ? seen_limit(qy.pos, pr.len, 1, prefix) : 0;
  qy.doc = 0;
  qy.slope2 = (MODE & kModeBias) ? a.p.slopes[hq] * kLog2e : 0.f;
  const int lim_lo = __builtin_amdgcn_readfirstlane(wr0 < n_rows ? lim_of(wr0) : pr.len);
  const int lim_hi = __builtin_amdgcn_readfirstlane(wr0 < n_rows ? lim_of(min(wr0 + 31, n_rows - 1)) : 0);
  const int wg_lo = lim_of(r0), wg_hi = lim_of(min(r0 + kTQ, n_rows) - 1);
  uint4 qf[D / 16];
  {
    const uint4* pq = reinterpret_cast<const uint4*>((const bf16_t*)a.p.q + t * a.p.q_token + hq * a.p.q_head + hb * 8);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = ok ? pq[2 * ks] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) asm volatile("" : "+v"(qf[ks].x), "+v"(qf[ks].y), "+v"(qf[ks].z), "+v"(qf[ks].w));
  int j0, j1;
  piece_keys(wg_hi, KT, piece, a.many_pieces, j0, j1);
  const int64_t head = int64_t(hk) * a.p.page * D;
  PagedSource<D, KT> src{(const bf16_t*)a.p.k + head, (const bf16_t*)a.p.v + head, a.p, pr.table, pr.len, 0};
  const TileDocs docs{nullptr, nullptr, make_int2(0, 0), make_int2(0, 0)};
  typename M::f16v O[D / 32];
  TileState st;
  int t0 = j0 / KT, t1 = (j1 + KT - 1) / KT;
  const bool again = tile_sweep<F16, D, MODE, false>(src, qf, qy, lim_lo, lim_hi, wg_lo, t0, t1, 0, 1, docs, a.score, lds, flag, O, st);
  if (again) {
    for (int rr = wr0; rr < min(wr0 + 32, n_rows); ++rr)
      paged_row_again<E>(a, pr, pr.q0 + rr / a.p.G, hk * a.p.G + rr % a.p.G, j0, j1,
                         many_index(a, pr.q0 + rr / a.p.G, hk * a.p.G + rr % a.p.G) + piece, a.many_pieces);
    return;
  }
  if (a.many_pieces == 1) {
    tile_write<F16, D>(O, st, ok ? (bf16_t*)a.p.out + t * a.p.o_token + hq * a.p.o_head : nullptr,
                       a.p.lse + t * a.p.l_token + hq * a.p.l_head);
    return;
  }
  if (!ok) return;
  const int64_t at = many_index(a, t, hq) + piece;
  tile_write_part<D>(O, st, a.part_o + at * D, a.part_ml + at);
}

// ---- the pieces of a query row, in order: 16 lanes a row, D / 16 dimensions each -----------------------------------------
// FEW: only the few-kernel's rows were cut, beside rows of many queries that are done; the launch counts as few_index does.
template <bool F16, int D, bool FEW>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedTileArgs a) {
  const int64_t unit = int64_t(blockIdx.x) * 16 + (threadIdx.x >> 4);
  PagedRow pr;
  int t, hk, r;
  if constexpr (FEW) {
    const int64_t u = unit / a.p.H;
    const int64_t slot = u / kFewRows;  // (the same in a wave: its four units are neighbours among 32 H)
    hk = int(unit - u * a.p.H), r = int(u % kFewRows);
    if (slot >= min(a.p.R, a.p.T)) return;
    pr = paged_row(a.p, few_row(a.p, int(slot)));
    const int n_rows = (pr.q1 - pr.q0) * a.p.G;
    if (n_rows > a.few_rows || r >= n_rows || slot != few_slot(a.p, pr.row, pr.q0)) return;
    t = pr.q0 + r / a.p.G;
  } else {
    const int HG = a.p.H * a.p.G;
    t = int(unit / HG);
    if (t >= a.p.T) return;
    const int hq = int(unit - int64_t(t) * HG);
    pr = paged_row_of_token(a.p, t);
    if (pr.row < 0) return;  // (written where nobody's tokens are)
    hk = hq / a.p.G, r = (t - pr.q0) * a.p.G + hq - hk * a.p.G;
  }
  const bool few = FEW || (pr.q1 - pr.q0) * a.p.G <= a.few_rows;
  const int pieces = few ? a.few_pieces : a.many_pieces, hq = hk * a.p.G + r % a.p.G;
  if (pieces == 1) return;
  const int64_t at = few ? few_index(a, few_slot(a.p, pr.row, pr.q0), r, hk, t, hq) : many_index(a, t, hq);
  tile_join<F16, D>(a.part_o + at * D, a.part_ml + at, pieces, (bf16_t*)a.p.out + t * a.p.o_token + hq * a.p.o_head,
                    a.p.lse + t * a.p.l_token + hq * a.p.l_head);
}

// ---- host: which launches, how many pieces -----------------------------------------------------------------------------
struct PagedPlan {
  bool few, many;
  int few_rows, few_pieces, many_pieces, slots;
  int64_t many_base;  // units of the few-kernel's pieces
  size_t part_ml, total;
};

// Pieces until there are about 1024 workgroups (four a compute unit), but none of less than 512 keys by the table's
// width.  Measured, 512 and 1024 workgroups (8 KV heads, d = 128): 32 ragged rows of up to 32 768 keys 623 and 607 us, ragged chunks of
// 1024 tokens 1075 and 1001 (finer pieces end more evenly); 16 equal rows of 4096 under 32 query rows each 53.5 and 59.3.
// 2048: as 1024.
inline PagedPlan paged_plan(int rows, int T, int max_new, int H, int G, int d, int64_t keys) {
  PagedPlan y{};
  const bool known = max_new > 0 && max_new <= T;
  y.few = !(known && rows == 1 && max_new == T && int64_t(T) * G > kFewRows);
  y.many = !(known && int64_t(max_new) * G <= kFewRows) && int64_t(T) * G > kFewRows;
  y.few_rows = !y.many ? 0x7fffffff : y.few ? kFewRows : 0;
  const int filled = std::min(rows, T);  // rows that may have tokens
  y.slots = int(int64_t(T) * G / kTQ) + filled;
  const int64_t most = std::min<int64_t>(ceil_div(keys, 512), 64);
  auto pieces = [&](int64_t groups) { return int(std::max<int64_t>(1, std::min(most, ceil_div(1024, groups)))); };
  // (where every row is the few-kernel's, by T as well: a max_new that is too small is no wrong answer, nor a large workspace)
  y.few_pieces = y.few ? pieces(std::max<int64_t>(filled, y.many ? 0 : int64_t(T) * G / kFewRows) * H) : 1;
  y.many_pieces = y.many ? pieces(std::max<int64_t>(1, int64_t(T) * G / kTQ) * H) : 1;
  y.many_base = y.few_pieces > 1 ? int64_t(y.many ? int64_t(filled) * kFewRows : int64_t(T) * G) * H * y.few_pieces : 0;
  const size_t units = size_t(y.many_base) + (y.many_pieces > 1 ? size_t(T) * H * G * y.many_pieces : 0);
  y.part_ml = align_up(units * d * 4, 256);
  y.total = y.part_ml + align_up(units * 8, 256);
  return y;
}

// of the fp32 products' kernel: 32 query rows a slot.  What a split costs is a write and a read of d values for each query row and
// piece, against 512 keys read: little.
inline PagedPlan paged_f32_plan(int rows, int T, int H, int G, int d, int64_t keys) {
  PagedPlan y{};
  y.many = true;
  y.slots = int(int64_t(T) * G / 32) + std::min(rows, T);
  const int64_t groups = std::max<int64_t>(std::min<int64_t>(rows, T), int64_t(T) * G / 32) * H;
  y.few_pieces = 1;
  y.many_pieces = int(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(ceil_div(keys, 512), 64), ceil_div(1024, groups))));
  const size_t units = y.many_pieces > 1 ? size_t(T) * H * G * y.many_pieces : 0;
  y.part_ml = align_up(units * d * 4, 256);
  y.total = y.part_ml + align_up(units * 8, 256);
  return y;
}

template <bool F16, int D, int NQ>
static int launch_few(const PagedTileArgs& a, int extra, hipStream_t st) {
  FM_ALLOW_LDS((paged_few_kernel<F16, D, NQ>), few_lds_bytes<D>(), "fm_paged_attn_fwd(lds)");
  hipLaunchKernelGGL((paged_few_kernel<F16, D, NQ>), dim3(unsigned(std::min(a.p.R, a.p.T) * a.p.H * a.few_pieces + extra)), dim3(256),
                     few_lds_bytes<D>(), st, a);
  return launch_status("fm_paged_attn_fwd(few)");
}

template <bool F16, int D, int MODE>
static int launch_many(const PagedTileArgs& a, int extra, hipStream_t st) {
  FM_ALLOW_LDS((paged_many_kernel<F16, D, MODE>), many_lds_bytes<D>(), "fm_paged_attn_fwd(lds)");
  hipLaunchKernelGGL((paged_many_kernel<F16, D, MODE>), dim3(unsigned(a.p.H * a.many_slots * a.many_pieces + extra)), dim3(256),
                     many_lds_bytes<D>(), st, a);
  return launch_status("fm_paged_attn_fwd(many)");
}

template <bool F16, int D>
static int launch_paged(const PagedTileArgs& a, const PagedPlan& y, int max_new, hipStream_t st) {
  const int extra = nobody_groups(a.p);
  int rc = FM_OK;
  if (y.few) {
    const bool one = max_new > 0 && int64_t(max_new) * a.p.G <= 16;
    rc = one ? launch_few<F16, D, 1>(a, extra, st) : launch_few<F16, D, 2>(a, extra, st);
    if (rc) return rc;
  }
  if (y.many) {
    const int more = y.few ? 0 : extra;
    switch ((a.p.softcap > 0.f ? kModeCap : 0) | (a.p.slopes ? kModeBias : 0)) {
      case 0: rc = launch_many<F16, D, 0>(a, more, st); break;
      case kModeCap: rc = launch_many<F16, D, kModeCap>(a, more, st); break;
      case kModeBias: rc = launch_many<F16, D, kModeBias>(a, more, st); break;
      default: rc = launch_many<F16, D, kModeCap | kModeBias>(a, more, st);
    }
    if (rc) return rc;
  }
  if (a.many_pieces > 1 || (a.few_pieces > 1 && a.few_rows != kFewRows)) {
    const int64_t units = int64_t(a.p.T) * a.p.H * a.p.G;
    hipLaunchKernelGGL((paged_join_kernel<F16, D, false>), dim3(unsigned(ceil_div(units, 16))), dim3(256), 0, st, a);
  } else if (a.few_pieces > 1) {
    const int64_t units = int64_t(std::min(a.p.R, a.p.T)) * kFewRows * a.p.H;
    hipLaunchKernelGGL((paged_join_kernel<F16, D, true>), dim3(unsigned(ceil_div(units, 16))), dim3(256), 0, st, a);
  }
  return launch_status("fm_paged_attn_fwd(join)");
}

template <int D>
int paged_tiles(const PagedTileArgs& a, const PagedPlan& y, int max_new, hipStream_t st) {
  return a.p.dtype == FM_F16 ? launch_paged<true, D>(a, y, max_new, st) : launch_paged<false, D>(a, y, max_new, st);
}

}  // namespace fm
