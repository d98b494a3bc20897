// Attention with score terms: the scores, what a query sees, and the row-at-a-time form of the operators.
//
//   x_ij = sm_scale q_i.k_j ;  softcap c > 0: x <- c tanh(x / c) ;  x <- x - slope_h |pos_i - j|
//   query i sees key j when j < lim_i and (documents) doc_q[i] == doc_k[j] >= 0
//   lim_i = min(n, max(causal ? pos_i + 1 : n, prefix_i)),  pos_i = i + n - (number of queries)
//   lse_i = log sum exp x_ij,  o_i = sum_j p_ij v_j,  p_ij = exp(x_ij - lse_i)   over the keys seen
//   D_i = do_i.o_i - dlse_i,  g_ij = p_ij (do_i.v_j - D_i) (1 - tanh^2) sm_scale
//   dq_i = sum_j g_ij k_j,  dk_j = sum_i g_ij q_i,  dv_j = sum_i p_ij do_i   (i over all heads of the key's group)
// A query that sees nothing has o = 0, lse = -FLT_MAX and no gradients (the marker of an empty bucket).
// Softmax in base 2 with fp32 scores, maxima, sums and accumulators throughout.
#pragma once
#include "common.hpp"

namespace fm {

// The terms of a call, by value to every kernel.
struct Terms {
  const float* slopes;     // [heads], may be null
  const int32_t* doc_q;    // [S], may be null
  const int32_t* doc_k;    // [L]
  const int32_t* prefix;   // [S] (paged: [rows]), may be null
  float softcap;           // 0: none
  int causal;
};

// tanh for |t| <= 1/2, t (1 + u P(u)) with u = t^2 and P a degree-4 Chebyshev fit of (tanh(t)/t - 1)/u on [0, 1/4]:
// within 2^-24 of the value, and no transcendental instruction.
__device__ __forceinline__ float tanh_small(float t) {
  const float u = t * t;
  float p = fmaf(u, -0.00694700312f, 0.021472721f);
  p = fmaf(u, p, -0.0539337893f);
  p = fmaf(u, p, 0.133332274f);
  p = fmaf(u, p, -0.333333328f);
  return fmaf(t * u, p, t);
}
// tanh = 1 - 2 / (e^2t + 1): within 2^-23 of the value in absolute terms, e^2t = inf included
__device__ __forceinline__ float tanh_large(float t) {
  const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(t * (2.f * kLog2e)) + 1.f);
  return fmaf(-2.f, r, 1.f);
}
constexpr float kTanhSmall = 0.5f;

// Score arithmetic in base 2: raw * in without a cap (in = sm_scale log2 e), out * tanh(raw * in) with one
// (in = sm_scale / c, out = c log2 e).
template <bool CAP>
struct Score {
  float in, out;
  __host__ __device__ Score(float sm_scale, float softcap) {
    in = CAP ? sm_scale / softcap : sm_scale * kLog2e;
    out = CAP ? softcap * kLog2e : 1.f;
  }
  // the score, and in `slack` the derivative of the cap, 1 - tanh^2
  __device__ __forceinline__ float operator()(float raw, float& slack) const {
    const float y = raw * in;
    if constexpr (!CAP) {
      slack = 1.f;
      return y;
    } else {
      const float t = fabsf(y) <= kTanhSmall ? tanh_small(y) : tanh_large(y);
      slack = fmaf(-t, t, 1.f);
      return out * t;
    }
  }
};

__device__ __forceinline__ int seen_limit(int pos, int n, int causal, int prefix) {
  return min(n, max(causal ? max(0, pos + 1) : n, prefix));
}

// Where the rows of one head's keys lie: one block of n rows, or the pages of a table.
template <typename T>
struct KeyRows {
  const T* base;           // this head's first row (paged: this head's block of page 0)
  const int32_t* table;    // null: contiguous
  int64_t page_stride;     // elements from a page to the next
  int log2p, n_pages, d;
  __device__ __forceinline__ const T* row(int j) const {
    if (!table) return base + int64_t(j) * d;
    const int page = min(max(table[j >> log2p], 0), n_pages - 1);
    return base + page * page_stride + int64_t(j & ((1 << log2p) - 1)) * d;
  }
};

template <typename T>
__device__ __forceinline__ float row_dot(const T* __restrict__ a, const T* __restrict__ b, int d) {
  float s = 0.f;
  int k = 0;
  for (; k + 8 <= d; k += 8) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = Elem<T>::load(b + k + u);
#pragma unroll
    for (int u = 0; u < 8; ++u) s = fmaf(Elem<T>::load(a + k + u), x[u], s);
  }
  for (; k < d; ++k) s = fmaf(Elem<T>::load(a + k), Elem<T>::load(b + k), s);
  return s;
}

// A query's position among the keys and what it sees.
struct QueryView {
  int pos, lim, doc;  // doc: -1 none, with use_doc
  bool use_doc;
  float slope2;       // slope * log2 e
  __device__ __forceinline__ bool sees(int j, const int32_t* doc_k) const {
    return j < lim && (!use_doc || (doc >= 0 && doc_k[j] == doc));
  }
};

__device__ __forceinline__ QueryView query_view(const Terms& t, int i, int S, int n, int hq) {
  QueryView v;
  v.pos = i + (n - S);
  v.lim = seen_limit(v.pos, n, t.causal, t.prefix ? t.prefix[i] : 0);
  v.use_doc = t.doc_q != nullptr;
  v.doc = v.use_doc ? t.doc_q[i] : -1;
  v.slope2 = t.slopes ? t.slopes[hq] * kLog2e : 0.f;
  return v;
}

// ---- the row-at-a-time form: one wave, lane = key (or query) in chunks of 64, lane = dimension in the sums.  Every
// sum visits only what is seen, so nothing that is masked -- not even a NaN or an infinity -- touches a result: the
// tiled kernels hand their rows to these when a tile with masked places holds such a value. ----

// (m, l) and this lane's four dimensions of the unnormalised output over keys [j0, j1)
struct RowState {
  float m, l, acc[4];
};

template <typename T, bool CAP>
__device__ __forceinline__ RowState row_forward(const T* __restrict__ q, const KeyRows<T>& K, const KeyRows<T>& V,
                                                const QueryView& qv, const int32_t* __restrict__ doc_k, int j0, int j1,
                                                const Score<CAP>& score) {
  const int lane = lane_id(), d = K.d;
  RowState st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r) st.acc[r] = 0.f;
  j1 = min(j1, qv.lim);
  for (int jb = j0; jb < j1; jb += kWave) {
    const int j = jb + lane;
    const bool ok = j < j1 && qv.sees(j, doc_k);
    float x = -INFINITY, slack;
    if (ok) x = fmaf(-qv.slope2, fabsf(float(qv.pos - j)), score(row_dot(q, K.row(j), d), slack));
    unsigned long long seen = __ballot(ok);
    if (!seen) continue;
    const float m_new = fmaxf(st.m, wave_max(x)), base = m_new == -INFINITY ? 0.f : m_new;
    const float p = ok ? __builtin_amdgcn_exp2f(x - base) : 0.f;
    const float alpha = __builtin_amdgcn_exp2f(st.m - base);
    st.l = st.l * alpha + wave_sum(p);
#pragma unroll
    for (int r = 0; r < 4; ++r) st.acc[r] *= alpha;
    st.m = m_new;
    while (seen) {
      const int t = __ffsll(seen) - 1;
      seen &= seen - 1;
      const float pt = __shfl(p, t);
      const T* vr = V.row(jb + t);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (lane + 64 * r < d) st.acc[r] = fmaf(pt, Elem<T>::load(vr + lane + 64 * r), st.acc[r]);
    }
  }
  return st;
}

template <typename T>
__device__ __forceinline__ void row_write(const RowState& st, int d, T* __restrict__ out, float* __restrict__ lse) {
  const int lane = lane_id();
  const bool none = st.l == 0.f;  // (NaN scores: l is NaN, and so is the row)
  const float inv = none ? 0.f : 1.f / st.l;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (lane + 64 * r < d) Elem<T>::store(out + lane + 64 * r, st.acc[r] * inv);
  if (lane == 0) *lse = none ? -FLT_MAX : (st.m + __builtin_amdgcn_logf(st.l)) * kLn2;
}

// what keys [j0, j1) leave in dq of one query; rd = {lse log2 e, D}
template <typename T, bool CAP, typename TO>
__device__ __forceinline__ void row_dq(const T* __restrict__ q, const T* __restrict__ dout, float2 rd, const KeyRows<T>& K, const KeyRows<T>& V, const QueryView& qv,
                                       const int32_t* __restrict__ doc_k, int j0, int j1, float sm_scale, const Score<CAP>& score,
                                       TO* __restrict__ dq) {
  const int lane = lane_id(), d = K.d;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  j1 = min(j1, qv.lim);
  for (int jb = j0; jb < j1; jb += kWave) {
    const int j = jb + lane;
    const bool ok = j < j1 && qv.sees(j, doc_k);
    float g = 0.f;
    if (ok) {
      float slack;
      const float x = fmaf(-qv.slope2, fabsf(float(qv.pos - j)), score(row_dot(q, K.row(j), d), slack));
      g = __builtin_amdgcn_exp2f(x - rd.x) * (row_dot(dout, V.row(j), d) - rd.y) * slack;
    }
    unsigned long long seen = __ballot(ok);
    while (seen) {
      const int t = __ffsll(seen) - 1;
      seen &= seen - 1;
      const float gt = __shfl(g, t);
      const T* kr = K.row(jb + t);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (lane + 64 * r < d) acc[r] = fmaf(gt, Elem<T>::load(kr + lane + 64 * r), acc[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (lane + 64 * r < d) Elem<TO>::store(dq + lane + 64 * r, acc[r] * sm_scale);
}

// The share of the at most 64 queries [i0, i1) of head hq in one key's gradients (not yet times sm_scale): lane = query, then dimension.
struct KeyGrads {
  float k[4], v[4];
};
__device__ __forceinline__ void key_grads_zero(KeyGrads& g) {
#pragma unroll
  for (int r = 0; r < 4; ++r) g.k[r] = 0.f, g.v[r] = 0.f;
}
template <typename T, bool CAP>
__device__ __forceinline__ void row_dkv_chunk(const T* __restrict__ k, const T* __restrict__ v, int j, int hq, int i0, int i1, int S, int L,
                                              int d, const T* __restrict__ q, const T* __restrict__ dout,
                                              const float2* __restrict__ rd, const Terms& t, const Score<CAP>& score,
                                              KeyGrads& a) {
  const int lane = lane_id(), i = i0 + lane;
  bool ok = false;
  float p = 0.f, gr = 0.f;
  if (i < i1) {
    const QueryView qv = query_view(t, i, S, L, hq);
    ok = qv.sees(j, t.doc_k);
    if (ok) {
      const int64_t row = int64_t(hq) * S + i;
      float slack;
      const float x = fmaf(-qv.slope2, fabsf(float(qv.pos - j)), score(row_dot(q + row * d, k, d), slack));
      p = __builtin_amdgcn_exp2f(x - rd[row].x);
      gr = p * (row_dot(dout + row * d, v, d) - rd[row].y) * slack;
    }
  }
  unsigned long long seen = __ballot(ok);
  while (seen) {
    const int u = __ffsll(seen) - 1;
    seen &= seen - 1;
    const float pu = __shfl(p, u), gu = __shfl(gr, u);
    const int64_t row = (int64_t(hq) * S + i0 + u) * d;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (lane + 64 * r < d) {
        a.k[r] = fmaf(gu, Elem<T>::load(q + row + lane + 64 * r), a.k[r]);
        a.v[r] = fmaf(pu, Elem<T>::load(dout + row + lane + 64 * r), a.v[r]);
      }
  }
}

}  // namespace fm
