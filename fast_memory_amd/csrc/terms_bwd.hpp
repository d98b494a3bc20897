// Local attention with score terms, backward, bf16 / fp16 at head dimensions 64, 128 and 256 (formulas in terms.hpp).
// Two launches behind a small one that forms D_i, none of them with atomics: every sum has one owner and one order.
//
//   dq     a workgroup of 128 queries sweeps the keys as the forward does:  S^T = K.Q^T, dP^T = V.dO^T (queries and
//          their dout in registers), g^T in place, dQ^T += K^T.g^T.
//   dk dv  a workgroup of 128 keys (32 per wave, keys and values in registers) sweeps the queries of all heads of its
//          group, 64 at a time:  S = Q.K^T, dP = dO.V^T, dV^T += dO^T.P, dK^T += Q^T.g.  A lane column is a key; its
//          16 rows are queries, whose lse, D and limits come through LDS.
// The score registers of a block are again the operand of the second product (terms_tile.hpp), and Q^T, dO^T and K^T are
// read out of the row-major tiles by ds_read_b64_tr_b16.
//
// 7 products of 2 d operations a pair where one launch with atomics for dq would do 5: the price of results that do not
// depend on scheduling.  The sweep over queries is cut into `splits` pieces where there are few blocks of keys (a
// workgroup fills a compute unit); the pieces leave fp32 partial sums that a last launch adds in order.
//
// fp16: p and g of a long row lie below fp16's normal numbers.  p is held times 2^12; g times 2^e, e from the largest
// |do_i|_2 max_j |v_j|_2 + |D_i| of the call (a bound of |g|), such that |g| 2^e <= 2^13.  bf16 has fp32's range: e = 0.
#pragma once
#include <type_traits>

#include "terms_masks.hpp"
#include "terms_tile.hpp"

namespace fm {

constexpr float kPScaleF16 = 4096.f;
constexpr int kNormRows = 256;  // rows whose norms a workgroup of the first launch takes the largest of

struct BwdTileArgs {
  const bf16_t *q, *k, *v, *dout;
  const float *lse, *delta;
  const float* norms;  // {largest |do|, largest |D|} per kNormRows query rows, then the largest |v| per kNormRows keys
  int n_q_norms, n_k_norms;
  bf16_t *dq, *dk, *dv;
  float* part;         // [splits][2][H][L][D], where splits > 1
  Terms t;
  Masks m;
  int use_masks, H, G, S, L, splits;
  float in, out_scale, sm_scale;
};

// 2^e for the fp16 gradients of the call, the same in every workgroup
__device__ __forceinline__ float grad_scale(const BwdTileArgs& a, float* smem) {
  float d = 0.f, D = 0.f, v = 0.f;
  for (int i = threadIdx.x; i < a.n_q_norms; i += 256) {
    d = fmaxf(d, a.norms[2 * i]);
    D = fmaxf(D, a.norms[2 * i + 1]);
  }
  for (int i = threadIdx.x; i < a.n_k_norms; i += 256) v = fmaxf(v, a.norms[2 * a.n_q_norms + i]);
  d = wave_max(d), D = wave_max(D), v = wave_max(v);
  const int w = threadIdx.x >> 6;
  if (lane_id() == 0) smem[3 * w] = d, smem[3 * w + 1] = D, smem[3 * w + 2] = v;
  __syncthreads();
  for (int i = 0; i < 4; ++i) d = fmaxf(d, smem[3 * i]), D = fmaxf(D, smem[3 * i + 1]), v = fmaxf(v, smem[3 * i + 2]);
  __syncthreads();
  const float bound = fmaf(d, v, D);
  if (!(bound > 0.f)) return 1.f;
  const int e = 12 - int(floorf(__builtin_amdgcn_logf(bound)));  // bound 2^e in [2^12, 2^13]
  return __builtin_amdgcn_exp2f(float(min(max(e, -60), 60)));
}

// D_i and, for fp16, the norms.  16 lanes a row, 4 rows a wave at a time; blocks behind the queries' take the values.
template <bool F16, int D>
__global__ __launch_bounds__(256) void terms_delta_tile_kernel(const bf16_t* __restrict__ out, const bf16_t* __restrict__ dout,
                                                               const float* __restrict__ dlse, const bf16_t* __restrict__ v,
                                                               float* __restrict__ delta, float* __restrict__ norms,
                                                               int64_t rows, int64_t keys, int q_blocks, int S, int L,
                                                               const int32_t* __restrict__ lim, const int32_t* __restrict__ dock) {
  using M = Mma<F16>;
  __shared__ float s_d[4], s_D[4];
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63, part = l & 15;
  const bool is_v = int(blockIdx.x) >= q_blocks;
  const int64_t n = is_v ? keys : rows, first = int64_t(is_v ? int(blockIdx.x) - q_blocks : int(blockIdx.x)) * kNormRows;
  const bf16_t* x = is_v ? v : dout;
  float big = 0.f, bigD = 0.f;
  for (int i = 4 * w + (l >> 4); i < kNormRows; i += 16) {
    const int64_t row = first + i;
    float s = 0.f, nn = 0.f;
    if (row < n) {
#pragma unroll
      for (int c = part; c < D / 8; c += 16) {
        const uint4 a = *reinterpret_cast<const uint4*>(x + row * D + c * 8);
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
        if (is_v) {
#pragma unroll
          for (int k = 0; k < 4; ++k) nn = fmaf(M::lo(aw[k]), M::lo(aw[k]), fmaf(M::hi(aw[k]), M::hi(aw[k]), nn));
        } else {
          const uint4 b = *reinterpret_cast<const uint4*>(out + row * D + c * 8);
          const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            s = fmaf(M::lo(aw[k]), M::lo(bw[k]), fmaf(M::hi(aw[k]), M::hi(bw[k]), s));
            if constexpr (F16) nn = fmaf(M::lo(aw[k]), M::lo(aw[k]), fmaf(M::hi(aw[k]), M::hi(aw[k]), nn));
          }
        }
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      s += __shfl_xor(s, o);
      if constexpr (F16) nn += __shfl_xor(nn, o);
    }
    if (!is_v && row < n) {
      s -= dlse ? dlse[row] : 0.f;
      if (part == 0) delta[row] = s;
    }
    // (a row that is not finite has no finite gradients, and padding has none at all; the others' precision does not
    // depend on either)
    if constexpr (F16) {
      const bool counts = row < n && (is_v ? !dock || dock[row % L] >= 0 : !lim || lim[row % S] > 0);
      if (counts && nn < INFINITY && fabsf(s) < INFINITY) big = fmaxf(big, nn), bigD = fmaxf(bigD, fabsf(s));
    }
  }
  if constexpr (!F16) return;
  big = wave_max(big), bigD = wave_max(bigD);
  if (l == 0) s_d[w] = big, s_D[w] = bigD;
  __syncthreads();
  if (threadIdx.x == 0) {
    big = sqrtf(fmaxf(fmaxf(s_d[0], s_d[1]), fmaxf(s_d[2], s_d[3])));
    bigD = fmaxf(fmaxf(s_D[0], s_D[1]), fmaxf(s_D[2], s_D[3]));
    if (is_v)
      norms[2 * q_blocks + int(blockIdx.x) - q_blocks] = big;
    else
      norms[2 * blockIdx.x] = big, norms[2 * blockIdx.x + 1] = bigD;
  }
}

// 16 scores x (base 2), their products dP and derivatives of the cap in, p and g out
template <bool F16, int MODE>
__device__ __forceinline__ void block_grads(float (&x)[16], float (&dp)[16], const float (&slack)[16], int r, float lse2,
                                            float delta, float g_scale) {
  const float p = __builtin_amdgcn_exp2f(x[r] - lse2);
  float g = p * (dp[r] - delta);
  if constexpr (MODE & kModeCap) g *= slack[r];
  if constexpr (F16) g *= g_scale;
  x[r] = p;
  dp[r] = g;
}

// ---- dq -------------------------------------------------------------------------------------------------
template <bool F16, int D, int MODE>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void terms_dq_kernel(BwdTileArgs a) {
  using M = Mma<F16>;
  typedef TileLds<D> T;
  typedef typename std::conditional<F16, f16_t, bf16_t>::type E;
  constexpr int NKS = D / 16, NDT = D / 32;
  extern __shared__ __attribute__((aligned(256))) bf16_t lds_all[];
  int* flag = reinterpret_cast<int*>(lds_all);
  lds_char_t* lds = (lds_char_t*)(lds_all + 128);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(lds)));
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5;
  if (tid == 0) *flag = 0;
  float g_scale = 1.f;
  if constexpr (F16) g_scale = grad_scale(a, reinterpret_cast<float*>(lds_all) + 16);
  __syncthreads();
  const int heads = a.H * a.G, bx = int(blockIdx.x) % heads;
  const int hk = bx % a.H, hq = hk * a.G + bx / a.H;
  const int qb = (a.S + kTQ - 1) / kTQ - 1 - int(blockIdx.x) / heads;
  const int i0 = qb * kTQ, wq0 = i0 + 32 * w, iq = wq0 + col;
  const bool q_ok = iq < a.S;
  const int pos = iq + (a.L - a.S);
  const float slope2 = (MODE & kModeBias) ? a.t.slopes[hq] * kLog2e : 0.f;
  const bool has_docs = a.use_masks && a.t.doc_q;
  int lim, doc = 0, lim_lo, lim_hi, wg_lo, wg_hi;
  int2 q_doc = make_int2(0, 0), wg_doc = make_int2(0, 0);
  if (a.use_masks) {
    lim = a.m.lim[iq];
    doc = a.m.docq[iq];
    const int4 q0 = a.m.qmeta[i0 / 32], q1 = a.m.qmeta[i0 / 32 + 1], q2 = a.m.qmeta[i0 / 32 + 2], q3 = a.m.qmeta[i0 / 32 + 3];
    const int4 mine = a.m.qmeta[wq0 / 32];
    lim_lo = mine.x, lim_hi = mine.y;
    wg_lo = min(min(q0.x, q1.x), min(q2.x, q3.x));
    wg_hi = max(max(q0.y, q1.y), max(q2.y, q3.y));
    q_doc = make_int2(mine.z, mine.w);
    wg_doc = make_int2(min(min(q0.z, q1.z), min(q2.z, q3.z)), max(max(q0.w, q1.w), max(q2.w, q3.w)));
  } else {
    auto lim_of = [&](int i) { return seen_limit(i + (a.L - a.S), a.L, a.t.causal, 0); };
    lim = lim_of(iq);
    lim_lo = wq0 < a.S ? lim_of(wq0) : a.L;
    lim_hi = wq0 < a.S ? lim_of(min(wq0 + 31, a.S - 1)) : 0;
    wg_lo = lim_of(i0);
    wg_hi = lim_of(min(i0 + kTQ, a.S) - 1);
  }
  lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);
  lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);

  const int64_t row = int64_t(hq) * a.S + iq;
  uint4 qf[NKS], df[NKS];
  {
    const int64_t r = (q_ok ? row : 0) * D + hb * 8;
    const uint4* pq = reinterpret_cast<const uint4*>(a.q + r);
    const uint4* pd = reinterpret_cast<const uint4*>(a.dout + r);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      qf[ks] = q_ok ? pq[2 * ks] : make_uint4(0, 0, 0, 0);
      df[ks] = q_ok ? pd[2 * ks] : make_uint4(0, 0, 0, 0);
    }
  }
  const float lse2 = q_ok ? a.lse[row] * kLog2e : 0.f, delta = q_ok ? a.delta[row] : 0.f;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    asm volatile("" : "+v"(qf[ks].x), "+v"(qf[ks].y), "+v"(qf[ks].z), "+v"(qf[ks].w));
    asm volatile("" : "+v"(df[ks].x), "+v"(df[ks].y), "+v"(df[ks].z), "+v"(df[ks].w));
  }
  typename M::f16v O[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[dt][r] = 0.f;

  FlatSource<D> src{a.k + int64_t(hk) * a.L * D, a.v + int64_t(hk) * a.L * D, a.L};
  const int t_end = (wg_hi + kTK - 1) / kTK;
  int mask_at = -64;
  unsigned long long mask = 0;
  auto next = [&](int t) {
    if (!has_docs) return t;
    while (t < t_end) {
      if (t >= mask_at + 64 || mask_at < 0) {
        mask_at = t;
        bool hit = false;
        if (t + l < t_end) {
          const int2 km = a.m.kmeta[t + l];
          hit = km.y >= wg_doc.x && km.x <= wg_doc.y && km.y >= 0;
        }
        mask = __ballot(hit);
      }
      const unsigned long long m = mask >> (t - mask_at);
      if (m) return t + __ffsll(m) - 1;
      t = mask_at + 64;
    }
    return t_end;
  };
  bool dirty = false;
  int t = next(0), par = 0;
  if (t < t_end) src.issue(t, lds0, lds0 + T::kBytes, w, l);
  while (t < t_end) {
    const int t_next = next(t + 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    ring_barrier();
    if (t_next < t_end) {
      const uint32_t to = lds0 + uint32_t(par ^ 1) * 2u * T::kBytes;
      src.issue(t_next, to, to + T::kBytes, w, l);
    }
    const lds_char_t* bK = lds + par * 2 * T::kBytes;
    const lds_char_t* bV = bK + T::kBytes;
    const int kp0 = t * kTK;
    bool wg_masked = kp0 + kTK > wg_lo, masked = kp0 + kTK > lim_lo, any = kp0 < lim_hi;
    if (has_docs) {
      const int2 km = a.m.kmeta[t];
      wg_masked |= km.x != km.y || wg_doc.x != wg_doc.y;
      masked |= km.x != km.y || q_doc.x != q_doc.y;
      any = any && km.y >= q_doc.x && km.x <= q_doc.y;
    }
    if (wg_masked) {
#pragma unroll
      for (int u = 0; u < T::kBytes / 4096; ++u) dirty |= any_nonfinite<F16>(lds_read16(bK + (u * 256 + tid) * 16));
    }
    if (any) {
#pragma unroll
      for (int sb = 0; sb < 2; ++sb) {
        typename M::f16v s, p;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f, p[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          s = M::m32(T::rows32(bK, 32 * sb, ks, l), qf[ks], s);
          p = M::m32(T::rows32(bV, 32 * sb, ks, l), df[ks], p);
        }
        float x[16], dp[16], slack[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = s[r], dp[r] = p[r];
        const int key0 = kp0 + 32 * sb + 4 * hb;
        block_scores<MODE, true>(x, slack, a.in, a.out_scale, float(pos - key0), slope2);
#pragma unroll
        for (int r = 0; r < 16; ++r) block_grads<F16, MODE>(x, dp, slack, r, lse2, delta, g_scale);
        if (masked) {
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            int4 dk = make_int4(0, 0, 0, 0);
            if (has_docs) dk = *reinterpret_cast<const int4*>(a.m.dock + key0 + 8 * r4);
            const int dd[4] = {dk.x, dk.y, dk.z, dk.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              bool ok = key0 + 8 * r4 + r < lim;
              if (has_docs) ok = ok && dd[r] == doc;
              if (!ok) dp[4 * r4 + r] = 0.f;
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 gf = make_uint4(M::pack2(dp[8 * h + 0], dp[8 * h + 1]), M::pack2(dp[8 * h + 2], dp[8 * h + 3]),
                                      M::pack2(dp[8 * h + 4], dp[8 * h + 5]), M::pack2(dp[8 * h + 6], dp[8 * h + 7]));
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) O[dt] = M::m32(T::cols32(bK, 32 * sb + 16 * h, dt, l), gf, O[dt]);
        }
      }
    }
    t = t_next;
    par ^= 1;
  }
  if (dirty) *flag = 1;
  __syncthreads();
  if (*flag == 0) {
    if (!q_ok) return;
    const float f = a.sm_scale / g_scale;
    bf16_t* to = a.dq + row * D;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        uint2 o;
        o.x = M::pack2(O[dt][4 * rq + 0] * f, O[dt][4 * rq + 1] * f);
        o.y = M::pack2(O[dt][4 * rq + 2] * f, O[dt][4 * rq + 3] * f);
        *reinterpret_cast<uint2*>(to + dt * 32 + 8 * rq + 4 * hb) = o;
      }
    return;
  }
  // keys that are not finite, in tiles with masked places: these rows one at a time
  const int64_t head = int64_t(hk) * a.L * D;
  const KeyRows<E> K{(const E*)a.k + head, nullptr, 0, 0, 0, D}, V{(const E*)a.v + head, nullptr, 0, 0, 0, D};
  const Score<(MODE & kModeCap) != 0> score(a.sm_scale, a.t.softcap);
  for (int i = wq0; i < min(wq0 + 32, a.S); ++i) {
    const int64_t r = int64_t(hq) * a.S + i;
    row_dq<E, (MODE & kModeCap) != 0>((const E*)a.q + r * D, (const E*)a.dout + r * D, a.lse[r], a.delta[r], K, V,
                                      query_view(a.t, i, a.S, a.L, hq), a.t.doc_k, a.sm_scale, score, (E*)a.dq + r * D);
  }
}

// ---- dk, dv ------------------------------------------------------------------------------------------------
constexpr int kDkvKeys = 128;  // keys of a workgroup
constexpr int kDkvQ = 64;      // queries of a tile

template <int D>
constexpr size_t dkv_lds_bytes() {
  return 512 + 4 * size_t(TileLds<D>::kBytes) + 2 * 4 * 256;  // two tiles of q and dout, two of lse, D, limits, documents
}

template <bool F16, int D, int MODE>
__global__ __launch_bounds__(256, 1) void terms_dkv_kernel(BwdTileArgs a) {
  using M = Mma<F16>;
  typedef TileLds<D> T;
  typedef typename std::conditional<F16, f16_t, bf16_t>::type E;
  constexpr int NKS = D / 16, NDT = D / 32;
  constexpr float p_scale = F16 ? kPScaleF16 : 1.f;
  extern __shared__ __attribute__((aligned(256))) bf16_t lds_all[];
  int* flag = reinterpret_cast<int*>(lds_all);
  lds_char_t* lds = (lds_char_t*)(lds_all + 256);
  lds_char_t* lds_row = lds + 4 * T::kBytes;  // [2]{lse, D, lim, doc}[64]
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(lds)));
  const uint32_t lds_row0 = __builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(lds_row)));
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5;
  if (tid == 0) *flag = 0;
  float g_scale = 1.f;
  if constexpr (F16) g_scale = grad_scale(a, reinterpret_cast<float*>(lds_all) + 16);
  __syncthreads();
  // the first keys, which a causal mask shows to the most queries, go first
  const int hk = int(blockIdx.x) % a.H, rest = int(blockIdx.x) / a.H;
  const int split = rest % a.splits, j0 = (rest / a.splits) * kDkvKeys;
  const int wj0 = j0 + 32 * w, j = wj0 + col;
  const bool j_ok = j < a.L;
  const bool has_docs = a.use_masks && a.t.doc_q;
  int doc = 0;
  int2 k_doc = make_int2(0, 0), wg_doc = make_int2(0, 0);  // of 64 keys (this wave's are half of them), of the workgroup's
  if (has_docs) {
    doc = a.m.dock[j];
    const int2 m0 = a.m.kmeta[j0 / 64], m1 = a.m.kmeta[j0 / 64 + 1];
    k_doc = w < 2 ? m0 : m1;
    wg_doc = make_int2(min(m0.x, m1.x), max(m0.y, m1.y));
  }
  uint4 kf[NKS], vf[NKS];
  {
    const int64_t r = (int64_t(hk) * a.L + (j_ok ? j : 0)) * D + hb * 8;
    const uint4* pk = reinterpret_cast<const uint4*>(a.k + r);
    const uint4* pv = reinterpret_cast<const uint4*>(a.v + r);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      kf[ks] = j_ok ? pk[2 * ks] : make_uint4(0, 0, 0, 0);
      vf[ks] = j_ok ? pv[2 * ks] : make_uint4(0, 0, 0, 0);
    }
  }
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    asm volatile("" : "+v"(kf[ks].x), "+v"(kf[ks].y), "+v"(kf[ks].z), "+v"(kf[ks].w));
    asm volatile("" : "+v"(vf[ks].x), "+v"(vf[ks].y), "+v"(vf[ks].z), "+v"(vf[ks].w));
  }
  typename M::f16v dK[NDT], dV[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) dK[dt][r] = 0.f, dV[dt][r] = 0.f;

  // Steps: tile qt of 64 queries of head g, counted from the first tile that can see the workgroup's keys:
  // step = g n + (qt - qt0), and this workgroup's are [s0, s1).
  const int nqt = (a.S + kDkvQ - 1) / kDkvQ;
  const int qt0 = (a.t.causal && !a.use_masks) ? min(max(0, j0 - (a.L - a.S)) / kDkvQ, nqt) : 0;
  const int n = nqt - qt0;
  const int64_t steps = int64_t(a.G) * n;
  const int s0 = int(steps * split / a.splits), s1 = int(steps * (split + 1) / a.splits);
  // the next step at or behind s whose queries see some key of the workgroup
  int mask_at = -64;
  unsigned long long mask = 0;
  auto next = [&](int s) {
    if (!a.use_masks) return s;
    while (s < s1) {
      if (s >= mask_at + 64 || mask_at < 0) {
        mask_at = s;
        bool hit = false;
        if (s + l < s1) {
          const int qt = qt0 + (s + l) % n;
          const int4 x = a.m.qmeta[2 * qt], y = a.m.qmeta[2 * qt + 1];
          hit = max(x.y, y.y) > j0;
          if (has_docs) hit = hit && wg_doc.y >= 0 && max(x.w, y.w) >= wg_doc.x && min(x.z, y.z) <= wg_doc.y;
        }
        mask = __ballot(hit);
      }
      const unsigned long long m = mask >> (s - mask_at);
      if (m) return s + __ffsll(m) - 1;
      s = mask_at + 64;
    }
    return s1;
  };
  auto issue = [&](int s, int par) {
    const int g = s / n, qt = qt0 + (s - g * n), hq = hk * a.G + g;
    const int i0 = qt * kDkvQ, last = a.S - 1 - i0;
    const int64_t row = int64_t(hq) * a.S + i0;
    const bf16_t* bq = ring_uniform_ptr(a.q + row * D);
    const bf16_t* bd = ring_uniform_ptr(a.dout + row * D);
    const uint32_t to = lds0 + uint32_t(par) * 2u * T::kBytes;
#pragma unroll
    for (int u = 0; u < T::kLoadsPerWave; ++u) {
      const int r = T::load_row(w + 4 * u, l);
      tile_load(to + uint32_t(w + 4 * u) * 1024u, uint32_t(min(r, last)) * T::kRowBytes + T::load_chunk(r, l), bq);
    }
#pragma unroll
    for (int u = 0; u < T::kLoadsPerWave; ++u) {
      const int r = T::load_row(w + 4 * u, l);
      tile_load(to + T::kBytes + uint32_t(w + 4 * u) * 1024u, uint32_t(min(r, last)) * T::kRowBytes + T::load_chunk(r, l), bd);
    }
    // wave 0: lse, 1: D, 2: limits, 3: documents (the last two without masks: nobody reads them)
    const void* base = w == 0 ? (const void*)(a.lse + row) : w == 1 ? (const void*)(a.delta + row)
                       : !a.use_masks ? (const void*)(a.lse + row)
                       : w == 2       ? (const void*)(a.m.lim + i0)
                                      : (const void*)(a.m.docq + i0);
    ring_load4(lds_row0 + uint32_t(par) * 1024u + uint32_t(w) * 256u, uint32_t(min(l, last)) * 4u, ring_uniform_ptr((const char*)base));
  };
  bool dirty = false;
  int s = next(s0), par = 0;
  if (s < s1) issue(s, 0);
  while (s < s1) {
    const int s_next = next(s + 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    ring_barrier();
    if (s_next < s1) issue(s_next, par ^ 1);
    const int g = s / n, qt = qt0 + (s - g * n), hq = hk * a.G + g;
    const int i0 = qt * kDkvQ;
    const float slope2 = (MODE & kModeBias) ? a.t.slopes[hq] * kLog2e : 0.f;
    const lds_char_t* bQ = lds + par * 2 * T::kBytes;
    const lds_char_t* bD = bQ + T::kBytes;
    const lds_char_t* rows = lds_row + par * 1024;
    // who sees what: fewest and most keys of the 64 queries, and of each 32
    int lo[2], hi[2];
    bool mixed[2] = {false, false};
    if (a.use_masks) {
      const int4 x = a.m.qmeta[2 * qt], y = a.m.qmeta[2 * qt + 1];
      lo[0] = x.x, hi[0] = x.y, lo[1] = y.x, hi[1] = y.y;
      if (has_docs) {
        mixed[0] = k_doc.x != k_doc.y || x.z != x.w || x.z != k_doc.x;
        mixed[1] = k_doc.x != k_doc.y || y.z != y.w || y.z != k_doc.x;
      }
    } else {
#pragma unroll
      for (int sb = 0; sb < 2; ++sb) {
        const int a0 = i0 + 32 * sb, a1 = min(a0 + 31, a.S - 1);
        lo[sb] = seen_limit(a0 + (a.L - a.S), a.L, a.t.causal, 0);
        hi[sb] = a0 < a.S ? seen_limit(a1 + (a.L - a.S), a.L, a.t.causal, 0) : 0;
      }
    }
    const bool ragged = i0 + kDkvQ > a.S;
    if (ragged || min(lo[0], lo[1]) < min(j0 + kDkvKeys, a.L) || mixed[0] || mixed[1] ||
        (has_docs && wg_doc.x != wg_doc.y)) {
#pragma unroll
      for (int u = 0; u < T::kBytes / 4096; ++u) {
        dirty |= any_nonfinite<F16>(lds_read16(bQ + (u * 256 + tid) * 16));
        dirty |= any_nonfinite<F16>(lds_read16(bD + (u * 256 + tid) * 16));
      }
    }
#pragma unroll
    for (int sb = 0; sb < 2; ++sb) {
      if (hi[sb] <= wj0) continue;
      typename M::f16v sc, pr;
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = 0.f, pr[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        sc = M::m32(T::rows32(bQ, 32 * sb, ks, l), kf[ks], sc);
        pr = M::m32(T::rows32(bD, 32 * sb, ks, l), vf[ks], pr);
      }
      float x[16], dp[16], slack[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = sc[r], dp[r] = pr[r];
      const int q0 = 32 * sb + 4 * hb;  // of the tile: this lane's rows are q0 + 8 (r / 4) + r % 4
      block_scores<MODE, true>(x, slack, a.in, a.out_scale, float(j - (i0 + q0 + (a.L - a.S))), slope2);
      const bool masked = mixed[sb] || ragged || wj0 + 32 > lo[sb];
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int at = (q0 + 8 * r4) * 4;
        const uint4 ls = lds_read16(rows + at), de = lds_read16(rows + 256 + at);
        const float lsv[4] = {__uint_as_float(ls.x), __uint_as_float(ls.y), __uint_as_float(ls.z), __uint_as_float(ls.w)};
        const float dev[4] = {__uint_as_float(de.x), __uint_as_float(de.y), __uint_as_float(de.z), __uint_as_float(de.w)};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          block_grads<F16, MODE>(x, dp, slack, 4 * r4 + r, lsv[r] * kLog2e, dev[r], g_scale);
        if (masked) {
          uint4 li = make_uint4(0, 0, 0, 0), dq4 = make_uint4(0, 0, 0, 0);
          if (a.use_masks) li = lds_read16(rows + 512 + at), dq4 = lds_read16(rows + 768 + at);
          const uint32_t liv[4] = {li.x, li.y, li.z, li.w}, dqv[4] = {dq4.x, dq4.y, dq4.z, dq4.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = i0 + q0 + 8 * r4 + r;
            bool ok = i < a.S && j < (a.use_masks ? int(liv[r]) : seen_limit(i + (a.L - a.S), a.L, a.t.causal, 0));
            if (has_docs) ok = ok && int(dqv[r]) == doc;
            if (!ok) x[4 * r4 + r] = 0.f, dp[4 * r4 + r] = 0.f;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (F16) {
#pragma unroll
          for (int r = 0; r < 8; ++r) x[8 * h + r] *= p_scale;
        }
        const uint4 pf = make_uint4(M::pack2(x[8 * h + 0], x[8 * h + 1]), M::pack2(x[8 * h + 2], x[8 * h + 3]),
                                    M::pack2(x[8 * h + 4], x[8 * h + 5]), M::pack2(x[8 * h + 6], x[8 * h + 7]));
        const uint4 gf = make_uint4(M::pack2(dp[8 * h + 0], dp[8 * h + 1]), M::pack2(dp[8 * h + 2], dp[8 * h + 3]),
                                    M::pack2(dp[8 * h + 4], dp[8 * h + 5]), M::pack2(dp[8 * h + 6], dp[8 * h + 7]));
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          dV[dt] = M::m32(T::cols32(bD, 32 * sb + 16 * h, dt, l), pf, dV[dt]);
          dK[dt] = M::m32(T::cols32(bQ, 32 * sb + 16 * h, dt, l), gf, dK[dt]);
        }
      }
    }
    s = s_next;
    par ^= 1;
  }
  if (dirty) *flag = 1;
  __syncthreads();
  const bool again = *flag != 0;
  const float fk = a.sm_scale / g_scale, fv = 1.f / p_scale;
  const int64_t plane = int64_t(a.H) * a.L * D;
  if (!again) {
    if (!j_ok) return;
    const int64_t to = (int64_t(hk) * a.L + j) * D;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int64_t at = to + dt * 32 + 8 * rq + 4 * hb;
        const float4 x = make_float4(dK[dt][4 * rq] * fk, dK[dt][4 * rq + 1] * fk, dK[dt][4 * rq + 2] * fk, dK[dt][4 * rq + 3] * fk);
        const float4 y = make_float4(dV[dt][4 * rq] * fv, dV[dt][4 * rq + 1] * fv, dV[dt][4 * rq + 2] * fv, dV[dt][4 * rq + 3] * fv);
        if (a.splits > 1) {
          *reinterpret_cast<float4*>(a.part + 2 * split * plane + at) = x;
          *reinterpret_cast<float4*>(a.part + (2 * split + 1) * plane + at) = y;
        } else {
          *reinterpret_cast<uint2*>(a.dk + at) = make_uint2(M::pack2(x.x, x.y), M::pack2(x.z, x.w));
          *reinterpret_cast<uint2*>(a.dv + at) = make_uint2(M::pack2(y.x, y.y), M::pack2(y.z, y.w));
        }
      }
    return;
  }
  // rows that are not finite, in tiles with masked places: these keys one at a time, over this workgroup's steps
  const Score<(MODE & kModeCap) != 0> score(a.sm_scale, a.t.softcap);
  for (int jj = wj0; jj < min(wj0 + 32, a.L); ++jj) {
    const int64_t at = (int64_t(hk) * a.L + jj) * D;
    KeyGrads kg;
    key_grads_zero(kg);
    for (int ss = s0; ss < s1; ++ss) {
      const int g = ss / n, qt = qt0 + (ss - g * n);
      row_dkv_chunk<E, (MODE & kModeCap) != 0>((const E*)a.k + at, (const E*)a.v + at, jj, hk * a.G + g, qt * kDkvQ, a.S, a.L, D,
                                               (const E*)a.q, (const E*)a.dout, a.lse, a.delta, a.t, score, kg);
    }
    for (int r = 0; r < (D + 63) / 64; ++r) {
      const int c = l + 64 * r;
      if (c >= D) continue;
      if (a.splits > 1) {
        a.part[2 * split * plane + at + c] = kg.k[r] * a.sm_scale;
        a.part[(2 * split + 1) * plane + at + c] = kg.v[r];
      } else {
        Elem<E>::store((E*)a.dk + at + c, kg.k[r] * a.sm_scale);
        Elem<E>::store((E*)a.dv + at + c, kg.v[r]);
      }
    }
  }
}

// the pieces' sums in order, each rounded once
template <bool F16>
__global__ __launch_bounds__(256) void terms_dkv_join_kernel(const float* __restrict__ part, bf16_t* __restrict__ dk,
                                                             bf16_t* __restrict__ dv, int64_t plane, int splits) {
  const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= 2 * plane) return;
  float4 s = *reinterpret_cast<const float4*>(part + i);
  for (int k = 1; k < splits; ++k) {
    const float4 x = *reinterpret_cast<const float4*>(part + 2 * k * plane + i);
    s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
  }
  bf16_t* to = i < plane ? dk + i : dv + (i - plane);
  *reinterpret_cast<uint2*>(to) = make_uint2(Mma<F16>::pack2(s.x, s.y), Mma<F16>::pack2(s.z, s.w));
}

template <bool F16, int D, int MODE>
static int launch_terms_bwd(const BwdTileArgs& a, hipStream_t st) {
  FM_ALLOW_LDS((terms_dq_kernel<F16, D, MODE>), 256 + 4 * size_t(TileLds<D>::kBytes), "fm_local_attn_terms_bwd(lds)");
  FM_ALLOW_LDS((terms_dkv_kernel<F16, D, MODE>), dkv_lds_bytes<D>(), "fm_local_attn_terms_bwd(lds)");
  hipLaunchKernelGGL((terms_dq_kernel<F16, D, MODE>), dim3(unsigned(a.H * a.G * ceil_div(a.S, kTQ))), dim3(256),
                     256 + 4 * size_t(TileLds<D>::kBytes), st, a);
  hipLaunchKernelGGL((terms_dkv_kernel<F16, D, MODE>), dim3(unsigned(a.H * a.splits * ceil_div(a.L, kDkvKeys))), dim3(256),
                     dkv_lds_bytes<D>(), st, a);
  if (a.splits > 1) {
    const int64_t plane = int64_t(a.H) * a.L * D;
    hipLaunchKernelGGL((terms_dkv_join_kernel<F16>), dim3(unsigned(ceil_div(2 * plane, 1024))), dim3(256), 0, st, a.part, a.dk,
                       a.dv, plane, a.splits);
  }
  return launch_status("fm_local_attn_terms_bwd(tiles)");
}

template <bool F16, int D>
static int launch_terms_bwd_type(const BwdTileArgs& a, const void* out, const float* dlse, float* delta, float* norms, hipStream_t st) {
  const int64_t rows = int64_t(a.H) * a.G * a.S, keys = int64_t(a.H) * a.L;
  const int qb = int(ceil_div(rows, kNormRows)), kb = F16 ? int(ceil_div(keys, kNormRows)) : 0;
  hipLaunchKernelGGL((terms_delta_tile_kernel<F16, D>), dim3(unsigned(qb + kb)), dim3(256), 0, st, (const bf16_t*)out, a.dout, dlse,
                     a.v, delta, norms, rows, keys, qb, a.S, a.L, a.use_masks ? a.m.lim : nullptr, a.use_masks ? a.m.dock : nullptr);
  switch ((a.t.softcap > 0.f ? kModeCap : 0) | (a.t.slopes ? kModeBias : 0)) {
    case 0: return launch_terms_bwd<F16, D, 0>(a, st);
    case kModeCap: return launch_terms_bwd<F16, D, kModeCap>(a, st);
    case kModeBias: return launch_terms_bwd<F16, D, kModeBias>(a, st);
    default: return launch_terms_bwd<F16, D, kModeCap | kModeBias>(a, st);
  }
}

template <int D>
int terms_bwd_tiles(const BwdTileArgs& a, bool f16, const void* out, const float* dlse, float* delta, float* norms, hipStream_t st) {
  return f16 ? launch_terms_bwd_type<true, D>(a, out, dlse, delta, norms, st)
             : launch_terms_bwd_type<false, D>(a, out, dlse, delta, norms, st);
}

}  // namespace fm
