// Local attention with score terms, backward, bf16 / fp16 at head dimensions 64, 128 and 256 (formulas in terms.hpp).
// One launch of two kinds of block, behind a small one that forms D_i, without atomics: every sum has one owner and one order.
//
//   dq     a workgroup of 128 queries sweeps the keys as the forward does:  S^T = K.Q^T, dP^T = V.dO^T (queries and
//          their dout in registers), g^T in place, dQ^T += K^T.g^T.
//   dk dv  a workgroup of 128 keys (32 per wave, keys in registers, values in LDS) sweeps the queries of all heads of its
//          group, 32 at a time:  S = Q.K^T, dP = dO.V^T, dV^T += dO^T.P, dK^T += Q^T.g.  A lane column is a key; its
//          16 rows are queries, whose lse, D and limits come through LDS.
// The score registers of a block are again the operand of the second product (terms_tile.hpp), and Q^T, dO^T and K^T are
// read out of the row-major tiles by ds_read_b64_tr_b16.
//
// 7 products of 2 d operations a pair where one launch with atomics for dq would do 5: the price of results that do not
// depend on scheduling.  The sweep over queries is cut into `splits` pieces where there are few blocks of keys (a
// workgroup fills a compute unit); the pieces leave fp32 partial sums that a last launch adds in order.  The two kinds of block
// are one launch: one after the other took 1.25 times as long (32 heads x 2048: 0.21 and 0.15 ms).
//
// Measured, 64 heads x 4096 causal, bf16: d = 128 1.23 ms = 560 TFLOP/s (of 10 d a pair), bias 1.16, cap 1.37, five documents
// 0.40; d = 64 0.77; d = 256 4.6 (an accumulator is 128 registers: the scores are formed twice and one wave runs on a SIMD).
// Bound at d = 128 (counters of 64 heads x 4096 with a bias and a prefix): the matrix pipes are busy 52 % of the time, the VALU 50 %, LDS
// 26 % without a bank conflict: two waves a SIMD take turns at products and arithmetic more than they overlap them.
//
// fp16: p and g of a long row lie below fp16's normal numbers.  p is held times 2^12; g times 2^e, e from the largest
// |do_i|_2 max_j |v_j|_2 + |D_i| of the call (a bound of |g|), such that |g| 2^e <= 2^13.  bf16 has fp32's range: e = 0.
#pragma once
#include <algorithm>
#include <type_traits>

#include "terms_masks.hpp"
#include "terms_tile.hpp"

namespace fm {

constexpr float kPScaleF16 = 4096.f;
constexpr int kNormRows = 64;   // rows whose norms a workgroup of the first launch takes the largest of

struct BwdTileArgs {
  const bf16_t *q, *k, *v, *dout;
  const float2* rd;    // {lse log2 e, D} of every query row
  const float* norms;  // {largest |do|, largest |D|} per kNormRows query rows, then the largest |v| per kNormRows keys
  int n_q_norms, n_k_norms;
  bf16_t *dq, *dk, *dv;
  float* part;         // [splits][2][H][L][D], where splits > 1
  Terms t;
  Masks m;
  int use_masks, H, G, S, L, splits;
  float sm_scale;
  TileScore score;
  int dq_pieces;
  float* part_dq;      // [dq_pieces][H G][S][D], where dq_pieces > 1
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
                                                               const float* __restrict__ lse, const float* __restrict__ dlse,
                                                               const bf16_t* __restrict__ v, float2* __restrict__ rd,
                                                               float* __restrict__ norms,
                                                               int64_t rows, int64_t keys, int q_blocks, int S, int L,
                                                               const int2* __restrict__ qinfo, const int32_t* __restrict__ dock) {
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
      if (part == 0) rd[row] = make_float2(lse[row] * kLog2e, s);
    }
    // (a row that is not finite has no finite gradients, and padding has none at all; the others' precision does not
    // depend on either)
    if constexpr (F16) {
      const bool counts = row < n && (is_v ? !dock || dock[row % L] >= 0 : !qinfo || qinfo[row % S].x > 0);
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

// Raw products of a block of 32 x 32 in, p and p (1 - tanh^2) out.  lse2 is read per register (a query is a lane column in
// the dq launch, a row in the dk / dv one); dist0 as for block_scores.
template <int MODE, class Rows>
__device__ __forceinline__ void block_probs(float (&x)[16], float (&y)[16], const TileScore& k, float dist0, float slope2,
                                            const Rows& rows) {
  auto dist = [&](int r) { return fabsf(dist0 - float(8 * (r >> 2) + (r & 3))); };
  auto finish = [&](int r, float z, float slack) {  // z: the score before the bias
    const float e = (MODE & kModeBias) ? fmaf(-slope2, dist(r), z) : z;
    x[r] = __builtin_amdgcn_exp2f(e - rows.lse2(r));
    y[r] = (MODE & kModeCap) ? x[r] * slack : x[r];
  };
  if constexpr (MODE & kModeCap) {
    if (__any(!(abs_max16(x) <= k.zmax))) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float z = x[r] * k.in, t = fabsf(z) <= kTanhSmall ? tanh_small(z) : tanh_large(z);
        finish(r, k.out * t, fmaf(-t, t, 1.f));
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float z = x[r] * capped_small(k, x[r]);
        finish(r, z, fmaf(z * k.k2, -z, 1.f));
      }
    }
  } else if constexpr (MODE & kModeBias) {
#pragma unroll
    for (int r = 0; r < 16; ++r) finish(r, x[r] * k.in, 1.f);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) y[r] = x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], k.in, -rows.lse2(r)));
  }
}
struct ColumnQuery {
  float l;
  __device__ __forceinline__ float lse2(int) const { return l; }
};
struct RowQueries {  // this lane's rows are queries 4 hb + 8 (r / 4) + r % 4 of the tile: 32 x lse log2 e, 32 x D from 4 hb on
  const lds_char_t* at;
  __device__ __forceinline__ float pick(const uint4& u, int r) const {
    return __uint_as_float((r & 3) == 0 ? u.x : (r & 3) == 1 ? u.y : (r & 3) == 2 ? u.z : u.w);
  }
  __device__ __forceinline__ float lse2(int r) const { return pick(lds_read16(at + 32 * (r >> 2)), r); }
  __device__ __forceinline__ float delta(int r) const { return pick(lds_read16(at + 128 + 32 * (r >> 2)), r); }
};

// keys of a tile of the dq launch
template <int D>
constexpr int dq_tile_keys() {
  return 64;
}
template <int D>
constexpr size_t dq_lds_bytes() {
  return 512 + 4 * size_t(TileLds<D, dq_tile_keys<D>()>::kBytes) + 512;
}

template <bool F16>
__device__ __forceinline__ uint4 pack8(const float (&x)[16], int h) {
  using M = Mma<F16>;
  return make_uint4(M::pack2(x[8 * h + 0], x[8 * h + 1]), M::pack2(x[8 * h + 2], x[8 * h + 3]),
                    M::pack2(x[8 * h + 4], x[8 * h + 5]), M::pack2(x[8 * h + 6], x[8 * h + 7]));
}

// What that rounding left: g goes to its products as a sum of two 16-bit numbers, 16 significant bits in bf16 (22 in fp16).
// With one number the error of dq and dk is that of g and the result's own rounding together, sqrt 2 of what it has to be.
// Measured, relative to 64 bits, 64 heads x 4096 in bf16: 2.4e-3 against 2.8e-3 (the rounding of the results alone: 1.7e-3; the
// rest comes with `out`, from which D is formed), at 1.13 against 0.97 ms.
template <bool F16>
__device__ __forceinline__ uint4 pack8_rest(const float (&x)[16], int h, const uint4& u) {
  using M = Mma<F16>;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = M::pack2(x[8 * h + 2 * i] - M::lo(w[i]), x[8 * h + 2 * i + 1] - M::hi(w[i]));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// ---- dq -------------------------------------------------------------------------------------------------
template <bool F16, int D, int MODE, bool DOCS>
__device__ __forceinline__ void dq_block(const BwdTileArgs& a, int block, bf16_t* lds_all) {
  using M = Mma<F16>;
  constexpr int KT = dq_tile_keys<D>(), NB = KT / 32;
  typedef TileLds<D, KT> T;
  typedef typename std::conditional<F16, f16_t, bf16_t>::type E;
  constexpr int NKS = D / 16, NDT = D / 32;
  int* flag = reinterpret_cast<int*>(lds_all);
  lds_char_t* lds = (lds_char_t*)(lds_all + 256);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(lds)));
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5;
  if (tid == 0) *flag = 0;
  float g_scale = 1.f;
  if constexpr (F16) g_scale = grad_scale(a, reinterpret_cast<float*>(lds_all) + 16);
  __syncthreads();
  const int heads = a.H * a.G, bx = block % heads;
  const int hk = bx % a.H, hq = hk * a.G + bx / a.H;
  const int rest = block / heads, piece = rest % a.dq_pieces, qb = (a.S + kTQ - 1) / kTQ - 1 - rest / a.dq_pieces;
  const int i0 = qb * kTQ, wq0 = i0 + 32 * w, iq = wq0 + col;
  const bool q_ok = iq < a.S;
  const int pos = iq + (a.L - a.S);
  const float slope2 = (MODE & kModeBias) ? scalar_load(a.t.slopes, hq) * kLog2e : 0.f;
  int lim, doc = 0, lim_lo, lim_hi, wg_lo, wg_hi;
  int2 q_doc = make_int2(0, 0), wg_doc = make_int2(0, 0);
  if (a.use_masks) {
    const int2 qi = a.m.qinfo[iq];
    lim = qi.x, doc = qi.y;
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
  wg_lo = __builtin_amdgcn_readfirstlane(wg_lo);
  const int qd_lo = __builtin_amdgcn_readfirstlane(q_doc.x), qd_hi = __builtin_amdgcn_readfirstlane(q_doc.y);
  const int wd_lo = __builtin_amdgcn_readfirstlane(wg_doc.x), wd_hi = __builtin_amdgcn_readfirstlane(wg_doc.y);

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
  const float2 rd = q_ok ? a.rd[row] : make_float2(0.f, 0.f);
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

  FlatSource<D, KT> src{a.k + int64_t(hk) * a.L * D, a.v + int64_t(hk) * a.L * D, a.L};
  int t_end = __builtin_amdgcn_readfirstlane((wg_hi + KT - 1) / KT);
  int mask_at = -64;
  unsigned long long mask = 0;
  auto next = [&](int t) {
    if constexpr (!DOCS) return t;
    while (t < t_end) {
      if (t >= mask_at + 64 || mask_at < 0) {
        mask_at = t;
        const int2 km = tile_docs<KT>(a.m.kmeta, min(t + l, t_end - 1));
        mask = __ballot(t + l < t_end && km.y >= wd_lo && km.x <= wd_hi && km.y >= 0);
      }
      const unsigned long long m = mask >> (t - mask_at);
      if (m) return t + __ffsll(m) - 1;
      t = mask_at + 64;
    }
    return t_end;
  };
  bool dirty = false;
  const typename T::Bases bases(l);
  const uint32_t lds_docs = lds0 + 4u * T::kBytes;
  auto compute = [&](int t, int buf, int2 km) {
    const int kp0 = t * KT;
    if (kp0 >= lim_hi) return;
    bool masked = kp0 + KT > lim_lo;
    if constexpr (DOCS) {
      if (km.y < qd_lo || km.x > qd_hi) return;
      masked |= km.x != km.y || qd_lo != qd_hi;
    }
    const auto at = bases.fresh(buf * 2 * T::kBytes);
#pragma unroll
    for (int sb = 0; sb < NB; ++sb) {
      typename M::f16v s, p;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f, p[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        s = M::m32(T::rows32(lds, at.rows, 32 * sb, ks), qf[ks], s);
        p = M::m32(T::rows32(lds + T::kBytes, at.rows, 32 * sb, ks), df[ks], p);
      }
      if constexpr ((MODE & kModeCap) != 0) tile_settle(s);
      float x[16], g[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = s[r];
      const int key0 = kp0 + 32 * sb + 4 * hb;
      block_probs<MODE>(x, g, a.score, float(pos - key0), slope2, ColumnQuery{rd.x});
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        g[r] *= p[r] - rd.y;
        if constexpr (F16) g[r] *= g_scale;
      }
      if (masked) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          uint4 dk = make_uint4(0, 0, 0, 0);
          if constexpr (DOCS) dk = lds_read16(lds + 4 * T::kBytes + buf * 256 + (key0 - kp0 + 8 * r4) * 4);
          const int dd[4] = {int(dk.x), int(dk.y), int(dk.z), int(dk.w)};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            bool ok = key0 + 8 * r4 + r < lim;
            if constexpr (DOCS) ok = ok && dd[r] == doc;
            if (!ok) g[4 * r4 + r] = 0.f;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 gf = pack8<F16>(g, h), gr = pack8_rest<F16>(g, h, gf);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const auto kt = T::cols32(lds, at.cols, 32 * sb + 16 * h, dt);
          O[dt] = M::m32(kt, gf, O[dt]);
          O[dt] = M::m32(kt, gr, O[dt]);
        }
      }
    }
  };
  int t = next(0), t_begin = 0;
  if (a.dq_pieces > 1) {
    tile_piece(t, t_end, piece, a.dq_pieces);
    t_begin = t;
    t = next(t);
  }
  if (t < t_end) {
    src.issue(t, lds0, lds0 + T::kBytes, w, l);
    if constexpr (DOCS) issue_docs<KT>(a.m.dock, t, lds_docs, w, l);
  }
  auto step = [&](int buf) {
    const int t_next = next(t + 1);
    int2 km = make_int2(0, 0);
    if constexpr (DOCS) km = tile_docs_scalar<KT>(a.m.kmeta, t);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    ring_barrier();
    if (t_next < t_end) {
      const uint32_t to = lds0 + uint32_t(buf ^ 1) * 2u * T::kBytes;
      src.issue(t_next, to, to + T::kBytes, w, l);
      if constexpr (DOCS) issue_docs<KT>(a.m.dock, t_next, lds_docs + uint32_t(buf ^ 1) * 256u, w, l);
    }
    bool wg_masked = t * KT + KT > wg_lo;
    if constexpr (DOCS) wg_masked |= km.x != km.y || wd_lo != wd_hi;
    if (wg_masked) {
      const lds_char_t* bK = lds + buf * 2 * T::kBytes;
#pragma unroll
      for (int u = 0; u < T::kBytes / 4096; ++u) dirty |= any_nonfinite<F16>(lds_read16(bK + (u * 256 + tid) * 16));
    }
    compute(t, buf, km);
    t = t_next;
  };
  if constexpr (D >= 128) {
    for (int buf = 0; t < t_end; buf ^= 1) step(buf);
  } else {
    while (t < t_end) {
      step(0);
      if (t >= t_end) break;
      step(1);
    }
  }
  if (dirty) *flag = 1;
  __syncthreads();
  if (*flag == 0) {
    if (!q_ok) return;
    const float f = a.sm_scale / g_scale;
    if (a.dq_pieces > 1) {
      float* to = a.part_dq + (int64_t(piece) * a.H * a.G * a.S + row) * D;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq)
          *reinterpret_cast<float4*>(to + dt * 32 + 8 * rq + 4 * hb) =
              make_float4(O[dt][4 * rq] * f, O[dt][4 * rq + 1] * f, O[dt][4 * rq + 2] * f, O[dt][4 * rq + 3] * f);
      return;
    }
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
    const E *q = (const E*)a.q + r * D, *o = (const E*)a.dout + r * D;
    const QueryView qv = query_view(a.t, i, a.S, a.L, hq);
    if (a.dq_pieces > 1)
      row_dq<E, (MODE & kModeCap) != 0>(q, o, a.rd[r], K, V, qv, a.t.doc_k, t_begin * KT, t_end * KT, a.sm_scale, score,
                                        a.part_dq + (int64_t(piece) * a.H * a.G * a.S + r) * D);
    else
      row_dq<E, (MODE & kModeCap) != 0>(q, o, a.rd[r], K, V, qv, a.t.doc_k, 0, a.L, a.sm_scale, score, (E*)a.dq + r * D);
  }
}

// ---- dk, dv ------------------------------------------------------------------------------------------------
constexpr int kDkvKeys = 128;  // keys of a workgroup
constexpr int kDkvQ = 32;      // queries of a tile

// the values of the workgroup's keys, two tiles of q and dout, two of {lse log2 e, D} and {limit, document} of the queries
template <int D>
constexpr size_t dkv_lds_bytes() {
  return 512 + size_t(TileLds<D, kDkvKeys>::kBytes) + 4 * size_t(TileLds<D, kDkvQ>::kBytes) + 2 * 2 * kDkvQ * 8;
}

// What a block of keys forms.  At head dimension 256 the accumulators of both gradients, 256 registers a lane, leave too
// few for the rest: dv and dk have workgroups of their own there, and the scores are formed twice.
constexpr int kDkAndDv = 0, kDvOnly = 1, kDkOnly = 2;

template <bool F16, int D, int MODE, bool DOCS, int PART>
__device__ __forceinline__ void dkv_block(const BwdTileArgs& a, int block, bf16_t* lds_all) {
  using M = Mma<F16>;
  typedef TileLds<D, kDkvQ> T;
  typedef TileLds<D, kDkvKeys> TV;
  typedef typename std::conditional<F16, f16_t, bf16_t>::type E;
  constexpr int NKS = D / 16, NDT = D / 32;
  constexpr float p_scale = F16 ? kPScaleF16 : 1.f;
  int* flag = reinterpret_cast<int*>(lds_all);
  lds_char_t* lds_v = (lds_char_t*)(lds_all + 256);
  lds_char_t* lds = lds_v + TV::kBytes;
  lds_char_t* lds_row = lds + 4 * T::kBytes;  // [2]{ lse log2 e [32], D [32], limit [32], document [32] }
  const uint32_t lds_v0 = __builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(lds_v)));
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(lds)));
  const uint32_t lds_row0 = __builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(lds_row)));
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5;
  if (tid == 0) *flag = 0;
  float g_scale = 1.f;
  if constexpr (F16) g_scale = grad_scale(a, reinterpret_cast<float*>(lds_all) + 16);
  __syncthreads();
  // the first keys, which a causal mask shows to the most queries, go first
  const int hk = block % a.H, rest = block / a.H;
  const int split = rest % a.splits, j0 = (rest / a.splits) * kDkvKeys;
  const int wj0 = j0 + 32 * w, j = wj0 + col;
  const bool j_ok = j < a.L;
  int doc = 0;
  int2 k_doc = make_int2(0, 0), wg_doc = make_int2(0, 0);  // of the wave's keys, of the workgroup's
  if constexpr (DOCS) {
    doc = a.m.dock[j];
    const int2 m0 = tile_docs_scalar<64>(a.m.kmeta, j0 / 64), m1 = tile_docs_scalar<64>(a.m.kmeta, j0 / 64 + 1);
    k_doc = scalar_load(a.m.kmeta, j0 / 32 + w);
    wg_doc = make_int2(min(m0.x, m1.x), max(m0.y, m1.y));
  }
  // keys in registers, values in LDS: with both in registers a wave would need more than half of its SIMD's
  uint4 kf[NKS];
  {
    const uint4* pk = reinterpret_cast<const uint4*>(a.k + (int64_t(hk) * a.L + (j_ok ? j : 0)) * D + hb * 8);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) kf[ks] = j_ok ? pk[2 * ks] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) asm volatile("" : "+v"(kf[ks].x), "+v"(kf[ks].y), "+v"(kf[ks].z), "+v"(kf[ks].w));
  if constexpr (PART != kDvOnly) {
    const bf16_t* bv = ring_uniform_ptr(a.v + (int64_t(hk) * a.L + j0) * D);
#pragma unroll
    for (int u = 0; u < TV::kLoadsPerWave; ++u) {
      const int r = TV::load_row(w + 4 * u, l);
      tile_load(lds_v0 + uint32_t(w + 4 * u) * 1024u, uint32_t(min(r, a.L - 1 - j0)) * TV::kRowBytes + TV::load_chunk(r, l), bv);
    }
  }
  typename M::f16v dK[NDT], dV[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) dK[dt][r] = 0.f, dV[dt][r] = 0.f;

  // Steps: tile qt of 32 queries of head g, from the last tile down to the first that can see the workgroup's keys (so
  // that workgroups with other keys, which see other first queries, read the same tiles at the same time):
  // step = g n + (last - qt), and this workgroup's are [s0, s1).
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
        const int4 x = a.m.qmeta[nqt - 1 - min(s + l, s1 - 1) % n];
        bool hit = s + l < s1 && x.y > j0;
        if constexpr (DOCS) hit = hit && wg_doc.y >= 0 && x.w >= wg_doc.x && x.z <= wg_doc.y;
        mask = __ballot(hit);
      }
      const unsigned long long m = mask >> (s - mask_at);
      if (m) return s + __ffsll(m) - 1;
      s = mask_at + 64;
    }
    return s1;
  };
  // a step's head and tile, kept by counting on
  struct Place {
    int s, g, qt;
  };
  auto place_at = [&](int s) {
    const int g = n > 0 ? s / n : 0;
    return Place{s, g, nqt - 1 - (s - g * n)};
  };
  auto move_to = [&](Place p, int s) {
    p.qt -= s - p.s;
    p.s = s;
    while (p.qt < qt0) p.qt += n, ++p.g;
    return p;
  };
  const int64_t head0 = int64_t(hk) * a.G * a.S;
  auto issue = [&](const Place& p, int buf) {
    const int i0 = p.qt * kDkvQ, last = a.S - 1 - i0;
    const int64_t row = head0 + (p.g * a.S + i0);
    const bf16_t* bq = ring_uniform_ptr(a.q + row * D);
    const bf16_t* bd = ring_uniform_ptr(a.dout + row * D);
    const uint32_t to = lds0 + uint32_t(buf) * 2u * T::kBytes;
#pragma unroll
    for (int u = 0; u < T::kLoadsPerWave; ++u) {
      const int r = T::load_row(w + 4 * u, l);
      const uint32_t voff = uint32_t(min(r, last)) * T::kRowBytes + T::load_chunk(r, l);
      tile_load(to + uint32_t(w + 4 * u) * 1024u, voff, bq);
      tile_load(to + T::kBytes + uint32_t(w + 4 * u) * 1024u, voff, bd);
    }
    // 8 bytes a query: wave 0 {lse log2 e, D}, wave 1 {limit, document} where there are masks; the halves of a wave take one each,
    // so that four queries' are 16 consecutive bytes in LDS
    const uint32_t voff = uint32_t(min(l & 31, last)) * 8u + uint32_t(l >> 5) * 4u;
    if (w == 0) ring_load4(lds_row0 + uint32_t(buf) * 512u, voff, ring_uniform_ptr(a.rd + row));
    if (w == 1 && a.use_masks) ring_load4(lds_row0 + uint32_t(buf) * 512u + 256u, voff, ring_uniform_ptr(a.m.qinfo + i0));
  };
  bool dirty = false;
  const typename T::Bases bases(l);
  const int L_end = min(j0 + kDkvKeys, a.L);
  auto compute = [&](const Place& p, int buf, const int4& qm) {
    const int i0 = p.qt * kDkvQ;
    const lds_char_t* bQ = lds + buf * 2 * T::kBytes;
    const lds_char_t* bD = bQ + T::kBytes;
    const lds_char_t* rows = lds_row + buf * 512;
    // who sees what: fewest and most keys of the 32 queries
    int lo, hi;
    bool mixed = false;
    if (a.use_masks) {
      lo = qm.x, hi = qm.y;
      if constexpr (DOCS) mixed = k_doc.x != k_doc.y || qm.z != qm.w || qm.z != k_doc.x || wg_doc.x != wg_doc.y;
    } else {
      lo = seen_limit(i0 + (a.L - a.S), a.L, a.t.causal, 0);
      hi = seen_limit(min(i0 + 31, a.S - 1) + (a.L - a.S), a.L, a.t.causal, 0);
    }
    const bool ragged = i0 + kDkvQ > a.S;
    if (ragged || mixed || lo < L_end) {
#pragma unroll
      for (int u = 0; u < (T::kBytes + 4095) / 4096; ++u) {
        const int at = (u * 256 + tid) * 16;
        if (T::kBytes % 4096 && at >= T::kBytes) continue;
        dirty |= any_nonfinite<F16>(lds_read16(bQ + at)) | any_nonfinite<F16>(lds_read16(bD + at));
      }
    }
    if (hi <= wj0) return;
    const float slope2 = (MODE & kModeBias) ? scalar_load(a.t.slopes, hk * a.G + p.g) * kLog2e : 0.f;
    const auto at = bases.fresh(buf * 2 * T::kBytes);
    int vrows = bases.rows + 32 * w * TV::kRowBytes;
    asm volatile("" : "+v"(vrows));
    // scores, p, and dv first, then dP, g and dk: of the two products' operands one is held at a time
    typename M::f16v sc;
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) sc = M::m32(T::rows32(lds, at.rows, 0, ks), kf[ks], sc);
    if constexpr ((MODE & kModeCap) != 0) tile_settle(sc);
    float x[16], y[16];  // p; p slack
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = sc[r];
    const RowQueries rq{rows + 4 * hb * 4};
    block_probs<MODE>(x, y, a.score, float(j - (i0 + 4 * hb + (a.L - a.S))), slope2, rq);
    const bool masked = mixed || ragged || wj0 + 32 > lo;
    constexpr float kUnseen = -4.f;  // in the place of p slack, which is 0 or (rounded) -2^-21 p at the least
    if (masked) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int iq = 4 * hb + 8 * q;
        uint4 lim = make_uint4(0, 0, 0, 0), docs = lim;
        if (a.use_masks) {
          lim = lds_read16(rows + 256 + iq * 4);
          if constexpr (DOCS) docs = lds_read16(rows + 384 + iq * 4);
        }
        const int ll[4] = {int(lim.x), int(lim.y), int(lim.z), int(lim.w)}, dd[4] = {int(docs.x), int(docs.y), int(docs.z), int(docs.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = i0 + iq + e;
          bool ok = i < a.S && j < (a.use_masks ? ll[e] : seen_limit(i + (a.L - a.S), a.L, a.t.causal, 0));
          if constexpr (DOCS) ok = ok && dd[e] == doc;
          if (!ok) x[4 * q + e] = 0.f, y[4 * q + e] = kUnseen;
        }
      }
    }
    if constexpr (PART != kDkOnly) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (F16) {
#pragma unroll
          for (int r = 0; r < 8; ++r) x[8 * h + r] *= p_scale;
        }
        const uint4 pf = pack8<F16>(x, h);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) dV[dt] = M::m32(T::cols32(lds + T::kBytes, at.cols, 16 * h, dt), pf, dV[dt]);
      }
    }
    if constexpr (PART == kDvOnly) return;
    typename M::f16v pr;
#pragma unroll
    for (int r = 0; r < 16; ++r) pr[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) pr = M::m32(T::rows32(lds + T::kBytes, at.rows, 0, ks), TV::rows32(lds_v, vrows, 0, ks), pr);
    float gr[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      gr[r] = (pr[r] - rq.delta(r)) * y[r];
      if constexpr (F16) gr[r] *= g_scale;
    }
    if (masked) {  // (where the mask is, not where p is 0: a seen pair's may be, beside a gradient that is not finite)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (y[r] == kUnseen) gr[r] = 0.f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 gf = pack8<F16>(gr, h), rest = pack8_rest<F16>(gr, h, gf);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const auto qt = T::cols32(lds, at.cols, 16 * h, dt);
        dK[dt] = M::m32(qt, gf, dK[dt]);
        dK[dt] = M::m32(qt, rest, dK[dt]);
      }
    }
  };
  int s = next(s0);
  Place here = place_at(min(s, s1 - 1 < s0 ? s0 : s1 - 1));
  if (s < s1) issue(here, 0);
  auto step = [&](int buf) {
    const int s_next = next(s + 1);
    int4 qm = make_int4(0, 0, 0, 0);
    if (a.use_masks) qm = scalar_load(a.m.qmeta, here.qt);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    ring_barrier();
    Place there = here;
    if (s_next < s1) {
      there = move_to(here, s_next);
      issue(there, buf ^ 1);
    }
    compute(here, buf, qm);
    here = there;
    s = s_next;
  };
  if constexpr (D >= 128) {  // (two copies of the step: the accumulators would not fit the registers)
    for (int buf = 0; s < s1; buf ^= 1) step(buf);
  } else {
    while (s < s1) {
      step(0);
      if (s >= s1) break;
      step(1);
    }
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
          if constexpr (PART != kDvOnly) *reinterpret_cast<float4*>(a.part + 2 * split * plane + at) = x;
          if constexpr (PART != kDkOnly) *reinterpret_cast<float4*>(a.part + (2 * split + 1) * plane + at) = y;
        } else {
          if constexpr (PART != kDvOnly) *reinterpret_cast<uint2*>(a.dk + at) = make_uint2(M::pack2(x.x, x.y), M::pack2(x.z, x.w));
          if constexpr (PART != kDkOnly) *reinterpret_cast<uint2*>(a.dv + at) = make_uint2(M::pack2(y.x, y.y), M::pack2(y.z, y.w));
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
      const int g = ss / n, qt = nqt - 1 - (ss - g * n);
      row_dkv_chunk<E, (MODE & kModeCap) != 0>((const E*)a.k + at, (const E*)a.v + at, jj, hk * a.G + g, qt * kDkvQ,
                                               min(a.S, (qt + 1) * kDkvQ), a.S, a.L, D,
                                               (const E*)a.q, (const E*)a.dout, a.rd, a.t, score, kg);
    }
    for (int r = 0; r < (D + 63) / 64; ++r) {
      const int c = l + 64 * r;
      if (c >= D) continue;
      if (a.splits > 1) {
        if constexpr (PART != kDvOnly) a.part[2 * split * plane + at + c] = kg.k[r] * a.sm_scale;
        if constexpr (PART != kDkOnly) a.part[(2 * split + 1) * plane + at + c] = kg.v[r];
      } else {
        if constexpr (PART != kDvOnly) Elem<E>::store((E*)a.dk + at + c, kg.k[r] * a.sm_scale);
        if constexpr (PART != kDkOnly) Elem<E>::store((E*)a.dv + at + c, kg.v[r]);
      }
    }
  }
}

// One launch: the blocks of keys first, heaviest first, then those of queries, which fill the card as the others end.
template <bool F16, int D, int MODE, bool DOCS>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void terms_bwd_kernel(BwdTileArgs a, int dkv_blocks) {
  extern __shared__ __attribute__((aligned(256))) bf16_t lds_all[];
  const int block = blockIdx.x;
  if constexpr (D == 256) {
    if (block < dkv_blocks) return dkv_block<F16, D, MODE, DOCS, kDkOnly>(a, block, lds_all);
    if (block < 2 * dkv_blocks) return dkv_block<F16, D, MODE, DOCS, kDvOnly>(a, block - dkv_blocks, lds_all);
    dq_block<F16, D, MODE, DOCS>(a, block - 2 * dkv_blocks, lds_all);
  } else {
    if (block < dkv_blocks) return dkv_block<F16, D, MODE, DOCS, kDkAndDv>(a, block, lds_all);
    dq_block<F16, D, MODE, DOCS>(a, block - dkv_blocks, lds_all);
  }
}

// The pieces' sums in order, each rounded once: dk and dv ([2][plane]) from `part`, then dq from `part_dq`, where they have any.
template <bool F16>
__global__ __launch_bounds__(256) void terms_bwd_join_kernel(BwdTileArgs a, int64_t plane, int64_t plane_q) {
  int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  const int64_t kv = a.splits > 1 ? 2 * plane : 0;
  const float* from = a.part + i;
  int64_t step = 2 * plane;
  int n = a.splits;
  bf16_t* to = i < plane ? a.dk + i : a.dv + (i - plane);
  if (i >= kv) {
    i -= kv;
    if (a.dq_pieces == 1 || i >= plane_q) return;
    from = a.part_dq + i, step = plane_q, n = a.dq_pieces, to = a.dq + i;
  }
  float4 s = *reinterpret_cast<const float4*>(from);
  for (int k = 1; k < n; ++k) {
    const float4 x = *reinterpret_cast<const float4*>(from + k * step);
    s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
  }
  *reinterpret_cast<uint2*>(to) = make_uint2(Mma<F16>::pack2(s.x, s.y), Mma<F16>::pack2(s.z, s.w));
}

template <bool F16, int D, int MODE, bool DOCS>
static int launch_terms_bwd_docs(const BwdTileArgs& a, hipStream_t st) {
  constexpr size_t lds = std::max(dq_lds_bytes<D>(), dkv_lds_bytes<D>());
  FM_ALLOW_LDS((terms_bwd_kernel<F16, D, MODE, DOCS>), lds, "fm_local_attn_terms_bwd(lds)");
  const int dkv = int(a.H * a.splits * ceil_div(a.L, kDkvKeys)), dq = int(a.H * a.G * ceil_div(a.S, kTQ) * a.dq_pieces);
  hipLaunchKernelGGL((terms_bwd_kernel<F16, D, MODE, DOCS>), dim3(unsigned((D == 256 ? 2 : 1) * dkv + dq)), dim3(256), lds, st, a, dkv);
  return launch_status("fm_local_attn_terms_bwd(tiles)");
}

template <bool F16, int D, int MODE>
static int launch_terms_bwd(const BwdTileArgs& a, hipStream_t st) {
  const int rc = a.t.doc_q ? launch_terms_bwd_docs<F16, D, MODE, true>(a, st) : launch_terms_bwd_docs<F16, D, MODE, false>(a, st);
  if (rc) return rc;
  if (a.splits > 1 || a.dq_pieces > 1) {
    const int64_t plane = int64_t(a.H) * a.L * D, plane_q = int64_t(a.H) * a.G * a.S * D;
    const int64_t n = (a.splits > 1 ? 2 * plane : 0) + (a.dq_pieces > 1 ? plane_q : 0);
    hipLaunchKernelGGL((terms_bwd_join_kernel<F16>), dim3(unsigned(ceil_div(n, 1024))), dim3(256), 0, st, a, plane, plane_q);
  }
  return launch_status("fm_local_attn_terms_bwd(join)");
}

template <bool F16, int D>
static int launch_terms_bwd_type(const BwdTileArgs& a, const void* out, const float* lse, const float* dlse, float2* rd, float* norms, hipStream_t st) {
  const int64_t rows = int64_t(a.H) * a.G * a.S, keys = int64_t(a.H) * a.L;
  const int qb = int(ceil_div(rows, kNormRows)), kb = F16 ? int(ceil_div(keys, kNormRows)) : 0;
  hipLaunchKernelGGL((terms_delta_tile_kernel<F16, D>), dim3(unsigned(qb + kb)), dim3(256), 0, st, (const bf16_t*)out, a.dout, lse,
                     dlse, a.v, rd, norms, rows, keys, qb, a.S, a.L, a.use_masks ? a.m.qinfo : nullptr, a.use_masks ? a.m.dock : nullptr);
  switch ((a.t.softcap > 0.f ? kModeCap : 0) | (a.t.slopes ? kModeBias : 0)) {
    case 0: return launch_terms_bwd<F16, D, 0>(a, st);
    case kModeCap: return launch_terms_bwd<F16, D, kModeCap>(a, st);
    case kModeBias: return launch_terms_bwd<F16, D, kModeBias>(a, st);
    default: return launch_terms_bwd<F16, D, kModeCap | kModeBias>(a, st);
  }
}

template <int D>
int terms_bwd_tiles(const BwdTileArgs& a, bool f16, const void* out, const float* lse, const float* dlse, float2* rd, float* norms, hipStream_t st) {
  return f16 ? launch_terms_bwd_type<true, D>(a, out, lse, dlse, rd, norms, st)
             : launch_terms_bwd_type<false, D>(a, out, lse, dlse, rd, norms, st);
}

}  // namespace fm
