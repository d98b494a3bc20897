// Attention of new tokens over a paged cache in fp32 products (terms_f32.hpp): fp32 caches at any head dimension up to 256 and
// any page size, and the 16-bit types where paged_attn.hpp's kernels are not laid out for the call.
//
// A workgroup per 32 query rows of a (row, KV head) and piece of the keys, found as paged_many_kernel finds its blocks; its four
// waves take tiles of 32 keys in turn.  A tile's 32 rows are looked up a tile ahead, one key a lane, so that a page may be as
// small as one key.  Bound: short calls by latency, long caches by their bytes, many query rows by the fp32 matrix products.
// Measured, fp32, 8 KV heads, d = 128: a token for each of 64 rows of up to 512 keys (32 query heads) 55 us = 3.5 TB/s, for each of 32
// rows of up to 16 384 (64 query heads) 712 = 4.8; chunks of 1024 behind up to 8192 (four rows, 32 query heads) 4.17 ms = 97 TFLOP/s; one
// token for one row of 512 27 us.  bf16: d = 96, the first of these 146 us, chunks 9.8 ms; d = 128 in pages of 8 keys, 65 us and 4.85 ms.
#pragma once
#include "paged_attn.hpp"
#include "terms_f32.hpp"

namespace fm {

constexpr int kF32Rows = 32;  // query rows of a workgroup

template <typename T, int VEC, int NDT>
__global__ __launch_bounds__(256, 1) void paged_f32_kernel(PagedTileArgs a, F32Score score) {
  extern __shared__ __attribute__((aligned(256))) float f32_lds[];
  int* flag = reinterpret_cast<int*>(f32_lds);
  float* lds = f32_lds + 64;
  float2* ml = reinterpret_cast<float2*>(lds + kMeetFloats<NDT>);
  const PagedArgs& p = a.p;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5, d = f32_dims<VEC, NDT>(p.d);
  const int units = p.H * a.many_slots * a.many_pieces;
  if (int(blockIdx.x) >= units) return paged_nobody<T>(a, int(blockIdx.x) - units, int(gridDim.x) - units);
  const int hk = int(blockIdx.x) % p.H, rest = int(blockIdx.x) / p.H;
  const int piece = rest % a.many_pieces, slot = a.many_slots - 1 - rest / a.many_pieces;
  int row, r0;
  paged_slot<kF32Rows>(p, slot, row, r0);
  const PagedRow pr = paged_row(p, row);
  const int n = pr.q1 - pr.q0, n_rows = n * p.G;
  if (n <= 0 || r0 < 0 || r0 >= n_rows) return;
  if (tid == 0) *flag = 0;
  __syncthreads();
  const int prefix = p.prefix ? p.prefix[row] : 0;
  const int r = r0 + col;
  const bool ok = r < n_rows;
  const int tok = ok ? r / p.G : 0, hq = hk * p.G + (ok ? r - tok * p.G : 0), t = pr.q0 + tok;
  auto lim_of = [&](int rr) { return seen_limit(pr.len - n + rr / p.G, pr.len, 1, prefix); };
  const int pos = pr.len - n + tok, lim = ok ? seen_limit(pos, pr.len, 1, prefix) : 0;
  const float slope2 = p.slopes ? p.slopes[hq] * kLog2e : 0.f;
  const int lim_lo = lim_of(r0), lim_hi = lim_of(min(r0 + kF32Rows, n_rows) - 1);
  float qf[16 * NDT];
  f32_resident<T, VEC, NDT>(qf, (const T*)p.q + t * p.q_token + hq * p.q_head, ok, d, hb);
  int j0, j1;
  piece_keys(lim_hi, 32, piece, a.many_pieces, j0, j1);
  const int64_t head = int64_t(hk) * p.page * d;
  auto row_of = [&](int j) {
    j = max(j, 0);
    return page_offset(p, pr.table[j >> p.log2p], d) + int64_t(j & (p.page - 1)) * d;
  };
  const F32Docs docs{nullptr, nullptr, 0, 0, 0, false};
  f32_acc O[NDT];
  float m, sum;
  bool dirty = false;
  f32_forward<T, VEC, NDT, false>(F32Regs<NDT>{qf}, pos, lim, slope2, lim_lo, (const T*)p.k + head, (const T*)p.v + head, row_of, pr.len, j0 / 32 + w,
                                  4, (j1 + 31) / 32, d, score, docs, O, m, sum, dirty);
  if (dirty) *flag = 1;
  sum += __shfl_xor(sum, 32);
  f32_put<NDT>(lds, O, 0, w, col, hb);
  if (hb == 0) ml[w * 32 + col] = make_float2(m, sum);
  __syncthreads();
  if (*flag) {
    for (int rr = r0 + w; rr < min(r0 + kF32Rows, n_rows); rr += 4)
      paged_row_again<T>(a, pr, pr.q0 + rr / p.G, hk * p.G + rr % p.G, j0, j1,
                         many_index(a, pr.q0 + rr / p.G, hk * p.G + rr % p.G) + piece, a.many_pieces);
    return;
  }
  const int rows = min(kF32Rows, n_rows - r0);
  auto place = [&](int i, int& tt, int& rq) {  // the token and query head of row i
    const int rt = (r0 + i) / p.G;
    tt = pr.q0 + rt, rq = hk * p.G + (r0 + i - rt * p.G);
  };
  if (l == 0)
    for (int i = w; i < rows; i += 4) {
      int tt, rq;
      place(i, tt, rq);
      const float2 st = f32_meet(ml, i);
      if (a.many_pieces > 1)
        a.part_ml[many_index(a, tt, rq) + piece] = st;
      else
        p.lse[tt * p.l_token + rq * p.l_head] = st.y == 0.f ? -FLT_MAX : (st.x + __builtin_amdgcn_logf(st.y)) * kLn2;
    }
  f32_meet_all<NDT>(lds, O, w, col, hb, rows, d, [&](int i, float (&g)[4]) { f32_weights(ml, i, a.many_pieces == 1, g); },
                    [&](int i, int c, float x) {
                      int tt, rq;
                      place(i, tt, rq);
                      if (a.many_pieces > 1)
                        a.part_o[(many_index(a, tt, rq) + piece) * d + c] = x;
                      else
                        Elem<T>::store((T*)p.out + tt * p.o_token + rq * p.o_head + c, x);
                    });
}

// the pieces of a query row, in order: a wave a row
template <typename T>
__global__ __launch_bounds__(256) void paged_f32_join_kernel(PagedTileArgs a) {
  const int HG = a.p.H * a.p.G;
  const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int t = int(unit / HG), hq = int(unit - int64_t(t) * HG);
  if (t >= a.p.T) return;
  const PagedRow pr = paged_row_of_token(a.p, t);
  if (pr.row < 0) return;  // (written where nobody's tokens are)
  const int64_t at = many_index(a, t, hq);
  f32_join_row(a.part_o + at * a.p.d, a.part_ml + at, a.many_pieces, a.p.d, (T*)a.p.out + t * a.p.o_token + hq * a.p.o_head,
               a.p.lse + t * a.p.l_token + hq * a.p.l_head);
}

template <typename T, int VEC, int NDT>
static int launch_paged_f32(const PagedTileArgs& a, hipStream_t st) {
  FM_ALLOW_LDS((paged_f32_kernel<T, VEC, NDT>), f32_lds_bytes<NDT>(), "fm_paged_attn_fwd(lds)");
  hipLaunchKernelGGL((paged_f32_kernel<T, VEC, NDT>), dim3(unsigned(a.p.H * a.many_slots * a.many_pieces + nobody_groups(a.p))), dim3(256),
                     f32_lds_bytes<NDT>(), st, a, f32_score(a.p.sm_scale, a.p.softcap));
  return launch_status("fm_paged_attn_fwd(f32)");
}

template <typename T>
int paged_f32(const PagedTileArgs& a, const PagedPlan& y, hipStream_t st) {
  const int vec = a.p.q_token % 4 == 0 && a.p.q_head % 4 == 0 ? f32_vec<T>(a.p.d, {a.p.q, a.p.k, a.p.v}) : kOne;
#define FM_F(V, N) launch_paged_f32<T, V, N>(a, st)
  const int rc = FM_F32_BY_DIM(a.p.d, vec, FM_F);
#undef FM_F
  if (rc || y.many_pieces == 1) return rc;
  const int64_t units = int64_t(a.p.T) * a.p.H * a.p.G;
  hipLaunchKernelGGL(paged_f32_join_kernel<T>, dim3(unsigned(ceil_div(units, 4))), dim3(256), 0, st, a);
  return launch_status("fm_paged_attn_fwd(join)");
}

}  // namespace fm
