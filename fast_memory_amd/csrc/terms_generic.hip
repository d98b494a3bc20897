// Attention with score terms, a wave per row: any type, any head dimension up to 256, any page size.  These define the
// operators (terms.hpp) and serve what the tiled kernels are not built for.  Bound: VALU (a multiply-add per lane, key
// and dimension, twice in the forward and five times in the backward, none of them on the matrix pipes).
#include "terms.hpp"
#include "terms_api.hpp"

namespace fm {

template <typename T, bool CAP>
__global__ __launch_bounds__(256) void terms_fwd_row_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                            const T* __restrict__ v, T* __restrict__ out,
                                                            float* __restrict__ lse, Terms t, int G, int S, int L, int d,
                                                            int64_t rows, Score<CAP> score) {
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int hq = int(row / S), i = int(row - int64_t(hq) * S);
  const int64_t head = int64_t(hq / G) * L * d;
  const KeyRows<T> K{k + head, nullptr, 0, 0, 0, d}, V{v + head, nullptr, 0, 0, 0, d};
  const RowState st = row_forward<T, CAP>(q + row * d, K, V, query_view(t, i, S, L, hq), t.doc_k, 0, L, score);
  row_write(st, d, out + row * d, lse + row);
}

template <typename T>
int terms_fwd_rows(const FwdArgs& a, hipStream_t st) {
  const int64_t rows = int64_t(a.H) * a.G * a.S;
  const dim3 grid = dim3(unsigned(ceil_div(rows, 4)));
  if (a.t.softcap > 0.f)
    hipLaunchKernelGGL((terms_fwd_row_kernel<T, true>), grid, dim3(256), 0, st, (const T*)a.q, (const T*)a.k, (const T*)a.v,
                       (T*)a.out, a.lse, a.t, a.G, a.S, a.L, a.d, rows, Score<true>(a.sm_scale, a.t.softcap));
  else
    hipLaunchKernelGGL((terms_fwd_row_kernel<T, false>), grid, dim3(256), 0, st, (const T*)a.q, (const T*)a.k, (const T*)a.v,
                       (T*)a.out, a.lse, a.t, a.G, a.S, a.L, a.d, rows, Score<false>(a.sm_scale, 0.f));
  return launch_status("fm_local_attn_terms_fwd(rows)");
}

// {lse_i log2 e, D_i = do_i.o_i - dlse_i}, a wave per row
template <typename T>
__global__ __launch_bounds__(256) void terms_delta_kernel(const T* __restrict__ out, const T* __restrict__ dout,
                                                          const float* __restrict__ lse, const float* __restrict__ dlse,
                                                          float2* __restrict__ rd, int d, int64_t rows) {
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  float s = 0.f;
  for (int k = lane_id(); k < d; k += 64) s = fmaf(Elem<T>::load(dout + row * d + k), Elem<T>::load(out + row * d + k), s);
  s = wave_sum(s);
  if (lane_id() == 0) rd[row] = make_float2(lse[row] * kLog2e, s - (dlse ? dlse[row] : 0.f));
}

template <typename T, bool CAP>
__global__ __launch_bounds__(256) void terms_dq_row_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                           const T* __restrict__ v, const T* __restrict__ dout,
                                                           const float2* __restrict__ rd, T* __restrict__ dq, Terms t, int G, int S, int L, int d,
                                                           int64_t rows, float sm_scale, Score<CAP> score) {
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int hq = int(row / S), i = int(row - int64_t(hq) * S);
  const int64_t head = int64_t(hq / G) * L * d;
  const KeyRows<T> K{k + head, nullptr, 0, 0, 0, d}, V{v + head, nullptr, 0, 0, 0, d};
  row_dq<T, CAP>(q + row * d, dout + row * d, rd[row], K, V, query_view(t, i, S, L, hq), t.doc_k, sm_scale, score,
                 dq + row * d);
}

template <typename T, bool CAP>
__global__ __launch_bounds__(256) void terms_dkv_row_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                            const T* __restrict__ v, const T* __restrict__ dout,
                                                            const float2* __restrict__ rd, T* __restrict__ dk, T* __restrict__ dv, Terms t, int G, int S,
                                                            int L, int d, int64_t rows, float sm_scale, Score<CAP> score) {
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int hk = int(row / L), j = int(row - int64_t(hk) * L);
  row_dkv<T, CAP>(k + row * d, v + row * d, j, hk, G, S, L, d, q, dout, rd, t, sm_scale, score, dk + row * d,
                  dv + row * d);
}

template <typename T>
int terms_delta(const BwdArgs& a, float2* rd, hipStream_t st) {
  const int64_t rows = int64_t(a.f.H) * a.f.G * a.f.S;
  hipLaunchKernelGGL(terms_delta_kernel<T>, dim3(unsigned(ceil_div(rows, 4))), dim3(256), 0, st, (const T*)a.f.out,
                     (const T*)a.dout, a.f.lse, a.dlse, rd, a.f.d, rows);
  return launch_status("fm_local_attn_terms_bwd(delta)");
}

template <typename T, bool CAP>
static void launch_bwd_rows(const BwdArgs& a, const float2* rd, Score<CAP> score, hipStream_t st) {
  const FwdArgs& f = a.f;
  const int64_t rows = int64_t(f.H) * f.G * f.S, keys = int64_t(f.H) * f.L;
  hipLaunchKernelGGL((terms_dq_row_kernel<T, CAP>), dim3(unsigned(ceil_div(rows, 4))), dim3(256), 0, st, (const T*)f.q,
                     (const T*)f.k, (const T*)f.v, (const T*)a.dout, rd, (T*)a.dq, f.t, f.G, f.S, f.L, f.d, rows,
                     f.sm_scale, score);
  hipLaunchKernelGGL((terms_dkv_row_kernel<T, CAP>), dim3(unsigned(ceil_div(keys, 4))), dim3(256), 0, st, (const T*)f.q,
                     (const T*)f.k, (const T*)f.v, (const T*)a.dout, rd, (T*)a.dk, (T*)a.dv, f.t, f.G, f.S, f.L, f.d,
                     keys, f.sm_scale, score);
}

template <typename T>
int terms_bwd_rows(const BwdArgs& a, const float2* rd, hipStream_t st) {
  if (a.f.t.softcap > 0.f)
    launch_bwd_rows<T, true>(a, rd, Score<true>(a.f.sm_scale, a.f.t.softcap), st);
  else
    launch_bwd_rows<T, false>(a, rd, Score<false>(a.f.sm_scale, 0.f), st);
  return launch_status("fm_local_attn_terms_bwd(rows)");
}

// A wave per (token, head) of a paged batch.
template <typename T, bool CAP>
__global__ __launch_bounds__(256) void paged_attn_row_kernel(PagedArgs a, Score<CAP> score) {
  const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int HG = a.H * a.G;
  const int t = int(unit / HG), hq = int(unit - int64_t(t) * HG);
  if (t >= a.T) return;
  const PagedRow pr = paged_row_of_token(a, t);
  T* out = (T*)a.out + t * a.o_token + hq * a.o_head;
  float* lse = a.lse + t * a.l_token + hq * a.l_head;
  QueryView qv;
  qv.pos = pr.len - (pr.q1 - t);
  qv.lim = pr.row < 0 ? 0 : seen_limit(qv.pos, pr.len, 1, a.prefix ? a.prefix[pr.row] : 0);
  qv.use_doc = false;
  qv.doc = -1;
  qv.slope2 = a.slopes ? a.slopes[hq] * kLog2e : 0.f;
  const int64_t head = int64_t(hq / a.G) * a.page * a.d, stride = int64_t(a.H) * a.page * a.d;
  const KeyRows<T> K{(const T*)a.k + head, pr.table, stride, a.log2p, a.n_pages, a.d};
  const KeyRows<T> V{(const T*)a.v + head, pr.table, stride, a.log2p, a.n_pages, a.d};
  const RowState st = row_forward<T, CAP>((const T*)a.q + t * a.q_token + hq * a.q_head, K, V, qv, nullptr, 0, qv.lim, score);
  row_write(st, a.d, out, lse);
}

template <typename T>
int paged_attn_rows(const PagedArgs& a, hipStream_t st) {
  const dim3 grid = dim3(unsigned(ceil_div(int64_t(a.T) * a.H * a.G, 4)));
  if (a.softcap > 0.f)
    hipLaunchKernelGGL((paged_attn_row_kernel<T, true>), grid, dim3(256), 0, st, a, Score<true>(a.sm_scale, a.softcap));
  else
    hipLaunchKernelGGL((paged_attn_row_kernel<T, false>), grid, dim3(256), 0, st, a, Score<false>(a.sm_scale, 0.f));
  return launch_status("fm_paged_attn_fwd(rows)");
}

#define FM_INST(T)                                                       \
  template int terms_fwd_rows<T>(const FwdArgs&, hipStream_t);           \
  template int terms_delta<T>(const BwdArgs&, float2*, hipStream_t);      \
  template int terms_bwd_rows<T>(const BwdArgs&, const float2*, hipStream_t); \
  template int paged_attn_rows<T>(const PagedArgs&, hipStream_t);
FM_INST(float)
FM_INST(bf16_t)
FM_INST(f16_t)
#undef FM_INST

}  // namespace fm
