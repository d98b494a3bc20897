// The masks of a call, one pass over its queries and keys (terms_masks.hpp).  A few hundred kilobytes at most: latency.
#include "terms_masks.hpp"

namespace fm {

__device__ __forceinline__ int wave_min_i(int v, int width) {
  for (int o = width / 2; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ int wave_max_i(int v, int width) {
  for (int o = width / 2; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
  return v;
}

__global__ __launch_bounds__(256) void terms_masks_kernel(Masks m, Terms t, int S, int L, int q_blocks) {
  if (int(blockIdx.x) < q_blocks) {
    const int i = int(blockIdx.x) * 256 + threadIdx.x;
    if (i >= (S + 127) / 128 * 128) return;
    const bool is = i < S;
    int lim = 0, doc = -1;
    if (is) {
      lim = seen_limit(i + (L - S), L, t.causal, t.prefix ? t.prefix[i] : 0);
      doc = t.doc_q ? t.doc_q[i] : 0;
      if (doc < 0) doc = -1, lim = 0;
    }
    m.qinfo[i] = make_int2(lim, doc);
    const int a = wave_min_i(is ? lim : 0x7fffffff, 32), b = wave_max_i(lim, 32);
    const int c = wave_min_i(is ? doc : 0x7fffffff, 32), e = wave_max_i(is ? doc : -1, 32);
    if ((threadIdx.x & 31) == 0) m.qmeta[i / 32] = make_int4(a, b, c, e);
    return;
  }
  const int j = (int(blockIdx.x) - q_blocks) * 256 + threadIdx.x;
  if (j >= (L + 127) / 128 * 128) return;
  int doc = -2;
  if (j < L) {
    doc = t.doc_k ? t.doc_k[j] : 0;
    if (doc < 0) doc = -2;
  }
  m.dock[j] = doc;
  const int a = wave_min_i(doc, 32), b = wave_max_i(doc, 32);
  if ((threadIdx.x & 31) == 0) m.kmeta[j / 32] = make_int2(a, b);
}

int make_masks(const Masks& m, const Terms& t, int S, int L, hipStream_t st) {
  const int S8 = (S + 127) / 128 * 128, L8 = (L + 127) / 128 * 128;
  const int q_blocks = (S8 + 255) / 256;
  hipLaunchKernelGGL(terms_masks_kernel, dim3(unsigned(q_blocks + (L8 + 255) / 256)), dim3(256), 0, st, m, t, S, L, q_blocks);
  return launch_status("fm_local_attn_terms(masks)");
}

}  // namespace fm
