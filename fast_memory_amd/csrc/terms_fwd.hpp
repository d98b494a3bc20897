// Local attention with score terms, forward, bf16 / fp16 at head dimensions 64, 128 and 256: the launch of the tiled
// sweep (terms_tile.hpp).  One instance a file and head dimension (terms_fwd_64.hip, ..).
//
// A workgroup takes 128 consecutive queries of one query head.  The launch hands out the last block of every head first
// (under a causal mask it sees the most keys), so that what starts last is short and the launch ends evenly; the heads
// go KV head first, so that the G query heads of a KV head run on one XCD (workgroups go to the 8 XCDs in turn) and
// share its K and V in that XCD's L2.
//
// Measured, 64 heads x 4096 causal, bf16, d = 128: no terms 0.31 ms = 890 TFLOP/s, distance bias 0.33, cap 0.38, both 0.40, five
// packed documents 0.11; a matrix product of 8192 reaches 1155 here.  Bound: the VALU beside the matrix pipes (a 32 x 32 block is
// 16 MFMAs of 32 cycles and about 100 vector instructions of 4, the cap 112 more; counters with a bias and a prefix: VALU busy 64 % of the
// time, matrix pipes 36 %, LDS 18 %).  Tiles of 32 keys instead of 64: 0.30 ms
// without terms, but 0.070 against 0.063 at 32 heads x 2048 with a bias, where the barrier a tile shows.
//
// Where the blocks are too few for the card (sweep_pieces, terms_api.hip) the tiles that a block sees are cut into pieces, each of
// which leaves (m, l, O) in fp32, and a second launch joins them in order.
#pragma once
#include <type_traits>

#include "terms_masks.hpp"
#include "terms_tile.hpp"

namespace fm {

template <int D>
constexpr size_t tile_lds_bytes() {
  return 256 + 4 * size_t(TileLds<D, fwd_tile_keys<D>()>::kBytes) + 512;  // flag, two tiles, their documents
}

struct FwdTileArgs {
  const bf16_t *q, *k, *v;
  bf16_t* out;
  float* lse;
  Terms t;
  Masks m;
  int use_masks, H, G, S, L;
  float sm_scale;
  TileScore score;
  int pieces;
  float* part_o;     // [H G S][pieces][D], where pieces > 1
  float2* part_ml;   // [H G S][pieces] {m, l}, m in base 2
};

template <bool F16, int D, int MODE, bool DOCS>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void terms_fwd_kernel(FwdTileArgs a) {
  using M = Mma<F16>;
  extern __shared__ __attribute__((aligned(256))) bf16_t lds_all[];
  int* flag = reinterpret_cast<int*>(lds_all);
  lds_char_t* lds = (lds_char_t*)(lds_all + 128);
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5;
  if (tid == 0) *flag = 0;
  __syncthreads();
  const int heads = a.H * a.G, bx = int(blockIdx.x) % heads;
  const int hk = bx % a.H, hq = hk * a.G + bx / a.H;
  const int rest = int(blockIdx.x) / heads, piece = rest % a.pieces, qb = (a.S + kTQ - 1) / kTQ - 1 - rest / a.pieces;
  const int i0 = qb * kTQ, wq0 = i0 + 32 * w, iq = wq0 + col;
  const bool q_ok = iq < a.S;
  TileQuery qy;
  qy.pos = iq + (a.L - a.S);
  qy.slope2 = (MODE & kModeBias) ? a.t.slopes[hq] * kLog2e : 0.f;
  TileDocs docs{nullptr, nullptr, make_int2(0, 0), make_int2(0, 0)};
  int lim_lo, lim_hi, wg_lo, wg_hi;
  if (a.use_masks) {
    const int2 qi = a.m.qinfo[iq];
    qy.lim = qi.x, qy.doc = qi.y;
    const int4 q0 = a.m.qmeta[i0 / 32], q1 = a.m.qmeta[i0 / 32 + 1], q2 = a.m.qmeta[i0 / 32 + 2], q3 = a.m.qmeta[i0 / 32 + 3];
    const int4 mine = a.m.qmeta[wq0 / 32];
    lim_lo = mine.x, lim_hi = mine.y;
    wg_lo = min(min(q0.x, q1.x), min(q2.x, q3.x));
    wg_hi = max(max(q0.y, q1.y), max(q2.y, q3.y));
    if constexpr (DOCS) {
      docs.dock = a.m.dock;
      docs.kmeta = a.m.kmeta;
      docs.q_doc = make_int2(mine.z, mine.w);
      docs.wg_doc = make_int2(min(min(q0.z, q1.z), min(q2.z, q3.z)), max(max(q0.w, q1.w), max(q2.w, q3.w)));
    }
  } else {
    auto lim = [&](int i) { return seen_limit(i + (a.L - a.S), a.L, a.t.causal, 0); };
    qy.lim = lim(iq);
    qy.doc = 0;
    lim_lo = wq0 < a.S ? lim(wq0) : a.L;
    lim_hi = wq0 < a.S ? lim(min(wq0 + 31, a.S - 1)) : 0;
    wg_lo = lim(i0);
    wg_hi = lim(min(i0 + kTQ, a.S) - 1);
  }
  lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);
  lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);

  const int64_t row = int64_t(hq) * a.S + iq;
  uint4 qf[D / 16];
  {
    const uint4* pq = reinterpret_cast<const uint4*>(a.q + (q_ok ? row : 0) * D + hb * 8);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = q_ok ? pq[2 * ks] : make_uint4(0, 0, 0, 0);
  }
  // (the wait for these loads goes here: the compiler, which does not see the tiles' loads, would wait for all of
  // them in front of the first product otherwise)
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) asm volatile("" : "+v"(qf[ks].x), "+v"(qf[ks].y), "+v"(qf[ks].z), "+v"(qf[ks].w));

  constexpr int KT = fwd_tile_keys<D>();
  const FlatSource<D, KT> src{a.k + int64_t(hk) * a.L * D, a.v + int64_t(hk) * a.L * D, a.L};
  typename M::f16v O[D / 32];
  TileState st;
  int t0 = 0, t1 = (wg_hi + KT - 1) / KT;
  const bool again = tile_sweep<F16, D, MODE, DOCS>(src, qf, qy, lim_lo, lim_hi, wg_lo, t0, t1, piece, a.pieces, docs, a.score, lds,
                                                    flag, O, st);
  if (!again) {
    if (a.pieces > 1) {
      if (q_ok) tile_write_part<D>(O, st, a.part_o + (row * a.pieces + piece) * D, a.part_ml + row * a.pieces + piece);
      return;
    }
    tile_write<F16, D>(O, st, q_ok ? a.out + row * D : nullptr, a.lse + row);
    return;
  }
  // values that are not finite, in tiles with masked places: these rows one at a time
  typedef typename std::conditional<F16, f16_t, bf16_t>::type E;
  const int64_t head = int64_t(hk) * a.L * D;
  const KeyRows<E> K{(const E*)a.k + head, nullptr, 0, 0, 0, D}, V{(const E*)a.v + head, nullptr, 0, 0, 0, D};
  const Score<(MODE & kModeCap) != 0> score(a.sm_scale, a.t.softcap);
  for (int i = wq0; i < min(wq0 + 32, a.S); ++i) {
    const int64_t r = int64_t(hq) * a.S + i;
    const RowState rs = row_forward<E, (MODE & kModeCap) != 0>((const E*)a.q + r * D, K, V, query_view(a.t, i, a.S, a.L, hq),
                                                               a.t.doc_k, t0 * KT, t1 * KT, score);
    if (a.pieces > 1) {
      const int64_t at = r * a.pieces + piece;
#pragma unroll
      for (int u = 0; u < D / 64; ++u) a.part_o[at * D + l + 64 * u] = rs.acc[u];
      if (l == 0) a.part_ml[at] = make_float2(rs.m, rs.l);
      continue;
    }
    row_write(rs, D, (E*)a.out + r * D, a.lse + r);
  }
}

// the pieces of a query, in order: 16 lanes a query, D / 16 dimensions each
template <bool F16, int D>
__global__ __launch_bounds__(256) void terms_fwd_join_kernel(FwdTileArgs a) {
  const int64_t row = int64_t(blockIdx.x) * 16 + (threadIdx.x >> 4);
  if (row >= int64_t(a.H) * a.G * a.S) return;
  tile_join<F16, D>(a.part_o + row * a.pieces * D, a.part_ml + row * a.pieces, a.pieces, a.out + row * D, a.lse + row);
}

template <bool F16, int D, int MODE, bool DOCS>
static int launch_terms_fwd_docs(const FwdTileArgs& a, hipStream_t st) {
  FM_ALLOW_LDS((terms_fwd_kernel<F16, D, MODE, DOCS>), tile_lds_bytes<D>(), "fm_local_attn_terms_fwd(lds)");
  hipLaunchKernelGGL((terms_fwd_kernel<F16, D, MODE, DOCS>), dim3(unsigned(a.H * a.G * ceil_div(a.S, kTQ) * a.pieces)), dim3(256),
                     tile_lds_bytes<D>(), st, a);
  return launch_status("fm_local_attn_terms_fwd(tiles)");
}
template <bool F16, int D, int MODE>
static int launch_terms_fwd(const FwdTileArgs& a, hipStream_t st) {
  return a.t.doc_q ? launch_terms_fwd_docs<F16, D, MODE, true>(a, st) : launch_terms_fwd_docs<F16, D, MODE, false>(a, st);
}

template <bool F16, int D>
static int launch_terms_fwd_mode(const FwdTileArgs& a, hipStream_t st) {
  switch ((a.t.softcap > 0.f ? kModeCap : 0) | (a.t.slopes ? kModeBias : 0)) {
    case 0: return launch_terms_fwd<F16, D, 0>(a, st);
    case kModeCap: return launch_terms_fwd<F16, D, kModeCap>(a, st);
    case kModeBias: return launch_terms_fwd<F16, D, kModeBias>(a, st);
    default: return launch_terms_fwd<F16, D, kModeCap | kModeBias>(a, st);
  }
}

template <bool F16, int D>
static int launch_terms_fwd_pieces(const FwdTileArgs& a, hipStream_t st) {
  const int rc = launch_terms_fwd_mode<F16, D>(a, st);
  if (rc || a.pieces == 1) return rc;
  hipLaunchKernelGGL((terms_fwd_join_kernel<F16, D>), dim3(unsigned(ceil_div(int64_t(a.H) * a.G * a.S, 16))), dim3(256), 0, st, a);
  return launch_status("fm_local_attn_terms_fwd(join)");
}

template <int D>
int terms_fwd_tiles(const FwdTileArgs& a, bool f16, hipStream_t st) {
  return f16 ? launch_terms_fwd_pieces<true, D>(a, st) : launch_terms_fwd_pieces<false, D>(a, st);
}

}  // namespace fm
