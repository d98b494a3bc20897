// C entry points of the local attention with score terms and of the attention over a paged cache.
#include <math.h>

#include <algorithm>
#include <initializer_list>

#include "paged_attn.hpp"
#include "terms_bwd.hpp"
#include "paged_f32.hpp"
#include "terms_f32.hpp"
#include "terms_fwd.hpp"

namespace fm {

extern std::atomic<int> g_force_generic;
extern template int terms_fwd_tiles<64>(const FwdTileArgs&, bool, hipStream_t);
extern template int terms_fwd_tiles<128>(const FwdTileArgs&, bool, hipStream_t);
extern template int terms_fwd_tiles<256>(const FwdTileArgs&, bool, hipStream_t);

extern template int terms_bwd_tiles<64>(const BwdTileArgs&, bool, const void*, const float*, const float*, float2*, float*, hipStream_t);
extern template int terms_bwd_tiles<128>(const BwdTileArgs&, bool, const void*, const float*, const float*, float2*, float*, hipStream_t);
extern template int terms_bwd_tiles<256>(const BwdTileArgs&, bool, const void*, const float*, const float*, float2*, float*, hipStream_t);

extern template int paged_tiles<64>(const PagedTileArgs&, const PagedPlan&, int, hipStream_t);
extern template int paged_tiles<128>(const PagedTileArgs&, const PagedPlan&, int, hipStream_t);
extern template int paged_tiles<256>(const PagedTileArgs&, const PagedPlan&, int, hipStream_t);

#define FM_EXTERN(T)                                                                            \
  extern template int terms_f32_fwd<T>(const F32Args&, hipStream_t);                             \
  extern template int terms_f32_bwd<T>(const F32Args&, const BwdArgs&, float2*, hipStream_t);    \
  extern template int paged_f32<T>(const PagedTileArgs&, const PagedPlan&, hipStream_t);
FM_EXTERN(float)
FM_EXTERN(bf16_t)
FM_EXTERN(f16_t)
#undef FM_EXTERN

static bool tiles_take(int d, int dtype) {
  return g_force_generic != 1 && dtype != FM_F32 && (d == 64 || d == 128 || d == 256);
}

// Into how many pieces the keys of a block of 128 queries are cut: until there are 512 workgroups, two a compute unit, none of
// less than 8 tiles of 64 keys.  Measured, whole and in pieces, bf16: 2 heads x 4096, d = 256: forward 220 and 64 us, backward
// 606 and 280; 8 heads x 128 over 4096 keys, d = 128: 122 and 28, 193 and 48; 16 x 2048: 66 and 52, 150 and 131; 32 x 1024
// (256 blocks): 37 and 37, 93 and 88.  At most 64 pieces: one token over 2^20 keys, d = 128, forward 344 us (16 pieces: 1271).
static int sweep_pieces(int H, int G, int S, int L) {
  const int64_t blocks = int64_t(H) * G * ceil_div(S, kTQ);
  return int(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(512 / blocks, ceil_div(L, 512)), 64)));
}

// Into how many pieces the sweep of a block is cut in the fp32 products' kernels, whose workgroups take 32 queries (or keys) and a tile
// of 32 on the other side a wave: until there is a workgroup for every compute unit, three for every two between d = 128 and 256 (where two
// fit one), none of less than four tiles, one a wave.  At d = 256 two for every one where a piece keeps 16 tiles.  Measured in fp32, causal,
// forward and backward, whole, in pieces for 256 workgroups and for 512: one head x 512, d = 64: 65, 44 and 43 us; 8 query heads on one KV
// head x 1024, d = 64: 500, 124, 134; d = 128: 898, 209, 220; 8 heads x 512, d = 128: 105, 98, 132; d = 256: 205, 142, 203; 4 heads on one
// x 2248 without a mask, d = 256: 2174, 1251, 1103.
static int f32_cut(int64_t blocks, int64_t tiles, int d) {
  const int64_t few = std::min(ceil_div(d > 128 && d < 256 ? 384 : 256, blocks), tiles / 4);
  const int64_t many = d == 256 ? std::min(ceil_div(512, blocks), tiles / 16) : 1;
  return int(std::max<int64_t>(1, std::min<int64_t>(std::max(few, many), 64)));
}
static int f32_pieces(int H, int G, int S, int L, int d) { return f32_cut(int64_t(H) * G * ceil_div(S, 32), ceil_div(L, 32), d); }
static int f32_splits(int H, int G, int S, int L, int d) { return f32_cut(int64_t(H) * ceil_div(L, 32), int64_t(G) * ceil_div(S, 32), d); }

// The workspace of a forward: masks | partial sums.  `tiles`: of the 16-bit products' kernels.
struct FwdLayout {
  int pieces;
  size_t part_o, part_ml, total;
};
static FwdLayout fwd_layout(int H, int G, int S, int L, int d, bool tiles) {
  FwdLayout y;
  y.pieces = tiles ? sweep_pieces(H, G, S, L) : f32_pieces(H, G, S, L, d);
  const size_t units = y.pieces > 1 ? size_t(H) * G * S * y.pieces : 0;
  y.part_o = masks_layout(nullptr, S, L).bytes;
  y.part_ml = y.part_o + align_up(units * d * 4, 256);
  y.total = y.part_ml + align_up(units * 8, 256);
  return y;
}

static int terms_fwd_run(const FwdArgs& a, void* ws, hipStream_t st) {
  const FwdLayout y = fwd_layout(a.H, a.G, a.S, a.L, a.d, true);
  char* p = static_cast<char*>(ws);
  FwdTileArgs t{(const bf16_t*)a.q, (const bf16_t*)a.k, (const bf16_t*)a.v, (bf16_t*)a.out, a.lse, a.t, masks_layout(ws, a.S, a.L),
                a.t.doc_q || a.t.prefix, a.H, a.G, a.S, a.L, a.sm_scale, tile_score(a.sm_scale, a.t.softcap), y.pieces, reinterpret_cast<float*>(p + y.part_o),
                reinterpret_cast<float2*>(p + y.part_ml)};
  if (t.use_masks) {
    const int rc = make_masks(t.m, a.t, a.S, a.L, st);
    if (rc) return rc;
  }
  const bool f16 = a.dtype == FM_F16;
  return a.d == 64 ? terms_fwd_tiles<64>(t, f16, st) : a.d == 128 ? terms_fwd_tiles<128>(t, f16, st) : terms_fwd_tiles<256>(t, f16, st);
}

static bool cap_ok(float sm_scale, float softcap) {
  return softcap == 0.f || (softcap > 0.f && isfinite(softcap * kLog2e) && isfinite(sm_scale / softcap));
}

static int terms_check(const char* name, const FwdArgs& a) {
  FM_REQUIRE(a.H >= 1 && a.G >= 1 && a.S >= 1 && a.L >= 1 && a.d >= 1 && a.d <= FM_MAX_D, FM_ERR_ARG,
             "%s: H=%d G=%d S=%d L=%d d=%d", name, a.H, a.G, a.S, a.L, a.d);
  FM_REQUIRE(dtype_ok(a.dtype), FM_ERR_ARG, "%s: dtype=%d", name, a.dtype);
  FM_REQUIRE(a.sm_scale > 0.f && isfinite(a.sm_scale), FM_ERR_ARG, "%s: sm_scale=%g", name, double(a.sm_scale));
  FM_REQUIRE(cap_ok(a.sm_scale, a.t.softcap), FM_ERR_ARG, "%s: softcap=%g", name, double(a.t.softcap));
  FM_REQUIRE((a.t.doc_q == nullptr) == (a.t.doc_k == nullptr), FM_ERR_ARG, "%s: doc_q and doc_k come together", name);
  FM_REQUIRE(a.q && a.k && a.v && a.out && a.lse, FM_ERR_ARG, "%s: null pointer", name);
  FM_REQUIRE(int64_t(a.H) * a.G <= 65535 && int64_t(a.H) * a.G * a.S <= 0x7fffffffLL && int64_t(a.H) * a.L <= 0x7fffffffLL &&
                 a.S <= (1 << 24) && a.L <= (1 << 24),
             FM_ERR_UNSUPPORTED, "%s: H*G=%lld S=%d L=%d", name, (long long)a.H * a.G, a.S, a.L);
  return FM_OK;
}

static int terms_fwd_f32(const FwdArgs& f, char* ws, hipStream_t st) {
  const FwdLayout y = fwd_layout(f.H, f.G, f.S, f.L, f.d, false);
  F32Args a{};
  a.f = f;
  a.m = masks_layout(ws, f.S, f.L);
  a.use_masks = f.t.doc_q || f.t.prefix;
  a.score = f32_score(f.sm_scale, f.t.softcap);
  a.pieces = y.pieces;
  a.part_o = reinterpret_cast<float*>(ws + y.part_o);
  a.part_ml = reinterpret_cast<float2*>(ws + y.part_ml);
  if (a.use_masks) {
    const int rc = make_masks(a.m, f.t, f.S, f.L, st);
    if (rc) return rc;
  }
  return f.dtype == FM_F32 ? terms_f32_fwd<float>(a, st) : f.dtype == FM_BF16 ? terms_f32_fwd<bf16_t>(a, st) : terms_f32_fwd<f16_t>(a, st);
}

// (the tiled kernels read rows of q, k, v in 16-byte pieces, 8 bytes at a time written)
static bool aligned16(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

static size_t row_data_bytes(int H, int G, int S) { return align_up(size_t(H) * G * S * 8, 256); }

// The workspace of a backward: {lse log2 e, D} | masks | norms | partial sums.
struct BwdLayout {
  size_t masks, norms, part, part_dq, total;
  int n_q_norms, n_k_norms, splits, dq_pieces;
};

// Into how many pieces the sweeps over the queries are cut: two workgroups a compute unit at least (512 in all), and four
// where a piece still has 64 tiles of queries (under a causal mask the first keys' sweeps are twice the average, and more
// pieces end more evenly); none of less than 4 tiles, 64 at most (2^18 queries over 64 keys, d = 128, forward and backward: 304 us, with
// 16 at most 882).  Measured, 512 against 1024 workgroups: 32 heads x 2048 tokens,
// d = 128: 0.153 and 0.198 ms (the pieces' partial sums are written and read); 64 x 4096, five documents: 0.59 and 0.48.
static int dkv_splits(int H, int G, int S, int L) {
  const int64_t blocks = int64_t(H) * ceil_div(L, kDkvKeys), steps = int64_t(G) * ceil_div(S, kDkvQ);
  const int64_t want = std::max(ceil_div(512, blocks), std::min(ceil_div(1024, blocks), steps / 64));
  return int(std::max<int64_t>(1, std::min<int64_t>(std::min(want, steps / 4), 64)));
}

static BwdLayout bwd_layout(int H, int G, int S, int L, int d, bool tiles) {
  BwdLayout b;
  b.masks = row_data_bytes(H, G, S);
  b.norms = b.masks + masks_layout(nullptr, S, L).bytes;
  b.n_q_norms = int(ceil_div(int64_t(H) * G * S, kNormRows));
  b.n_k_norms = int(ceil_div(int64_t(H) * L, kNormRows));
  b.part = b.norms + align_up(size_t(2 * b.n_q_norms + b.n_k_norms) * 4, 256);
  b.splits = tiles ? dkv_splits(H, G, S, L) : f32_splits(H, G, S, L, d);
  b.dq_pieces = tiles ? sweep_pieces(H, G, S, L) : f32_pieces(H, G, S, L, d);
  b.part_dq = b.part + (b.splits > 1 ? size_t(b.splits) * 2 * H * L * d * 4 : 0);
  b.total = b.part_dq + (b.dq_pieces > 1 ? size_t(b.dq_pieces) * H * G * S * d * 4 : 0);
  return b;
}

static int terms_bwd_f32(const BwdArgs& b, char* ws, hipStream_t st) {
  const FwdArgs& f = b.f;
  const BwdLayout y = bwd_layout(f.H, f.G, f.S, f.L, f.d, false);
  float2* rd = reinterpret_cast<float2*>(ws);
  F32Args a{};
  a.f = f;
  a.dout = b.dout, a.rd = rd;
  a.dq = b.dq, a.dk = b.dk, a.dv = b.dv;
  a.m = masks_layout(ws + y.masks, f.S, f.L);
  a.use_masks = f.t.doc_q || f.t.prefix;
  a.score = f32_score(f.sm_scale, f.t.softcap);
  a.pieces = y.dq_pieces, a.splits = y.splits;
  a.part_kv = reinterpret_cast<float*>(ws + y.part);
  a.part_dq = reinterpret_cast<float*>(ws + y.part_dq);
  if (a.use_masks) {
    const int rc = make_masks(a.m, f.t, f.S, f.L, st);
    if (rc) return rc;
  }
  return f.dtype == FM_F32    ? terms_f32_bwd<float>(a, b, rd, st)
         : f.dtype == FM_BF16 ? terms_f32_bwd<bf16_t>(a, b, rd, st)
                              : terms_f32_bwd<f16_t>(a, b, rd, st);
}

static int terms_bwd_run(const BwdArgs& b, void* ws, hipStream_t st) {
  const FwdArgs& a = b.f;
  const BwdLayout y = bwd_layout(a.H, a.G, a.S, a.L, a.d, true);
  char* p = static_cast<char*>(ws);
  float2* rd = reinterpret_cast<float2*>(p);
  float* norms = reinterpret_cast<float*>(p + y.norms);
  BwdTileArgs t{(const bf16_t*)a.q, (const bf16_t*)a.k, (const bf16_t*)a.v, (const bf16_t*)b.dout, rd, norms, y.n_q_norms,
                y.n_k_norms, (bf16_t*)b.dq, (bf16_t*)b.dk, (bf16_t*)b.dv, reinterpret_cast<float*>(p + y.part), a.t,
                masks_layout(p + y.masks, a.S, a.L), a.t.doc_q || a.t.prefix, a.H, a.G, a.S, a.L, y.splits, a.sm_scale,
                tile_score(a.sm_scale, a.t.softcap), y.dq_pieces, reinterpret_cast<float*>(p + y.part_dq)};
  if (t.use_masks) {
    const int rc = make_masks(t.m, a.t, a.S, a.L, st);
    if (rc) return rc;
  }
  const bool f16 = a.dtype == FM_F16;
  return a.d == 64    ? terms_bwd_tiles<64>(t, f16, a.out, a.lse, b.dlse, rd, norms, st)
         : a.d == 128 ? terms_bwd_tiles<128>(t, f16, a.out, a.lse, b.dlse, rd, norms, st)
                      : terms_bwd_tiles<256>(t, f16, a.out, a.lse, b.dlse, rd, norms, st);
}

}  // namespace fm

extern "C" size_t fm_local_attn_terms_fwd_workspace(int H, int G, int S, int L, int d, int dtype) {
  if (H < 1 || G < 1 || S < 1 || L < 1 || d < 1) return 0;
  // (rows that are not on 16 bytes go the fp32 products' way)
  const size_t tiles = fm::tiles_take(d, dtype) ? fm::fwd_layout(H, G, S, L, d, true).total : 0;
  return std::max(tiles, fm::fwd_layout(H, G, S, L, d, false).total);
}

extern "C" int fm_local_attn_terms_fwd(const void* q, const void* k, const void* v, void* out, float* lse, float softcap,
                                       const float* slopes, const int32_t* doc_q, const int32_t* doc_k,
                                       const int32_t* prefix, int H, int G, int S, int L, int d, float sm_scale, int causal,
                                       int dtype, void* ws, size_t ws_bytes, void* stream) {
  using namespace fm;
  const FwdArgs a{q, k, v, out, lse, {slopes, doc_q, doc_k, prefix, softcap, causal != 0}, H, G, S, L, d, dtype, sm_scale};
  int rc = terms_check("fm_local_attn_terms_fwd", a);
  if (rc) return rc;
  const size_t need = fm_local_attn_terms_fwd_workspace(H, G, S, L, d, dtype);
  FM_REQUIRE(ws, FM_ERR_ARG, "fm_local_attn_terms_fwd: null pointer");
  FM_REQUIRE(ws_bytes >= need, FM_ERR_WORKSPACE, "fm_local_attn_terms_fwd: workspace %zu < %zu", ws_bytes, need);
  if (tiles_take(d, dtype) && aligned16({q, k, v, out, ws})) return terms_fwd_run(a, ws, as_stream(stream));
  return terms_fwd_f32(a, static_cast<char*>(ws), as_stream(stream));
}

extern "C" size_t fm_local_attn_terms_bwd_workspace(int H, int G, int S, int L, int d, int dtype) {
  if (H < 1 || G < 1 || S < 1 || L < 1 || d < 1) return 0;
  const size_t tiles = fm::tiles_take(d, dtype) ? fm::bwd_layout(H, G, S, L, d, true).total : 0;
  return std::max(tiles, fm::bwd_layout(H, G, S, L, d, false).total);
}

extern "C" int fm_local_attn_terms_bwd(const void* q, const void* k, const void* v, const void* out, const float* lse,
                                       const void* dout, const float* dlse, void* dq, void* dk, void* dv, float softcap,
                                       const float* slopes, const int32_t* doc_q, const int32_t* doc_k,
                                       const int32_t* prefix, int H, int G, int S, int L, int d, float sm_scale, int causal,
                                       int dtype, void* ws, size_t ws_bytes, void* stream) {
  using namespace fm;
  const BwdArgs a{{q, k, v, const_cast<void*>(out), const_cast<float*>(lse), {slopes, doc_q, doc_k, prefix, softcap, causal != 0},
                   H, G, S, L, d, dtype, sm_scale},
                  dout, dlse, dq, dk, dv};
  int rc = terms_check("fm_local_attn_terms_bwd", a.f);
  if (rc) return rc;
  FM_REQUIRE(dout && dq && dk && dv && ws, FM_ERR_ARG, "fm_local_attn_terms_bwd: null pointer");
  const size_t need = fm_local_attn_terms_bwd_workspace(H, G, S, L, d, dtype);
  FM_REQUIRE(ws_bytes >= need, FM_ERR_WORKSPACE, "fm_local_attn_terms_bwd: workspace %zu < %zu", ws_bytes, need);
  if (tiles_take(d, dtype) && aligned16({q, k, v, out, dout, dq, dk, dv, ws})) return terms_bwd_run(a, ws, as_stream(stream));
  return terms_bwd_f32(a, static_cast<char*>(ws), as_stream(stream));
}

extern "C" size_t fm_paged_attn_fwd_workspace(int rows, int T, int max_new, int H, int G, int d, int width, int page, int dtype) {
  if (rows < 1 || T < 1 || H < 1 || G < 1 || d < 1 || width < 1 || page < 1) return 0;
  const int64_t keys = int64_t(width) * page;
  const size_t tiles = fm::tiles_take(d, dtype) ? fm::paged_plan(rows, T, max_new, H, G, d, keys).total : 0;
  return std::max<size_t>(256, std::max(tiles, fm::paged_f32_plan(rows, T, H, G, d, keys).total));
}

extern "C" int fm_paged_attn_fwd(const void* q, int64_t q_token, int64_t q_head, const void* k_pages, const void* v_pages,
                                 const int32_t* book, int n_pages, int rows, int width, int page, const int32_t* cu, void* out,
                                 int64_t out_token, int64_t out_head, float* lse, int64_t lse_token, int64_t lse_head, int T,
                                 int max_new, int H, int G, int d, float sm_scale, float softcap, const float* slopes,
                                 const int32_t* prefix, int dtype, void* ws, size_t ws_bytes, void* stream) {
  using namespace fm;
  FM_REQUIRE(n_pages >= 1 && rows >= 1 && width >= 1 && H >= 1 && G >= 1 && d >= 1 && d <= FM_MAX_D && T >= 0 && max_new >= 0,
             FM_ERR_ARG, "fm_paged_attn_fwd: n_pages=%d rows=%d width=%d H=%d G=%d d=%d T=%d max_new=%d", n_pages, rows, width, H,
             G, d, T, max_new);
  FM_REQUIRE(page <= FM_CACHE_MAX_PAGE && log2_exact(page) >= 0, FM_ERR_ARG,
             "fm_paged_attn_fwd: page size %d is no power of two up to %d", page, FM_CACHE_MAX_PAGE);
  FM_REQUIRE(dtype_ok(dtype), FM_ERR_ARG, "fm_paged_attn_fwd: dtype=%d", dtype);
  FM_REQUIRE(sm_scale > 0.f && isfinite(sm_scale) && cap_ok(sm_scale, softcap), FM_ERR_ARG,
             "fm_paged_attn_fwd: sm_scale=%g softcap=%g", double(sm_scale), double(softcap));
  FM_REQUIRE(int64_t(H) * G <= 65535 && int64_t(T) * H * G <= 0x7fffffffLL && rows <= (1 << 24) &&
                 (int64_t(width) * page) <= (1 << 24),
             FM_ERR_UNSUPPORTED, "fm_paged_attn_fwd: T=%d H*G=%lld rows=%d width*page=%lld", T, (long long)H * G, rows,
             (long long)width * page);
  if (T == 0) return FM_OK;
  FM_REQUIRE(q && k_pages && v_pages && book && cu && out && lse && ws, FM_ERR_ARG, "fm_paged_attn_fwd: null pointer");
  const size_t need = fm_paged_attn_fwd_workspace(rows, T, max_new, H, G, d, width, page, dtype);
  FM_REQUIRE(ws_bytes >= need, FM_ERR_WORKSPACE, "fm_paged_attn_fwd: workspace %zu < %zu", ws_bytes, need);
  const PagedArgs a{q, q_token, q_head, k_pages, v_pages, book, n_pages, rows, width, page, log2_exact(page), cu, out, out_token,
                    out_head, lse, lse_token, lse_head, T, H, G, d, sm_scale, softcap, slopes, prefix, dtype};
  const int64_t e = dtype_bytes(dtype), keys = int64_t(width) * page;
  const bool tiles = tiles_take(d, dtype) && page >= 16 && aligned16({q, k_pages, v_pages, out, ws}) && q_token * e % 16 == 0 &&
                     q_head * e % 16 == 0 && out_token * e % 8 == 0 && out_head * e % 8 == 0;
  const PagedPlan y = tiles ? paged_plan(rows, T, max_new, H, G, d, keys) : paged_f32_plan(rows, T, H, G, d, keys);
  const int64_t groups = int64_t(H) * std::max(int64_t(std::min(rows, T)) * y.few_pieces, int64_t(y.slots) * y.many_pieces) + 1024;
  FM_REQUIRE(groups <= 0x7fffffffLL, FM_ERR_UNSUPPORTED, "fm_paged_attn_fwd: %lld workgroups", (long long)groups);
  char* w = static_cast<char*>(ws);
  const PagedTileArgs t{a, tile_score(sm_scale, softcap), y.few_rows, y.few_pieces, y.many_pieces, reinterpret_cast<float*>(w),
                        reinterpret_cast<float2*>(w + y.part_ml), y.many_base, y.slots};
  hipStream_t st = as_stream(stream);
  if (!tiles) return dtype == FM_F32 ? paged_f32<float>(t, y, st) : dtype == FM_BF16 ? paged_f32<bf16_t>(t, y, st) : paged_f32<f16_t>(t, y, st);
  return d == 64 ? paged_tiles<64>(t, y, max_new, st) : d == 128 ? paged_tiles<128>(t, y, max_new, st) : paged_tiles<256>(t, y, max_new, st);
}
