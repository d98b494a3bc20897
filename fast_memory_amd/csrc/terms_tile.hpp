// The tiled forward of the attention with score terms (bf16 / fp16, head dimension 64, 128 or 256): 128 query rows per
// workgroup, 32 per wave, over tiles of keys.  The training forward (terms_fwd.hpp) and the chunks over a paged cache
// (paged_attn.hpp) run it; they differ in where a key's row lies and in what a query row is.
//
//   S^T = K.Q^T   v_mfma_f32_32x32x16: A = 32 keys of the tile from LDS, B = this wave's queries, in registers for the
//                 whole sweep.  Lane (query l % 32, half l / 32) ends up with the scores of keys 8 (r / 4) + 4 (l / 32) +
//                 r % 4: a query is a lane column, its softmax statistics are plain registers and one exchange between
//                 the halves per tile makes a maximum whole.
//   O^T += V^T.P^T  same instruction.  Registers 8 s .. 8 s + 7 of a score block are the B operand of step s with the 16
//                 keys of the step in the order 0-3, 8-11 | 4-7, 12-15, and ds_read_b64_tr_b16 reads V^T in just that
//                 order out of row-major V: nothing is shuffled or transposed in registers.
//
// K and V go from global memory straight into LDS (global_load_lds_dwordx4, two tiles: one read, one on its way), a
// 1 KiB block of whole rows per load.  16-byte chunk c of row r lies at position c ^ f(r): the lanes that read one chunk
// of 16 rows (K) and the 4 rows x 64 bytes that half a wave reads of V then hit every bank once.
//
// Masks cost only the tiles that have masked places: the others (keys that all queries of a wave see) run without a
// compare.  Where a tile does have masked places and its values hold a NaN or an infinity, the product 0 x NaN would
// reach queries that do not see the row: the workgroup notes it and, after the sweep, does its rows again a row at a
// time (terms.hpp), which visits only what is seen.
#pragma once
#include "attn_ring.hpp"
#include "mma16.hpp"
#include "terms_api.hpp"

namespace fm {

constexpr int kTQ = 128;  // query rows of a workgroup
// keys of a tile of the forward
template <int D>
constexpr int fwd_tile_keys() { return D == 256 ? 32 : 64; }

// The probabilities of the product with the values are held times 2^kPUp in fp16, and against a running maximum that is at most
// 2^kPLazy behind the true one: at most 2^15 of fp16's 65504, and a key that weighs 2^-37 of the largest is half the smallest number
// fp16 holds, so that what falls below is off by at most 2^-37 of it a key: 2^-13 in all for the 2^24 keys a row may have, under the
// rounding of the result.  (Unscaled, 65 535 keys 17.5 under one key without a value gave 0 where 1.6e-3 is right.)  bf16 has fp32's
// range.  The factor costs nothing: it sits in the maximum that the exponents are taken against, and in the sums as well.  (A
// maximum followed from 2^5 or 2^8 on instead of 2^3 is no faster.)
template <bool F16>
constexpr float kPUp = F16 ? 12.f : 0.f;
template <bool F16>
constexpr float kPLazy = F16 ? 3.f : 8.f;

// The log-sum-exp of sums against m.  (m + kPUp and the scaled l are exact; a logarithm of about 12 would cost bits of a small result.)
template <bool F16>
__device__ __forceinline__ float tile_lse(float m, float l) {
  return ((m + kPUp<F16>) + __builtin_amdgcn_logf(F16 ? l * 0x1p-12f : l)) * kLn2;
}

// what the scores have, beside the product: bit 0 the cap, bit 1 the distance bias
constexpr int kModeCap = 1, kModeBias = 2;

template <int D>
__device__ __forceinline__ constexpr int tile_swz(int r) {
  if constexpr (D == 64)
    return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);  // 8 chunks a row, two rows span the banks
  else
    return ((r & 3) << 2) | ((r >> 2) & 3);  // (head dimension 256: among 16 of the 32 chunks)
}

// 16-bit values that are infinite or NaN: any in the 8 of a register quad
template <bool F16>
__device__ __forceinline__ bool any_nonfinite(const uint4& x) {
  constexpr uint32_t e = F16 ? 0x7c007c00u : 0x7f807f80u, one = F16 ? 0x04000400u : 0x00800080u;
  const uint32_t a = ((x.x & e) + one) | ((x.y & e) + one) | ((x.z & e) + one) | ((x.w & e) + one);
  return (a & 0x80008000u) != 0;  // an exponent of all ones carries into the (masked) sign
}

// One direct load: lane i's 16 bytes from base + voff to LDS byte `lds_addr` + 16 i (both wave-uniform)
__device__ __forceinline__ void tile_load(uint32_t lds_addr, uint32_t voff, const void* base) { ring_load16(lds_addr, voff, base); }

__device__ __forceinline__ uint4 lds_read16(const lds_char_t* p) {
  const ring_u32x4 a = *reinterpret_cast<const __attribute__((address_space(3))) ring_u32x4*>(p);
  return make_uint4(a[0], a[1], a[2], a[3]);
}
__device__ __forceinline__ ring_short4 lds_read_tr(const lds_char_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ring_short4*)p);
}
__device__ __forceinline__ uint4 tr_pair(const lds_char_t* p, const lds_char_t* q) {
  union {
    ring_short4 s[2];
    uint4 u;
  } a;
  a.s[0] = lds_read_tr(p);
  a.s[1] = lds_read_tr(q);
  return a.u;
}

// Loads through the scalar cache, from a place that is the same in the whole wave and that nothing writes meanwhile.  A
// vector load in a tile's loop would be waited for with all direct loads in flight (they share a counter, in order).
typedef int tile_int2 __attribute__((ext_vector_type(2)));
typedef int tile_int4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ int2 scalar_load(const int2* p, int i) {
  const tile_int2 v = reinterpret_cast<const __attribute__((address_space(4))) tile_int2*>(reinterpret_cast<uintptr_t>(p))[__builtin_amdgcn_readfirstlane(i)];
  return make_int2(v[0], v[1]);
}
__device__ __forceinline__ int4 scalar_load(const int4* p, int i) {
  const tile_int4 v = reinterpret_cast<const __attribute__((address_space(4))) tile_int4*>(reinterpret_cast<uintptr_t>(p))[__builtin_amdgcn_readfirstlane(i)];
  return make_int4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ float scalar_load(const float* p, int i) {
  return reinterpret_cast<const __attribute__((address_space(4))) float*>(reinterpret_cast<uintptr_t>(p))[__builtin_amdgcn_readfirstlane(i)];
}
__device__ __forceinline__ int scalar_load(const int32_t* p, int i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int*>(reinterpret_cast<uintptr_t>(p))[__builtin_amdgcn_readfirstlane(i)];
}

// LDS of one tile of ROWS rows: where a wave's lanes load, and where the operands are read
template <int D, int ROWS>
struct TileLds {
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kBytes = ROWS * kRowBytes;
  static constexpr int kRowsPerLoad = 1024 / kRowBytes;         // whole rows in a load of 1 KiB
  static constexpr int kLoads = kBytes / 1024;                   // loads of a tile ..
  static constexpr int kLoadsPerWave = kLoads / 4;               // .. and of a wave's share: loads w, w + 4, ..
  // the row of load i this lane fills, and the byte offset in that row it asks global memory for
  __device__ static __forceinline__ int load_row(int i, int lane) { return i * kRowsPerLoad + lane / (D / 8); }
  __device__ static __forceinline__ uint32_t load_chunk(int row, int lane) {
    return uint32_t((lane % (D / 8)) ^ tile_swz<D>(row)) << 4;
  }
  // Operand addresses.  A chunk's position is c ^ f(r) and f looks at r % 16 only, so that the bytes of step ks (or of
  // dimensions 32 dt ..) are the lane's first address with some of its low bits flipped: one XOR each from a base that
  // is formed once -- and re-formed by `fresh` in every tile, or the compiler would keep all of them in registers.
  struct Bases {
    int rows, cols;
    __device__ __forceinline__ Bases(int lane) {
      const int row = lane & 31, hb = lane >> 5, i = lane & 15, r = 4 * hb + (i >> 2);
      rows = row * kRowBytes + ((hb ^ tile_swz<D>(row)) << 4);
      cols = r * kRowBytes + (((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ tile_swz<D>(r)) << 4) + (i & 1) * 8;
    }
    __device__ __forceinline__ Bases fresh(int offset) const {
      Bases b = *this;
      b.rows += offset;
      b.cols += offset;
      asm volatile("" : "+v"(b.rows), "+v"(b.cols));
      return b;
    }
  };
  // 32 rows from row0 (row = l % 32), contraction step ks: 8 elements from 16 ks + 8 (l / 32)
  __device__ static __forceinline__ uint4 rows32(const lds_char_t* tile, int base, int row0, int ks) {
    return lds_read16(tile + (base ^ (ks << 5)) + row0 * kRowBytes);
  }
  // transposed: dimensions 32 dt + l % 32, contraction over the 16 rows from row0 in the order 0-3, 8-11 | 4-7, 12-15
  // (f(r + 8) = f(r) ^ 2)
  __device__ static __forceinline__ uint4 cols32(const lds_char_t* tile, int base, int row0, int dt) {
    return tr_pair(tile + (base ^ (dt << 6)) + row0 * kRowBytes, tile + (base ^ (dt << 6) ^ 32) + (row0 + 8) * kRowBytes);
  }
};

// Score arithmetic of a launch (base 2, see Score in terms.hpp).  With w = raw^2 the small-argument cap is
// raw (c0 + w (c1 + w (..))): terms.hpp's polynomial in y = raw in, its coefficients times out in^(2 i + 1), which spares the
// product raw in (of about 12 instructions a score).  It serves |raw| <= zmax (|y| <= 1/2); zmax is -1, and every score goes the
// general way, where the last coefficient would leave fp32's normal range (sm_scale / softcap below 1e-3 or above 1e3 or so).
// 1 - tanh^2 = 1 - k2 x^2 from the capped score x.
struct TileScore {
  float in, out, c0, c1, c2, c3, c4, c5, zmax, k2;
};

inline TileScore tile_score(float sm_scale, float softcap) {
  TileScore t{};
  if (!(softcap > 0.f)) {
    t.in = sm_scale * kLog2e;
    t.out = 1.f;
    return t;
  }
  t.in = sm_scale / softcap;
  t.out = softcap * kLog2e;
  t.k2 = 1.f / t.out / t.out;
  const double in = double(t.in), w = in * in, c0 = double(t.out) * in;
  const double c5 = -0.00694700312 * c0 * w * w * w * w * w;
  t.c0 = float(c0);
  t.c1 = float(-0.333333328 * c0 * w);
  t.c2 = float(0.133332274 * c0 * w * w);
  t.c3 = float(-0.0539337893 * c0 * w * w * w);
  t.c4 = float(0.021472721 * c0 * w * w * w * w);
  t.c5 = float(c5);
  const bool fits = -c5 >= 1e-36 && -c5 <= 1e36 && c0 >= 1e-36 && c0 <= 1e36;
  t.zmax = fits ? kTanhSmall / t.in : -1.f;
  return t;
}

__device__ __forceinline__ float capped_small(const TileScore& k, float x) {
  const float w = x * x;
  float p = fmaf(w, k.c5, k.c4);
  p = fmaf(w, p, k.c3);
  p = fmaf(w, p, k.c2);
  p = fmaf(w, p, k.c1);
  return fmaf(w, p, k.c0);  // times x
}

typedef float tile_f16v __attribute__((__vector_size__(16 * sizeof(float))));
// What an MFMA of 8 passes wrote may be read by inline assembly (the maxima below) 11 slots after it at the earliest, and
// the compiler does not look into assembly: these spend the slots (see mma16.hpp) and take the registers through.
__device__ __forceinline__ void tile_settle(tile_f16v& a) { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(a)); }

// maximum of 16 registers in 8 instructions (attn_staged.hpp: the assembly spares the quieting of each operand)
__device__ __forceinline__ float max16(const float (&x)[16], float m) {
#pragma unroll
  for (int r = 0; r < 16; r += 2) m = st_max3(m, x[r], x[r + 1]);
  return m;
}
__device__ __forceinline__ float abs_max16(const float (&x)[16]) {
  float m = 0.f;
#pragma unroll
  for (int r = 0; r < 16; r += 2) asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(x[r]), "v"(x[r + 1]));
  return m;
}

// maximum over the two halves of the wave, without a round trip through LDS (attn_staged.hpp)
__device__ __forceinline__ float max_halves(float x) {
  const unsigned u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return st_max(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// Scores of a block of 32 x 32 in place: raw products in; out come the scores in base 2, or, where there is neither cap
// nor bias, the products as they are (x in = the score).  dist0 = pos - (first key of the block) - 4 (l / 32), slope2 =
// slope log2 e.  Register r is key (or query) 8 (r / 4) + r % 4 behind that.
template <int MODE>
__device__ __forceinline__ void block_scores(float (&x)[16], const TileScore& k, float dist0, float slope2) {
  auto dist = [&](int r) { return fabsf(dist0 - float(8 * (r >> 2) + (r & 3))); };
  if constexpr (MODE & kModeCap) {
    if (__any(!(abs_max16(x) <= k.zmax))) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float y = x[r] * k.in;
        const float t = fabsf(y) <= kTanhSmall ? tanh_small(y) : tanh_large(y);
        x[r] = (MODE & kModeBias) ? fmaf(-slope2, dist(r), k.out * t) : k.out * t;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = capped_small(k, x[r]);
        x[r] = (MODE & kModeBias) ? fmaf(x[r], p, -slope2 * dist(r)) : x[r] * p;
      }
    }
  } else if constexpr (MODE & kModeBias) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = fmaf(-slope2, dist(r), x[r] * k.in);
  }
}

}  // namespace fm

namespace fm {

// ---- where the rows of a tile lie ------------------------------------------------------------------------
// contiguous [n][D]: rows behind the last repeat it (their scores are masked)
template <int D, int KT>
struct FlatSource {
  const bf16_t *k, *v;
  int n;
  __device__ __forceinline__ void prefetch(int) {}
  __device__ __forceinline__ void issue(int t, uint32_t lds_k, uint32_t lds_v, int w, int lane) const {
    typedef TileLds<D, KT> T;
    const int kp0 = t * KT;
    const int64_t off = int64_t(kp0) * D;
    const bf16_t* bk = ring_uniform_ptr(k + off);
    const bf16_t* bv = ring_uniform_ptr(v + off);
    const int last = n - 1 - kp0;
#pragma unroll
    for (int u = 0; u < T::kLoadsPerWave; ++u) {
      const int row = T::load_row(w + 4 * u, lane);
      const uint32_t voff = uint32_t(min(row, last)) * T::kRowBytes + T::load_chunk(row, lane);
      tile_load(lds_k + uint32_t(w + 4 * u) * 1024u, voff, bk);
    }
#pragma unroll
    for (int u = 0; u < T::kLoadsPerWave; ++u) {
      const int row = T::load_row(w + 4 * u, lane);
      const uint32_t voff = uint32_t(min(row, last)) * T::kRowBytes + T::load_chunk(row, lane);
      tile_load(lds_v + uint32_t(w + 4 * u) * 1024u, voff, bv);
    }
  }
};

// What a lane's query sees, in the tile's terms.
struct TileQuery {
  int pos, lim, doc;   // doc: -1 sees nothing (only read where there are documents)
  float slope2;
};

// The sweep of a workgroup: tiles [t_begin, t_end) of the keys, this lane's query `qy` (column l % 32 of wave w).
//   lim_lo, lim_hi   fewest and most keys a query of this wave sees; wg_lo: fewest of the workgroup
//   docs             null, or the documents of the keys (padded to whole tiles, negative: -2) and their {min, max} a tile
//   q_doc            {min, max} document of the wave's queries, wg_doc of the workgroup's
struct TileDocs {
  const int32_t* dock;
  const int2* kmeta;
  int2 q_doc, wg_doc;
};

// {min, max} document of a tile of KT keys out of those of 32
template <int KT>
__device__ __forceinline__ int2 tile_docs(const int2* kmeta, int t) {
  if constexpr (KT == 32) return kmeta[t];
  const int2 a = kmeta[2 * t], b = kmeta[2 * t + 1];
  return make_int2(min(a.x, b.x), max(a.y, b.y));
}
template <int KT>
__device__ __forceinline__ int2 tile_docs_scalar(const int2* kmeta, int t) {
  if constexpr (KT == 32) return scalar_load(kmeta, t);
  const int2 a = scalar_load(kmeta, 2 * t), b = scalar_load(kmeta, 2 * t + 1);
  return make_int2(min(a.x, b.x), max(a.y, b.y));
}
// the documents of a tile's keys on their way to LDS beside its rows (wave 3's share)
template <int KT>
__device__ __forceinline__ void issue_docs(const int32_t* dock, int t, uint32_t lds_addr, int w, int lane) {
  if (w == 3) ring_load4(lds_addr, uint32_t(min(lane, KT - 1)) * 4u, ring_uniform_ptr(dock + int64_t(t) * KT));
}

// piece i of n of the tiles [t, t_end); the last ones may be empty
__device__ __forceinline__ void tile_piece(int& t, int& t_end, int i, int n) {
  const int each = (max(t_end - t, 0) + n - 1) / n;
  t = min(t + i * each, t_end);
  t_end = min(t + each, t_end);
}

struct TileState {
  float m, l;
};

template <bool F16, int D, int MODE, bool DOCS, class Source>
__device__ __forceinline__ bool tile_sweep(Source src, const uint4 (&qf)[D / 16], const TileQuery& qy, int lim_lo, int lim_hi,
                                           int wg_lo, int& t_begin, int& t_end, int piece, int pieces, const TileDocs& docs, const TileScore& score,
                                           lds_char_t* lds, int* dirty_flag, typename Mma<F16>::f16v (&O)[D / 32], TileState& st) {
  constexpr int KT = fwd_tile_keys<D>(), NB = KT / 32;
  typedef TileLds<D, KT> T;
  using M = Mma<F16>;
  constexpr int NKS = D / 16, NDT = D / 32;
  constexpr float kLazyGrow = kPLazy<F16>;  // growth of a running maximum (in powers of two) that is left unfollowed
  const int tid = threadIdx.x, l = tid & 63, hb = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(uint32_t(uintptr_t(lds)));
  lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);
  lim_hi = __builtin_amdgcn_readfirstlane(lim_hi);
  wg_lo = __builtin_amdgcn_readfirstlane(wg_lo);
  t_end = __builtin_amdgcn_readfirstlane(t_end);
  const int qd_lo = __builtin_amdgcn_readfirstlane(docs.q_doc.x), qd_hi = __builtin_amdgcn_readfirstlane(docs.q_doc.y);
  const int wd_lo = __builtin_amdgcn_readfirstlane(docs.wg_doc.x), wd_hi = __builtin_amdgcn_readfirstlane(docs.wg_doc.y);
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[dt][r] = 0.f;
  st.m = -INFINITY;
  st.l = 0.f;
  bool dirty = false;

  // the next tile at or behind t that some query of the workgroup sees a document of
  int mask_at = -64;
  unsigned long long mask = 0;
  auto next = [&](int t) {
    if constexpr (!DOCS) return t;
    while (t < t_end) {
      if (t >= mask_at + 64 || mask_at < 0) {
        mask_at = t;
        const int tt = min(t + l, t_end - 1);
        const int2 km = tile_docs<KT>(docs.kmeta, tt);
        mask = __ballot(t + l < t_end && km.y >= wd_lo && km.x <= wd_hi && km.y >= 0);
      }
      const unsigned long long m = mask >> (t - mask_at);
      if (m) return t + __ffsll(m) - 1;
      t = mask_at + 64;
    }
    return t_end;
  };

  const typename T::Bases bases(l);
  auto compute = [&](int t, int buf, int2 km) {
    const lds_char_t* bK = lds + buf * 2 * T::kBytes;
    const lds_char_t* bV = bK + T::kBytes;
    const int kp0 = t * KT;
    if (kp0 >= lim_hi) return;
    bool masked = kp0 + KT > lim_lo;
    if constexpr (DOCS) {
      if (km.y < qd_lo || km.x > qd_hi) return;
      masked |= km.x != km.y || qd_lo != qd_hi;
    }
    const auto at = bases.fresh(0);
    float x[NB][16];
#pragma unroll
    for (int sb = 0; sb < NB; ++sb) {
      typename M::f16v s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) s = M::m32(T::rows32(bK, at.rows, 32 * sb, ks), qf[ks], s);
      tile_settle(s);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[sb][r] = s[r];
      block_scores<MODE>(x[sb], score, float(qy.pos - (kp0 + 32 * sb + 4 * hb)), qy.slope2);
    }
    if (masked) {
#pragma unroll
      for (int sb = 0; sb < NB; ++sb)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int key0 = kp0 + 32 * sb + 8 * r4 + 4 * hb;
          uint4 dk = make_uint4(0, 0, 0, 0);
          if constexpr (DOCS) dk = lds_read16(lds + 4 * T::kBytes + buf * 256 + (key0 - kp0) * 4);
          const int dd[4] = {int(dk.x), int(dk.y), int(dk.z), int(dk.w)};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            bool ok = key0 + r < qy.lim;
            if constexpr (DOCS) ok = ok && dd[r] == qy.doc;
            if (!ok) x[sb][4 * r4 + r] = -INFINITY;
          }
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int sb = 0; sb < NB; ++sb) mx = max16(x[sb], mx);
    mx = max_halves(mx);
    if constexpr (MODE == 0) mx *= score.in;  // (in > 0: scaling commutes with the maximum)
    // The running maximum follows only when some query's grew by more than 2^kLazyGrow (or it sees its first key): until
    // then p stays below 2^kLazyGrow against the older maximum, which neither the fp32 sums nor the relative rounding
    // of p notice, and the accumulator's multiplications are spared in most tiles.
    // (st.m is held kPUp below the maximum it stands for: what the exponents are taken against)
    if (__any(mx > st.m + (kPUp<F16> + kLazyGrow))) {
      const float m_new = fmaxf(st.m, mx - kPUp<F16>), m_to = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(st.m - m_to);
      st.l *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] *= alpha;
      st.m = m_new;
    }
    const float m_sub = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int sb = 0; sb < NB; ++sb) {
      uint4 pf[2];
      float l_block;  // (a block's probabilities are summed by themselves first: one by one a large sum would swallow small ones)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[sb][r] = __builtin_amdgcn_exp2f(MODE == 0 ? fmaf(x[sb][r], score.in, -m_sub) : x[sb][r] - m_sub);
        l_block = r == 0 ? x[sb][0] : l_block + x[sb][r];
      }
      st.l += l_block;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        pf[h] = make_uint4(M::pack2(x[sb][8 * h + 0], x[sb][8 * h + 1]), M::pack2(x[sb][8 * h + 2], x[sb][8 * h + 3]),
                           M::pack2(x[sb][8 * h + 4], x[sb][8 * h + 5]), M::pack2(x[sb][8 * h + 6], x[sb][8 * h + 7]));
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) O[dt] = M::m32(T::cols32(bV, at.cols, 32 * sb + 16 * h, dt), pf[h], O[dt]);
    }
  };

  const uint32_t lds_docs = lds0 + 4u * T::kBytes;
  int t = next(t_begin);
  if (pieces > 1) {
    tile_piece(t, t_end, piece, pieces);
    t_begin = t;
    t = next(t);
  }
  if (t < t_end) {
    src.prefetch(t);
    src.issue(t, lds0, lds0 + T::kBytes, w, l);
    if constexpr (DOCS) issue_docs<KT>(docs.dock, t, lds_docs, w, l);
    src.prefetch(t + 1);
  }
  auto step = [&](int buf) {
    const int t_next = next(t + 1);
    int2 km = make_int2(0, 0);
    if constexpr (DOCS) km = tile_docs_scalar<KT>(docs.kmeta, t);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    ring_barrier();  // tile t is in place, and every wave has finished the tile before it, whose buffer is free
    if (t_next < t_end) {
      const uint32_t to = lds0 + uint32_t(buf ^ 1) * 2u * T::kBytes;
      src.issue(t_next, to, to + T::kBytes, w, l);
      if constexpr (DOCS) issue_docs<KT>(docs.dock, t_next, lds_docs + uint32_t(buf ^ 1) * 256u, w, l);
      src.prefetch(t_next + 1);  // (what a source looks up for its rows: a tile ahead of them)
    }
    // masked places for some query of the workgroup: are there values that 0 x would not erase?
    bool wg_masked = t * KT + KT > wg_lo;
    if constexpr (DOCS) wg_masked |= km.x != km.y || wd_lo != wd_hi;
    if (wg_masked) {
      const lds_char_t* bV = lds + (buf * 2 + 1) * T::kBytes;
#pragma unroll
      for (int u = 0; u < T::kBytes / 4096; ++u) dirty |= any_nonfinite<F16>(lds_read16(bV + (u * 256 + tid) * 16));
    }
    compute(t, buf, km);
    t = t_next;
  };
  if constexpr (D == 256) {  // (one copy of the step: two would not fit the instruction cache)
    for (int buf = 0; t < t_end; buf ^= 1) step(buf);
  } else {  // two tiles a round, so that the buffers are constants
    while (t < t_end) {
      step(0);
      if (t >= t_end) break;
      step(1);
    }
  }
  if (dirty) *dirty_flag = 1;  // (every writer writes the same)
  __syncthreads();
  return *dirty_flag != 0;
}

// This lane's share of a finished query: dimensions 32 dt + 8 (r / 4) + 4 (l / 32) + r % 4.
template <bool F16, int D>
__device__ __forceinline__ void tile_write(const typename Mma<F16>::f16v (&O)[D / 32], const TileState& st, bf16_t* out,
                                           float* lse) {
  const int hb = (threadIdx.x >> 5) & 1;
  const float l = st.l + __shfl_xor(st.l, 32);
  const bool none = st.m == -INFINITY && !(l > 0.f) && l == 0.f;
  const float inv = none ? 0.f : 1.f / l;
  if (!out) return;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      uint2 o;
      o.x = Mma<F16>::pack2(O[dt][4 * rq + 0] * inv, O[dt][4 * rq + 1] * inv);
      o.y = Mma<F16>::pack2(O[dt][4 * rq + 2] * inv, O[dt][4 * rq + 3] * inv);
      *reinterpret_cast<uint2*>(out + dt * 32 + 8 * rq + 4 * hb) = o;
    }
  if (hb == 0) *lse = none ? -FLT_MAX : tile_lse<F16>(st.m, l);
}

// A piece's state of a query, in fp32 and not yet divided.
template <int D, class Acc>
__device__ __forceinline__ void tile_write_part(const Acc (&O)[D / 32], const TileState& st, float* o, float2* ml) {
  const int hb = (threadIdx.x >> 5) & 1;
  const float l = st.l + __shfl_xor(st.l, 32);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq)
      *reinterpret_cast<float4*>(o + dt * 32 + 8 * rq + 4 * hb) =
          make_float4(O[dt][4 * rq], O[dt][4 * rq + 1], O[dt][4 * rq + 2], O[dt][4 * rq + 3]);
  if (hb == 0) *ml = make_float2(st.m, l);
}

// The pieces of a query, in order: 16 lanes a query, D / 16 dimensions each.
template <bool F16, int D>
__device__ __forceinline__ void tile_join(const float* __restrict__ po, const float2* __restrict__ ml, int pieces, bf16_t* __restrict__ out,
                                          float* __restrict__ lse) {
  using M = Mma<F16>;
  const int part = threadIdx.x & 15;
  float mt = -INFINITY;
  for (int i = 0; i < pieces; ++i) mt = fmaxf(mt, ml[i].x);
  const float base = mt == -INFINITY ? 0.f : mt;
  float lt = 0.f, o[D / 16];
#pragma unroll
  for (int k = 0; k < D / 16; ++k) o[k] = 0.f;
  for (int i = 0; i < pieces; ++i) {
    const float2 x = ml[i];
    const float f = __builtin_amdgcn_exp2f(x.x - base);
    lt = fmaf(x.y, f, lt);
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const float4 v = *reinterpret_cast<const float4*>(po + int64_t(i) * D + 64 * u + 4 * part);
      o[4 * u] = fmaf(v.x, f, o[4 * u]), o[4 * u + 1] = fmaf(v.y, f, o[4 * u + 1]);
      o[4 * u + 2] = fmaf(v.z, f, o[4 * u + 2]), o[4 * u + 3] = fmaf(v.w, f, o[4 * u + 3]);
    }
  }
  const bool none = lt == 0.f;
  const float inv = none ? 0.f : 1.f / lt;
#pragma unroll
  for (int u = 0; u < D / 64; ++u)
    *reinterpret_cast<uint2*>(out + 64 * u + 4 * part) =
        make_uint2(M::pack2(o[4 * u] * inv, o[4 * u + 1] * inv), M::pack2(o[4 * u + 2] * inv, o[4 * u + 3] * inv));
  if (part == 0) *lse = none ? -FLT_MAX : tile_lse<F16>(mt, lt);
}

}  // namespace fm
