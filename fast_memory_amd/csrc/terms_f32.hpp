// Attention with score terms in fp32 products: fp32 inputs at any head dimension up to 256, and the 16-bit types at the
// dimensions and page sizes that the 16-bit matrix instructions are not laid out for.  v_mfma_f32_32x32x2_f32.
//
// These instructions take 16 times as long as the 16-bit ones for the same product, so that the streamed operands can come
// straight from global memory (L1 and L2 serve the repeats): no barriers in the sweep, every wave on its own.  A workgroup
// owns 32 queries (or 32 keys) and its four waves take the tiles of 32 on the other side in turn; their sums meet in LDS
// at the end, in wave order.  Short rows are spread over four waves this way; too few blocks are cut into pieces (terms_api.hip).
//
//   operand of 32 rows   lane (row l % 32, half l / 32) holds half of the row's dimensions, four of eight: the order of a
//                        contraction is free, a lane then reads 16 consecutive bytes for four products, and both halves the
//                        same cache line
//   scores               as in terms_tile.hpp: lane column = query (key), register r = row 8 (r / 4) + 4 (l / 32) + r % 4
//   second product       register r of both halves is the operand of one instruction: rows k and k + 4; its partner is
//                        one element per lane of those two rows, 32 neighbouring dimensions
// Head dimensions are padded with zeros to Dp = 32 NDT in registers and LDS only.
//
// Masked places are cleared by selects on bits that are formed beforehand (F32Docs::seen), never by an assignment inside a branch on
// the mask: with such a branch around the array of scores the compiler left the store of one of them out (documents were ignored).
//
// Measured in fp32 (a product of 8192 reaches 154 TFLOP/s): 16 heads x 2048 causal, d = 64 130 us forward = 66 TFLOP/s and 356
// backward, d = 128 199 = 86 and 612, d = 256 (1024 tokens) 109 = 79 and 377; one head of 512 tokens 16 and 24 us, 8 query heads on one
// KV head x 1024, d = 128, 49 and 104.  bf16 at d = 96, 32 heads x 2048: 768 and 2420 us.  Bound: the loads' latency between the
// products, at one wave a SIMD (d > 64) or two.  Eight waves a workgroup instead of four: 20 and 54 us for 8 heads x 512, where four
// take 18 and 36 (the backward's registers no longer hold).
#pragma once
#include <type_traits>

#include "terms_masks.hpp"
#include "terms_tile.hpp"

namespace fm {

typedef float f32_acc __attribute__((__vector_size__(16 * sizeof(float))));
__device__ __forceinline__ f32_acc mfma_f32(float a, float b, f32_acc c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32_acc f32_zero() {
  f32_acc a;
#pragma unroll
  for (int r = 0; r < 16; ++r) a[r] = 0.f;
  return a;
}
// the row of register r of a block, without the half's 4 hb
__device__ __forceinline__ constexpr int f32_row(int r) { return 8 * (r >> 2) + (r & 3); }

// VEC: how rows are read.  kOne: an element at a time; kFour: four (d a multiple of 4, rows aligned to four elements); kWhole: four,
// and d is the instance's 32 NDT, so that no load asks where its row ends (every offset is then a constant of its instruction)
constexpr int kOne = 0, kFour = 1, kWhole = 2;
template <int VEC, int NDT>
__device__ __forceinline__ int f32_dims(int d) { return VEC == kWhole ? 32 * NDT : d; }

// four elements of a row from dimension c, zero behind the row's d
template <typename T, int VEC>
__device__ __forceinline__ float4 f32_load4(const T* __restrict__ row, int c, int d) {
  if constexpr (VEC != kOne) {
    if (c >= d) return make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (std::is_same<T, float>::value) {
      return *reinterpret_cast<const float4*>(row + c);
    } else {
      typedef Mma<std::is_same<T, f16_t>::value> M;
      const uint2 u = *reinterpret_cast<const uint2*>(row + c);
      return make_float4(M::lo(u.x), M::hi(u.x), M::lo(u.y), M::hi(u.y));
    }
  } else {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = c + i < d ? Elem<T>::load(row + c + i) : 0.f;
    return make_float4(x[0], x[1], x[2], x[3]);
  }
}

// this lane's half of a row (dimensions 8 j + 4 hb ..), to stay in registers
template <typename T, int VEC, int NDT>
__device__ __forceinline__ void f32_resident(float (&x)[16 * NDT], const T* row, bool ok, int d, int hb) {
#pragma unroll
  for (int j = 0; j < 4 * NDT; ++j) {
    const float4 v = ok ? f32_load4<T, VEC>(row, 8 * j + 4 * hb, d) : make_float4(0.f, 0.f, 0.f, 0.f);
    x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
  }
}

// The resident operand of a product, 4 NDT quads of a lane: registers, or LDS in the backward at 32 NDT = 256, where two operands and a
// sum would take three quarters of a wave's registers and 455 spilled (16 heads x 1024, fp32, d = 256: 606 us, with LDS 378).  The waves'
// sums meet in LDS 128 dimensions at a time, so that two workgroups of such a kernel fit a compute unit: with loads that ask where a row
// ends, two waves a SIMD (and the forward's operand in LDS as well) are the faster (2 x 4 heads x 900, d = 192: forward 87 against 96 us,
// backward 268 against 295), without one (16 heads x 1024, d = 256: 112 against 168, 378 against 478).
// A row in LDS has four words more than dimensions, so that eight neighbouring rows lie on different banks.
template <int NDT>
struct F32Regs {
  const float (&x)[16 * NDT];
  __device__ __forceinline__ float4 quad(int j) const { return make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]); }
};
template <int NDT>
constexpr bool kF32Lds = NDT == 8;
// whether two waves are to run on a SIMD there: where the loads have their bounds to ask for
template <int VEC, int NDT>
constexpr bool f32_two_waves() { return kF32Lds<NDT> && VEC != kWhole; }
template <int NDT>
struct F32Lds {
  static constexpr int kRow = 32 * NDT + 4;
  const float* at;
  __device__ __forceinline__ F32Lds(const float* lds, int col, int hb) : at(lds + col * kRow + 4 * hb) {}
  __device__ __forceinline__ float4 quad(int j) const { return *reinterpret_cast<const float4*>(at + 8 * j); }
  // 32 rows from `rows`, of which the first n are there; all threads of the workgroup
  template <typename T, int VEC>
  __device__ static __forceinline__ void fill(float* lds, const T* rows, int n, int d) {
    for (int i = threadIdx.x; i < 32 * 8 * NDT; i += 256) {
      const int r = i / (8 * NDT), c = 4 * (i % (8 * NDT));
      *reinterpret_cast<float4*>(lds + r * kRow + c) = r < n ? f32_load4<T, VEC>(rows + int64_t(r) * d, c, d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
};

// products of 32 streamed rows (this lane's is `row`) with the resident ones.  Sixteen elements are in flight while the
// products of the sixteen before them run (1024 cycles); the barriers keep the compiler from loading everything at once.
template <typename T, int VEC, int NDT, class Resident>
__device__ __forceinline__ f32_acc f32_products_of(const T* row, const Resident& x, int d, int hb) {
  f32_acc s = f32_zero();
  float4 v[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[0][i] = f32_load4<T, VEC>(row, 8 * i + 4 * hb, d);
#pragma unroll
  for (int g = 0; g < NDT; ++g) {
    float4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = x.quad(4 * g + i);
    if (g + 1 < NDT)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[(g + 1) & 1][i] = f32_load4<T, VEC>(row, 32 * (g + 1) + 8 * i + 4 * hb, d);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 a = v[g & 1][i], b = u[i];
      s = mfma_f32(a.x, b.x, s);
      s = mfma_f32(a.y, b.y, s);
      s = mfma_f32(a.z, b.z, s);
      s = mfma_f32(a.w, b.w, s);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  return s;
}
template <typename T, int VEC, int NDT>
__device__ __forceinline__ f32_acc f32_products(const T* row, const float (&x)[16 * NDT], int d, int hb) {
  return f32_products_of<T, VEC, NDT>(row, F32Regs<NDT>{x}, d, hb);
}

// acc += sum over the 32 rows of a block of row^T w, w = 16 registers.  offset_of(k): of row k from base, in elements
template <typename T, int NDT, class OffsetOf>
__device__ __forceinline__ void f32_accumulate(f32_acc (&acc)[NDT], const float (&w)[16], const T* __restrict__ base,
                                               const OffsetOf& offset_of, int d, int hb, int col, bool watch, bool& dirty) {
  constexpr int kRows = 16 / NDT;  // a group: 16 elements
  float v[2][16];
  auto load = [&](int g) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const auto at = offset_of(f32_row(kRows * g + i) + 4 * hb);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) v[g & 1][NDT * i + dt] = 32 * dt + col < d ? Elem<T>::load(base + at + (32 * dt + col)) : 0.f;
    }
  };
  load(0);
#pragma unroll
  for (int g = 0; g < NDT; ++g) {
    if (g + 1 < NDT) load(g + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) acc[dt] = mfma_f32(v[g & 1][NDT * i + dt], w[kRows * g + i], acc[dt]);
    if (watch)
#pragma unroll
      for (int i = 0; i < 16; ++i) dirty |= !(fabsf(v[g & 1][i]) < INFINITY);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// score arithmetic, chosen at run time (the products hide it)
struct F32Score {
  float in, out;  // terms.hpp; out = 0: no cap
};
// x = the block's scores in base 2; slack = 1 - tanh^2 where asked for.  dist: query's place - key's, of register 0, whose
// sign in r is `along` (-1: registers are keys, 1: queries).
template <bool SLACK>
__device__ __forceinline__ void f32_scores(float (&x)[16], float (&slack)[16], const f32_acc& s, const F32Score& score, float slope2,
                                           int dist, int along) {
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = s[r] * score.in, slack[r] = 1.f;
  if (score.out != 0.f) {
    float big = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(x[r]));
    const bool small = !__any(!(big <= kTanhSmall));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float large = small ? 0.f : tanh_large(x[r]);
      const float t = fabsf(x[r]) <= kTanhSmall ? tanh_small(x[r]) : large;
      if (SLACK) slack[r] = fmaf(-t, t, 1.f);
      x[r] = score.out * t;
    }
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = fmaf(-slope2, fabsf(float(dist + along * f32_row(r))), x[r]);
}
__device__ __forceinline__ bool wave_any(bool b) { return __any(b); }
inline F32Score f32_score(float sm_scale, float softcap) {
  if (softcap > 0.f) return F32Score{sm_scale / softcap, softcap * kLog2e};
  return F32Score{sm_scale * kLog2e, 0.f};
}

struct F32Args {
  FwdArgs f;
  const void* dout;
  const float2* rd;
  void *dq, *dk, *dv;
  Masks m;
  int use_masks;
  F32Score score;
  // where the blocks are too few for the card: pieces of a block's keys (forward, dq) and of its queries (dk dv), each of which
  // leaves its sums, and a launch that joins them in order
  int pieces, splits;
  float* part_o;     // [H G S][pieces][d], forward
  float2* part_ml;   // [H G S][pieces] {m, l}, m in base 2
  float* part_kv;    // [splits][2][H][L][d]
  float* part_dq;    // [pieces][H G][S][d]
};

// {fewest, most keys} and {smallest, largest document} of 32 queries
__device__ __forceinline__ int4 f32_query_meta(const F32Args& a, int i0) {
  if (a.use_masks) return a.m.qmeta[i0 / 32];
  const FwdArgs& f = a.f;
  return make_int4(seen_limit(i0 + (f.L - f.S), f.L, f.t.causal, 0),
                   seen_limit(min(i0 + 31, f.S - 1) + (f.L - f.S), f.L, f.t.causal, 0), 0, 0);
}
__device__ __forceinline__ int2 f32_query_info(const F32Args& a, int i) {  // {limit, document}
  if (a.use_masks) return a.m.qinfo[i];
  return make_int2(i < a.f.S ? seen_limit(i + (a.f.L - a.f.S), a.f.L, a.f.t.causal, 0) : 0, 0);
}

// The waves' sums meet in LDS, 128 dimensions at a time at most.
constexpr int kMeetBlocks = 4;
template <int NDT>
constexpr int meet_blocks() { return NDT < kMeetBlocks ? NDT : kMeetBlocks; }
template <int NDT>
constexpr int kMeetRow = 32 * meet_blocks<NDT>() + 4;
template <int NDT>
constexpr int kMeetFloats = 4 * 32 * kMeetRow<NDT>;  // (two operands of 256 dimensions in LDS take 260 x 64 of these 264 x 64)

template <int NDT>
constexpr size_t f32_lds_bytes() {
  return 256 + size_t(kMeetFloats<NDT>) * 4 + 4 * 32 * 8;
}

// Part h of a wave's sums into LDS ([wave][32][dimensions + 4]), then dimension c of a row's part summed over the waves with weights f
template <int NDT>
__device__ __forceinline__ void f32_put(float* lds, const f32_acc (&acc)[NDT], int h, int w, int col, int hb) {
  float* mine = lds + (w * 32 + col) * kMeetRow<NDT> + 4 * hb;
#pragma unroll
  for (int dt = 0; dt < meet_blocks<NDT>(); ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32_acc& x = acc[meet_blocks<NDT>() * h + dt];
      *reinterpret_cast<float4*>(mine + 32 * dt + 8 * q) = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
    }
}
template <int NDT>
__device__ __forceinline__ float f32_get(const float* lds, int row, int c, const float (&f)[4]) {
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) s = fmaf(lds[(w * 32 + row) * kMeetRow<NDT> + c], f[w], s);
  return s;
}
// All rows' sums over the waves, part 0 of which is in LDS already: write(row, dimension, value) a wave a row, dims of rows [0, n).
// weights(row, f): what the waves weigh.
template <int NDT, class Weights, class Write>
__device__ __forceinline__ void f32_meet_all(float* lds, const f32_acc (&acc)[NDT], int w, int col, int hb, int n, int d, const Weights& weights,
                                             const Write& write) {
  constexpr int kDims = 32 * meet_blocks<NDT>();
#pragma unroll
  for (int h = 0; h < NDT / meet_blocks<NDT>(); ++h) {
    if (h > 0) {
      if (kDims * h >= d) return;
      __syncthreads();
      f32_put<NDT>(lds, acc, h, w, col, hb);
      __syncthreads();
    }
    for (int i = w; i < n; i += 4) {
      float f[4];
      weights(i, f);
      for (int c = lane_id(); c < kDims && kDims * h + c < d; c += 64) write(i, kDims * h + c, f32_get<NDT>(lds, i, c, f));
    }
  }
}
__device__ __forceinline__ void f32_ones(int, float (&f)[4]) { f[0] = f[1] = f[2] = f[3] = 1.f; }

// what wave k's sums of a query weigh under the maximum m, and the query's {maximum, sum} over the waves
__device__ __forceinline__ float f32_weight(const float2* ml, int i, int k, float m) {
  return __builtin_amdgcn_exp2f(ml[k * 32 + i].x - (m == -INFINITY ? 0.f : m));
}
__device__ __forceinline__ float2 f32_meet(const float2* ml, int i) {
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) m = fmaxf(m, ml[k * 32 + i].x);
#pragma unroll
  for (int k = 0; k < 4; ++k) l = fmaf(ml[k * 32 + i].y, f32_weight(ml, i, k, m), l);
  return make_float2(m, l);
}

// the waves' weights in a query's result, which is divided by its sum where it is whole
__device__ __forceinline__ void f32_weights(const float2* ml, int i, bool whole, float (&g)[4]) {
  const float2 st = f32_meet(ml, i);
  const float inv = !whole ? 1.f : st.y == 0.f ? 0.f : 1.f / st.y;
#pragma unroll
  for (int k = 0; k < 4; ++k) g[k] = f32_weight(ml, i, k, st.x) * inv;
}

// The sweep of a wave over tiles of 32 keys t = first, first + step, .. < t_end of one head.  row_of(j): where key j's row
// begins, the same function for keys and values.  FLAT: rows follow one another.
template <typename T, int VEC, int NDT, bool FLAT, class Resident, class RowOf, class Docs>
__device__ __forceinline__ void f32_forward(const Resident& q, int pos, int lim, float slope2, int lim_lo, const T* K,
                                            const T* V, const RowOf& row_of, int n, int first, int step, int t_end, int d,
                                            const F32Score& score, const Docs& docs, f32_acc (&O)[NDT], float& m, float& sum,
                                            bool& dirty) {
  const int l = lane_id(), col = l & 31, hb = l >> 5;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) O[dt] = f32_zero();
  m = -INFINITY;
  sum = 0.f;
  int64_t next = row_of(min(32 * first + col, n - 1));
  for (int t = first; t < t_end; t += step) {
    const int kp0 = 32 * t;
    const int64_t at = next;
    next = row_of(min(kp0 + 32 * step + col, n - 1));
    bool masked = kp0 + 32 > lim_lo;
    if (!docs.meets(t, masked)) continue;
    masked = wave_any(masked);
    const f32_acc s = f32_products_of<T, VEC, NDT>(K + at, q, d, hb);
    float x[16], slack[16], mx = -INFINITY;
    f32_scores<false>(x, slack, s, score, slope2, pos - kp0 - 4 * hb, -1);
    if (masked) {
      const unsigned seen = docs.seen(kp0 + 4 * hb, lim);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = seen >> r & 1 ? x[r] : -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.f : m_new;
    if (__any(m_new > m)) {
      const float alpha = __builtin_amdgcn_exp2f(m - base);
      sum *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[dt][r] *= alpha;
    }
    m = m_new;
    float s_tile = 0.f;  // (by itself first, see tile_sweep)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = __builtin_amdgcn_exp2f(x[r] - base);
      s_tile += x[r];
    }
    sum += s_tile;
    if constexpr (FLAT) {
      const int last = n - 1 - kp0;
      f32_accumulate<T, NDT>(O, x, V + int64_t(kp0) * d, [&](int k) { return unsigned(min(k, last) * d); }, d, hb, col, masked, dirty);
    } else {
      f32_accumulate<T, NDT>(O, x, V, [&](int k) { return __shfl(at, k); }, d, hb, col, masked, dirty);
    }
  }
}

struct F32Docs {
  const int2* kmeta;
  const int32_t* dock;
  int lo, hi, mine;  // of the 32 queries; of this lane's
  bool has;
  __device__ __forceinline__ bool meets(int t, bool& masked) const {
    if (!has) return true;
    const int2 km = kmeta[t];
    masked |= km.x != km.y || lo != hi;
    return wave_any(km.y >= 0 && km.y >= lo && km.x <= hi);
  }
  // bit r: the query sees key + f32_row(r); dock is padded to whole tiles
  __device__ __forceinline__ unsigned seen(int key, int lim) const {
    unsigned bits = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      int4 dk = make_int4(mine, mine, mine, mine);
      if (has) dk = *reinterpret_cast<const int4*>(dock + key + 8 * q);
      const int x[4] = {dk.x, dk.y, dk.z, dk.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) bits |= unsigned(int(key + 8 * q + e < lim) & int(x[e] == mine)) << (4 * q + e);
    }
    return bits;
  }
};

template <typename T, int VEC, int NDT>
__global__ __launch_bounds__(256, (f32_two_waves<VEC, NDT>() ? 2 : 1)) void terms_f32_fwd_kernel(F32Args a) {
  extern __shared__ __attribute__((aligned(256))) float f32_lds[];
  int* flag = reinterpret_cast<int*>(f32_lds);
  float* lds = f32_lds + 64;
  float2* ml = reinterpret_cast<float2*>(lds + kMeetFloats<NDT>);
  const FwdArgs& f = a.f;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5, d = f32_dims<VEC, NDT>(f.d);
  const int heads = f.H * f.G, bx = int(blockIdx.x) % heads;
  const int hk = bx % f.H, hq = hk * f.G + bx / f.H;
  const int rest = int(blockIdx.x) / heads, piece = rest % a.pieces;
  const int i0 = ((f.S + 31) / 32 - 1 - rest / a.pieces) * 32, iq = i0 + col;
  if (tid == 0) *flag = 0;
  __syncthreads();
  const bool ok = iq < f.S;
  const int2 qi = f32_query_info(a, iq);
  const int4 qm = f32_query_meta(a, i0);
  const float slope2 = f.t.slopes ? f.t.slopes[hq] * kLog2e : 0.f;
  constexpr bool kLds = f32_two_waves<VEC, NDT>();
  float qf[kLds ? 1 : 16 * NDT];
  if constexpr (kLds) {
    F32Lds<NDT>::template fill<T, VEC>(lds, (const T*)f.q + (int64_t(hq) * f.S + i0) * d, f.S - i0, d);
    __syncthreads();
  } else {
    f32_resident<T, VEC, NDT>(qf, (const T*)f.q + (int64_t(hq) * f.S + (ok ? iq : 0)) * d, ok, d, hb);
  }
  const T* K = (const T*)f.k + int64_t(hk) * f.L * d;
  const T* V = (const T*)f.v + int64_t(hk) * f.L * d;
  const F32Docs docs{a.m.kmeta, a.m.dock, qm.z, qm.w, qi.y, f.t.doc_q != nullptr};
  f32_acc O[NDT];
  float m, sum;
  bool dirty = false;
  int t0 = 0, t1 = (qm.y + 31) / 32;
  tile_piece(t0, t1, piece, a.pieces);
  auto sweep = [&](const auto& q) {
    f32_forward<T, VEC, NDT, true>(q, iq + (f.L - f.S), qi.x, slope2, qm.x, K, V, [&](int j) { return int64_t(j) * d; }, f.L, t0 + w, 4,
                                   t1, d, a.score, docs, O, m, sum, dirty);
  };
  if constexpr (kLds)
    sweep(F32Lds<NDT>(lds, col, hb));
  else
    sweep(F32Regs<NDT>{qf});
  if (dirty) *flag = 1;
  sum += __shfl_xor(sum, 32);
  if constexpr (kLds) __syncthreads();
  f32_put<NDT>(lds, O, 0, w, col, hb);
  if (hb == 0) ml[w * 32 + col] = make_float2(m, sum);
  __syncthreads();
  if (*flag) {  // values that are not finite, in tiles with masked places: a row at a time (terms.hpp)
    const KeyRows<T> KR{K, nullptr, 0, 0, 0, d}, VR{V, nullptr, 0, 0, 0, d};
    for (int i = i0 + w; i < min(i0 + 32, f.S); i += 4) {
      const int64_t r = int64_t(hq) * f.S + i;
      const QueryView qv = query_view(f.t, i, f.S, f.L, hq);
      const RowState rs = f.t.softcap > 0.f
                              ? row_forward<T, true>((const T*)f.q + r * d, KR, VR, qv, f.t.doc_k, 32 * t0, 32 * t1, Score<true>(f.sm_scale, f.t.softcap))
                              : row_forward<T, false>((const T*)f.q + r * d, KR, VR, qv, f.t.doc_k, 32 * t0, 32 * t1, Score<false>(f.sm_scale, 0.f));
      if (a.pieces == 1) {
        row_write(rs, d, (T*)f.out + r * d, f.lse + r);
        continue;
      }
      const int64_t at = r * a.pieces + piece;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (l + 64 * u < d) a.part_o[at * d + l + 64 * u] = rs.acc[u];
      if (l == 0) a.part_ml[at] = make_float2(rs.m, rs.l);
    }
    return;
  }
  const int n = min(32, f.S - i0);
  const int64_t r0 = int64_t(hq) * f.S + i0;
  if (l == 0)
    for (int i = w; i < n; i += 4) {
      const float2 st = f32_meet(ml, i);
      if (a.pieces > 1)
        a.part_ml[(r0 + i) * a.pieces + piece] = st;
      else
        f.lse[r0 + i] = st.y == 0.f ? -FLT_MAX : (st.x + __builtin_amdgcn_logf(st.y)) * kLn2;
    }
  f32_meet_all<NDT>(lds, O, w, col, hb, n, d, [&](int i, float (&g)[4]) { f32_weights(ml, i, a.pieces == 1, g); }, [&](int i, int c, float x) {
    if (a.pieces > 1)
      a.part_o[((r0 + i) * a.pieces + piece) * d + c] = x;
    else
      Elem<T>::store((T*)f.out + (r0 + i) * d + c, x);
  });
}

// the pieces of a query row, in order: a wave a row
template <typename T>
__device__ __forceinline__ void f32_join_row(const float* __restrict__ po, const float2* __restrict__ ml, int pieces, int d, T* __restrict__ out,
                                             float* __restrict__ lse) {
  const int l = lane_id();
  RowState st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r) st.acc[r] = 0.f;
  for (int i = 0; i < pieces; ++i) st.m = fmaxf(st.m, ml[i].x);
  const float base = st.m == -INFINITY ? 0.f : st.m;
  for (int i = 0; i < pieces; ++i) {
    const float2 x = ml[i];
    const float f = __builtin_amdgcn_exp2f(x.x - base);
    st.l = fmaf(x.y, f, st.l);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (l + 64 * r < d) st.acc[r] = fmaf(po[int64_t(i) * d + l + 64 * r], f, st.acc[r]);
  }
  row_write(st, d, out, lse);
}
template <typename T>
__global__ __launch_bounds__(256) void terms_f32_join_kernel(F32Args a) {
  const FwdArgs& f = a.f;
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= int64_t(f.H) * f.G * f.S) return;
  f32_join_row(a.part_o + row * a.pieces * f.d, a.part_ml + row * a.pieces, a.pieces, f.d, (T*)f.out + row * f.d, f.lse + row);
}

// ---- backward ---------------------------------------------------------------------------------------------------------
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

template <typename T, int VEC, int NDT>
__device__ __forceinline__ void f32_dq_block(const F32Args& a, int block, float* f32_lds) {
  int* flag = reinterpret_cast<int*>(f32_lds);
  float* lds = f32_lds + 64;
  const FwdArgs& f = a.f;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5, d = f32_dims<VEC, NDT>(f.d);
  const int heads = f.H * f.G, bx = block % heads;
  const int hk = bx % f.H, hq = hk * f.G + bx / f.H;
  const int rest = block / heads, piece = rest % a.pieces;
  const int i0 = ((f.S + 31) / 32 - 1 - rest / a.pieces) * 32, iq = i0 + col;
  if (tid == 0) *flag = 0;
  __syncthreads();
  const bool ok = iq < f.S;
  const int2 qi = f32_query_info(a, iq);
  const int4 qm = f32_query_meta(a, i0);
  const float slope2 = f.t.slopes ? f.t.slopes[hq] * kLog2e : 0.f;
  const int64_t row = int64_t(hq) * f.S + (ok ? iq : 0);
  constexpr bool kLds = kF32Lds<NDT>;
  float qf[kLds ? 1 : 16 * NDT], df[kLds ? 1 : 16 * NDT];
  if constexpr (kLds) {
    F32Lds<NDT>::template fill<T, VEC>(lds + 32 * F32Lds<NDT>::kRow, (const T*)f.q + (int64_t(hq) * f.S + i0) * d, f.S - i0, d);
    F32Lds<NDT>::template fill<T, VEC>(lds, (const T*)a.dout + (int64_t(hq) * f.S + i0) * d, f.S - i0, d);
    __syncthreads();
  } else {
    f32_resident<T, VEC, NDT>(qf, (const T*)f.q + row * d, ok, d, hb);
    f32_resident<T, VEC, NDT>(df, (const T*)a.dout + row * d, ok, d, hb);
  }
  const float2 rd = ok ? a.rd[row] : make_float2(0.f, 0.f);
  const T* K = (const T*)f.k + int64_t(hk) * f.L * d;
  const T* V = (const T*)f.v + int64_t(hk) * f.L * d;
  const F32Docs docs{a.m.kmeta, a.m.dock, qm.z, qm.w, qi.y, f.t.doc_q != nullptr};
  const int pos = iq + (f.L - f.S);
  f32_acc O[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) O[dt] = f32_zero();
  bool dirty = false;
  int t0 = 0, t1 = (qm.y + 31) / 32;
  tile_piece(t0, t1, piece, a.pieces);
  float* part = a.pieces > 1 ? a.part_dq + (int64_t(piece) * heads + hq) * f.S * d : nullptr;
  for (int t = t0 + w; t < t1; t += 4) {
    const int kp0 = 32 * t;
    bool masked = kp0 + 32 > qm.x;
    if (!docs.meets(t, masked)) continue;
    const int64_t at = int64_t(min(kp0 + col, f.L - 1)) * d;
    f32_acc s, p;
    if constexpr (kLds)
      s = f32_products_of<T, VEC, NDT>(K + at, F32Lds<NDT>(lds + 32 * F32Lds<NDT>::kRow, col, hb), d, hb);
    else
      s = f32_products<T, VEC, NDT>(K + at, qf, d, hb);
    if constexpr (kLds)
      p = f32_products_of<T, VEC, NDT>(V + at, F32Lds<NDT>(lds, col, hb), d, hb);
    else
      p = f32_products<T, VEC, NDT>(V + at, df, d, hb);
    float g[16], slack[16];
    f32_scores<true>(g, slack, s, a.score, slope2, pos - kp0 - 4 * hb, -1);
#pragma unroll
    for (int r = 0; r < 16; ++r) g[r] = __builtin_amdgcn_exp2f(g[r] - rd.x) * (p[r] - rd.y) * slack[r];
    if (masked) {
      const unsigned seen = docs.seen(kp0 + 4 * hb, qi.x);
#pragma unroll
      for (int r = 0; r < 16; ++r) g[r] = seen >> r & 1 ? g[r] : 0.f;
    }
    const int last = f.L - 1 - kp0;
    f32_accumulate<T, NDT>(O, g, K + int64_t(kp0) * d, [&](int k) { return unsigned(min(k, last) * d); }, d, hb, col, masked, dirty);
  }
  if (dirty) *flag = 1;
  if constexpr (kLds) __syncthreads();
  f32_put<NDT>(lds, O, 0, w, col, hb);
  __syncthreads();
  if (*flag) {
    const KeyRows<T> KR{K, nullptr, 0, 0, 0, d}, VR{V, nullptr, 0, 0, 0, d};
    for (int i = i0 + w; i < min(i0 + 32, f.S); i += 4) {
      const int64_t r = int64_t(hq) * f.S + i;
      const QueryView qv = query_view(f.t, i, f.S, f.L, hq);
      const T *q = (const T*)f.q + r * d, *o = (const T*)a.dout + r * d;
      auto row = [&](auto* to) {
        if (f.t.softcap > 0.f)
          row_dq<T, true>(q, o, a.rd[r], KR, VR, qv, f.t.doc_k, 32 * t0, 32 * t1, f.sm_scale, Score<true>(f.sm_scale, f.t.softcap), to);
        else
          row_dq<T, false>(q, o, a.rd[r], KR, VR, qv, f.t.doc_k, 32 * t0, 32 * t1, f.sm_scale, Score<false>(f.sm_scale, 0.f), to);
      };
      if (part)
        row(part + int64_t(i) * d);
      else
        row((T*)a.dq + r * d);
    }
    return;
  }
  f32_meet_all<NDT>(lds, O, w, col, hb, min(32, f.S - i0), d, f32_ones, [&](int i, int c, float x) {
    x *= f.sm_scale;
    if (part)
      part[int64_t(i0 + i) * d + c] = x;
    else
      Elem<T>::store((T*)a.dq + (int64_t(hq) * f.S + i0 + i) * d + c, x);
  });
}

// dk and dv of 32 keys; PART as in terms_bwd.hpp (both sums and both operands of a padded dimension of 256 are 512 registers)
constexpr int kF32Both = 0, kF32Dv = 1, kF32Dk = 2;

template <typename T, int VEC, int NDT, int PART>
__device__ __forceinline__ void f32_dkv_block(const F32Args& a, int block, float* f32_lds) {
  constexpr bool kDk = PART != kF32Dv, kDv = PART != kF32Dk;
  int* flag = reinterpret_cast<int*>(f32_lds);
  float* lds = f32_lds + 64;
  const FwdArgs& f = a.f;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, col = l & 31, hb = l >> 5, d = f32_dims<VEC, NDT>(f.d);
  const int hk = block % f.H, part = block / f.H, split = part % a.splits, j0 = part / a.splits * 32, j = j0 + col;
  if (tid == 0) *flag = 0;
  __syncthreads();
  const bool ok = j < f.L, has_docs = f.t.doc_q != nullptr;
  const int doc = has_docs ? a.m.dock[j] : 0;
  const int2 km = has_docs ? a.m.kmeta[j0 / 32] : make_int2(0, 0);
  const int64_t row = (int64_t(hk) * f.L + (ok ? j : 0)) * d;
  constexpr bool kLds = kF32Lds<NDT>;
  float kf[kLds ? 1 : 16 * NDT], vf[kDk && !kLds ? 16 * NDT : 1];
  if constexpr (!kLds) f32_resident<T, VEC, NDT>(kf, (const T*)f.k + row, ok, d, hb);
  if constexpr (kLds) {
    F32Lds<NDT>::template fill<T, VEC>(lds + 32 * F32Lds<NDT>::kRow, (const T*)f.k + (int64_t(hk) * f.L + j0) * d, f.L - j0, d);
    if constexpr (kDk) F32Lds<NDT>::template fill<T, VEC>(lds, (const T*)f.v + (int64_t(hk) * f.L + j0) * d, f.L - j0, d);
    __syncthreads();
  } else if constexpr (kDk) {
    f32_resident<T, VEC, NDT>(vf, (const T*)f.v + row, ok, d, hb);
  }
  f32_acc dK[kDk ? NDT : 1], dV[kDv ? NDT : 1];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    if constexpr (kDk) dK[dt] = f32_zero();
    if constexpr (kDv) dV[dt] = f32_zero();
  }
  bool dirty = false;
  // the (head, tile of queries) pairs from the last tile down to the first that can see the keys; of this workgroup's, every
  // fourth is this wave's
  const int nqt = (f.S + 31) / 32, qt0 = (f.t.causal && !a.use_masks) ? min(max(0, j0 - (f.L - f.S)) / 32, nqt) : 0, n = nqt - qt0;
  const int64_t steps = int64_t(f.G) * n;
  const int s0 = int(steps * split / a.splits), s1 = int(steps * (split + 1) / a.splits);
  // (a loop over heads and one over tiles: as a single one over pairs it takes 100 registers more)
  int g = n > 0 ? s0 / n : 0, step = s0 - g * n + w;
  for (; g * n < s1; ++g) {
    const int hq = hk * f.G + g, end = min(n, s1 - g * n);
    const float slope2 = f.t.slopes ? f.t.slopes[hq] * kLog2e : 0.f;
    const T* Q = (const T*)f.q + int64_t(hq) * f.S * d;
    const T* DO = (const T*)a.dout + int64_t(hq) * f.S * d;
    const float2* RD = a.rd + int64_t(hq) * f.S;
    for (; step < end; step += 4) {
      const int i0 = (nqt - 1 - step) * 32;
      const int4 qm = f32_query_meta(a, i0);
      if (qm.y <= j0) continue;
      bool masked = i0 + 32 > f.S || j0 + 32 > qm.x;
      if (has_docs) {
        if (km.y < 0 || km.y < qm.z || km.x > qm.w) continue;
        masked |= km.x != km.y || qm.z != qm.w;
      }
      masked = wave_any(masked);
      const int i = min(i0 + col, f.S - 1);
      const float2 mine = RD[i];
      f32_acc s;
      if constexpr (kLds)
        s = f32_products_of<T, VEC, NDT>(Q + int64_t(i) * d, F32Lds<NDT>(lds + 32 * F32Lds<NDT>::kRow, col, hb), d, hb);
      else
        s = f32_products<T, VEC, NDT>(Q + int64_t(i) * d, kf, d, hb);
      float x[16], y[16];  // p; slack, then g
      f32_scores<true>(x, y, s, a.score, slope2, i0 + 4 * hb + (f.L - f.S) - j, 1);
      unsigned seen = 0xffff;
      if (masked) {
        seen = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int iq = i0 + f32_row(r) + 4 * hb;
          const int2 qi = f32_query_info(a, iq);
          seen |= unsigned(int(iq < f.S) & int(j < qi.x) & int(!has_docs | (qi.y == doc))) << r;
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = __builtin_amdgcn_exp2f(x[r] - __shfl(mine.x, f32_row(r) + 4 * hb));
        x[r] = seen >> r & 1 ? e : 0.f;
      }
      const int last = f.S - 1 - i0;
      auto offset = [&](int k) { return unsigned(min(k, last) * d); };
      if constexpr (kDv) f32_accumulate<T, NDT>(dV, x, DO + int64_t(i0) * d, offset, d, hb, col, masked, dirty);
      if constexpr (kDk) {
        f32_acc p;
        if constexpr (kLds)
          p = f32_products_of<T, VEC, NDT>(DO + int64_t(i) * d, F32Lds<NDT>(lds, col, hb), d, hb);
        else
          p = f32_products<T, VEC, NDT>(DO + int64_t(i) * d, vf, d, hb);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = x[r] * y[r] * (p[r] - __shfl(mine.y, f32_row(r) + 4 * hb));
          y[r] = seen >> r & 1 ? e : 0.f;
        }
        f32_accumulate<T, NDT>(dK, y, Q + int64_t(i0) * d, offset, d, hb, col, masked, dirty);
      }
    }
    step -= n;
  }
  if (dirty) *flag = 1;
  if constexpr (kLds) __syncthreads();
  if constexpr (kDk) f32_put<NDT>(lds, dK, 0, w, col, hb);
  __syncthreads();
  const int last = min(32, f.L - j0);
  // element c of key jj's gradients, x of dk (times sm_scale here) and of dv
  const int64_t plane = int64_t(f.H) * f.L * d;
  auto put = [&](bool dv, int jj, int c, float x) {
    const int64_t at = (int64_t(hk) * f.L + jj) * d + c;
    if (!dv) x *= f.sm_scale;
    if (a.splits > 1)
      a.part_kv[(2 * split + dv) * plane + at] = x;
    else
      Elem<T>::store((T*)(dv ? a.dv : a.dk) + at, x);
  };
  if (*flag) {
    for (int jj = j0 + w; jj < j0 + last; jj += 4) {
      const int64_t at = (int64_t(hk) * f.L + jj) * d;
      const T *k = (const T*)f.k + at, *v = (const T*)f.v + at;
      KeyGrads kg;
      key_grads_zero(kg);
      for (int step = s0; step < s1; ++step) {
        const int g = step / n, ib = (nqt - 1 - (step - g * n)) * 32;
        if (f.t.softcap > 0.f)
          row_dkv_chunk<T, true>(k, v, jj, hk * f.G + g, ib, min(f.S, ib + 32), f.S, f.L, d, (const T*)f.q, (const T*)a.dout, a.rd,
                                 f.t, Score<true>(f.sm_scale, f.t.softcap), kg);
        else
          row_dkv_chunk<T, false>(k, v, jj, hk * f.G + g, ib, min(f.S, ib + 32), f.S, f.L, d, (const T*)f.q, (const T*)a.dout, a.rd,
                                  f.t, Score<false>(f.sm_scale, 0.f), kg);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int c = l + 64 * r;
        if (c >= d) continue;
        if constexpr (kDk) put(false, jj, c, kg.k[r]);
        if constexpr (kDv) put(true, jj, c, kg.v[r]);
      }
    }
    return;
  }
  if constexpr (kDk) f32_meet_all<NDT>(lds, dK, w, col, hb, last, d, f32_ones, [&](int i, int c, float x) { put(false, j0 + i, c, x); });
  if constexpr (kDv) {
    if constexpr (kDk) __syncthreads();
    f32_put<NDT>(lds, dV, 0, w, col, hb);
    __syncthreads();
    f32_meet_all<NDT>(lds, dV, w, col, hb, last, d, f32_ones, [&](int i, int c, float x) { put(true, j0 + i, c, x); });
  }
}

// The pieces' sums in order, each rounded once: dk and dv from part_kv, then dq from part_dq, where they have any.
template <typename T>
__global__ __launch_bounds__(256) void terms_f32_bwd_join_kernel(F32Args a, int64_t plane, int64_t plane_q) {
  int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int64_t kv = a.splits > 1 ? 2 * plane : 0;
  const bool is_q = i >= kv;
  if (is_q) i -= kv;
  if (is_q && (a.pieces == 1 || i >= plane_q)) return;
  const float* from = (is_q ? a.part_dq : a.part_kv) + i;
  const int64_t step = is_q ? plane_q : 2 * plane;
  float x = *from;
  for (int k = 1; k < (is_q ? a.pieces : a.splits); ++k) x += from[k * step];
  Elem<T>::store(is_q ? (T*)a.dq + i : i < plane ? (T*)a.dk + i : (T*)a.dv + (i - plane), x);
}

template <typename T, int VEC, int NDT>
__global__ __launch_bounds__(256, (f32_two_waves<VEC, NDT>() ? 2 : 1)) void terms_f32_bwd_kernel(F32Args a, int dkv_blocks) {
  extern __shared__ __attribute__((aligned(256))) float f32_lds[];
  const int block = blockIdx.x;
  if constexpr (NDT == 8) {
    if (block < dkv_blocks) return f32_dkv_block<T, VEC, NDT, kF32Dk>(a, block, f32_lds);
    if (block < 2 * dkv_blocks) return f32_dkv_block<T, VEC, NDT, kF32Dv>(a, block - dkv_blocks, f32_lds);
    f32_dq_block<T, VEC, NDT>(a, block - 2 * dkv_blocks, f32_lds);
  } else {
    if (block < dkv_blocks) return f32_dkv_block<T, VEC, NDT, kF32Both>(a, block, f32_lds);
    f32_dq_block<T, VEC, NDT>(a, block - dkv_blocks, f32_lds);
  }
}

template <typename T, int VEC, int NDT>
static int launch_f32_fwd(const F32Args& a, hipStream_t st) {
  FM_ALLOW_LDS((terms_f32_fwd_kernel<T, VEC, NDT>), f32_lds_bytes<NDT>(), "fm_local_attn_terms_fwd(lds)");
  hipLaunchKernelGGL((terms_f32_fwd_kernel<T, VEC, NDT>), dim3(unsigned(a.f.H * a.f.G * ceil_div(a.f.S, 32) * a.pieces)), dim3(256),
                     f32_lds_bytes<NDT>(), st, a);
  return launch_status("fm_local_attn_terms_fwd(f32)");
}
template <typename T>
static int launch_delta(const BwdArgs& a, float2* rd, hipStream_t st) {
  const int64_t rows = int64_t(a.f.H) * a.f.G * a.f.S;
  hipLaunchKernelGGL(terms_delta_kernel<T>, dim3(unsigned(ceil_div(rows, 4))), dim3(256), 0, st, (const T*)a.f.out,
                     (const T*)a.dout, a.f.lse, a.dlse, rd, a.f.d, rows);
  return launch_status("fm_local_attn_terms_bwd(delta)");
}

template <typename T, int VEC, int NDT>
static int launch_f32_bwd(const F32Args& a, hipStream_t st) {
  FM_ALLOW_LDS((terms_f32_bwd_kernel<T, VEC, NDT>), f32_lds_bytes<NDT>(), "fm_local_attn_terms_bwd(lds)");
  const int dkv = int(a.f.H * ceil_div(a.f.L, 32) * a.splits), dq = int(a.f.H * a.f.G * ceil_div(a.f.S, 32) * a.pieces);
  hipLaunchKernelGGL((terms_f32_bwd_kernel<T, VEC, NDT>), dim3(unsigned((NDT == 8 ? 2 : 1) * dkv + dq)), dim3(256),
                     f32_lds_bytes<NDT>(), st, a, dkv);
  return launch_status("fm_local_attn_terms_bwd(f32)");
}

// how rows of d elements are read
template <typename T>
static int f32_vec(int d, std::initializer_list<const void*> ptrs) {
  bool ok = d % 4 == 0;
  for (const void* p : ptrs) ok = ok && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0;
  return !ok ? kOne : d == 64 || d == 128 || d == 256 ? kWhole : kFour;
}
#define FM_F32_BY_VEC(vec, F, N) ((vec) == kWhole ? F(kWhole, N) : (vec) == kFour ? F(kFour, N) : F(kOne, N))
#define FM_F32_BY_DIM(d, vec, F) \
  ((d) <= 64 ? FM_F32_BY_VEC(vec, F, 2) : (d) <= 128 ? FM_F32_BY_VEC(vec, F, 4) : FM_F32_BY_VEC(vec, F, 8))

template <typename T>
int terms_f32_fwd(const F32Args& a, hipStream_t st) {
  const int vec = f32_vec<T>(a.f.d, {a.f.q, a.f.k, a.f.v});
#define FM_F(V, N) launch_f32_fwd<T, V, N>(a, st)
  const int rc = FM_F32_BY_DIM(a.f.d, vec, FM_F);
#undef FM_F
  if (rc || a.pieces == 1) return rc;
  hipLaunchKernelGGL(terms_f32_join_kernel<T>, dim3(unsigned(ceil_div(int64_t(a.f.H) * a.f.G * a.f.S, 4))), dim3(256), 0, st, a);
  return launch_status("fm_local_attn_terms_fwd(join)");
}
template <typename T>
int terms_f32_bwd(const F32Args& a, const BwdArgs& b, float2* rd, hipStream_t st) {
  int rc = launch_delta<T>(b, rd, st);
  if (rc) return rc;
  const int vec = f32_vec<T>(a.f.d, {a.f.q, a.f.k, a.f.v, a.dout});
#define FM_F(V, N) launch_f32_bwd<T, V, N>(a, st)
  rc = FM_F32_BY_DIM(a.f.d, vec, FM_F);
#undef FM_F
  if (rc || (a.splits == 1 && a.pieces == 1)) return rc;
  const int64_t plane = int64_t(a.f.H) * a.f.L * a.f.d, plane_q = int64_t(a.f.H) * a.f.G * a.f.S * a.f.d;
  const int64_t n = (a.splits > 1 ? 2 * plane : 0) + (a.pieces > 1 ? plane_q : 0);
  hipLaunchKernelGGL(terms_f32_bwd_join_kernel<T>, dim3(unsigned(ceil_div(n, 256))), dim3(256), 0, st, a, plane, plane_q);
  return launch_status("fm_local_attn_terms_bwd(join)");
}

}  // namespace fm
