// What the queries of a call see, laid out for the tiled kernels by one small launch (terms_masks.hip); only made where
// there are documents or prefixes -- a causal or full attention needs none of it.
//   qinfo [S8]   {keys query i sees as far as order goes (the rows behind the last query: 0), its document or -1}
//   dock [L8]    a key's document, -2 where it has none or lies behind the last key
//   qmeta [S8 / 32]   {fewest, most keys, smallest, largest document} of 32 queries (of those there are)
//   kmeta [L8 / 32]   {smallest, largest document} of 32 keys
// S8, L8: S and L rounded up to 128.
#pragma once
#include "terms_api.hpp"

namespace fm {

struct Masks {
  int2* qinfo;
  int32_t* dock;
  int4* qmeta;
  int2* kmeta;
  size_t bytes;
};

inline Masks masks_layout(void* ws, int S, int L) {
  const size_t S8 = align_up(size_t(S), 128), L8 = align_up(size_t(L), 128);
  Masks m;
  char* p = static_cast<char*>(ws);
  size_t at = 0;
  auto take = [&](size_t n) {
    char* r = p + at;
    at += align_up(n, 256);
    return r;
  };
  m.qinfo = reinterpret_cast<int2*>(take(S8 * 8));
  m.dock = reinterpret_cast<int32_t*>(take(L8 * 4));
  m.qmeta = reinterpret_cast<int4*>(take(S8 / 32 * 16));
  m.kmeta = reinterpret_cast<int2*>(take(L8 / 32 * 8));
  m.bytes = at;
  return m;
}

int make_masks(const Masks& m, const Terms& t, int S, int L, hipStream_t st);

}  // namespace fm
