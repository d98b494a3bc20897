// Attention of new tokens over a paged cache at head dimension 64 (paged_attn.hpp).
#include <algorithm>

#include "paged_attn.hpp"

namespace fm {
template int paged_tiles<64>(const PagedTileArgs&, const PagedPlan&, int, hipStream_t);
}  // namespace fm
