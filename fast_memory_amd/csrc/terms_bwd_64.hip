// The tiled backward with score terms at head dimension 64 (terms_bwd.hpp).
#include "terms_bwd.hpp"

namespace fm {
template int terms_bwd_tiles<64>(const BwdTileArgs&, bool, const void*, const float*, const float*, float2*, float*, hipStream_t);
}  // namespace fm
