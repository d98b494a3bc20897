// The tiled forward with score terms at head dimension 256 (terms_fwd.hpp).
#include "terms_fwd.hpp"

namespace fm {
template int terms_fwd_tiles<256>(const FwdTileArgs&, bool, hipStream_t);
}  // namespace fm
