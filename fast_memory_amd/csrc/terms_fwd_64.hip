// The tiled forward with score terms at head dimension 64 (terms_fwd.hpp).
#include "terms_fwd.hpp"

namespace fm {
template int terms_fwd_tiles<64>(const FwdTileArgs&, bool, hipStream_t);
}  // namespace fm
