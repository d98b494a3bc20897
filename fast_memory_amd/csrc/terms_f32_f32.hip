// Attention with score terms in fp32 products, f32 inputs (terms_f32.hpp, paged_f32.hpp).
#include <algorithm>

#include "paged_f32.hpp"
#include "terms_f32.hpp"

namespace fm {
template int terms_f32_fwd<float>(const F32Args&, hipStream_t);
template int terms_f32_bwd<float>(const F32Args&, const BwdArgs&, float2*, hipStream_t);
template int paged_f32<float>(const PagedTileArgs&, const PagedPlan&, hipStream_t);
}  // namespace fm
