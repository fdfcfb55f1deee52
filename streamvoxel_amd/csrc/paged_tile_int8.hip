#include "paged_tile.hpp"

namespace svhip {

template void launch_paged_tiles<kInt8, false>(const PagedArgs&, const PagedPlan&, bool, hipStream_t);
template void launch_paged_tiles<kInt8, true>(const PagedArgs&, const PagedPlan&, bool, hipStream_t);

}  // namespace svhip
