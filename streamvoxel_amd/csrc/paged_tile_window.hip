#include "paged_tile.hpp"

namespace svhip {

template void launch_paged_tiles<kBf16, true>(const PagedArgs&, const PagedPlan&, bool, hipStream_t);
template void launch_paged_tiles<kE4m3, true>(const PagedArgs&, const PagedPlan&, bool, hipStream_t);

}  // namespace svhip
