#include "paged_mixed.hpp"

namespace svhip {

template void launch_paged_mixed<kBf16, true>(const PagedArgs&, const PagedPlan&, hipStream_t);
template void launch_paged_mixed<kE4m3, true>(const PagedArgs&, const PagedPlan&, hipStream_t);

}  // namespace svhip
