#include "paged_row.hpp"

namespace svhip {

template void launch_paged_rows<kBf16, true>(const PagedArgs&, const PagedPlan&, hipStream_t);
template void launch_paged_rows<kE4m3, true>(const PagedArgs&, const PagedPlan&, hipStream_t);

}  // namespace svhip
