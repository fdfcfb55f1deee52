#include "paged_row.hpp"

namespace svhip {

template void launch_paged_rows<kBf16, false>(const PagedArgs&, const PagedPlan&, hipStream_t);
template void launch_paged_rows<kE4m3, false>(const PagedArgs&, const PagedPlan&, hipStream_t);

}  // namespace svhip
