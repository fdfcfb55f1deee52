#include "paged_row.hpp"

namespace svhip {

template void launch_paged_rows<kInt8, false>(const PagedArgs&, const PagedPlan&, hipStream_t);
template void launch_paged_rows<kInt8, true>(const PagedArgs&, const PagedPlan&, hipStream_t);

}  // namespace svhip
