#include "paged_row.hpp"

namespace svhip {

// Windows that are all of the row form.
template <bool FP8, int KS>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_row_kernel(PagedArgs a, unsigned first_group) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kFirst = FP8 ? 4 : 2;
  typedef RowLds<FP8, KS, kFirst> L;
  __shared__ __attribute__((aligned(16))) char s0[L::k0], s1[L::k1];
  __shared__ float s_ml[4][2][kRows];
  row_work<FP8, KS, kFirst>(a, static_cast<int>(first_group + blockIdx.x), s0, s1, s_ml);
#endif
}

template <bool FP8, int KS>
void launch_rows(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  in_launches(p.row_slots, [&](unsigned first, unsigned grid) {
    paged_row_kernel<FP8, KS><<<grid, kPagedThreads, 0, s>>>(a, first);
  });
}

void launch_paged_rows(const PagedArgs& a, const PagedPlan& p, bool fp8, hipStream_t s) {
  if (fp8) {
    SVHIP_PAGED_WIDTH(launch_rows, true)
  }
  SVHIP_PAGED_WIDTH(launch_rows, false)
}

}  // namespace svhip
