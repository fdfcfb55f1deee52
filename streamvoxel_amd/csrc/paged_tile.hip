#include "paged_tile.hpp"

namespace svhip {

// Windows that are all of the tile form.
template <bool FP8, bool WHOLE, int KS>
__global__ __launch_bounds__(kPagedThreads, FP8 || KS > 4 ? 2 : 4) void paged_tile_kernel(PagedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ __attribute__((aligned(16))) char s0[TileLds<KS>::kBuffer], s1[TileLds<KS>::kBuffer];
  __shared__ int s_odd;
  tile_work<FP8, WHOLE, KS>(a, static_cast<int>(blockIdx.x), s0, s1, &s_odd);
#endif
}

template <bool FP8, bool WHOLE, int KS>
void launch_tiles(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  paged_tile_kernel<FP8, WHOLE, KS><<<static_cast<unsigned>(p.tile_grid), kPagedThreads, 0, s>>>(a);
}

void launch_paged_tiles(const PagedArgs& a, const PagedPlan& p, bool fp8, bool whole, hipStream_t s) {
  SVHIP_PAGED_LAUNCH(launch_tiles)
}

}  // namespace svhip
