#include "paged_tile.hpp"

namespace svhip {

// Windows that are all of the tile form. Up to 64 head_dim elements a bf16 pool's kernel fits 128 registers and four
// workgroups a CU (8 windows of 1024 queries, head_dim 64: 203.6 us, 204.5 with room for two); wider or decoding ones
// spill there.
template <bool FP8, bool WHOLE, int KS>
__global__ __launch_bounds__(kPagedThreads, FP8 || KS > 4 ? 2 : 4) void paged_tile_kernel(PagedArgs a, unsigned first_group) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ __attribute__((aligned(16))) char s0[TileLds<KS>::kBuffer], s1[TileLds<KS>::kBuffer];
  __shared__ int s_odd;
  tile_work<FP8, WHOLE, KS>(a, static_cast<int>(first_group + blockIdx.x), s0, s1, &s_odd);
#endif
}

template <bool FP8, bool WHOLE, int KS>
void launch_tiles(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  in_launches(p.tile_grid, [&](unsigned first, unsigned grid) {
    paged_tile_kernel<FP8, WHOLE, KS><<<grid, kPagedThreads, 0, s>>>(a, first);
  });
}

void launch_paged_tiles(const PagedArgs& a, const PagedPlan& p, bool fp8, bool whole, hipStream_t s) {
  if (fp8) {
    if (whole) {
      SVHIP_PAGED_WIDTH(launch_tiles, true, true)
    }
    SVHIP_PAGED_WIDTH(launch_tiles, true, false)
  }
  if (whole) {
    SVHIP_PAGED_WIDTH(launch_tiles, false, true)
  }
  SVHIP_PAGED_WIDTH(launch_tiles, false, false)
}

}  // namespace svhip
