#include "paged_row.hpp"
#include "paged_tile.hpp"

namespace svhip {

// Packed windows, which may be of either form: tile_grid workgroups for tiles, which take longest, then those of the
// row form, which fill the CUs as the tiles end. One launch for both: 24 windows, 6 of them chunks (head_dim 96,
// pages of 16, 335 MB) 110 us; the two kernels one after the other 116, and 18 us of host time for 16. Workgroups of
// both forms in turn, one tile's to one, two and four of rows: 122, 112 and 125 us, since a tile with a CU to share
// takes no less time.
template <bool FP8, int KS>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_mixed_kernel(PagedArgs a, int tile_grid, unsigned first_group) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef RowLds<FP8, KS, 2> R;
  constexpr int kTile = TileLds<KS>::kBuffer;
  __shared__ __attribute__((aligned(16))) char s0[R::k0 > kTile ? R::k0 : kTile], s1[R::k1 > kTile ? R::k1 : kTile];
  __shared__ float s_ml[4][2][kRows];
  __shared__ int s_odd;
  const int place = static_cast<int>(first_group + blockIdx.x);
  if (place < tile_grid) {
    tile_work<FP8, false, KS>(a, place, s0, s1, &s_odd);
  } else {
    row_work<FP8, KS, 2>(a, place - tile_grid, s0, s1, s_ml);
  }
#endif
}

template <bool FP8, int KS>
void launch_mixed(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  in_launches(p.tile_grid + p.row_slots, [&](unsigned first, unsigned grid) {
    paged_mixed_kernel<FP8, KS><<<grid, kPagedThreads, 0, s>>>(a, static_cast<int>(p.tile_grid), first);
  });
}

void launch_paged_mixed(const PagedArgs& a, const PagedPlan& p, bool fp8, hipStream_t s) {
  if (fp8) {
    SVHIP_PAGED_WIDTH(launch_mixed, true)
  }
  SVHIP_PAGED_WIDTH(launch_mixed, false)
}

}  // namespace svhip
