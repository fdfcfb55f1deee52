// The launch of svhip_paged_attention (paged_attention.hip) for windows of both forms.
#pragma once

#include "paged_row.hpp"
#include "paged_tile.hpp"

namespace svhip {

// Packed windows, which may be of either form: tile_grid workgroups for tiles, which take longest, then those of the
// row form, which fill the CUs as the tiles end. One launch for both: 24 windows, 6 of them chunks (head_dim 96,
// pages of 16, 335 MB) 110 us; the two kernels one after the other 116, and 18 us of host time for 16. Workgroups of
// both forms in turn, one tile's to one, two and four of rows: 122, 112 and 125 us, since a tile with a CU to share
// takes no less time.
template <int ST, bool WIN, int KS>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_mixed_kernel(PagedArgs a, int tile_grid, unsigned first_group) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef RowLds<ST, KS, 2> R;
  constexpr int kTile = TileLds<KS>::kBuffer;
  __shared__ __attribute__((aligned(16))) char s0[R::k0 > kTile ? R::k0 : kTile], s1[R::k1 > kTile ? R::k1 : kTile];
  __shared__ float s_ml[4][2][kRows];
  __shared__ __attribute__((aligned(16))) float s_scale[coded(ST) ? 2 : 1][4];
  __shared__ int s_odd;
  const int place = static_cast<int>(first_group + blockIdx.x);
  if (place < tile_grid) {
    tile_work<ST, WIN, false, KS>(a, place, s0, s1, &s_odd, s_scale);
  } else {
    row_work<ST, WIN, KS, 2>(a, place - tile_grid, s0, s1, s_ml);
  }
#endif
}

template <int ST, bool WIN, int KS>
void launch_mixed(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  in_launches(p.tile_grid + p.row_slots, [&](unsigned first, unsigned grid) {
    paged_mixed_kernel<ST, WIN, KS><<<grid, kPagedThreads, 0, s>>>(a, static_cast<int>(p.tile_grid), first);
  });
}

template <int ST, bool WIN>
void launch_paged_mixed(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  SVHIP_PAGED_WIDTH(launch_mixed, ST, WIN)
}

}  // namespace svhip
