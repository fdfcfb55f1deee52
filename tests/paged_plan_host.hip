// The plans of svhip_paged_attention on the host, by the kernels' own functions (tests/test_paged_plan.py).
#include "../streamvoxel_amd/csrc/paged_row.hpp"
#include "../streamvoxel_amd/csrc/paged_tile.hpp"

#include <vector>

namespace svhip {
void set_error(const char*, ...) {}
void clear_error() {}
}  // namespace svhip

using namespace svhip;

namespace {
// One thread that plans for all windows.
struct HostTeam {
  static constexpr int kSize = 1;
  __host__ __device__ int id() const { return 0; }
  __host__ __device__ float sum(float v) const { return v; }
};
}  // namespace

// out: places of tiles and their workgroups, places that no workgroup takes, slots that cut tiles use and that there are;
// the same of the row form but for the third.
extern "C" void plan_places(int64_t B, int64_t H, int64_t Hkv, int64_t N, const int32_t* cu, const int32_t* lengths, int64_t D,
                            int64_t max_pages, int64_t page, int fp8, int64_t* out) {
  const int row_most = fp8 ? kRowMostFp8 : kRowMost;
  const PagedPlan p = paged_plan(B, H, Hkv, N, cu != nullptr, D, max_pages * page, row_most);
  PagedArgs a{};
  a.tokens = Tokens{cu, B, N};
  a.pages = Pages{nullptr, 0, max_pages, 1, page_shift(page), lengths, nullptr};
  a.H = static_cast<int>(H);
  a.Hkv = static_cast<int>(Hkv);
  a.G = static_cast<int>(H / Hkv);
  a.row_most = row_most;
  const HostTeam team;
  for (int i = 0; i < 9; ++i) out[i] = 0;
  if (p.tiles && p.split) {
    int tiles, blocks;
    float total;
    const int each = tile_length(a, team, tiles, blocks, total);
    int64_t places = 0, slots = 0;
    for (int64_t c = 0; c < B; ++c) {
      tiles_of_window(a, c, tiles, blocks);
      const int64_t n = static_cast<int64_t>(tiles) * Hkv * tile_parts(blocks, each);
      places += n;
      slots += n > static_cast<int64_t>(tiles) * Hkv ? n : 0;
    }
    std::vector<char> taken(static_cast<size_t>(places));
    for (int64_t g = 0; g < p.tile_grid; ++g) {
      const int at = shared_place(static_cast<int>(g), static_cast<int>(places), each);
      if (at >= 0) ++taken[static_cast<size_t>(at)];
    }
    int64_t lost = 0;
    for (const char n : taken) lost += n == 1 ? 0 : 1;
    out[0] = places;
    out[1] = p.tile_grid;
    out[2] = lost;
    out[3] = slots;
    out[4] = p.tile_slots;
  }
  if (p.rows && p.row_parts) {
    int mine;
    const int each = row_length(a, team, 0, mine);
    for (int64_t c = 0; c < B; ++c) {
      const int64_t parts = row_parts(row_keys(a, c), each);
      out[5] += Hkv * parts;
      out[7] += parts > 1 ? Hkv * parts : 0;
    }
    out[6] = out[8] = p.row_slots;
  }
}
