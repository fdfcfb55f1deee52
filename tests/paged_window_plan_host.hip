// The plans of svhip_paged_window_attention on the host, by the kernels' own functions (tests/test_paged_window_plan.py).
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

// The key blocks that a tile of `count` tokens whose first is `i` walks, from the definition: those with a key that one of its
// tokens sees (counted over the first keys' blocks and the windows', which may be one run).
static int64_t walked(int64_t held, int64_t last, int64_t first, int64_t tokens, int64_t window, int64_t sinks) {
  int64_t n = 0;
  const int64_t top = last + first + tokens - 1;       // the last token's own key
  for (int64_t blk = 0; blk * kKB < held; ++blk) {
    const int64_t from = blk * kKB, to = from + kKB - 1;
    bool any = false;
    for (int64_t i = first; i < first + tokens && !any; ++i) {
      const int64_t p = last + i, low = p - window + 1;
      const int64_t end = p < held - 1 ? p : held - 1;
      any = (from <= end && to >= low) || (from < sinks && from <= end);
    }
    n += any ? 1 : 0;
  }
  (void)top;
  return n;
}

// out: as plan_places (paged_plan_host.hip), then tiles whose blocks are more than the plan's, and row-form windows whose
// parts do not hold the keys that they see.
extern "C" void window_places(int64_t B, int64_t H, int64_t Hkv, int64_t N, const int32_t* cu, const int32_t* lengths, int64_t D,
                              int64_t max_pages, int64_t page, int codes, int64_t window, int64_t sinks, int64_t* out) {
  const int row_most = codes ? kRowMostFp8 : kRowMost;
  const PagedPlan p = paged_plan(B, H, Hkv, N, cu != nullptr, D, window_keys(max_pages * page, window, sinks), row_most);
  const PagedPlan whole = paged_plan(B, H, Hkv, N, cu != nullptr, D, max_pages * page, row_most);
  PagedArgs a{};
  a.tokens = Tokens{cu, B, N};
  a.pages = Pages{nullptr, 0, max_pages, 1, page_shift(page), lengths, nullptr};
  a.H = static_cast<int>(H);
  a.Hkv = static_cast<int>(Hkv);
  a.G = static_cast<int>(H / Hkv);
  a.row_most = row_most;
  a.causal = true;
  a.window = static_cast<int>(window);
  a.sinks = static_cast<int>(sinks);
  const HostTeam team;
  for (int i = 0; i < 12; ++i) out[i] = 0;
  if (p.tiles && p.split) {
    int tiles, blocks;
    float total;
    const int each = tile_length<true>(a, team, tiles, blocks, total);
    int64_t places = 0, slots = 0;
    for (int64_t c = 0; c < B; ++c) {
      tiles_of_window<true>(a, c, tiles, blocks);
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
    const int each = row_length<true>(a, team, 0, mine);
    for (int64_t c = 0; c < B; ++c) {
      const int64_t parts = row_parts(row_keys<true>(a, c), each);
      out[5] += Hkv * parts;
      out[7] += parts > 1 ? Hkv * parts : 0;
    }
    out[6] = out[8] = p.row_slots;
  }
  out[9] = p.bytes() > whole.bytes() ? 1 : 0;
  for (int64_t c = 0; c < B; ++c) {
    int64_t first, count;
    window_tokens(a.tokens, c, first, count);
    if (count <= 0) continue;
    const int64_t held = held_keys(a.pages, c), last = lengths[c] - count;
    if (row_form(a, count)) {
      // Keys that are not walked are seen by none of the tokens.
      const int64_t keys = row_keys<true>(a, c), skipped = held - keys, from = sink_keys(static_cast<int>(sinks));
      if (skipped < 0 || (skipped > 0 && (from + skipped > (last - window + 1 < held ? last - window + 1 : held)))) ++out[11];
      continue;
    }
    int tiles, blocks;
    tiles_of_window<true>(a, c, tiles, blocks);
    for (int t = 0; t < tiles; t += tiles > 8 ? tiles / 4 : 1) {
      const int64_t i0 = static_cast<int64_t>(t) * kTileRows / a.G;
      int64_t i1 = ((t + 1) * static_cast<int64_t>(kTileRows) - 1) / a.G;
      i1 = i1 < count - 1 ? i1 : count - 1;
      if (walked(held, last, i0, i1 - i0 + 1, window, sinks) > blocks) ++out[10];
    }
  }
}
