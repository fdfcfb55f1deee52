// svhip_paged_attention: attention of the windows' new tokens over their keys and values in a paged cache
// (paged.hpp), bf16 matrix cores, fp32 sums.
//
// A key head's queries are its G heads' rows of every token, row r = token r / G, head r % G; a wave takes 32 of them
// as the columns of S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_32x32x16_bf16), so that the softmax of a row stays in
// two lanes and P^T leaves the first product in the second one's operand layout (K rows lie in LDS under sigma_row;
// xattn_kernel.hpp). V rows lie as they come and are read transposed (ds_read_b64_tr_b16). Two forms of work:
//   * windows of more than kRowMost rows (tile, paged_tile.hpp): a workgroup takes 128 rows, 32 a wave; the 4 waves
//     stage each block of 64 keys together, the next one in flight while the current one is computed. Bound: the
//     matrix cores and the exponentials, which overlap little. Measured: 8 windows x 1024 queries, 1552 to 9744 keys,
//     12 x 64 (153 GFLOP) 195 us, 785 TFLOP/s (e4m3 209); 4 causal chunks of 512, 16 heads to 4 of 128, up to 16 384
//     keys (241 GFLOP) 279 us, 12 of them the join (e4m3 298); a causal prompt of 8192 tokens, 16 heads of 64 208 us
//     (e4m3 235), of 128 345 (395); 32 queries of 64 windows over 2048 to 4096 keys, 8 heads of 64 86 us (e4m3 75).
//   * windows of up to kRowMost rows, single tokens among them (row, paged_row.hpp): the 4 waves share the rows and
//     split the keys, each staging its own blocks of 32 keys in its own LDS; no barrier until the waves' sums are
//     joined. Bound: HBM. Measured: 64 tokens over 1.18 GB of keys 216 us, 5.4 TB/s; over 754 MB of e4m3 pages 148
//     us, 5.1 TB/s; one token over 30 MB 9.1 us, a chain of loads. One wave a row of its own, with shuffles instead
//     of the products, took 14.9 ms.
// Packed windows may be of both (paged_mixed.hip). Either form may cut a window's keys into parts for several
// workgroups; a part leaves O, its running maximum and its sum in fp32 and paged_join_kernel joins them in order (4.5
// us for one token, 12 for 34 MB of parts). What is cut is planned on the device, where the lengths are: by every
// workgroup for up to 64 windows, one a lane, else by paged_plan_kernel (6.6 us; every workgroup for itself: 4096
// windows of one token 2348 us for 491).
//
// Staging: 16 keys lie in one page (pages are of 16 keys or more), so the wave's load of 8 rows has one base, a
// scalar buffer descriptor whose bound is the number of its keys that exist: keys past the window's end, bad pages
// and the chunks past head_dim read as zeros and nothing is read outside a page.
#include "paged_row.hpp"
#include "paged_tile.hpp"

namespace svhip {

// The plan of more windows than a wave has lanes, by one workgroup: part lengths, and every window's places in the
// lists of row-form parts and of tiles. (Up to 64 windows a workgroup's own plan is one load a lane, less than this
// launch.)
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedArgs a, bool rows, bool tiles) {
  __shared__ float of_wave[kPlanThreads / 64];
  __shared__ int4 counts[kPlanThreads / 64];
  const BlockTeam team{of_wave};
  const int tid = static_cast<int>(threadIdx.x), Hkv = a.Hkv;
  int unused, more;
  float total;
  const int row_each = rows && a.row_part ? row_length(a, team, 0, unused) : kUncut;
  const int tile_each = tiles ? tile_length(a, team, unused, more, total) : kUncut;
  int2 at = make_int2(0, 0), slot = at;
  int cut = 0;  // 1: windows of the row form, 2: tiles
  for (int64_t c0 = 0; c0 < a.tokens.B; c0 += kPlanThreads) {
    const int64_t c = c0 + tid;
    int row = 0, tile = 0, parts = 1, t = 0, blocks = 0;
    if (c < a.tokens.B) {
      if (tiles) tiles_of_window(a, c, t, blocks);
      if (t > 0) {
        parts = tile_parts(blocks, tile_each);
        tile = t * Hkv * parts;
      } else if (rows) {
        parts = row_parts(row_keys(a, c), row_each);
        row = Hkv * parts;
      }
    }
    cut |= parts > 1 ? (t > 0 ? 2 : 1) : 0;
    const int row_n = parts > 1 ? row : 0, tile_n = parts > 1 ? tile : 0;
    int4 sums;  // of places, then of slots
    int4 before = make_int4(wave_prefix(row, sums.x), 0, 0, 0);
    before.y = wave_prefix(tile, sums.y);
    before.z = wave_prefix(row_n, sums.z);
    before.w = wave_prefix(tile_n, sums.w);
    if ((tid & 63) == 0) counts[tid >> 6] = sums;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPlanThreads / 64; ++i) {
      if (i == tid >> 6) {
        before.x += at.x;
        before.y += at.y;
        before.z += slot.x;
        before.w += slot.y;
      }
      at.x += counts[i].x;
      at.y += counts[i].y;
      slot.x += counts[i].z;
      slot.y += counts[i].w;
    }
    if (c < a.tokens.B) {
      a.plan[c] = t > 0 ? make_int4(before.w, parts, tile_each, t) : make_int4(before.z, parts, row_each, 1);
      a.running[c] = make_int2(before.x + row, before.y + tile);
    }
    __syncthreads();
  }
  const bool row_cut = __syncthreads_or(cut & 1), tile_cut = __syncthreads_or(cut & 2);
  if (tid == 0) a.plan[a.tokens.B] = make_int4(at.x, at.y, row_cut ? row_each : kUncut, tile_cut ? tile_each : kUncut);
}

// The parts of a row joined in order. kGroups 32-lane groups a row, 4 elements a lane: one group where the rows are
// many (it has kAhead parts in flight), all 8 of the workgroup where they are few (every part of up to 64 in flight
// at once).
constexpr int kAhead = 8;

template <int kGroups>
__global__ __launch_bounds__(kPagedThreads) void paged_join_kernel(PagedArgs a, unsigned first_group) {
  __shared__ float4 s_o[kGroups > 1 ? kGroups : 1][32];
  __shared__ float2 s_ml[kGroups > 1 ? kGroups : 1];
  if (a.running) {
    const int4 sums = a.plan[a.tokens.B];
    if (sums.z == kUncut && sums.w == kUncut) return;  // no parts
  }
  const int group = threadIdx.x / 32, d0 = 4 * (threadIdx.x % 32);
  const unsigned place = first_group + blockIdx.x;
  const int id = static_cast<int>(kGroups > 1 ? place : place * (kPagedThreads / 32) + group);
  const int total = static_cast<int>(a.tokens.cu ? a.tokens.N : a.tokens.B * a.tokens.N);
  const int token = id / a.H, h = id - token * a.H;
  int64_t b = -1;
  if (token < total && !a.tokens.cu) b = token / static_cast<int>(a.tokens.N);
  if (token < total && a.tokens.cu && a.tokens.B > 64) b = window_of(a.tokens, token);
  if (a.tokens.cu && a.tokens.B <= 64) {
    // Up to 64 borders are read at once; a wave has the tokens of its two groups.
    const int lane = threadIdx.x & 63, B = static_cast<int>(a.tokens.B);
    const int from = a.tokens.cu[0], to = lane < B ? a.tokens.cu[1 + lane] : INT_MAX;
    const int other = __shfl(token, lane ^ 32);
    const int n0 = __builtin_popcountll(__builtin_amdgcn_ballot_w64(to <= (lane < 32 ? token : other)));
    const int n1 = __builtin_popcountll(__builtin_amdgcn_ballot_w64(to <= (lane < 32 ? other : token)));
    const int n = lane < 32 ? n0 : n1;
    if (token < total && token >= from && n < B) b = n;
  }
  // With several groups a row every one of them takes the same way to the barrier.
  if (b < 0) return;
  const int4 plan = a.plan[b];
  const Window w = window_at(a, b);
  if (w.count <= 0) return;
  if (token < w.first || token - w.first >= w.count) return set_bad(a.pages);  // borders not ascending
  const int i = static_cast<int>(token - w.first), kvh = h / a.G, r = i * a.G + (h - kvh * a.G);
  const float* slot;
  int64_t step;
  int count;
  if (row_form(a, w.count)) {
    if (!a.row_part) return;
    count = plan.y;
    if (plan.x < 0 || count < 0 || plan.x + static_cast<int64_t>(a.Hkv) * count > a.row_slots) {
      return set_bad(a.pages);  // borders not ascending
    }
    slot = a.row_part + (static_cast<int64_t>(plan.x + kvh * count) * a.slot_rows + r) * (a.D + 2);
    step = static_cast<int64_t>(a.slot_rows) * (a.D + 2);
  } else {
    if (!a.split) return;
    const int qt = r / kTileRows, blocks = (tile_keys(a, w, qt) + kKB - 1) / kKB;
    const int each = plan.z, tiles = plan.w;
    if (each < 1) return set_bad(a.pages);
    count = blocks > each ? (blocks - 1) / each + 1 : 1;
    if (count < 2) return;
    if (plan.x < 0 || plan.y < count || plan.y > a.tile_slots || tiles <= qt || tiles > a.tile_slots ||
        plan.x + static_cast<int64_t>(a.Hkv) * plan.y * tiles > a.tile_slots) {
      return set_bad(a.pages);
    }
    const int64_t first = static_cast<int64_t>(plan.x + kvh * plan.y * tiles + qt) * kTileRows;
    slot = a.tile_part + (first + (r - qt * kTileRows)) * (a.D + 2);
    step = static_cast<int64_t>(tiles) * kTileRows * (a.D + 2);
  }
  if (count < 2) return;
  float m = kNoMax, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  const int e0 = d0 < a.D ? d0 : 0;
  for (int p0 = kGroups > 1 ? group : 0; p0 < count; p0 += kAhead * kGroups) {
    float2 ml[kAhead], oa[kAhead], ob[kAhead];
#pragma unroll
    for (int p = 0; p < kAhead; ++p) {  // the last part again behind the end: no branch around the loads
      const int at = p0 + p * kGroups;
      const float* from = slot + (at < count ? at : count - 1) * step;
      ml[p] = *reinterpret_cast<const float2*>(from + a.D);
      oa[p] = *reinterpret_cast<const float2*>(from + e0);
      ob[p] = *reinterpret_cast<const float2*>(from + e0 + 2);
    }
#pragma unroll
    for (int p = 0; p < kAhead; ++p) {
      if (p0 + p * kGroups >= count) break;
      const float mn = fmaxf(m, ml[p].x), x = __builtin_amdgcn_exp2f(m - mn), y = __builtin_amdgcn_exp2f(ml[p].x - mn);
      m = mn;
      l = join_value(l, ml[p].y, x, y);
      o[0] = join_value(o[0], oa[p].x, x, y);
      o[1] = join_value(o[1], oa[p].y, x, y);
      o[2] = join_value(o[2], ob[p].x, x, y);
      o[3] = join_value(o[3], ob[p].y, x, y);
    }
  }
  if constexpr (kGroups > 1) {
    s_o[group][threadIdx.x % 32] = make_float4(o[0], o[1], o[2], o[3]);
    if (threadIdx.x % 32 == 0) s_ml[group] = make_float2(m, l);
    __syncthreads();
    if (group > 0) return;
    for (int g = 1; g < kGroups; ++g) {
      const float2 ml = s_ml[g];
      const float4 og = s_o[g][threadIdx.x];
      const float mn = fmaxf(m, ml.x), x = __builtin_amdgcn_exp2f(m - mn), y = __builtin_amdgcn_exp2f(ml.x - mn);
      m = mn;
      l = join_value(l, ml.y, x, y);
      o[0] = join_value(o[0], og.x, x, y);
      o[1] = join_value(o[1], og.y, x, y);
      o[2] = join_value(o[2], og.z, x, y);
      o[3] = join_value(o[3], og.w, x, y);
    }
  }
  if (d0 >= a.D) return;
  const float inv = last_key(a, w, i) >= 0 ? 1.f / l : 0.f;
  uint16_t* out = a.o + row_at(a, w, b, h, i, a.so_b, a.so_h, a.so_n);
  *reinterpret_cast<uint2*>(out + d0) = make_uint2(bf16_pack2(o[0] * inv, o[1] * inv), bf16_pack2(o[2] * inv, o[3] * inv));
}

// Rows up to which a row has a workgroup of its own (one token, 12 rows: 15.8 us, 25.7 without; 64 tokens, 1024 rows:
// 217.6 and 222.9; 32 768 rows in two parts: 323 with, 281 without; 16 304 rows 116 and 104).
constexpr int64_t kJoinFew = 4096;

}  // namespace svhip

using namespace svhip;

extern "C" size_t svhip_paged_attention_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t N, int packed,
                                                        int64_t D, int64_t max_keys) {
  if (B < 1 || B >= 1ll << 31 || Hkv < 1 || H < 1 || H > 1 << 20 || H % Hkv != 0 || N < 1 || N >= 1ll << 31 ||
      N * H >= 1ll << 40 || D < 1 || D > kMaxPagedDim || max_keys < 0 || max_keys > 1ll << 30) {
    return 0;
  }
  const size_t bf16 = paged_plan(B, H, Hkv, N, packed != 0, D, max_keys, kRowMost).bytes();
  const size_t fp8 = paged_plan(B, H, Hkv, N, packed != 0, D, max_keys, kRowMostFp8).bytes();
  return bf16 > fp8 ? bf16 : fp8;
}

extern "C" int svhip_paged_attention(const svhip_paged_cache* cache, const svhip_paged_attention_args* args,
                                     void* stream) {
  const char* name = "svhip_paged_attention";
  clear_error();
  if (const int rc = check_cache(name, cache)) return rc;
  SVHIP_REQUIRE(args, "%s: null arguments", name);
  const svhip_paged_cache& pc = *cache;
  const svhip_paged_attention_args& c = *args;
  const int64_t B = pc.windows, H = c.H, Hkv = pc.heads, N = c.N, D = pc.head_dim;
  SVHIP_REQUIRE(H >= 0 && H <= 1 << 20 && N >= 0 && N < (1ll << 31) && N * H < (1ll << 40), "%s: bad sizes", name);
  SVHIP_REQUIRE(Hkv >= 1 && H % Hkv == 0, "%s: %lld heads do not share %lld key heads evenly", name, (long long)H,
                (long long)Hkv);
  const float scale = static_cast<float>(c.scale);
  SVHIP_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", name);
  if (B == 0 || H == 0 || N == 0) return SVHIP_OK;
  if (const int rc = check_pool(name, pc)) return rc;
  SVHIP_REQUIRE(c.q && c.out, "%s: null pointer", name);
  const int64_t even = c.cu_queries ? 0 : B;
  SVHIP_REQUIRE(rows_on(8, c.q, even, H, N, c.sq_b, c.sq_h, c.sq_n), "%s: query rows must start on 16-byte boundaries", name);
  SVHIP_REQUIRE(rows_on(4, c.out, even, H, N, c.so_b, c.so_h, c.so_n),
                "%s: rows of out must start on 8-byte boundaries", name);
  const bool fp8 = pc.kv_dtype == SVHIP_FP8_E4M3;
  const int row_most = fp8 ? kRowMostFp8 : kRowMost;
  const PagedPlan p = paged_plan(B, H, Hkv, N, c.cu_queries != nullptr, D, pc.max_pages * pc.page_size, row_most);
  SVHIP_REQUIRE(p.bytes() == 0 || (c.workspace && c.workspace_bytes >= static_cast<int64_t>(p.bytes()) &&
                                   reinterpret_cast<uintptr_t>(c.workspace) % 16 == 0),
                "%s: workspace too small or misaligned (%lld < %zu bytes)", name, (long long)c.workspace_bytes, p.bytes());
  const int64_t rows = (c.cu_queries ? N : B * N) * H, join = cdiv(rows, kPagedThreads / 32);
  SVHIP_REQUIRE(p.row_slots + p.tile_grid < (1ll << 31) && rows < (1ll << 31) - kPagedThreads &&
                    N * (H / Hkv) < (1ll << 31) - kPagedThreads, "%s: sizes too large", name);
  const int64_t es = fp8 ? 1 : 2;
  float* const part = static_cast<float*>(c.workspace);
  int4* const plan = reinterpret_cast<int4*>(part + p.row_floats + p.tile_floats);
  const PagedArgs a{static_cast<const uint16_t*>(c.q), pc.k_pages, pc.v_pages, pc.k_exponents, pc.v_exponents,
                    static_cast<uint16_t*>(c.out), Tokens{c.cu_queries, B, N}, pages_of(pc),
                    static_cast<int>(H), static_cast<int>(Hkv), static_cast<int>(H / Hkv), static_cast<int>(D), c.sq_b,
                    c.sq_h, c.sq_n, pc.sk_h, pc.sv_h, pc.sek_h, pc.sev_h, c.so_b, c.so_h, c.so_n,
                    static_cast<uint32_t>(pc.sk_p * es), static_cast<uint32_t>(pc.sk_r * es),
                    static_cast<uint32_t>(pc.sv_p * es), static_cast<uint32_t>(pc.sv_r * es),
                    static_cast<uint32_t>(pc.sek_p), static_cast<uint32_t>(pc.sev_p), c.causal != 0, scale * kLog2e,
                    row_most, p.q_tiles, p.split, static_cast<int>(p.row_slots), static_cast<int>(p.tile_slots),
                    static_cast<int>(p.slot_rows), p.row_parts ? part : nullptr, part + p.row_floats,
                    p.plan_windows ? plan : nullptr, p.planned ? reinterpret_cast<int2*>(plan + B + 1) : nullptr};
  hipStream_t s = as_stream(stream);
  if (p.planned) paged_plan_kernel<<<1, kPlanThreads, 0, s>>>(a, p.rows, p.tiles);
  if (p.rows && p.tiles) {
    launch_paged_mixed(a, p, fp8, s);
  } else if (p.rows) {
    launch_paged_rows(a, p, fp8, s);
  } else {
    launch_paged_tiles(a, p, fp8, pc.page_size >= kWholePages, s);
  }
  if (p.plan_windows) {
    if (rows <= kJoinFew) {
      paged_join_kernel<8><<<static_cast<unsigned>(rows), kPagedThreads, 0, s>>>(a, 0u);
    } else {
      in_launches(join, [&](unsigned first, unsigned grid) {
        paged_join_kernel<1><<<grid, kPagedThreads, 0, s>>>(a, first);
      });
    }
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
