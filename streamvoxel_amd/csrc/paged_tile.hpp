// The tile form of svhip_paged_attention (paged_attention.hip): windows of more than row_most rows.
#pragma once

#include "paged_attention.hpp"

namespace svhip {

// A window's tiles (0: the row form) and key blocks (0: no tokens).
__host__ __device__ __forceinline__ void tiles_of_window(const PagedArgs& a, int64_t c, int& tiles, int& blocks) {
  int64_t first, count;
  window_tokens(a.tokens, c, first, count);
  tiles = row_form(a, count) ? 0 : static_cast<int>(cdiv(count * a.G, kTileRows));
  const int held = static_cast<int>((held_keys(a.pages, c) + kKB - 1) / kKB);  // (read beside the borders, not after them)
  blocks = count > 0 ? held : 0;
}

__host__ __device__ __forceinline__ int tile_parts(int blocks, int length) {
  return blocks > length ? (blocks - 1) / length + 1 : 1;
}

// Even windows that fill the chip by themselves (split false): XCD id % 8 takes every 8th (window, key head) with all
// its tiles, so that its L2 reads the keys once; the windows longest first (up to 64 of them), and every other round
// of an XCD's CUs in reverse, which evens out the CUs' sums.
__device__ __forceinline__ PagedItem whole_item(const PagedArgs& a, int place) {
  const int seq = place >> 3, q_tiles = a.q_tiles;
  int k = seq / q_tiles;
  const int units = static_cast<int>(a.tokens.B * a.Hkv), per_round = kCusPerXcd / q_tiles;
  if (kCusPerXcd % q_tiles == 0 && per_round > 1) {
    const int round = k / per_round;
    if ((round & 1) && round < units / kXcds / per_round) k = (2 * round + 1) * per_round - 1 - k;
  }
  const int unit = k * kXcds + (place & 7);
  PagedItem item{-1, 0, 0, 1, seq - seq / q_tiles * q_tiles, q_tiles, 0, 0};
  if (unit >= units) return item;
  const int rank = unit / a.Hkv;
  item.kvh = unit - rank * a.Hkv;
  item.b = rank;
  if (a.tokens.B > 1 && a.tokens.B <= 64) {
    const int lane = threadIdx.x & 63, B = static_cast<int>(a.tokens.B);
    const int mine = lane < B ? static_cast<int>(held_keys(a.pages, lane)) : -1;
    int place = 0;
    for (int o = 0; o < B; ++o) {
      const int other = __builtin_amdgcn_readlane(mine, o);
      place += other > mine || (other == mine && o < lane) ? 1 : 0;
    }
    item.b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < B && place == rank));
  }
  return item;
}

// Otherwise the tiles stand one window after the other. Fewer than kTileTarget of them share out their keys: into
// parts of the least number of blocks, kTileLeast at least, for which the parts are at most kTileTarget and run side
// by side; at most kTileBeside where the row form's windows read half as many blocks or more (they then have the
// other half of every CU: a block takes about 1 us of either's CU; 24 mixed windows 101 us for 110). kUncut: no
// parts. `tiles`, `blocks`: of the team's own window; `total`: the tiles.
template <typename Team>
__host__ __device__ __forceinline__ int tile_length(const PagedArgs& a, const Team& team, int& tiles, int& blocks, float& total) {
  const float Hkv = static_cast<float>(a.Hkv);
  float units = 0.f, work = 0.f, beside = 0.f;
  tiles = blocks = 0;
  for (int64_t c = team.id(); c < a.tokens.B; c += Team::kSize) {
    tiles_of_window(a, c, tiles, blocks);
    units += static_cast<float>(tiles);
    work += static_cast<float>(tiles) * static_cast<float>(blocks);
    beside += tiles == 0 ? static_cast<float>(blocks) : 0.f;
  }
  total = team.sum(units) * Hkv;
  if (total == 0.f) return kUncut;
  work = team.sum(work) * Hkv;
  const int target = 2.f * Hkv * team.sum(beside) >= work ? kTileBeside : kTileTarget;
  const int own_tiles = tiles, own_blocks = blocks;
  // As many tiles or more: only those of windows longer than 1.5 times an equal share are cut, and their parts alone
  // counted (64 windows of 40 queries, 8 heads of 128, 1024 keys and one of 60 000: 204 us, uncut 1157).
  const bool full = total >= static_cast<float>(target);
  if (full) work *= 1.5f;
  return part_length(a, team, work, target, 1, kTileLeast, [&](int c, int length) __attribute__((always_inline)) {
    int t = own_tiles, n = own_blocks;
    if (a.tokens.B > Team::kSize) tiles_of_window(a, c, t, n);
    return full && n <= length ? 0.f : Hkv * static_cast<float>(t) * static_cast<float>(tile_parts(n, length));
  });
}

// An XCD takes a run of consecutive places of parts, so that the tiles of a part meet in its L2.
__host__ __device__ __forceinline__ int shared_place(int place, int total, int each) {
  if (each == kUncut) return place < total ? place : -1;
  const int run = (total + kXcds - 1) / kXcds, at = (place & 7) * run + (place >> 3);
  return (place >> 3) < run && at < total ? at : -1;
}

__device__ __forceinline__ PagedItem shared_item(const PagedArgs& a, int place, int& each) {
  const PagedItem none{-1, 0, 0, 1, 0, 1, 0, 0};
  if (a.running) {
    const int4 sums = a.plan[a.tokens.B];
    each = sums.w;
    const int at = shared_place(place, sums.y, each);
    return at < 0 ? none : planned_item(a, at, &a.running->y);
  }
  const int Hkv = a.Hkv;
  int tiles, blocks;
  float total;
  each = __builtin_amdgcn_readfirstlane(tile_length(a, WaveTeam{}, tiles, blocks, total));
  if (total == 0.f) return none;
  const int parts = tile_parts(blocks, each);
  int sum;
  wave_prefix(tiles * Hkv * parts, sum);
  const int at = shared_place(place, sum, each);
  return at < 0 ? none : item_at(Hkv, at, tiles, parts);
}

// Two buffers of a block of K and a block of V.
template <int KS>
struct TileLds {
  static constexpr int kSubBytes = kKB * kRow * 2, kTileBytes = Width<tiles_of(KS)>::kSubTiles * kSubBytes;
  static constexpr int kBuffer = 2 * kTileBytes;
};

#if defined(__HIP_DEVICE_COMPILE__)

template <bool FP8, bool WHOLE, int KS>
__device__ __forceinline__ void tile_work(const PagedArgs& a, int place, char* s0, char* s1, int* s_odd) {
  constexpr int DT = tiles_of(KS), ES = FP8 ? 1 : 2;
  constexpr int kSubBytes = TileLds<KS>::kSubBytes, kTileBytes = TileLds<KS>::kTileBytes;
  char *sK0 = s0, *sV0 = s0 + kTileBytes, *sK1 = s1, *sV1 = s1 + kTileBytes;
  int each = kUncut;
  const PagedItem item = a.split ? shared_item(a, place, each) : whole_item(a, place);
  const int b = __builtin_amdgcn_readfirstlane(item.b);
  if (b < 0) return;
  const int qt = __builtin_amdgcn_readfirstlane(item.qt), kvh = __builtin_amdgcn_readfirstlane(item.kvh);
  const int part = __builtin_amdgcn_readfirstlane(item.part);
  const Window w = window_at(a, b);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
  const int r0 = qt * kTileRows, r = r0 + wave * kRows + col, rows = w.count * a.G;
  const int keys = __builtin_amdgcn_readfirstlane(tile_keys(a, w, qt));
  const int blocks = (keys + kKB - 1) / kKB;
  const int count = blocks > each ? (blocks - 1) / each + 1 : 1;
  if (a.split && !a.running && part == 0 && kvh == 0 && qt == 0 && threadIdx.x == 0) {
    a.plan[b] = make_int4(item.first, item.parts, each, item.tiles);
  }
  if (part >= count || (count > 1 && item.slot >= a.tile_slots)) return;  // (borders not ascending)
  const int blk0 = part == 0 ? 0 : part * each, blk1 = blocks - blk0 > each ? blk0 + each : blocks;

  Rows<KS> s;
  load_rows<KS>(a, w, b, kvh, r, s);
  // Where the lane's row goes, found now: what it takes would stay in scalar registers through the loop.
  const bool cut = count > 1;
  const int D = a.D;
  void* dest = nullptr;
  if (r < rows) {
    const int i = r / a.G;
    dest = cut ? static_cast<void*>(a.tile_part + (static_cast<int64_t>(item.slot) * kTileRows + (r - r0)) * (a.D + 2))
               : static_cast<void*>(a.o + row_at(a, w, b, kvh * a.G + (r - i * a.G), i, a.so_b, a.so_h, a.so_n));
  }
  // K rows: lane (col, hh) takes logical chunk 2 k + hh of rows col and 32 + col, which share their swizzle.
  uint32_t rd[4], rvt[DT];
#pragma unroll
  for (int k = 0; k < 4; ++k) rd[k] = static_cast<uint32_t>(col * kRow * 2 + swz(col, 2 * k + hh) * 16);
  v_offsets<DT>(rvt);
  const Source ks = k_source<ES>(a, kvh), vs = v_source<ES>(a, kvh);
  const int32_t* row = a.pages.table + b * a.pages.st_b;
  // The wave's rows see every key up to `all` and none past `any`.
  const int wr0 = r0 + wave * kRows, wr1 = wr0 + kRows < rows ? wr0 + kRows : rows;
  const int all = __builtin_amdgcn_readfirstlane(wr0 < rows ? last_key(a, w, wr0 / a.G) : -1);
  const int any = __builtin_amdgcn_readfirstlane(wr0 < rows ? last_key(a, w, (wr1 - 1) / a.G) : -1);
  // Every row of the tile sees the keys up to `seen`; blocks past it are seen in part (clean_values).
  const int seen = __builtin_amdgcn_readfirstlane(last_key(a, w, r0 / a.G));
  const int clean_from = seen + 1 < keys ? (seen + 1) / kKB : kUncut;

  // The wave stages rows 8 wave .. and 8 wave + 32 .. of a block: of one page (WHOLE), or of the 16 keys around each.
  constexpr int kGroup = WHOLE ? 64 : 16, kGroups = WHOLE ? 1 : 2;
  Staged<DT, FP8 ? 2 : 1> kst, vst;
  const int in_mask = (1 << a.pages.shift) - 1, row_bytes = D * ES;
  const int g0 = WHOLE ? 0 : 16 * (wave >> 1);
  Lane8 kl[2], vl[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    kl[i] = k_lane<ES>(a, 8 * wave + 32 * i, WHOLE ? 0 : g0 + 32 * i);
    vl[i] = v_lane<ES>(a, 8 * wave + 32 * i, WHOLE ? 0 : g0 + 32 * i);
  }
  int page[kGroups];
  auto find = [&](int kv0) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) page[g] = page_number(a, row, kv0 + g0 + 32 * g);
  };
  auto issue = [&](int kv0, char* sK, char* sV) __attribute__((always_inline)) {
    __amdgpu_buffer_rsrc_t kr, vr, ek, ev;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i < kGroups) {
        const int j = kv0 + g0 + 32 * i, in_page = j & in_mask;
        const int valid = valid_keys<kGroup>(a, keys, j, page[i]);
        kr = rows_of(ks.rows, ks.sp, ks.sr, page[i], in_page, valid, row_bytes);
        vr = rows_of(vs.rows, vs.sp, vs.sr, page[i], in_page, valid, row_bytes);
        if constexpr (FP8) {
          ek = rows_of(reinterpret_cast<const char*>(ks.exponents), ks.se, 1, page[i], in_page, valid, 1);
          ev = rows_of(reinterpret_cast<const char*>(vs.exponents), vs.se, 1, page[i], in_page, valid, 1);
        }
      }
      const int to = (8 * wave + 32 * i) * kRow * 2;
      stage_rows8<FP8, DT, kSubBytes>(kr, ek, kl[i], i, sK + to, kst);
      stage_rows8<FP8, DT, kSubBytes>(vr, ev, vl[i], i, sV + to, vst);
    }
  };
  auto commit = [&](char* sK, char* sV) __attribute__((always_inline)) {
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        commit_rows8<DT, kSubBytes>(kst, i, sK + (8 * wave + 32 * i) * kRow * 2);
        commit_rows8<DT, kSubBytes>(vst, i, sV + (8 * wave + 32 * i) * kRow * 2);
      }
    }
  };
  auto compute = [&](int kv0, const char* sK, const char* sV) __attribute__((always_inline)) {
    if (kv0 > any) return;
    f32x16_t x[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      bf16x8_t ka[KS];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        ka[k] = *reinterpret_cast<const bf16x8_t*>(sK + (k >> 2) * kSubBytes + rd[k & 3] + 32 * t * kRow * 2);
      }
      x[t] = scores<KS>(s, ka);
    }
    bound_scores<KS, 2>(s, x, a.scale_log2, kv0 + kKB - 1 > all, kv0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      bf16x8_t pb[2];
      weights_of<KS>(s, x[t], a.scale_log2, pb);
      add_values<KS, kSubBytes>(s, pb, sV + 32 * t * kRow * 2, rvt);
    }
  };
  if (blk0 < blk1) {
    if (threadIdx.x == 0) *s_odd = 0;
    find(kKB * blk0);
    issue(kKB * blk0, sK0, sV0);
    find(kKB * (blk0 + 1));
    commit(sK0, sV0);
    wait_vmem();
    __syncthreads();
    auto step = [&](int blk, char* cK, char* cV, char* nK, char* nV) __attribute__((always_inline)) {
      const bool more = blk + 1 < blk1;
      if (more) issue(kKB * (blk + 1), nK, nV);
      find(kKB * (blk + 2));
      if (blk >= clean_from) {
        if (clean_values(cV, kTileBytes, 16 * static_cast<int>(threadIdx.x), 16 * kPagedThreads)) *s_odd = 1;
        __syncthreads();
      }
      compute(kKB * blk, cK, cV);
      if (more) {
        commit(nK, nV);
        wait_vmem();
        __syncthreads();
      }
    };
    for (int blk = blk0; blk < blk1; blk += 2) {
      step(blk, sK0, sV0, sK1, sV1);
      if (blk + 1 < blk1) step(blk + 1, sK1, sV1, sK0, sV0);
    }
    if (clean_from < blk1 && *s_odd != 0) {
      add_odd_values<FP8, KS>(a, vs, row, kKB * (clean_from > blk0 ? clean_from : blk0),
                              kKB * blk1 < keys ? kKB * blk1 : keys, s);
    }
  }
  const float l = row_sum(s.l[0]);
  if (dest == nullptr) return;
  const float inv = s.last >= 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int j = 0; j < DT; ++j) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d0 = 32 * j + 8 * g + 4 * hh;
      if (d0 >= D) continue;
      const float4 o = make_float4(s.o[j][4 * g], s.o[j][4 * g + 1], s.o[j][4 * g + 2], s.o[j][4 * g + 3]);
      if (cut) {
        float2* slot = reinterpret_cast<float2*>(static_cast<float*>(dest) + d0);
        slot[0] = make_float2(o.x, o.y);
        slot[1] = make_float2(o.z, o.w);
      } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(dest) + d0) =
            make_uint2(bf16_pack2(o.x * inv, o.y * inv), bf16_pack2(o.z * inv, o.w * inv));
      }
    }
  }
  if (cut && hh == 0) *reinterpret_cast<float2*>(static_cast<float*>(dest) + D) = make_float2(s.m, l);
}

#endif  // __HIP_DEVICE_COMPILE__

}  // namespace svhip
