// The row form of svhip_paged_attention (paged_attention.hip): windows of up to row_most rows, single tokens among
// them.
#pragma once

#include <type_traits>

#include "paged_attention.hpp"

namespace svhip {

[[maybe_unused]] constexpr int kRowKeys = 32;  // keys of a half of a wave's block

// Keys of window c that its tokens see, or -1: not of this form.
template <bool WIN = false>
__host__ __device__ __forceinline__ int row_keys(const PagedArgs& a, int64_t c) {
  int64_t first, count;
  window_tokens(a.tokens, c, first, count);
  const int held = static_cast<int>(held_keys(a.pages, c));  // (read beside the borders, not after them)
  if (!(count > 0 && row_form(a, count))) return -1;
  if constexpr (WIN) return held - left_out(a.sinks, first_key(a.window, a.pages.lengths[c] - count, held, 0));
  return held;
}
__host__ __device__ __forceinline__ int row_parts(int keys, int length) {
  return keys < 0 ? 0 : (keys > length ? (keys - 1) / length + 1 : 1);
}

// The length of a part: the least, a multiple of kRowLeast (4 waves' blocks), for which the parts are at most
// kRowTarget more than the (window, key head) pairs; kUncut if there are no places from `place` on. `mine`: keys of
// the team's own window.
template <bool WIN = false, typename Team>
__host__ __device__ __forceinline__ int row_length(const PagedArgs& a, const Team& team, int place, int& mine) {
  float keys = 0.f, units = 0.f;
  mine = -1;
  for (int64_t c = team.id(); c < a.tokens.B; c += Team::kSize) {
    mine = row_keys<WIN>(a, c);
    keys += mine > 0 ? static_cast<float>(mine) : 0.f;
    units += mine >= 0 ? 1.f : 0.f;
  }
  const float Hkv = static_cast<float>(a.Hkv);
  keys = team.sum(keys) * Hkv;
  units = team.sum(units) * Hkv;
  // (At most that many parts; a little more, since the sum of the keys is rounded.)
  if (static_cast<float>(place) > units + keys * (1.01f / kRowLeast)) return kUncut;
  const int own = mine;
  return part_length(a, team, keys, static_cast<int>(units) + kRowTarget, kRowLeast, kRowLeast,
                     [&](int c, int length) __attribute__((always_inline)) {
                       const int n = a.tokens.B <= Team::kSize ? own : row_keys<WIN>(a, c);
                       return Hkv * static_cast<float>(row_parts(n, length));
                     });
}

// The lengths are on the device, so the workgroups form the plan themselves, or read it.
template <bool WIN>
__device__ __forceinline__ PagedItem row_item(const PagedArgs& a, int place, int& each) {
  const int Hkv = a.Hkv;
  if (!a.row_part) {
    const int b = place / Hkv;
    return PagedItem{b < a.tokens.B ? b : -1, place - b * Hkv, 0, 1, 0, 1, 0, 0};
  }
  if (a.running) {
    const int4 sums = a.plan[a.tokens.B];
    each = sums.z;
    if (place >= sums.x) return PagedItem{-1, 0, 0, 1, 0, 1, 0, 0};
    return planned_item(a, place, &a.running->x);
  }
  int mine;
  each = __builtin_amdgcn_readfirstlane(row_length<WIN>(a, WaveTeam{}, place, mine));
  const int parts = row_parts(mine, each);
  return item_at(Hkv, place, parts > 0 ? 1 : 0, parts);
}

// A wave takes every 4th block of 32 keys of its part (codes up to head_dim 64: of 64 keys, as many bytes). K rows go
// straight from memory to the A operands, a lane its own key's chunks, the next block's while the current one's
// softmax and second product run; V rows go through the wave's LDS, since they are read transposed. Its LDS: V of the
// four waves, bf16 two blocks of each; O of them at the end, 32 DT x 32 floats each, of the first `kFirst` in the one
// buffer and of the others in the other.
template <int ST, int KS, int kFirst>
struct RowLds {
  static constexpr bool kCodes = coded(ST);
  static constexpr int kHalves = kCodes && KS <= 4 ? 2 : 1, kKeys = kRowKeys * kHalves;  // of a wave's block
  static constexpr int kSubBytes = kKeys * kRow * 2, kTileBytes = Width<tiles_of(KS)>::kSubTiles * kSubBytes;
  static constexpr int kWaveO = 32 * tiles_of(KS) * kRows;
  static constexpr int kO0 = kFirst * kWaveO * 4, kO1 = (4 - kFirst) * kWaveO * 4, kV = 4 * kTileBytes;
  static constexpr int k0 = kV > kO0 ? kV : kO0, k1 = kCodes ? (kO1 > 16 ? kO1 : 16) : (kV > kO1 ? kV : kO1);
};

#if defined(__HIP_DEVICE_COMPILE__)

template <int ST, bool WIN, int KS, int kFirst>
__device__ __forceinline__ void row_work(const PagedArgs& a, int place, char* sV0, char* sV1, float (*s_ml)[2][kRows]) {
  constexpr int DT = tiles_of(KS), ES = bytes_of(ST);
  constexpr bool kCodes = coded(ST);
  typedef RowLds<ST, KS, kFirst> L;
  constexpr int kHalves = L::kHalves, kKeys = L::kKeys, kSubBytes = L::kSubBytes, kTileBytes = L::kTileBytes;
  constexpr int kWaveO = L::kWaveO;
  const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int each = kUncut;
  const PagedItem item = row_item<WIN>(a, place, each);
  const int b = __builtin_amdgcn_readfirstlane(item.b);
  if (b < 0) return;
  const int kvh = __builtin_amdgcn_readfirstlane(item.kvh), part = __builtin_amdgcn_readfirstlane(item.part);
  const int parts = __builtin_amdgcn_readfirstlane(item.parts);
  if (a.row_part && !a.running && part == 0 && kvh == 0 && threadIdx.x == 0) {
    a.plan[b] = make_int4(item.first, parts, each, 1);
  }
  const Window w = window_at(a, b);
  if (w.count <= 0 || !row_form(a, w.count)) return;  // (uncut windows stand by their numbers)
  const int rows = w.count * a.G;
  const int keys = __builtin_amdgcn_readfirstlane(w.keys);
  // From here on a key's place `kv` is among those that the tokens see, out_of_sight of them left out behind sink_end.
  int low = 0, low_last = 0, sink_end = 0, out_of_sight = 0;
  if constexpr (WIN) {
    low = __builtin_amdgcn_readfirstlane(first_key(a, w, 0));
    low_last = __builtin_amdgcn_readfirstlane(first_key(a, w, w.count - 1));
    sink_end = sink_keys(a.sinks);
    out_of_sight = left_out(a.sinks, low);
  }
  auto real = [&](int kv) __attribute__((always_inline)) { return WIN ? real_key(kv, sink_end, out_of_sight) : kv; };
  const int walked = keys - out_of_sight;
  const int k0 = part * each, k1 = walked - k0 > each ? k0 + each : walked;

  Rows<KS> s;
  load_rows<WIN, KS>(a, w, b, kvh, col, s);
  uint32_t rvt[DT];
  v_offsets<DT>(rvt);
  const Source ks = k_source<ES>(a, kvh), vs = v_source<ES>(a, kvh);
  const int32_t* row = a.pages.table + b * a.pages.st_b;
  const int all = __builtin_amdgcn_readfirstlane(last_key(a, w, 0));
  // Blocks that end past it are seen in part (clean_values), if a later token sees more.
  const int clean_from = all + 1 < keys ? all + 1 - kKeys : kUncut;
  // The keys from `at` on are not all in sight of the last token.
  auto past_low = [&](int at) __attribute__((always_inline)) { return WIN && at < low_last && at + kKeys > a.sinks; };
  bool odd = false;
  const int in_mask = (1 << a.pages.shift) - 1, D = a.D;
  constexpr int kGroup = 16, kGroups = kKeys / kGroup;  // keys that lie in one page for sure
  Lane8 vl[4 * kHalves];
#pragma unroll
  for (int i = 0; i < 4 * kHalves; ++i) vl[i] = v_lane<ST>(a, 8 * i, 16 * (i >> 1));
  // The lane's key of each half and its offsets in a K row (the last step's chunk may lie past head_dim: any chunk of
  // the row then, and zeros in its place, since an infinity there times Q's zeros would be NaN).
  const int own = sigma_row(col);
  const bool past = 16 * (KS - 1) + 8 * hh >= D;
  const int k_last = past ? -8 * hh * ES : 16 * (KS - 1) * ES;

  using KWord = typename std::conditional<kCodes, uint2, uint4>::type;
  KWord kw[kHalves][KS];
  // e4m3: the exponent of the lane's key of each half (the V rows' lie beside them); int8: one of every 16 keys, K and V.
  uint32_t ke[ST == kInt8 ? 2 * kHalves : (kCodes ? kHalves : 1)], ve[ST == kInt8 ? 2 * kHalves : 1];
  Staged<DT, kCodes ? 4 * kHalves : 1> vst;
  int page[kGroups], valid[kGroups];   // of the groups of the block to load
  bool broken = false;                 // the block in kw has keys on a bad page
  auto find = [&](int kv) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) page[g] = page_number(a, row, real(kv) + kGroup * g);
  };
  auto check = [&](int kv) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) valid[g] = valid_keys<kGroup>(a, k1, kv + kGroup * g, page[g]);
  };
  auto load_v = [&](int kv, char* to) __attribute__((always_inline)) {
    __amdgpu_buffer_rsrc_t r, er;
#pragma unroll
    for (int i = 0; i < 4 * kHalves; ++i) {
      const int g = 8 * i / kGroup;
      if (8 * i % kGroup == 0) {
        const int in_page = (real(kv) + kGroup * g) & in_mask;
        r = rows_of(vs.rows, vs.sp, vs.sr, page[g], in_page, valid[g], D * ES);
        if constexpr (ST == kE4m3) er = exponents_of<ST>(a, vs, page[g], in_page, valid[g]);
        if constexpr (ST == kInt8) {
          ve[g] = vs.exponents[static_cast<uint64_t>(static_cast<uint32_t>(page[g])) * vs.se + (in_page >> a.block_shift)];
        }
      }
      stage_rows8<ST, ST == kE4m3, DT, kSubBytes>(r, er, vl[i], i, to + 8 * i * kRow * 2, vst);
    }
  };
  // Keys that do not exist are never loaded (the group's first one is read instead, or page 0 where there is none):
  // their scores are masked, but for bad pages, which count as zeros.
  auto load_k = [&](int kv) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kHalves; ++t) {
      const int g = 2 * t;
      const int in0 = (real(kv) + 16 * g) & in_mask, in1 = (real(kv) + 16 * g + 16) & in_mask;
      const bool second = col >= 16;
      const uint32_t pg = second ? page[g + 1] : page[g], in = second ? in1 : in0;
      const int there = (own & 15) < (second ? valid[g + 1] : valid[g]) ? own & 15 : 0;
      const char* at = ks.rows + static_cast<uint64_t>(pg) * ks.sp + ((in + there) * ks.sr + 8 * hh * ES);
      if constexpr (ST == kE4m3) ke[t] = ks.exponents[static_cast<uint64_t>(pg) * ks.se + in + there];
      if constexpr (ST == kInt8) {
        ke[2 * t] = ks.exponents[static_cast<uint64_t>(static_cast<uint32_t>(page[g])) * ks.se + (in0 >> a.block_shift)];
        ke[2 * t + 1] = ks.exponents[static_cast<uint64_t>(static_cast<uint32_t>(page[g + 1])) * ks.se + (in1 >> a.block_shift)];
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        kw[t][k] = *reinterpret_cast<const KWord*>(at + (k < KS - 1 ? 16 * k * ES : k_last));
      }
    }
    broken = false;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) broken |= valid[g] == 0 && kv + kGroup * g < k1;
  };
  const int stride = 4 * kKeys;
  int kv = k0 + wave * kKeys;
  char *c0 = sV0 + wave * kTileBytes, *c1 = kCodes ? c0 : sV1 + wave * kTileBytes;
  if (kv < k1) {
    find(kv);
    check(kv);
    load_v(kv, c0);
    load_k(kv);
    int kvn = kv + stride;
    find(kvn);
    auto step = [&](char* cur, char* next) __attribute__((always_inline)) {
      const bool more = kvn < k1;
      if constexpr (kCodes) {
#pragma unroll
        for (int i = 0; i < 4 * kHalves; ++i) {
          commit_rows8<ST, true, DT, kSubBytes>(vst, i, ST == kInt8 ? ve[8 * i / kGroup] : vst.e[i], cur + 8 * i * kRow * 2);
        }
      }
      if (more) {
        check(kvn);
        load_v(kvn, next);
      }
      f32x16_t x[kHalves];
#pragma unroll
      for (int t = 0; t < kHalves; ++t) {
        bf16x8_t ka[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          if constexpr (kCodes) {
            ka[k] = __builtin_bit_cast(bf16x8_t, decode8<ST, false>(kw[t][k], ke[t]));
          } else {
            ka[k] = __builtin_bit_cast(bf16x8_t, kw[t][k]);
          }
        }
        if (past) ka[KS - 1] = bf16x8_t{};
        x[t] = scores<KS>(s, ka);
        if (__builtin_expect(broken, 0)) {
          // (The pages' numbers are the next block's by now: looked up again.)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int g = real(kv) + 32 * t + (i < 8 ? 0 : 16);
            if (static_cast<uint32_t>(page_number(a, row, g)) >= static_cast<uint32_t>(a.pages.pages)) x[t][i] = 0.f;
          }
        }
      }
      KeyScales<kHalves> f;
      if constexpr (ST == kInt8) {
#pragma unroll
        for (int i = 0; i < 2 * kHalves; ++i) f.of[i] = int8_power(ke[i]);
      }
      if (more) {
        load_k(kvn);
        find(kvn + stride);
      }
      // V of this block was on its way before K of this block, which has arrived: at most the next block's loads are
      // left.
      if constexpr (!kCodes) {
        if (more) {
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * Width<DT>::kSubTiles + KS) : "memory");
        } else {
          wait_vmem();
        }
      }
      const int key0 = real(kv);
      if (ST != kInt8 && (key0 > clean_from || past_low(key0))) {
        odd |= __builtin_amdgcn_ballot_w64(clean_values(cur, kTileBytes, 16 * lane, 16 * 64)) != 0ull;
      }
      bound_scores<ST, WIN, KS, kHalves>(a, s, x, f, key0 + kKeys - 1 > all || past_low(key0), key0);
#pragma unroll
      for (int t = 0; t < kHalves; ++t) {
        bf16x8_t pb[2];
        weights_of<ST, false, KS>(s, x[t], a.scale_log2, f.of + 2 * t, pb);
        add_values<KS, kSubBytes>(s, pb, cur + 32 * t * kRow * 2, rvt);
      }
      kv = kvn;
      kvn += stride;
    };
    while (kv < k1) {
      step(c0, c1);
      if (!kCodes && kv < k1) step(c1, c0);
    }
  }
  if (odd) {
    for (kv = k0 + wave * kKeys; kv < k1; kv += stride) {
      const int key0 = real(kv);
      if (key0 > clean_from || past_low(key0)) {
        add_odd_values<ST, WIN, KS>(a, vs, row, key0, key0 + (kKeys < k1 - kv ? kKeys : k1 - kv), s);
      }
    }
  }
  // The waves' sums joined, in order: O of wave w [head_dim][row].
  const float l = row_sum(s.l[0]);
  __syncthreads();
  float* so = reinterpret_cast<float*>(wave < kFirst ? sV0 : sV1) + (wave % kFirst) * kWaveO;
  if (hh == 0) {
    s_ml[wave][0][col] = s.m;
    s_ml[wave][1][col] = l;
  }
#pragma unroll
  for (int j = 0; j < DT; ++j) {
#pragma unroll
    for (int e = 0; e < 16; ++e) so[(32 * j + 8 * (e >> 2) + 4 * hh + (e & 3)) * kRows + col] = s.o[j][e];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * (D / 2); e += kPagedThreads) {
    const int rr = e / (D / 2), d = 2 * (e - rr * (D / 2));
    float m = s_ml[0][0][rr];
#pragma unroll
    for (int x = 1; x < 4; ++x) m = fmaxf(m, s_ml[x][0][rr]);
    float total = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = __builtin_amdgcn_exp2f(s_ml[x][0][rr] - m);
      const float* from = reinterpret_cast<const float*>(x < kFirst ? sV0 : sV1) + (x % kFirst) * kWaveO;
      total = __builtin_fmaf(s_ml[x][1][rr], f, total);
      o0 = __builtin_fmaf(from[d * kRows + rr], f, o0);
      o1 = __builtin_fmaf(from[(d + 1) * kRows + rr], f, o1);
    }
    if (parts > 1) {
      float* slot = a.row_part + (static_cast<int64_t>(item.slot) * a.slot_rows + rr) * (D + 2);
      *reinterpret_cast<float2*>(slot + d) = make_float2(o0, o1);
      if (d == 0) *reinterpret_cast<float2*>(slot + D) = make_float2(m, total);
    } else {
      const int i = rr / a.G, g = rr - i * a.G;
      uint16_t* out = a.o + row_at(a, w, b, kvh * a.G + g, i, a.so_b, a.so_h, a.so_n);
      const float inv = sees_any<WIN>(a, w, i) ? 1.f / total : 0.f;
      *reinterpret_cast<uint32_t*>(out + d) = bf16_pack2(o0 * inv, o1 * inv);
    }
  }
}

#endif  // __HIP_DEVICE_COMPILE__

// Workgroups a CU that the registers leave room for: int8 three up to head_dim 96, four up to 32 (64 tokens through windows of
// 1024, head_dim 32: 43 us, three 48).
template <int ST, int KS>
constexpr int kRowGroups = ST == kInt8 && KS <= 6 ? (KS <= 2 ? 4 : 3) : 2;

// Windows that are all of the row form.
template <int ST, bool WIN, int KS>
__global__ __launch_bounds__(kPagedThreads, (kRowGroups<ST, KS>)) void paged_row_kernel(PagedArgs a, unsigned first_group) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kFirst = coded(ST) ? 4 : 2;
  typedef RowLds<ST, KS, kFirst> L;
  __shared__ __attribute__((aligned(16))) char s0[L::k0], s1[L::k1];
  __shared__ float s_ml[4][2][kRows];
  row_work<ST, WIN, KS, kFirst>(a, static_cast<int>(first_group + blockIdx.x), s0, s1, s_ml);
#endif
}

template <int ST, bool WIN, int KS>
void launch_rows(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  in_launches(p.row_slots, [&](unsigned first, unsigned grid) {
    paged_row_kernel<ST, WIN, KS><<<grid, kPagedThreads, 0, s>>>(a, first);
  });
}

template <int ST, bool WIN>
void launch_paged_rows(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  SVHIP_PAGED_WIDTH(launch_rows, ST, WIN)
}

}  // namespace svhip
