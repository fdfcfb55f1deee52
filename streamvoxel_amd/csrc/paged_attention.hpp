// What the kernels of svhip_paged_attention share (paged_attention.hip describes them).
#pragma once

#include "paged.hpp"
#include "xattn_kernel.hpp"

namespace svhip {

constexpr int kPagedThreads = 256;
constexpr int kRows = 32;          // rows of a wave
// Rows of a window up to which it is of the row form, bf16 and codes. At 4, 8, 16, 32 rows a key head the row form
// takes 47, 57, 59, 85 us and tiles 42, 46, 41, 46 (64 windows of 512 to 1024 keys, 8 key heads of 128); 16 windows
// of 2048 to 4096 keys: 42, 50, 59, 82 and 38, 41, 44, 48; e4m3, 64 windows of 2048 to 4096 keys of 64: 51, 57, 56,
// 71 and 72, 73, 73, 76. int8 has e4m3's limit: at 5, 8 and 16 rows 71, 72, 76 and 94, 96, 93 us, with 8 heads of 128 123, 130,
// 138 and 130, 131, 128; through windows of 1000 keys tiles are the faster ones, 43, 47, 49 and 40, 42, 38, and a limit of its
// own there is left. With one of 64 windows 60 times as long as the others, 4 rows: 113 and 160; 200 windows of 1024 keys: 161 and 183.
constexpr int kRowMost = 4, kRowMostFp8 = 16;
constexpr int kTileRows = 128;     // rows of a tile workgroup
// Tile workgroups below which keys are split, two for every CU (one, four: a causal chunk of 4 x 512 tokens, head_dim
// 128, 313 and 278 us for 281; the same with all keys seen 198 and 180 for 167; 1024 queries over 9744 keys 82 and 61
// for 60).
constexpr int kTileTarget = 512;
// The same beside the row form: one for every CU. With 512 in its place: 24 windows, 6 of them chunks (head_dim 96) 110 us
// for 101; 8 heads of 64, 4 chunks of 512 and 60 tokens over 8192 keys 237 for 218, 32 chunks of 64 over 4096 and 8 tokens
// over 32 768 175 for 168, 16 chunks of 256 over 2048 and 48 tokens over 4096 123 for 110, a chunk of 128 over 16 384 and
// 63 tokens over 4096 123 for 116; 12 heads, 3 chunks of 512 over 4096 and 100 tokens over 2048 169 for 152; but 8 heads of
// 96, 6 chunks of 300 and 18 tokens over 8192, as much of one form as of the other, 163 for 180.
constexpr int kTileBeside = 256;
constexpr int kTileLong = 96;      // key blocks of a part beside the row form, through a window (tile_length)
constexpr int kTileLeast = 6;      // least key blocks of a tile's part (1024 queries over 9744 keys 60 us; 3, 12: 61)
// Row-form parts beyond one for each (window, key head): eight for every CU (64 tokens, four heads to a key head, 218
// us, 512 parts: 248; over e4m3 pages 158 and 180).
constexpr int kRowTarget = 2048;
constexpr int kRowLeast = 256;     // keys that a row-form part has a multiple of: 2 blocks of each wave (512: no difference)
constexpr int kWholePages = 64;    // pages from this size on hold whole blocks of keys: found once a block (tiles 1.4 % less)
constexpr int kUncut = 0x40000000; // a part length that cuts nothing
constexpr float kNoMax = -3.0e38f; // running maximum before any key: finite, so that a row that sees nothing stays finite
[[maybe_unused]] constexpr uint32_t kOutside = 0x7ffffff0u;  // byte offset past every descriptor's bound

struct PagedArgs {
  const uint16_t* q;
  const void *k, *v;
  const uint8_t *ek, *ev;
  uint16_t* o;
  Tokens tokens;
  Pages pages;
  int H, Hkv, G, D;     // G: heads of a key head (a window has less than 2^31 rows: a 64-bit division takes 0.3 us)
  int64_t sq_b, sq_h, sq_n, sk_h, sv_h, sek_h, sev_h, so_b, so_h, so_n;
  uint32_t sk_p, sk_r, sv_p, sv_r, sek_p, sev_p;  // bytes from page to page and row to row
  bool causal;
  float scale_log2;
  // The plan.
  int row_most;         // rows of a window up to which it is of the row form
  int q_tiles;          // tiles of a window (even windows)
  bool split;           // tiles: whether parts of keys may be dealt out
  int row_slots, tile_slots;  // slots of parts at most
  int slot_rows;        // rows of a row-form slot
  float *row_part, *tile_part;  // row_part null: the row form's windows are not cut
  int4* plan;           // (null: no parts) a window's first slot, its parts, a part's length (tiles: blocks) and its tiles
  int2* running;        // (null: every workgroup plans for itself) places of row form and of tiles up to and with a window;
                        // plan[B] then has their sums and the part lengths
  int block_shift;      // int8: log2 of the keys that share an exponent
  int window, sinks;    // keys that a token sees up to its own, and first keys that it sees beside them (window 0: all)
};

// The window as a workgroup sees it.
struct Window {
  int64_t first;         // its tokens
  int count;
  int64_t last;          // the last key that its first token sees (causal), or its last key
  int keys;              // its keys
};

__device__ __forceinline__ Window window_at(const PagedArgs& a, int64_t b) {
  Window w;
  int64_t count;
  window_tokens(a.tokens, b, w.first, count);
  w.count = static_cast<int>(count);
  const int64_t L = held_keys(a.pages, b);
  w.keys = static_cast<int>(L);
  w.last = a.causal ? a.pages.lengths[b] - w.count : L - 1;
  return w;
}

// Last key that token i sees (below 0: none).
__device__ __forceinline__ int last_key(const PagedArgs& a, const Window& w, int64_t i) {
  const int64_t j = a.causal ? w.last + i : w.last;
  return static_cast<int>(j < w.keys - 1 ? (j < -1 ? -1 : j) : w.keys - 1);
}

// First key of token i's window, the last keys that it sees.
__host__ __device__ __forceinline__ int first_key(int window, int64_t last, int keys, int64_t i) {
  const int64_t j = last + i - window + 1;
  return static_cast<int>(j < 0 ? 0 : (j < keys ? j : keys));
}
__device__ __forceinline__ int first_key(const PagedArgs& a, const Window& w, int64_t i) {
  return first_key(a.window, w.last, w.keys, i);
}

// The first keys that stay visible, in whole blocks of tiles; and the keys between them and the window's first block,
// which a workgroup whose first window begins at `low` leaves out: it walks the others as if they stood one behind the
// other (`real_key`).
__host__ __device__ __forceinline__ int sink_keys(int sinks) { return (sinks + kKB - 1) / kKB * kKB; }
__host__ __device__ __forceinline__ int left_out(int sinks, int low) {
  const int n = low / kKB * kKB - sink_keys(sinks);
  return n > 0 ? n : 0;
}
__device__ __forceinline__ int real_key(int j, int sink_end, int out) { return j < sink_end ? j : j + out; }

// True where token i sees a key.
template <bool WIN>
__device__ __forceinline__ bool sees_any(const PagedArgs& a, const Window& w, int64_t i) {
  const int last = last_key(a, w, i);
  if constexpr (WIN) return last >= 0 && (a.sinks > 0 || first_key(a, w, i) <= last);
  return last >= 0;
}

__host__ __device__ __forceinline__ bool row_form(const PagedArgs& a, int64_t count) { return count * a.G <= a.row_most; }

// Keys that the rows of tile qt see, the last of them the most.
__device__ __forceinline__ int tile_keys(const PagedArgs& a, const Window& w, int qt) {
  const int r1 = (qt + 1) * kTileRows, rows = w.count * a.G;
  return last_key(a, w, ((r1 < rows ? r1 : rows) - 1) / a.G) + 1;
}

// Those of them that the tile leaves out.
template <bool WIN>
__device__ __forceinline__ int tile_left_out(const PagedArgs& a, const Window& w, int qt) {
  if constexpr (WIN) return left_out(a.sinks, first_key(a, w, qt * kTileRows / a.G));
  return 0;
}

// Row of `out` (or, with its strides, of the queries) that token i and head h have.
__device__ __forceinline__ int64_t row_at(const PagedArgs& a, const Window& w, int64_t b, int64_t h, int64_t i, int64_t sb,
                                          int64_t sh, int64_t sn) {
  return a.tokens.cu ? h * sh + (w.first + i) * sn : b * sb + h * sh + i * sn;
}

// The wave's sum, in every lane: the plans' counts, exact up to 2^24 (where a plan cuts, its places are fewer). DPP
// steps: a shuffle through LDS takes as long as all of them.
__device__ __forceinline__ float wave_sum(float v) {
  v = row16_sum(v);
  const auto at = [&](int lane) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
  };
  return (at(0) + at(16)) + (at(32) + at(48));
}

// Exclusive prefix over the wave's lanes; `total` the sum.
__device__ __forceinline__ int wave_prefix(int v, int& total) {
  int incl = v;
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x112, 0xf, 0xf, true);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x114, 0xf, 0xf, true);
  incl += __builtin_amdgcn_update_dpp(0, incl, 0x118, 0xf, 0xf, true);
  const int r0 = __builtin_amdgcn_readlane(incl, 15), r1 = __builtin_amdgcn_readlane(incl, 31);
  const int r2 = __builtin_amdgcn_readlane(incl, 47), r3 = __builtin_amdgcn_readlane(incl, 63);
  const int row = (threadIdx.x & 63) >> 4;
  incl += row > 0 ? r0 : 0;
  incl += row > 1 ? r1 : 0;
  incl += row > 2 ? r2 : 0;
  total = r0 + r1 + r2 + r3;
  return incl - v;
}

// What a workgroup takes: part `part` of `parts` of key head kvh of window b (tiles: of tile qt). The windows that
// are cut have slots for their parts, one after the other: this one's is `slot`, its window's first `first`. b < 0:
// nothing.
struct PagedItem {
  int b, kvh, part, parts, qt, tiles, slot, first;
};

// Place `in` of window b's list: for every key head its parts, for every part its tiles; slots from `first` on.
__device__ __forceinline__ PagedItem item_of(int b, int first, int in, int parts, int tiles) {
  const int u = in / tiles, kvh = u / parts;
  return PagedItem{b, kvh, u - kvh * parts, parts, in - u * tiles, tiles, first + in, first};
}

// The item at place `at` of the lists of up to 64 windows, one after the other; the lane's window has `tiles` and
// `parts`.
__device__ __forceinline__ PagedItem item_at(int Hkv, int at, int tiles, int parts) {
  int total;
  const int n = tiles * Hkv * parts, before = wave_prefix(n, total);
  if (at >= total) return PagedItem{-1, 0, 0, 1, 0, 1, 0, 0};
  int slots;
  const int first = wave_prefix(parts > 1 ? n : 0, slots);
  const int c = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before <= at && at < before + n));
  return item_of(c, __builtin_amdgcn_readlane(first, c), at - __builtin_amdgcn_readlane(before, c),
                 __builtin_amdgcn_readlane(parts, c), __builtin_amdgcn_readlane(tiles, c));
}

// The same from paged_plan_kernel's lists; `ends` the running sums of the form, two numbers apart. 64 windows a step.
__device__ __forceinline__ PagedItem planned_item(const PagedArgs& a, int at, const int* ends) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = static_cast<int>(a.tokens.B), c;
  do {
    const int step = (hi - lo + 63) / 64, end = lo + (lane + 1) * step, last = end < hi ? end : hi;
    const uint64_t past = __builtin_amdgcn_ballot_w64(ends[2 * (last - 1)] > at);
    if (past == 0ull) return PagedItem{-1, 0, 0, 1, 0, 1, 0, 0};
    c = __builtin_ctzll(past);
    lo += c * step;
    hi = hi - lo > step ? lo + step : hi;
  } while (hi - lo > 1);
  const int4 plan = a.plan[lo];
  return item_of(lo, plan.x, at - (lo > 0 ? ends[2 * (lo - 1)] : 0), plan.y, plan.w);
}

// Who plans: a wave, for up to 64 windows (one a lane), or a workgroup.
struct WaveTeam {
  static constexpr int kSize = 64;
  __device__ __forceinline__ int id() const { return threadIdx.x & 63; }
  __device__ __forceinline__ float sum(float v) const { return wave_sum(v); }
};
constexpr int kPlanThreads = 1024;
struct BlockTeam {
  static constexpr int kSize = kPlanThreads;
  float* of_wave;  // LDS, one for every wave
  __device__ __forceinline__ int id() const { return threadIdx.x; }
  __device__ __forceinline__ float sum(float v) const {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 64; ++i) total += of_wave[i];
    __syncthreads();
    return total;
  }
};

// The least length of a part, a multiple of `grain` and `least` at least, for which the windows' parts are at most
// `target`: they then run side by side, and none longer than it must. places(c, length): parts of window c, all key
// heads and tiles.
template <typename Team, typename Places>
__host__ __device__ __forceinline__ int part_length(const PagedArgs& a, const Team& team, float work, int target, int grain,
                                           int least, Places places) {
  // An equal share is too short, or all but; twice as long again and again until it fits, then halves between.
  const float share = work / static_cast<float>(target) / static_cast<float>(grain);
  int low = share < static_cast<float>(kUncut / 4) / static_cast<float>(grain) ? static_cast<int>(share) : kUncut / 4 / grain;
  if (low * grain < least) low = least / grain - 1;
  int high = low + 1;
  auto fits = [&](int length) __attribute__((always_inline)) {
    float n = 0.f;
    for (int64_t c = team.id(); c < a.tokens.B; c += Team::kSize) n += places(static_cast<int>(c), length * grain);
    return team.sum(n) <= static_cast<float>(target);
  };
  while (high < kUncut / grain / 2 && !fits(high)) {
    low = high;
    high += high;
  }
  while (high - low > 1) {
    const int mid = low + (high - low) / 2;
    (fits(mid) ? high : low) = mid;
  }
  return high * grain;
}

// Page of the keys at j of the window whose table row this is, through the scalar cache; the number as it stands in the
// table (j may lie past the window's keys: its last entry then).
__device__ __forceinline__ int page_number(const PagedArgs& a, const int32_t* row, int j) {
  typedef const __attribute__((address_space(4))) int32_t* table_t;
  const int at = j >> a.pages.shift, last = static_cast<int>(a.pages.max_pages) - 1;
  return __builtin_amdgcn_readfirstlane(((table_t)row)[at < last ? at : last]);
}

// Keys of the kGroup at j that exist: inside the window and on a page of the pool.
template <int kGroup>
__device__ __forceinline__ int valid_keys(const PagedArgs& a, int keys, int j, int& page) {
  int valid = j + kGroup <= keys ? kGroup : (j < keys ? keys - j : 0);
  if (__builtin_expect(static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages.pages), 0)) {
    if (valid > 0) set_bad(a.pages);
    valid = 0;
    page = 0;
  }
  return valid;
}

// Head widths: KS steps of 16 head_dim elements in the score product, and output tiles of 32.
constexpr int tiles_of(int KS) { return (KS + 1) / 2; }

#if defined(__HIP_DEVICE_COMPILE__)

// One key head's part of a pool (of keys or of values): bytes from page to page and row to row.
struct Source {
  const char* rows;
  const uint8_t* exponents;
  uint32_t sp, sr, se;
};
template <int ES>
__device__ __forceinline__ Source k_source(const PagedArgs& a, int64_t kvh) {
  return Source{static_cast<const char*>(a.k) + kvh * a.sk_h * ES, ES == 1 ? a.ek + kvh * a.sek_h : nullptr, a.sk_p,
                a.sk_r, a.sek_p};
}
template <int ES>
__device__ __forceinline__ Source v_source(const PagedArgs& a, int64_t kvh) {
  return Source{static_cast<const char*>(a.v) + kvh * a.sv_h * ES, ES == 1 ? a.ev + kvh * a.sev_h : nullptr, a.sv_p,
                a.sv_r, a.sev_p};
}

// Descriptor of the rows of a group of keys, row in_page of `page` the first: `valid` of them, `bytes` of each. A
// read past them gives zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const char* head, uint32_t sp, uint32_t sr, int page, int in_page,
                                                         int valid, int bytes) {
  const char* base = head + static_cast<uint64_t>(static_cast<uint32_t>(page)) * sp + static_cast<uint32_t>(in_page) * sr;
  const uint32_t bound = valid > 0 ? static_cast<uint32_t>(valid - 1) * sr + bytes : 0u;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, bound, kRsrcFlags);
}

// A wave's 32 rows: the queries as B operands, O^T, running maximum and sum.
template <int KS>
struct Rows {
  bf16x8_t qf[KS];
  f32x16_t o[tiles_of(KS)];
  f32x4_t l;   // four equal entries: the lane's share of its row's sum
  float m;     // running maximum, log2 units
  int last;    // last key that the lane's row sees
  int low;     // first key of its window (WIN)
};

// True where the lane's row sees key j, or any.
template <bool WIN, int KS>
__device__ __forceinline__ bool sees(const PagedArgs& a, const Rows<KS>& s, int j) {
  if constexpr (WIN) return j <= s.last && (j >= s.low || j < a.sinks);
  return j <= s.last;
}
template <bool WIN, int KS>
__device__ __forceinline__ bool sees_any(const PagedArgs& a, const Rows<KS>& s) {
  if constexpr (WIN) return s.last >= 0 && (a.sinks > 0 || s.low <= s.last);
  return s.last >= 0;
}

template <bool WIN, int KS>
__device__ __forceinline__ void load_rows(const PagedArgs& a, const Window& w, int64_t b, int kvh, int r,
                                          Rows<KS>& s) {
  const int hh = (threadIdx.x & 63) >> 5;
  const int i = r / a.G, g = r - i * a.G;
  const bool ok = i < w.count;
  const uint16_t* q = a.q + row_at(a, w, b, kvh * a.G + g, i, a.sq_b, a.sq_h, a.sq_n);
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int d0 = 16 * k + 8 * hh;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (ok && d0 < a.D) raw = *reinterpret_cast<const uint4*>(q + d0);
    s.qf[k] = __builtin_bit_cast(bf16x8_t, raw);
  }
#pragma unroll
  for (int j = 0; j < tiles_of(KS); ++j) s.o[j] = f32x16_t{0};
  s.l = f32x4_t{0.f, 0.f, 0.f, 0.f};
  s.m = kNoMax;
  s.last = ok ? last_key(a, w, i) : -1;
  if constexpr (WIN) s.low = first_key(a, w, i);
}

// S^T of 32 keys: ka the K rows as A operands, row R of the tile key sigma_row(R).
template <int KS>
__device__ __forceinline__ f32x16_t scores(const Rows<KS>& s, const bf16x8_t (&ka)[KS]) {
  f32x16_t x;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[k], s.qf[k], k == 0 ? f32x16_t{0} : x, 0, 0, 0);
  }
  return x;
}

// int8: a block's keys enter the score product as their codes; what 16 of them stand for, a power of two, is put to the scores
// (an FMA's factor where the weights are formed) and not to every element of the keys: 32 kHalves keys, 16 each. (So a
// query's products with codes must fit fp32: elements up to 2^114.)
template <int kHalves>
struct KeyScales {
  float of[2 * kHalves];
};

// That factor with the call's scale. Not 0, which would make a masked score's -inf NaN: 2^-149 in a smaller one's place adds less
// than 2^-21 to an exponent for any finite score. Not infinite, which a score of 0 would be NaN with: with the largest number in
// its place scores from 2^-98 on pass 2^30 either way (weights_of). The row form bounds the product, the tile form, where
// one lane forms a block's power of two for all, that power, from its byte (the row form so: 64 tokens through windows of 1024
// 57.4 us for 56.5; the tile form by the product: 4 chunks of 512 337 us for 334).
__device__ __forceinline__ float bounded_scale(float scale, float f) {
  return __builtin_amdgcn_fmed3f(scale * f, 0x1p-149f, kFltMax);
}
__device__ __forceinline__ float bounded_power(float scale, uint32_t byte) {
  const int x = __builtin_amdgcn_frexp_expf(scale);  // scale in [2^(x - 1), 2^x)
  const int low = -21 - x > 1 ? -21 - x : 1, top = 255 - x < kInt8Top ? 255 - x : kInt8Top, e = static_cast<int>(byte);
  return exponent_value(e < low ? low : (e < top ? e : top));
}

// Scores x of a block of 32 kHalves keys, `key0` the first: those that a row does not see masked, and the running
// maximum moved for a score more than kMaxHigh above it (the weights then stay below 2^20, which fp32 sums and bf16
// hold alike). One such branch a block: a second one in a loop makes the compiler merge two register sets of O behind
// it, a copy that the common path pays.
template <int ST, bool WIN, int KS, int kHalves>
__device__ __forceinline__ void bound_scores(const PagedArgs& a, Rows<KS>& s, f32x16_t (&x)[kHalves], const KeyScales<kHalves>& f,
                                             bool masked, int key0) {
  const float sl2 = a.scale_log2;
  const int hh = (threadIdx.x & 63) >> 5;
  if (masked) {
#pragma unroll
    for (int t = 0; t < kHalves; ++t) {
      const int seen = s.last - key0 - 32 * t - 8 * hh;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if ((i < 8 ? i : i + 8) > seen) x[t][i] = -INFINITY;
      }
      if constexpr (WIN) {
        const int low = s.low - key0 - 32 * t - 8 * hh, sinks = a.sinks - key0 - 32 * t - 8 * hh;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if ((i < 8 ? i : i + 8) < low && (i < 8 ? i : i + 8) >= sinks) x[t][i] = -INFINITY;
        }
      }
    }
  }
  const auto max3 = [](float p, float q, float r) __attribute__((always_inline)) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(p, q), r);
  };
  float mx = 0.f;
#pragma unroll
  for (int t = 0; t < kHalves; ++t) {
    const f32x16_t& y = x[t];
    if constexpr (ST == kInt8) {
      const float lo = max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), __builtin_elementwise_maximum(y[6], y[7]));
      const float hi = max3(max3(y[8], y[9], y[10]), max3(y[11], y[12], y[13]), __builtin_elementwise_maximum(y[14], y[15]));
      const float h = __builtin_elementwise_maximum(lo * f.of[2 * t], hi * f.of[2 * t + 1]);
      mx = t == 0 ? h : __builtin_elementwise_maximum(mx, h);
      continue;
    }
    const float h = max3(max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), max3(y[6], y[7], y[8])),
                         max3(y[9], y[10], y[11]), max3(max3(y[12], y[13], y[14]), y[15], y[15]));
    mx = t == 0 ? h : __builtin_elementwise_maximum(mx, h);
  }
  if (__builtin_amdgcn_ballot_w64(__builtin_fmaf(mx, sl2, -s.m) > kMaxHigh) != 0ull) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    const float top = fmaxf(__int_as_float(sw[0]), __int_as_float(sw[1]));
    const float cand = (top < kFltMax ? top : kFltMax) * sl2;
    const float mn = cand > s.m ? cand : s.m;
    const float alpha = __builtin_amdgcn_exp2f(s.m - mn);
    s.m = mn;
#pragma unroll
    for (int i = 0; i < 4; ++i) s.l[i] *= alpha;
#pragma unroll
    for (int j = 0; j < tiles_of(KS); ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s.o[j][i] *= alpha;
    }
  }
}

// 32 keys' weights P^T = exp2(sl2 x - m) as B operands of the second product's two steps. They are rounded to bf16, since
// the product runs on the bf16 matrix cores, and the row's sum is taken over the rounded weights (add_values), so that
// what a rounding adds to the one it adds to the other: 0.0022 from 64 bits, relative, where weights in
// fp32 leave the result's own rounding, 0.0017. m is the rounded product of a score: beyond scores of
// 2^30 what its rounding leaves of the largest weight's exponent no longer fits fp32, and the row is NaN.
// BOUNDED: int8's factors f are bounded_power's.
template <int ST, bool BOUNDED, int KS>
__device__ __forceinline__ void weights_of(const Rows<KS>& s, const f32x16_t& x, float scale, const float* f,
                                           bf16x8_t (&pb)[2]) {
  const float nm = -s.m;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const float sl2 = ST != kInt8 ? scale : (BOUNDED ? scale * f[ks] : bounded_scale(scale, f[ks]));
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const f32x2_t two = {__builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * ks + j], sl2, nm)),
                           __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * ks + j + 1], sl2, nm))};
      const bf16x2_t c = __builtin_convertvector(two, bf16x2_t);
      pb[ks][j] = c[0];
      pb[ks][j + 1] = c[1];
    }
  }
}

// O^T += V^T P^T and the row's sum for 32 keys whose V rows are staged at vp (sub-tiles of 64 head_dim elements
// kSubBytes apart). The sum is taken over the bf16 weights that the product reads, by v_mfma_f32_4x4x4_16b_bf16 with
// ones in A, whose columns are single lanes: no row's NaN reaches another's sum.
template <int KS, int kSubBytes>
__device__ __forceinline__ void add_values(Rows<KS>& s, const bf16x8_t (&pb)[2], const char* vp,
                                           const uint32_t (&rvt)[tiles_of(KS)]) {
  constexpr int DT = tiles_of(KS);
  typedef short i16x4_t __attribute__((ext_vector_type(4)));
  typedef short i16x8_t __attribute__((ext_vector_type(8)));
  const i16x4_t ones = {0x3F80, 0x3F80, 0x3F80, 0x3F80};
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const i16x8_t p8 = __builtin_bit_cast(i16x8_t, pb[ks]);
    s.l = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(ones, __builtin_shufflevector(p8, p8, 0, 1, 2, 3), s.l, 0, 0, 0);
    s.l = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(ones, __builtin_shufflevector(p8, p8, 4, 5, 6, 7), s.l, 0, 0, 0);
  }
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    bf16x8_t va[DT];
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;
      char* at = const_cast<char*>(vp) + (j >> 1) * kSubBytes + rvt[j] + 16 * ks * kRow * 2;
      const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t*)(at));
      const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t*)(at + 4 * kRow * 2));
      va[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma unroll
    for (int j = 0; j < DT; ++j) s.o[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[j], pb[ks], s.o[j], 0, 0, 0);
  }
}

// Byte offsets of the reads of V rows, transposed: output tile j inside its sub-tile (xattn_kernel.hpp).
template <int DT>
__device__ __forceinline__ void v_offsets(uint32_t (&rvt)[DT]) {
  const int lane = threadIdx.x & 63, hh = lane >> 5;
  const int row = 8 * hh + ((lane & 15) >> 2), flip = (row >> 1) & 1;
  const int c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
  for (int j = 0; j < DT; ++j) {
    rvt[j] = static_cast<uint32_t>(row * kRow * 2 + 16 * (4 * ((j & 1) ^ flip) + c) + 8 * (lane & 1));
  }
}

// The lane's sum of its row, both lanes' shares.
__device__ __forceinline__ float row_sum(float l) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_int(l), __float_as_int(l), false, false);
  return __int_as_float(sw[0]) + __int_as_float(sw[1]);
}

// Rows of codes on their way to LDS: a wave's kLoads loads of 8 rows, and the rows' exponents.
template <int DT, int kLoads>
struct Staged {
  uint2 w[kLoads * Width<DT>::kSubTiles];
  uint32_t e[kLoads];
};

// A lane's place in a load of 8 rows whose first is row `first` of a block's tile (a multiple of 8), `base` being the
// tile row of the descriptor's first key: row lane / 8 and its chunk; K under sigma_row and swz, V under swzv.
struct Lane8 {
  uint32_t at[2];   // byte offset in the descriptor in each sub-tile, or kOutside past head_dim
  uint32_t key;     // the place of the key's exponent in theirs
};

// Exponents in front of that of the `key`th of a group of keys: one a key, or int8's one a block. (A group begins with a
// block, or lies in one.)
template <int ST>
__device__ __forceinline__ int exponent_at(const PagedArgs& a, int key) {
  return ST == kInt8 ? key >> a.block_shift : key;
}

template <int ST>
__device__ __forceinline__ Lane8 lane_of_load(const PagedArgs& a, uint32_t sr, int key, int chunk) {
  Lane8 n;
  n.key = static_cast<uint32_t>(exponent_at<ST>(a, key));
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int d = 64 * u + 8 * chunk;
    n.at[u] = d < a.D ? static_cast<uint32_t>(key) * sr + static_cast<uint32_t>(d * bytes_of(ST)) : kOutside;
  }
  return n;
}
template <int ST>
__device__ __forceinline__ Lane8 k_lane(const PagedArgs& a, int first, int base) {
  const int lane = threadIdx.x & 63, R = first + (lane >> 3);
  return lane_of_load<ST>(a, a.sk_r, sigma_row(R) - base, swz(R, lane & 7));
}
template <int ST>
__device__ __forceinline__ Lane8 v_lane(const PagedArgs& a, int first, int base) {
  const int lane = threadIdx.x & 63, R = first + (lane >> 3);
  return lane_of_load<ST>(a, a.sv_r, R - base, swzv(R, lane & 7));
}

// Descriptor of the exponents of a group of keys, as rows_of.
template <int ST>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t exponents_of(const PagedArgs& a, const Source& s, int page, int in_page,
                                                              int valid) {
  const char* e = reinterpret_cast<const char*>(s.exponents);
  if constexpr (ST == kInt8) {
    const int some = valid > 0 ? ((valid - 1) >> a.block_shift) + 1 : 0;
    return rows_of(e, s.se, 1, page, in_page >> a.block_shift, some, 1);
  }
  return rows_of(e, s.se, 1, page, in_page, valid, 1);
}

// Issues a load of 8 rows: bf16 straight into LDS at `to` (row 0 of the 8 in sub-tile 0), codes into registers at
// index i, with their exponents (EXPONENTS).
template <int ST, bool EXPONENTS, int DT, int kSubBytes, int kLoads>
__device__ __forceinline__ void stage_rows8(const __amdgpu_buffer_rsrc_t r, const __amdgpu_buffer_rsrc_t er, const Lane8& n,
                                            int i, char* to, Staged<DT, kLoads>& st) {
#pragma unroll
  for (int u = 0; u < Width<DT>::kSubTiles; ++u) {
    if constexpr (coded(ST)) {
      st.w[i * Width<DT>::kSubTiles + u] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, n.at[u], 0, 0));
    } else {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)(to + u * kSubBytes), 16, n.at[u], 0, 0, 0);
    }
  }
  if constexpr (EXPONENTS) st.e[i] = __builtin_amdgcn_raw_buffer_load_b8(er, n.key, 0, 0);
}

// 8 codes times 2^(exponent - 127) as bf16 (int8: SCALED), exact.
template <int ST, bool SCALED>
__device__ __forceinline__ uint4 decode8(uint2 w, uint32_t exponent) {
  if constexpr (ST == kInt8) return int8_values<SCALED>(w, SCALED ? int8_power(exponent) : 1.f);
  const float f = exponent_value(static_cast<int>(exponent));
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, f, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, f, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, f, true);
  return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                    __builtin_bit_cast(uint32_t, d));
}

// Codes: load i of `st` into its 8 rows at `to`; SCALED: times their powers of two.
template <int ST, bool SCALED, int DT, int kSubBytes, int kLoads>
__device__ __forceinline__ void commit_rows8(const Staged<DT, kLoads>& st, int i, uint32_t exponent, char* to) {
#pragma unroll
  for (int u = 0; u < Width<DT>::kSubTiles; ++u) {
    *reinterpret_cast<uint4*>(to + u * kSubBytes + 16 * (threadIdx.x & 63)) =
        decode8<ST, SCALED>(st.w[i * Width<DT>::kSubTiles + u], exponent);
  }
}

// Values that are not finite (int8 has none), in a block whose keys some rows of the product see and some do not: their weight 0
// times such a value is NaN. So they are zeroed in LDS before the product (true: one was), a thread 16 bytes of
// `bytes` every `step`, and added to the rows that see them at the end, from the pool.
__device__ __forceinline__ bool clean_values(char* v, int bytes, int at, int step) {
  bool odd = false;
  for (; at < bytes; at += step) {
    uint4* const p = reinterpret_cast<uint4*>(v + at);
    const uint4 w = *p;
    uint32_t u[4] = {w.x, w.y, w.z, w.w};
    bool here = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool lo = (u[i] & 0x7f80u) == 0x7f80u, hi = (u[i] & 0x7f800000u) == 0x7f800000u;
      here |= lo || hi;
      u[i] &= (lo ? 0xffff0000u : ~0u) & (hi ? 0xffffu : ~0u);
    }
    if (here) *p = make_uint4(u[0], u[1], u[2], u[3]);
    odd |= here;
  }
  return odd;
}

// Those of keys [from, to) to O^T of the rows that see them. (Their weights are above 0, and an infinity or NaN stays
// one.)
template <int ST, bool WIN, int KS>
__device__ __forceinline__ void add_odd_values(const PagedArgs& a, const Source& vs, const int32_t* row, int from, int to,
                                               Rows<KS>& s) {
  const int hh = (threadIdx.x & 63) >> 5, in_mask = (1 << a.pages.shift) - 1;
  for (int j = from; j < to; ++j) {
    const int page = page_number(a, row, j);
    if (static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages.pages) && sees<WIN>(a, s, j)) {
      const uint32_t in_page = j & in_mask;
      const char* at = vs.rows + static_cast<uint64_t>(page) * vs.sp + in_page * vs.sr;
      float f = 0.f;
      if constexpr (ST == kE4m3) f = exponent_value(vs.exponents[static_cast<uint64_t>(page) * vs.se + in_page]);
#pragma unroll
      for (int i = 0; i < 4 * tiles_of(KS); ++i) {
        const int d0 = 8 * i + 4 * hh;
        if (d0 >= a.D) continue;
        uint2 w;
        if constexpr (ST == kE4m3) {
          const uint32_t codes = *reinterpret_cast<const uint32_t*>(at + d0);
          w = make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, f, false)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, f, true)));
        } else {
          w = *reinterpret_cast<const uint2*>(at + 2 * d0);
        }
        const float v[4] = {__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                            __uint_as_float(w.y & 0xffff0000u)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((__float_as_uint(v[e]) & 0x7f800000u) == 0x7f800000u) s.o[i >> 2][4 * (i & 3) + e] += v[e];
        }
      }
    }
  }
}

#endif  // __HIP_DEVICE_COMPILE__

// What a call launches, by its sizes alone.
struct PagedPlan {
  bool rows, tiles, row_parts, split;  // the forms that its windows may take, and which may be cut into parts
  int q_tiles;
  bool planned;                        // by paged_plan_kernel: more windows than a wave has lanes
  int64_t tile_grid, tile_slots, row_slots, slot_rows, row_floats, tile_floats, plan_windows;
  size_t bytes() const {
    return static_cast<size_t>(row_floats + tile_floats) * 4 +
           static_cast<size_t>(planned ? plan_windows * 24 + 16 : plan_windows * 16);
  }
};

inline PagedPlan paged_plan(int64_t B, int64_t H, int64_t Hkv, int64_t N, bool packed, int64_t D, int64_t max_keys,
                             int row_most) {
  PagedPlan p{};
  const int64_t G = H / Hkv;
  p.rows = packed || N * G <= row_most;
  p.tiles = N * G > row_most;
  if (p.tiles) {
    p.q_tiles = packed ? 1 : static_cast<int>(cdiv(N * G, kTileRows));
    // Tiles of all windows and key heads: exactly, or packed at most (a window of them has more than row_most rows).
    const int64_t windows = N * G / (row_most + 1) < B ? N * G / (row_most + 1) : B;
    const int64_t units = (packed ? N * G / kTileRows + windows : B * p.q_tiles) * Hkv;
    // Even windows that fill the chip are cut, where one is far longer than the others, if they have one wave's rows
    // (64 windows x 8 key heads of 128, 16 heads each, 1024 keys and one of 60 000: 162 us); with more the plan and
    // the join would cost calls of even lengths a quarter (64 windows x 8 heads, 64 queries, 512 keys: 18.4 us, 23.9
    // planned).
    p.split = packed || ((units < kTileTarget || N * G <= kRows) && max_keys > kTileLeast * kKB);
    if (!p.split) {
      p.tile_grid = cdiv(B * Hkv, kXcds) * kXcds * p.q_tiles;
      p.tile_slots = p.tile_grid;
    } else {
      p.tile_slots = kTileTarget;
      // A share of parts, or tiles that are as many and a share of parts of the long windows among them: of kTileTarget,
      // and packed, where there may be windows of the row form, also of kTileBeside (tile_length).
      int64_t places = units < kTileTarget ? kTileTarget : units + kTileTarget;
      if (packed && units >= kTileBeside && places < units + kTileBeside) places = units + kTileBeside;
      p.tile_grid = cdiv(places, kXcds) * kXcds;
      p.tile_floats = p.tile_slots * kTileRows * (D + 2);
    }
  }
  if (p.rows) {
    // One for each (window, key head), and the parts: at most kRowTarget more, and no shorter than kRowLeast.
    // (From 2^22 pairs on there is no need, and the plan's sums stay exact.)
    const int64_t more = B * Hkv > 1 << 22 ? 0 : B * Hkv * (cdiv(max_keys, kRowLeast) - 1);
    p.row_parts = more > 0;
    p.row_slots = (more < 0 ? 0 : (more < kRowTarget ? more : kRowTarget)) + B * Hkv;
    p.slot_rows = packed ? (N * G < row_most ? N * G : row_most) : N * G;
    if (p.row_parts) p.row_floats = (p.row_slots * p.slot_rows * (D + 2) + 3) / 4 * 4;
  }
  p.plan_windows = p.row_parts || p.split ? B : 0;
  p.planned = p.plan_windows > 64;
  return p;
}

// Keys that a tile's tokens, or those of a window of the row form, see at most of `max_keys` through a window.
inline int64_t window_keys(int64_t max_keys, int64_t window, int64_t sinks) {
  const int64_t most = window + 2 * kTileRows + 2 * kKB + sink_keys(static_cast<int>(sinks));
  return max_keys < most ? max_keys : most;
}

// The launches of a storage, WIN: with a window (KS: steps of 16 head_dim elements; whole: pages of kWholePages keys or more).
template <int ST, bool WIN>
void launch_paged_rows(const PagedArgs& a, const PagedPlan& p, hipStream_t s);
template <int ST, bool WIN>
void launch_paged_tiles(const PagedArgs& a, const PagedPlan& p, bool whole, hipStream_t s);
template <int ST, bool WIN>
void launch_paged_mixed(const PagedArgs& a, const PagedPlan& p, hipStream_t s);

// The instantiations of `launch` by head width; the others of its template arguments in front.
#define SVHIP_PAGED_WIDTH(launch, ...)                       \
  switch ((a.D + 15) / 16) {                                 \
    case 8: return launch<__VA_ARGS__, 8>(a, p, s);          \
    case 7: return launch<__VA_ARGS__, 7>(a, p, s);          \
    case 6: return launch<__VA_ARGS__, 6>(a, p, s);          \
    case 5: return launch<__VA_ARGS__, 5>(a, p, s);          \
    case 4: return launch<__VA_ARGS__, 4>(a, p, s);          \
    case 3: return launch<__VA_ARGS__, 3>(a, p, s);          \
    case 2: return launch<__VA_ARGS__, 2>(a, p, s);          \
    default: return launch<__VA_ARGS__, 1>(a, p, s);         \
  }

}  // namespace svhip
