// svhip_paged_append into int8 pools: whole numbers of at most 127 times one power of two for a block of 16, 32 or 64 rows
// and head (paged.hpp).
//
// A block's power of two is the least that holds its new rows, and not below the one it has if older rows of the window are in
// the block; those are halved with it where it grows. So a block of one head, of keys or of values, is one piece of work,
// whichever of its rows are new: its rows are read once, kept (rotated) in registers until the largest magnitude is known
// across all lanes, and written as codes. A wave takes a piece of few rows (single tokens); the four waves of a workgroup share
// the rows of a longer one and meet over the magnitude in LDS (a wave for all 64 rows held 256 registers: 32 chunks 53 us, a
// turned one spilled: 196). The workgroups of a slot of consecutive tokens (blockIdx.y of them) find the blocks whose
// first new token is among them and share out (block, slice of the heads); a workgroup forms a block's (cos, sin) in LDS once
// for the heads of its slice. Bound: HBM, and for few blocks the chain length, page, rows, magnitude. Measured on
// pools in turn: 32 ragged chunks of up to 1024 tokens of 8 x 128, blocks of 32 (105 MB) 35.1 us, 3.1 TB/s (28.6 on one pool,
// which the caches hold in part), turned 41.4 and 41.9, blocks of 64 35.3 and 47.5: a piece's rows are asked for behind its angles and a
// barrier; 64 chunks of 2048 (805 MB) 164 us, 4.9 TB/s, turned 169; 64 tokens of 16 x 64 6 to 7 us. Three axes: 8480 tokens of
// 8 x 48 22.4 us, 32 chunks of 16 x 48 50 (as they are 32); where pairs are no multiple of 8 rows go element by element, which
// lie 16 apart from lane to lane: 12 x 72 151 us (as they are 38).
#include "paged_append.hpp"

namespace svhip {

constexpr int kLeadersMost = 64;  // tokens of a workgroup at most, a lane of its first wave for each

// Byte of the least power of two with most <= 127 2^(byte - 127).
__device__ __forceinline__ int block_exponent(float most) {
  const uint32_t u = __float_as_uint(most);
  const int e = static_cast<int>(u >> 23) - ((u & 0x7fffffu) <= 0x7e0000u ? 6 : 5);
  return e < 1 ? 1 : (e > kInt8Top ? kInt8Top : e);
}

__device__ __forceinline__ float wave_max(float v) {
  v = row16_max(v);
  const auto at = [&](int lane) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
  };
  return fmaxf(fmaxf(at(0), at(16)), fmaxf(at(32), at(48)));
}

// 4 values of at most 127 / f times f as bytes, rounded to nearest even: added to 1.5 2^23, where the step is 1, a whole
// number stands in the low bits, two's complement.
__device__ __forceinline__ uint32_t int8_codes(float a, float b, float c, float d, float f) {
  const auto code = [&](float x) __attribute__((always_inline)) { return __float_as_uint(__builtin_fmaf(x, f, 12582912.f)); };
  const uint32_t lo = __builtin_amdgcn_perm(code(b), code(a), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(code(d), code(c), 0x04000c0cu);
  return lo | hi;
}

// A block that gets rows.
struct Block {
  int64_t src[2], page, pos;  // places of the first new row (key, value) and of its position, or, without one, its key's index
  int rows, older, row;       // new rows, older ones in front of them, the block's first row in its page
};

// What a wave needs of a piece: a block of one head, keys (side 0) or values.
struct Piece {
  const uint16_t* from;
  uint8_t *rows, *exponent;
  int64_t step, sr;
};

__device__ __forceinline__ Piece piece_of(const AppendArgs& a, const Block& blk, int shift, int h, int side) {
  if (side == 0) {
    return Piece{a.key + blk.src[0] + h * a.sk_h,
                 static_cast<uint8_t*>(a.ck) + blk.page * a.sck_p + h * a.sck_h + blk.row * a.sck_r,
                 a.ek + blk.page * a.sek_p + h * a.sek_h + (blk.row >> shift), a.sk_n, a.sck_r};
  }
  return Piece{a.value + blk.src[1] + h * a.sv_h,
               static_cast<uint8_t*>(a.cv) + blk.page * a.scv_p + h * a.scv_h + blk.row * a.scv_r,
               a.ev + blk.page * a.sev_p + h * a.sev_h + (blk.row >> shift), a.sv_n, a.scv_r};
}

// A lane's item of a row: whole runs at once, else element by element.
struct Raw {
  uint4 u, v;
};

__device__ __forceinline__ Raw load_item(const uint16_t* row, const Places& at, bool runs) {
  Raw r{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  if (runs) {
    if (at.n0) r.u = *reinterpret_cast<const uint4*>(row + at.first);
    if (at.n1) r.v = *reinterpret_cast<const uint4*>(row + at.second);
  } else {
    uint32_t e[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e[i] = i < at.n0 ? row[at.first + i] : 0u;
      e[8 + i] = i < at.n1 ? row[at.second + i] : 0u;
    }
    r.u = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    r.v = make_uint4(e[8] | e[9] << 16, e[10] | e[11] << 16, e[12] | e[13] << 16, e[14] | e[15] << 16);
  }
  return r;
}

__device__ __forceinline__ void unpack16(const Raw& r, float (&x)[16]) {
  const uint32_t w[8] = {r.u.x, r.u.y, r.u.z, r.u.w, r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// The lane's pairs turned by the row's angles.
template <int TURN>
__device__ __forceinline__ void turn_item(float (&x)[16], const float2* angle, const Places& at) {
  constexpr bool INTER = TURN != kTurnHalf;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= at.pairs) break;
    const float2 r = angle[i];
    float &p = x[INTER ? 2 * i : i], &q = x[INTER ? 2 * i + 1 : 8 + i];
    const float u = turned<TURN>(p, q, r, false), v = turned<TURN>(q, p, r, true);
    p = u;
    q = v;
  }
}

__device__ __forceinline__ uint32_t most_bits(const float (&x)[16]) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
    bits = u > bits ? u : bits;
  }
  return bits;
}

// The most that a block can hold, and its bits.
__device__ __forceinline__ float int8_reach() { return kInt8Most * exponent_value(kInt8Top); }

// What int8 cannot hold: finite values are cut to the reach, NaN becomes 0. Infinities stay (their code is that of 0 until
// mark_infinities) and take no part in the block's magnitude, since one would round all other rows of the block to 0, older ones
// for good. The bits of the largest finite magnitude.
__device__ __forceinline__ uint32_t cut_item(float (&x)[16]) {
  const float reach = int8_reach();
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float v = x[i] == x[i] ? x[i] : 0.f, w = fminf(fmaxf(v, -reach), reach);
    const bool finite = fabsf(v) < INFINITY;
    x[i] = finite ? w : v;
    const uint32_t u = finite ? __float_as_uint(w) & 0x7fffffffu : 0u;
    bits = u > bits ? u : bits;
  }
  return bits;
}

__device__ __forceinline__ void store_item(uint8_t* row, const Places& at, bool runs, const float (&x)[16], float f) {
  const uint32_t w[4] = {int8_codes(x[0], x[1], x[2], x[3], f), int8_codes(x[4], x[5], x[6], x[7], f),
                         int8_codes(x[8], x[9], x[10], x[11], f), int8_codes(x[12], x[13], x[14], x[15], f)};
  if (runs) {
    if (at.n0) *reinterpret_cast<uint2*>(row + at.first) = make_uint2(w[0], w[1]);
    if (at.n1) *reinterpret_cast<uint2*>(row + at.second) = make_uint2(w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < at.n0) row[at.first + i] = static_cast<uint8_t>(w[i >> 2] >> 8 * (i & 3));
      if (i < at.n1) row[at.second + i] = static_cast<uint8_t>(w[2 + (i >> 2)] >> 8 * (i & 3));
    }
  }
}

// Infinities of a row that is written: the largest number of their block, whatever it stands for.
__device__ __forceinline__ void mark_infinities(uint8_t* row, const Places& at, const float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int j = i & 7;
    if (fabsf(x[i]) == INFINITY && j < (i < 8 ? at.n0 : at.n1)) {
      row[(i < 8 ? at.first : at.second) + j] = static_cast<uint8_t>(x[i] > 0.f ? 127 : 0x81);
    }
  }
}

// 0 where all lanes' bits are finite; bit 0: a lane has an infinity, bit 1: or NaN.
constexpr uint32_t kInfinite = 0x7f800000u;
__device__ __forceinline__ uint32_t wild_bits(uint32_t bits) {
  return (__builtin_amdgcn_ballot_w64(bits == kInfinite) != 0ull ? 1u : 0u) |
         (__builtin_amdgcn_ballot_w64(bits >= kInfinite) != 0ull ? 2u : 0u);
}

// The exponent of a block whose new rows' largest finite magnitude has these bits (cut to the reach) and that had `had`; a
// block of zeros and infinities alone (`infinite`) takes the largest. The rows that are there, `first`, first + step, .. of the
// lane's 8-byte runs, go with it where it grows (127 2^-8 and less round to 0).
__device__ __forceinline__ int settle(const AppendArgs& a, const Block& blk, const Piece& p, uint32_t bits, bool infinite, int had,
                                      int lanes, int lane, bool writes) {
  int code = infinite && bits == 0 && blk.older == 0 ? kInt8Top : block_exponent(__uint_as_float(bits));
  if (blk.older > 0) {
    if (had >= code) {
      code = had < kInt8Top ? had : kInt8Top;
    } else {
      const float f = exponent_value(127 - (code - had < 30 ? code - had : 30));
      const int per_row = a.D / 8, all = blk.older * per_row;
      constexpr int kAtOnce = 2;
      for (int i0 = lane; i0 < all; i0 += kAtOnce * lanes) {
        uint2 w[kAtOnce];
        int at[kAtOnce];  // (a page's rows of a head lie within 2^31 bytes)
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int i = i0 + k * lanes, r = i / per_row;
          at[k] = r * static_cast<int>(p.sr) + 8 * (i - r * per_row);
          if (i < all) w[k] = *reinterpret_cast<const uint2*>(p.rows + at[k]);
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          if (i0 + k * lanes >= all) break;
          float c[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) c[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? w[k].x : w[k].y) >> 8 * (e & 3)));
          *reinterpret_cast<uint2*>(p.rows + at[k]) =
              make_uint2(int8_codes(c[0], c[1], c[2], c[3], f), int8_codes(c[4], c[5], c[6], c[7], f));
        }
      }
    }
  }
  if (writes) *p.exponent = static_cast<uint8_t>(code);
  return code;
}

// A piece of at most PASSES * 64 / LPR rows, by a wave.
template <int TURN, int LPR, int PASSES>
__device__ __forceinline__ void hold_few(const AppendArgs& a, const RowItems& items, const Block& blk, const Piece& p, bool turns,
                                         const float2* table, const Places& at) {
  const int lane = static_cast<int>(threadIdx.x & 63), r0 = lane / LPR;
  const int had = blk.older > 0 ? *p.exponent : 0;
  float x[PASSES][16];
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < PASSES; ++k) {
    const int r = r0 + 64 / LPR * k;
    Raw raw{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (r < blk.rows) raw = load_item(p.from + r * p.step, at, TURN == kTurnNone || a.runs);
    unpack16(raw, x[k]);
  }
#pragma unroll
  for (int k = 0; k < PASSES; ++k) {
    const int r = r0 + 64 / LPR * k;
    if (TURN != kTurnNone && turns && r < blk.rows) turn_item<TURN>(x[k], table + r * items.half + at.pair, at);
    const uint32_t b = most_bits(x[k]);
    bits = b > bits ? b : bits;
  }
  uint32_t wild = 0;
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(bits > __float_as_uint(int8_reach())) != 0ull, 0)) {
    wild = wild_bits(bits);
    if (wild) set_bad(a.pages);
    bits = 0;
#pragma unroll
    for (int k = 0; k < PASSES; ++k) {
      const uint32_t b = cut_item(x[k]);
      bits = b > bits ? b : bits;
    }
  }
  const int code = settle(a, blk, p, __float_as_uint(wave_max(__uint_as_float(bits))), wild & 1, __builtin_amdgcn_readfirstlane(had),
                          64, lane, lane == 0);
#pragma unroll
  for (int k = 0; k < PASSES; ++k) {
    const int r = r0 + 64 / LPR * k;
    if (r < blk.rows) store_item(p.rows + (blk.older + r) * p.sr, at, TURN == kTurnNone || a.runs, x[k], exponent_value(254 - code));
  }
  if (__builtin_expect(wild, 0)) {
#pragma unroll
    for (int k = 0; k < PASSES; ++k) {
      const int r = r0 + 64 / LPR * k;
      if (r < blk.rows) mark_infinities(p.rows + (blk.older + r) * p.sr, at, x[k]);
    }
  }
}

// LPR: lanes of a row. `heads`: of a slice, `slices` of them.
// Where a wave has one row of every lane there is room for six workgroups a CU (32 chunks 34.3 us, five 36.2); more spill.
template <int TURN, int LPR, int kBlock>
__global__ __launch_bounds__(kAppendThreads, kBlock > 16 && kBlock * LPR <= kAppendThreads ? 6 : 2) void
paged_append_int8_kernel(AppendArgs a, RowItems items, unsigned first_group, int heads, int slices) {
  constexpr int kShift = kBlock == 64 ? 6 : (kBlock == 32 ? 5 : 4), kWaves = kAppendThreads / 64;
  constexpr int kFew = 64 / LPR, kPasses = kBlock > kWaves * kFew ? kBlock / (kWaves * kFew) : 1;
  constexpr int kOwn = kBlock == 16 && kFew < 16 ? 16 / kFew : 1;  // passes of a wave by itself: all of a short block
  // (4 lanes have 32 pairs at most.)
  __shared__ float2 table[TURN == kTurnNone ? 1 : kBlock * (LPR == 4 ? 32 : kMaxPagedDim / 2)];
  __shared__ uint32_t s_most[2][kWaves];
  __shared__ Block blocks[kLeadersMost];
  __shared__ int s_count;
  const int64_t t0 = static_cast<int64_t>(first_group + blockIdx.x) * a.per_group;
  const int tokens = static_cast<int>(a.total - t0 < a.per_group ? a.total - t0 : a.per_group);
  const int tid = static_cast<int>(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (wave == 0) {
    const int64_t mine = t0 + tid;
    int64_t b = -1, n = mine;
    bool leads = false;
    Block blk{};
    if (tid < tokens) {
      if (!a.tokens.cu) {
        b = static_cast<int>(mine) / static_cast<int>(a.tokens.N);
        n = mine - b * a.tokens.N;
      } else {
        b = window_of(a.tokens, mine);
      }
    }
    if (b >= 0) {
      int64_t start, count;
      window_tokens(a.tokens, b, start, count);
      const int64_t i = mine - start, j = a.pages.lengths[b] - a.before - count + i;
      if (j < 0 || j >= a.pages.max_pages << a.pages.shift) {
        set_bad(a.pages);
      } else if (i == 0 || (i > 0 && i < count && (j & (kBlock - 1)) == 0)) {  // (i outside: borders not ascending)
        const int older = static_cast<int>(j & (kBlock - 1));
        blk.page = page_of(a.pages, b, j);
        leads = blk.page >= 0;
        // (packed: a row's index alone places it)
        blk.src[0] = (a.tokens.cu ? 0 : b * a.sk_b) + n * a.sk_n;
        blk.src[1] = (a.tokens.cu ? 0 : b * a.sv_b) + n * a.sv_n;
        blk.pos = a.positions ? (a.tokens.cu ? 0 : b * a.sp_b) + n * a.sp_n : j;
        blk.older = older;
        blk.rows = static_cast<int>(count - i < kBlock - older ? count - i : kBlock - older);
        blk.row = static_cast<int>(j & ((1ll << a.pages.shift) - 1)) - older;
      }
    }
    const uint64_t all = __builtin_amdgcn_ballot_w64(leads);
    if (leads) blocks[__builtin_popcountll(all & ((1ull << tid) - 1))] = blk;
    if (tid == 0) s_count = __builtin_popcountll(all);
  }
  __syncthreads();
  const int lane = tid & 63, r0 = lane / LPR;
  const Places at = places_of<TURN != kTurnHalf>(items, lane % LPR);
  const int pieces = __builtin_amdgcn_readfirstlane(s_count) * slices;
  int turn = 0;
  for (int piece = static_cast<int>(blockIdx.y); piece < pieces; piece += static_cast<int>(gridDim.y)) {
    const int i = piece / slices, h0 = (piece - i * slices) * heads, h1 = h0 + heads < a.H ? h0 + heads : a.H;
    const Block blk = blocks[i];
    if constexpr (TURN != kTurnNone) {
      __syncthreads();  // the table is read until here
      int r = tid / items.half, pr = tid - r * items.half;
      const int step_r = kAppendThreads / items.half, step_p = kAppendThreads - step_r * items.half;
      while (r < blk.rows) {
        float2 angle;
        if constexpr (TURN == kTurnAxial) {
          const int per_axis = items.half / 3, axis = pr / per_axis;
          const float* pos = static_cast<const float*>(a.positions) + blk.pos + r * a.sp_n;
          const float phase = pos[axis] * static_cast<const float*>(a.freq)[pr - axis * per_axis];
          angle = make_float2(bf16_round1(cosf(phase)), bf16_round1(sinf(phase)));
        } else {
          const double place = a.positions ? rotary_position(a.positions, a.wide, blk.pos + r * a.sp_n)
                                           : static_cast<double>(blk.pos + r);
          angle = rotary_phase(place, static_cast<const double*>(a.freq)[pr], a.amplitude);
        }
        table[r * items.half + pr] = angle;
        r += step_r;
        pr += step_p;
        if (pr >= items.half) {
          pr -= items.half;
          ++r;
        }
      }
      __syncthreads();
    }
    const int units = 2 * (h1 - h0);
    if (blk.rows <= kFew * kOwn) {
      for (int u = wave; u < units; u += kWaves) {
        hold_few<TURN, LPR, kOwn>(a, items, blk, piece_of(a, blk, kShift, h0 + (u >> 1), u & 1), (u & 1) == 0, table, at);
      }
      continue;
    }
    // The waves share the rows: wave w has rows kFew w .., kFew (w + 4) .. The next unit's rows are on their way while the
    // waves meet.
    Raw raw[kPasses];
    int had = 0;
    auto load = [&](int u) __attribute__((always_inline)) {
      const Piece p = piece_of(a, blk, kShift, h0 + (u >> 1), u & 1);
      had = blk.older > 0 ? *p.exponent : 0;
#pragma unroll
      for (int k = 0; k < kPasses; ++k) {
        const int r = kFew * (wave + kWaves * k) + r0;
        if (r < blk.rows) raw[k] = load_item(p.from + r * p.step, at, TURN == kTurnNone || a.runs);
      }
    };
    load(0);
    for (int u = 0; u < units; ++u) {
      const Piece p = piece_of(a, blk, kShift, h0 + (u >> 1), u & 1);
      float x[kPasses][16];
      uint32_t bits = 0;
#pragma unroll
      for (int k = 0; k < kPasses; ++k) {
        const int r = kFew * (wave + kWaves * k) + r0;
        if (r < blk.rows) {
          unpack16(raw[k], x[k]);
          if (TURN != kTurnNone && (u & 1) == 0) turn_item<TURN>(x[k], table + r * items.half + at.pair, at);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) x[k][e] = 0.f;
        }
        const uint32_t b = most_bits(x[k]);
        bits = b > bits ? b : bits;
      }
      const int were = __builtin_amdgcn_readfirstlane(had);
      if (u + 1 < units) load(u + 1);
      uint32_t wild = 0;
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(bits > __float_as_uint(int8_reach())) != 0ull, 0)) {
        wild = wild_bits(bits);
        if (wild) set_bad(a.pages);
        bits = 0;
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          const uint32_t b = cut_item(x[k]);
          bits = b > bits ? b : bits;
        }
      }
      uint32_t mine = __float_as_uint(wave_max(__uint_as_float(bits)));
      if (__builtin_expect(wild & 1, 0) && mine == 0) mine = kInfinite;
      if (lane == 0) s_most[turn][wave] = mine;
      __syncthreads();
      uint32_t most = s_most[turn][0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) most = s_most[turn][w] > most ? s_most[turn][w] : most;
      bool infinite = false;
      if (__builtin_expect(__builtin_amdgcn_readfirstlane(most) == kInfinite, 0)) {  // of a wave that has nothing else but zeros
        infinite = true;
        most = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const uint32_t other = s_most[turn][w];
          most = other < kInfinite && other > most ? other : most;
        }
      }
      turn ^= 1;  // (a wave is behind the next unit's barrier before it writes here again)
      const float f = exponent_value(254 - settle(a, blk, p, most, infinite, were, kAppendThreads, tid, tid == 0));
#pragma unroll
      for (int k = 0; k < kPasses; ++k) {
        const int r = kFew * (wave + kWaves * k) + r0;
        if (r < blk.rows) store_item(p.rows + (blk.older + r) * p.sr, at, TURN == kTurnNone || a.runs, x[k], f);
      }
      if (__builtin_expect(wild, 0)) {
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          const int r = kFew * (wave + kWaves * k) + r0;
          if (r < blk.rows) mark_infinities(p.rows + (blk.older + r) * p.sr, at, x[k]);
        }
      }
    }
  }
}

template <int TURN, int LPR>
void launch_int8(const AppendArgs& a, const RowItems& r, int shift, dim3 grid, unsigned first, int heads, int slices, hipStream_t s) {
  switch (shift) {
    case 6: paged_append_int8_kernel<TURN, LPR, 64><<<grid, kAppendThreads, 0, s>>>(a, r, first, heads, slices); break;
    case 5: paged_append_int8_kernel<TURN, LPR, 32><<<grid, kAppendThreads, 0, s>>>(a, r, first, heads, slices); break;
    default: paged_append_int8_kernel<TURN, LPR, 16><<<grid, kAppendThreads, 0, s>>>(a, r, first, heads, slices);
  }
}

template <int TURN>
void launch_int8(const AppendArgs& a, const RowItems& r, int shift, dim3 grid, unsigned first, int heads, int slices, hipStream_t s) {
  switch (row_lanes(r)) {
    case 4: return launch_int8<TURN, 4>(a, r, shift, grid, first, heads, slices, s);
    case 8: return launch_int8<TURN, 8>(a, r, shift, grid, first, heads, slices, s);
    default: return launch_int8<TURN, 16>(a, r, shift, grid, first, heads, slices, s);  // (128 elements: 9 items at most)
  }
}

// (Block, slice) pieces that a launch aims at (512, 1024, 4096: 32 chunks 73, 64, 66 us with their reading back, blocks of
// 16 70 with 1024 and 74 with 2048).
constexpr int64_t kBlockPieces = 1024;

void launch_append_int8(const AppendArgs& args, int turn, int shift, hipStream_t s) {
  AppendArgs a = args;
  const RowItems r = row_items(a.D, a.half);
  a.runs = a.half % 8 == 0;
  a.per_group = static_cast<int>(tokens_per_group(a.total, kLeadersMost));
  const int64_t groups = cdiv(a.total, a.per_group), block = 1ll << shift;
  // Slices of heads, two heads (a unit for each wave) at least, until the pieces are enough.
  const int64_t blocks = a.total / block + (a.tokens.B < a.total ? a.tokens.B : a.total);
  int64_t slices = cdiv(kBlockPieces, blocks);
  if (slices > (a.H + 1) / 2) slices = (a.H + 1) / 2;
  const int heads = static_cast<int>(cdiv(a.H, slices));
  slices = cdiv(a.H, heads);
  // A slot of a long window has so many blocks; one of single tokens more.
  const int64_t rows = cdiv(a.per_group, block) * slices;
  const int64_t y = rows < 65535 ? rows : 65535, most = kLaunchGroups / y;
  for (int64_t from = 0; from < groups; from += most) {
    const dim3 grid(static_cast<unsigned>(groups - from < most ? groups - from : most), static_cast<unsigned>(y));
    const unsigned first = static_cast<unsigned>(from);
    const int n = static_cast<int>(slices);
    switch (turn) {
      case SVHIP_ROTARY_HALF: launch_int8<kTurnHalf>(a, r, shift, grid, first, heads, n, s); break;
      case SVHIP_ROTARY_INTERLEAVED: launch_int8<kTurnInterleaved>(a, r, shift, grid, first, heads, n, s); break;
      case SVHIP_ROTARY_AXIAL: launch_int8<kTurnAxial>(a, r, shift, grid, first, heads, n, s); break;
      default: launch_int8<kTurnNone>(a, r, shift, grid, first, heads, n, s);
    }
  }
}

}  // namespace svhip
