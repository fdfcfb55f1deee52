// Rotary positions: what the rotation of activations and the append to a paged cache share.
//
// Pair i < half of a head turns by theta = p f_i: y_a = A (x_a cos - x_b sin), y_b = A (x_b cos + x_a sin), with (a,
// b) = (i, i + half) in the half layout and (2 i, 2 i + 1) in the interleaved one; elements from 2 half on are kept.
// A phase in fp32 is off by p f 2^-24: a thirtieth of a radian at position 2^19. So the turns p f / 2 pi are formed
// in 64 bits and cut to half a turn there (off by 2^-52 of the turns, below fp32's step up to position 2^30), and
// only what is left goes to fp32's sin and cos; both are shared by all heads of a token, so the table costs little.
#pragma once

#include "common.hpp"

namespace svhip {

constexpr int kMaxRotaryPairs = 128;

// cos and sin of p turned by frequency f (radians a position), times the amplitude.
__device__ __forceinline__ float2 rotary_phase(double p, double f, float amplitude) {
  const double turns = p * (f * 0.15915494309189533577);
  const double cut = turns - __builtin_rint(turns);
  float s, c;
  sincospif(static_cast<float>(2.0 * cut), &s, &c);
  return make_float2(amplitude * c, amplitude * s);
}

__device__ __forceinline__ double rotary_position(const void* positions, bool wide, int64_t i) {
  return wide ? static_cast<double>(static_cast<const int64_t*>(positions)[i])
              : static_cast<double>(static_cast<const int32_t*>(positions)[i]);
}

// One pair (a, b) by r = (cos, sin), fp32.
__device__ __forceinline__ void rotary_turn(float& a, float& b, float2 r) {
  const float x = a;
  a = __builtin_fmaf(x, r.x, -(b * r.y));
  b = __builtin_fmaf(b, r.x, x * r.y);
}

// A row of D elements, its first `half` pairs turning, as items of 16 elements each: item e < turning has pairs 8 e .., two
// runs of 8 elements half apart (half layout) or side by side (interleaved); the others have 16 elements that are kept. A
// lane that carries an item turns its pairs by itself.
struct RowItems {
  int D, half, turning, items;
};
inline RowItems row_items(int D, int half) {
  const int turning = (half + 7) / 8;
  return RowItems{D, half, turning, turning + (D - 2 * half + 15) / 16};
}
// Lanes of a row: a power of two that holds its items.
inline int row_lanes(const RowItems& r) { return r.items <= 4 ? 4 : (r.items <= 8 ? 8 : (r.items <= 16 ? 16 : 32)); }

struct Places {
  int first, second;  // of elements 0 .. 7 and 8 .. 15
  int n0, n1;         // how many of each there are (whole runs: 0 or 8)
  int pair, pairs;    // the first pair, and how many (0: kept)
};

template <bool INTER>
__device__ __forceinline__ Places places_of(const RowItems& r, int e) {
  Places p{0, 0, 0, 0, 0, 0};
  if (e >= r.items) return p;
  if (e < r.turning) {
    p.pair = 8 * e;
    p.pairs = r.half - 8 * e < 8 ? r.half - 8 * e : 8;
  }
  if (!INTER && e < r.turning) {
    p.first = 8 * e;
    p.second = r.half + 8 * e;
    p.n0 = p.n1 = p.pairs;
  } else {
    p.first = e < r.turning ? 16 * e : 2 * r.half + 16 * (e - r.turning);
    p.second = p.first + 8;
    const int n = e < r.turning ? 2 * p.pairs : (r.D - p.first < 16 ? r.D - p.first : 16);
    p.n0 = n < 8 ? n : 8;
    p.n1 = n - p.n0;
  }
  return p;
}

// Tokens of a workgroup: as many as leave two workgroups for every CU, up to `most` (1024 tokens of 16 x 128: rotation
// 4.1 us, append 5.6; eight in every workgroup 5.4 and 8.9; 520 tokens 3.8 and 4.4, 5.1 and 8.2).
inline int64_t tokens_per_group(int64_t total, int64_t most) {
  const int64_t n = total / 512;
  return n < 1 ? 1 : (n < most ? n : most);
}

}  // namespace svhip
