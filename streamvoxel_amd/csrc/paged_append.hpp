// What the appends to a paged cache share (paged_append.hip, paged_append_int8.hip).
#pragma once

#include "paged.hpp"
#include "rotary.hpp"

namespace svhip {

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 8;
constexpr int kAppendAhead = 2;  // rows a thread has in flight

enum AppendTurn { kTurnNone = 0, kTurnHalf = 1, kTurnInterleaved = 2, kTurnAxial = 3 };

struct AppendArgs {
  const uint16_t *key, *value;
  int64_t sk_b, sk_h, sk_n, sv_b, sv_h, sv_n;
  Tokens tokens;
  int64_t total, before;
  int H, D, per_group;  // per_group: tokens of a workgroup
  void *ck, *cv;
  int64_t sck_p, sck_h, sck_r, scv_p, scv_h, scv_r;
  uint8_t *ek, *ev;
  int64_t sek_p, sek_h, sev_p, sev_h;
  Pages pages;
  const void* positions;
  int64_t sp_b, sp_n;
  const void* freq;
  int half;             // pairs that turn
  bool wide, runs;      // runs: the pairs of 8 elements lie in 8 elements each
  float amplitude, reach;  // reach: |turned| <= reach max |key|
};

__device__ __forceinline__ void unpack_run(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ float max_run(const float (&x)[8]) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
  return m;
}

// x = element d of a row turned with its partner y by r = (cos, sin); `second`: it is the pair's second one.
template <int TURN>
__device__ __forceinline__ float turned(float x, float y, float2 r, bool second) {
  if constexpr (TURN == kTurnAxial) {
    const float p = bf16_round1(x * r.x), q = bf16_round1(y * r.y);
    return bf16_round1(second ? q + p : p - q);
  }
  return __builtin_fmaf(x, r.x, second ? y * r.y : -(y * r.y));
}

// 8 elements d0 .. of a key row turned: x the row's, `other` the 8 that hold their partners (half layout: half
// further on or back; else unused).
template <int TURN>
__device__ __forceinline__ void turn_run(const AppendArgs& a, float (&x)[8], const uint4& other, const uint16_t* row,
                                         const float2* table, int d0) {
  if constexpr (TURN == kTurnNone) {
    return;
  } else if (!a.runs) {
    // Pairs anywhere: the partners are read one by one.
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      if (d >= 2 * a.half) continue;
      const bool second = TURN == kTurnHalf ? d >= a.half : (d & 1);
      const int pair = TURN == kTurnHalf ? (second ? d - a.half : d) : d >> 1;
      const float y = bf16_bits_to_float(row[TURN == kTurnHalf ? (second ? d - a.half : d + a.half) : d ^ 1]);
      x[e] = turned<TURN>(x[e], y, table[pair], second);
    }
  } else if (d0 < 2 * a.half) {
    if constexpr (TURN == kTurnHalf) {
      const bool second = d0 >= a.half;
      float y[8];
      unpack_run(other, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = turned<TURN>(x[e], y[e], table[(second ? d0 - a.half : d0) + e], second);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float2 r = table[(d0 + e) / 2];
        const float u = x[e], v = x[e + 1];
        x[e] = turned<TURN>(u, v, r, false);
        x[e + 1] = turned<TURN>(v, u, r, true);
      }
    }
  }
}

// The int8 pools' append.
void launch_append_int8(const AppendArgs& a, int turn, int block_shift, hipStream_t s);

}  // namespace svhip
