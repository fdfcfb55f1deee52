// svhip_rotary: rotary positions of activations [B, H, N, D] (rotary.hpp), and with `inverse` the gradient: the
// transposed rotation, sin negated.
//
// Bound: HBM, every element read and written once (3 operations each). Workgroup = (window, up to kRotaryTokens
// tokens), all heads: the tile's (cos, sin) of every (token, pair) go to LDS once, since they are the same for every
// head, and a thread then turns pairs of 16-byte runs, kRotaryAhead of them in flight before the table is formed.
// Rows that are not made of such runs (odd numbers of pairs, unaligned rows) go pair by pair. Measured: 32 768 x 16 x
// 128 in fp32 (537 MB) 105 us, 5.1 TB/s, what a large copy reaches; 8 x 1024 x 12 x 64 in bf16 (25 MB) 8.1 us; 64
// tokens 3.6 us. Loads behind the table, one run a thread: 136 and 19 us. 4 and 16 tokens a workgroup: 8.8 and 8.5 us
// for the 25 MB. Pair by pair (30 pairs of the same rows, from call to call): 11.0 us for 7.7 of 32, in fp32 11.5 for
// 9.7.
#include "rotary.hpp"

namespace svhip {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 8;
constexpr int kRotaryAhead = 2;

struct RotaryArgs {
  const void* x;
  void* out;
  const void* positions;
  const double* freq;
  int64_t B, N, sx_b, sx_h, sx_n, so_b, so_h, so_n, sp_b, sp_n;
  int H, D, half, tokens;  // tokens: of a workgroup
  bool wide, interleaved;
  float amplitude, sign;
};

// Elements of T in 16 bytes, as fp32.
template <typename T>
struct Run {
  static constexpr int n = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = w; }
  __device__ __forceinline__ void get(float (&x)[n]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (n == 4) {
        x[i] = __uint_as_float(u[i]);
      } else {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ void set(const float (&x)[n]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = n == 4 ? __float_as_uint(x[i]) : bf16_pack2(x[2 * i], x[2 * i + 1]);
    w = make_uint4(u[0], u[1], u[2], u[3]);
  }
};

template <typename T>
__device__ __forceinline__ void store_as(T* p, float v) {
  if constexpr (sizeof(T) == 4) {
    *p = v;
  } else {
    *p = bf16_bits(v);
  }
}

// VEC: an item is Run::n pairs (two runs), or one run past the pairs; else one pair, or one element.
template <typename T, bool VEC>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a, unsigned first_group) {
  __shared__ float2 table[kRotaryTokens * kMaxRotaryPairs];
  constexpr int E = VEC ? Run<T>::n : 1, kAhead = VEC ? kRotaryAhead : 1;
  // (In 32 bits: a 64-bit division takes 0.3 us.)
  const unsigned N = static_cast<unsigned>(a.N), per = static_cast<unsigned>(a.tokens), tiles = (N + per - 1) / per;
  const unsigned group = first_group + blockIdx.x, window = group / tiles, from = (group - window * tiles) * per;
  const int64_t b = window, n0 = from;
  const int tokens = static_cast<int>(N - from < per ? N - from : per);
  const T* x = static_cast<const T*>(a.x) + b * a.sx_b + n0 * a.sx_n;
  T* out = static_cast<T*>(a.out) + b * a.so_b + n0 * a.so_n;
  const int turning = a.half / E, per_row = turning + (a.D - 2 * a.half) / E;
  // Item e of (token, head) row th = t H + h; kRotaryThreads items further on without a division.
  int th = static_cast<int>(threadIdx.x) / per_row, e = static_cast<int>(threadIdx.x) - th * per_row;
  int t = th / a.H, h = th - t * a.H;
  const int step_th = kRotaryThreads / per_row, step_e = kRotaryThreads - step_th * per_row;
  const int step_t = step_th / a.H, step_h = step_th - step_t * a.H;
  auto advance = [&]() __attribute__((always_inline)) {
    e += step_e;
    h += step_h;
    t += step_t;
    if (e >= per_row) {
      e -= per_row;
      ++h;
    }
    if (h >= a.H) {
      h -= a.H;
      ++t;
    }
  };
  struct Item {
    int t, h, first, second, pair;  // elements of the two runs; pair < 0: one run, kept
    Run<T> u, v;
    float p, q;
  };
  Item items[kAhead];
  auto load = [&](Item& it) __attribute__((always_inline)) {
    it.t = t;
    it.h = h;
    it.pair = e < turning ? E * e : -1;
    it.first = e < turning ? (a.interleaved ? 2 * E * e : E * e) : 2 * a.half + E * (e - turning);
    it.second = e < turning ? (a.interleaved ? it.first + E : a.half + E * e) : it.first;
    if (t < tokens) {
      const T* row = x + h * a.sx_h + t * a.sx_n;
      if constexpr (VEC) {
        it.u.load(row + it.first);
        it.v.load(row + it.second);
      } else {
        it.p = to_float<T>(row[it.first]);
        it.q = to_float<T>(row[it.second]);
      }
    }
    advance();
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(items[i]);
  for (int i = threadIdx.x; i < tokens * a.half; i += kRotaryThreads) {
    const int row = i / a.half, pr = i - row * a.half;
    float2 r = rotary_phase(rotary_position(a.positions, a.wide, b * a.sp_b + (n0 + row) * a.sp_n), a.freq[pr], a.amplitude);
    r.y *= a.sign;
    table[i] = r;
  }
  __syncthreads();
  while (items[0].t < tokens) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      Item& it = items[i];
      if (it.t >= tokens) break;
      T* row = out + it.h * a.so_h + it.t * a.so_n;
      const float2* angle = table + it.t * a.half + it.pair;
      if constexpr (VEC) {
        if (it.pair < 0) {
          it.u.store(row + it.first);
          continue;
        }
        float p[E], q[E];
        it.u.get(p);
        it.v.get(q);
        if (a.interleaved) {
#pragma unroll
          for (int j = 0; j < E; j += 2) {
            rotary_turn(p[j], p[j + 1], angle[j / 2]);
            rotary_turn(q[j], q[j + 1], angle[(E + j) / 2]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) rotary_turn(p[j], q[j], angle[j]);
        }
        it.u.set(p);
        it.v.set(q);
        it.u.store(row + it.first);
        it.v.store(row + it.second);
      } else {
        float p = it.p, q = it.q;
        if (it.pair >= 0) {
          rotary_turn(p, q, angle[0]);
          store_as<T>(row + it.second, q);
        }
        store_as<T>(row + it.first, p);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(items[i]);
  }
}

template <typename T>
void launch_rotary(const RotaryArgs& a, bool vec, hipStream_t s) {
  in_launches(a.B * cdiv(a.N, a.tokens), [&](unsigned first, unsigned grid) {
    if (vec) {
      rotary_kernel<T, true><<<grid, kRotaryThreads, 0, s>>>(a, first);
    } else {
      rotary_kernel<T, false><<<grid, kRotaryThreads, 0, s>>>(a, first);
    }
  });
}

}  // namespace svhip

using namespace svhip;

extern "C" int svhip_rotary(const svhip_rotary_args* args, void* stream) {
  const char* name = "svhip_rotary";
  clear_error();
  SVHIP_REQUIRE(args, "%s: null arguments", name);
  const svhip_rotary_args& c = *args;
  SVHIP_REQUIRE(c.B >= 0 && c.B < (1ll << 31) && c.H >= 0 && c.N >= 0 && c.N < (1ll << 31) && c.D >= 1, "%s: bad sizes",
                name);
  SVHIP_REQUIRE(c.dtype == SVHIP_F32 || c.dtype == SVHIP_BF16, "%s: dtype %d unsupported", name, (int)c.dtype);
  SVHIP_REQUIRE(c.layout == SVHIP_ROTARY_HALF || c.layout == SVHIP_ROTARY_INTERLEAVED, "%s: layout %d unsupported", name,
                (int)c.layout);
  SVHIP_REQUIRE(c.pairs >= 1 && c.pairs <= kMaxRotaryPairs && 2 * c.pairs <= c.D,
                "%s: %lld pairs do not fit head_dim %lld (at most %d)", name, (long long)c.pairs, (long long)c.D,
                kMaxRotaryPairs);
  SVHIP_REQUIRE(c.D <= 1 << 20 && c.H <= 1 << 20, "%s: sizes too large", name);
  if (c.B == 0 || c.H == 0 || c.N == 0) return SVHIP_OK;
  SVHIP_REQUIRE(c.x && c.out && c.positions && c.freq, "%s: null pointer", name);
  const int64_t tokens = tokens_per_group(c.B * c.N, kRotaryTokens);
  SVHIP_REQUIRE(c.B * cdiv(c.N, tokens) < (1ll << 31), "%s: grid too large", name);
  const RotaryArgs a{c.x, c.out, c.positions, c.freq, c.B, c.N, c.sx_b, c.sx_h, c.sx_n, c.so_b, c.so_h, c.so_n, c.sp_b,
                     c.sp_n, static_cast<int>(c.H), static_cast<int>(c.D), static_cast<int>(c.pairs),
                     static_cast<int>(tokens), c.positions_wide != 0, c.layout == SVHIP_ROTARY_INTERLEAVED,
                     static_cast<float>(c.amplitude), c.inverse ? -1.f : 1.f};
  const int64_t run = c.dtype == SVHIP_F32 ? 4 : 8;
  const bool vec = c.pairs % run == 0 && c.D % run == 0 && reinterpret_cast<uintptr_t>(c.x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(c.out) % 16 == 0 &&
                   (used_stride(c.B, c.sx_b | c.so_b) | used_stride(c.H, c.sx_h | c.so_h) |
                    used_stride(c.N, c.sx_n | c.so_n)) % run == 0;
  hipStream_t s = as_stream(stream);
  if (c.dtype == SVHIP_F32) {
    launch_rotary<float>(a, vec, s);
  } else {
    launch_rotary<uint16_t>(a, vec, s);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
