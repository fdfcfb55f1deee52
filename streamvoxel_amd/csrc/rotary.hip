// svhip_rotary: rotary positions of activations [B, H, N, D] (rotary.hpp), and with `inverse` the gradient: the transposed
// rotation, sin negated.
//
// Bound: HBM, every element read and written once (3 operations each). Workgroup = (window, kRotaryTokens tokens), all
// heads: the tile's (cos, sin) of every (token, pair) go to LDS once, since they are the same for every head, and a thread
// then turns runs of 16 bytes; its first loads are in flight while the table is formed.
#include "rotary.hpp"

namespace svhip {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 8;

struct RotaryArgs {
  const void* x;
  void* out;
  const void* positions;
  const double* freq;
  int64_t B, H, N, D;
  int half;
  bool wide, interleaved;
  float amplitude, sign;
  int64_t sx_b, sx_h, sx_n, so_b, so_h, so_n, sp_b, sp_n;
};

template <typename T>
__device__ __forceinline__ void store_as(T* p, float v) {
  if constexpr (sizeof(T) == 4) {
    *p = v;
  } else {
    *p = bf16_bits(v);
  }
}

// An item is one pair, or one element past the pairs.
template <typename T>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 table[kRotaryTokens * kMaxRotaryPairs];
  const int64_t tiles = cdiv(a.N, kRotaryTokens);
  const int64_t b = blockIdx.x / tiles, n0 = (blockIdx.x % tiles) * kRotaryTokens;
  const int tokens = static_cast<int>(a.N - n0 < kRotaryTokens ? a.N - n0 : kRotaryTokens);
  for (int i = threadIdx.x; i < tokens * a.half; i += kRotaryThreads) {
    const int t = i / a.half, pr = i - t * a.half;
    const double p = rotary_position(a.positions, a.wide, b * a.sp_b + (n0 + t) * a.sp_n);
    float2 r = rotary_phase(p, a.freq[pr], a.amplitude);
    r.y *= a.sign;
    table[i] = r;
  }
  __syncthreads();
  const int per_row = static_cast<int>(a.D) - a.half, H = static_cast<int>(a.H);
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(tokens) * H * per_row; i += kRotaryThreads) {
    const int e = static_cast<int>(i % per_row), th = static_cast<int>(i / per_row);
    const int h = th % H, t = th / H;
    const T* src = static_cast<const T*>(a.x) + b * a.sx_b + h * a.sx_h + (n0 + t) * a.sx_n;
    T* dst = static_cast<T*>(a.out) + b * a.so_b + h * a.so_h + (n0 + t) * a.so_n;
    if (e < a.half) {
      const int i0 = a.interleaved ? 2 * e : e, i1 = a.interleaved ? 2 * e + 1 : e + a.half;
      float u = to_float<T>(src[i0]), v = to_float<T>(src[i1]);
      rotary_turn(u, v, table[t * a.half + e]);
      store_as<T>(dst + i0, u);
      store_as<T>(dst + i1, v);
    } else {
      dst[e + a.half] = src[e + a.half];
    }
  }
}

}  // namespace svhip

using namespace svhip;

extern "C" int svhip_rotary(const svhip_rotary_args* args, void* stream) {
  const char* name = "svhip_rotary";
  clear_error();
  SVHIP_REQUIRE(args, "%s: null arguments", name);
  const svhip_rotary_args& c = *args;
  SVHIP_REQUIRE(c.B >= 0 && c.H >= 0 && c.N >= 0 && c.D >= 1, "%s: bad sizes", name);
  SVHIP_REQUIRE(c.dtype == SVHIP_F32 || c.dtype == SVHIP_BF16, "%s: dtype %d unsupported", name, (int)c.dtype);
  SVHIP_REQUIRE(c.layout == SVHIP_ROTARY_HALF || c.layout == SVHIP_ROTARY_INTERLEAVED, "%s: layout %d unsupported", name,
                (int)c.layout);
  SVHIP_REQUIRE(c.pairs >= 1 && c.pairs <= kMaxRotaryPairs && 2 * c.pairs <= c.D,
                "%s: %lld pairs do not fit head_dim %lld (at most %d)", name, (long long)c.pairs, (long long)c.D,
                kMaxRotaryPairs);
  SVHIP_REQUIRE(c.D <= 1 << 20 && c.H <= 1 << 20, "%s: sizes too large", name);
  if (c.B == 0 || c.H == 0 || c.N == 0) return SVHIP_OK;
  SVHIP_REQUIRE(c.x && c.out && c.positions && c.freq, "%s: null pointer", name);
  const int64_t grid = c.B * cdiv(c.N, kRotaryTokens);
  SVHIP_REQUIRE(grid < (1ll << 31), "%s: grid too large", name);
  const RotaryArgs a{c.x, c.out, c.positions, c.freq, c.B, c.H, c.N, c.D, static_cast<int>(c.pairs),
                     c.positions_wide != 0, c.layout == SVHIP_ROTARY_INTERLEAVED, static_cast<float>(c.amplitude),
                     c.inverse ? -1.f : 1.f, c.sx_b, c.sx_h, c.sx_n, c.so_b, c.so_h, c.so_n, c.sp_b, c.sp_n};
  hipStream_t s = as_stream(stream);
  if (c.dtype == SVHIP_F32) {
    rotary_kernel<float><<<static_cast<unsigned>(grid), kRotaryThreads, 0, s>>>(a);
  } else {
    rotary_kernel<uint16_t><<<static_cast<unsigned>(grid), kRotaryThreads, 0, s>>>(a);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
