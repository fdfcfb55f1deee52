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

extern "C" int svhip_rotary(const void* x, void* out, int dtype, const void* positions, int positions_wide,
                            const double* freq, int64_t pairs, int layout, float amplitude, int inverse, int64_t B,
                            int64_t H, int64_t N, int64_t D, int64_t sx_b, int64_t sx_h, int64_t sx_n, int64_t so_b,
                            int64_t so_h, int64_t so_n, int64_t sp_b, int64_t sp_n, void* stream) {
  const char* name = "svhip_rotary";
  clear_error();
  SVHIP_REQUIRE(B >= 0 && H >= 0 && N >= 0 && D >= 1, "%s: bad sizes", name);
  SVHIP_REQUIRE(dtype == SVHIP_F32 || dtype == SVHIP_BF16, "%s: dtype %d unsupported", name, dtype);
  SVHIP_REQUIRE(layout == SVHIP_ROTARY_HALF || layout == SVHIP_ROTARY_INTERLEAVED, "%s: layout %d unsupported", name,
                layout);
  SVHIP_REQUIRE(pairs >= 1 && pairs <= kMaxRotaryPairs && 2 * pairs <= D,
                "%s: %lld pairs do not fit head_dim %lld (at most %d)", name, (long long)pairs, (long long)D,
                kMaxRotaryPairs);
  SVHIP_REQUIRE(D <= 1 << 20 && H <= 1 << 20, "%s: sizes too large", name);
  if (B == 0 || H == 0 || N == 0) return SVHIP_OK;
  SVHIP_REQUIRE(x && out && positions && freq, "%s: null pointer", name);
  const int64_t grid = B * cdiv(N, kRotaryTokens);
  SVHIP_REQUIRE(grid < (1ll << 31), "%s: grid too large", name);
  const RotaryArgs a{x, out, positions, freq, B, H, N, D, static_cast<int>(pairs), positions_wide != 0,
                     layout == SVHIP_ROTARY_INTERLEAVED, amplitude, inverse ? -1.f : 1.f, sx_b, sx_h, sx_n, so_b, so_h,
                     so_n, sp_b, sp_n};
  hipStream_t s = as_stream(stream);
  if (dtype == SVHIP_F32) {
    rotary_kernel<float><<<static_cast<unsigned>(grid), kRotaryThreads, 0, s>>>(a);
  } else {
    rotary_kernel<uint16_t><<<static_cast<unsigned>(grid), kRotaryThreads, 0, s>>>(a);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
