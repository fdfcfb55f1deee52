// svhip_norm_rotary: queries and keys normed for each head and turned by their rotary positions (rotary.hpp) in one pass, and
// its gradient.
//
// u = x / sqrt(mean x^2 + eps), y = R(p) (w u), R the rotation (times the amplitude) of the first 2 half elements. With g =
// R(p)^T dy and c = w g: dw = sum over rows of g u, dx = (c - u mean(c u)) / sqrt(mean x^2 + eps). Sums in fp32, results rounded
// once. The gradient forms u again from x: a pass over x is read anyway, and nothing is kept between the passes.
//
// Bound: HBM, every row read once and written once (gradient: x and dy read, dx written). Workgroup = up to kNormTokens
// tokens of a window, all heads of queries and keys; their (cos, sin) go to LDS once. A group of LPR lanes carries a row, a
// lane its pairs' 16 elements (two 8-element runs, half apart in the half layout), so that the row's sums are steps within
// the group and a pair turns within its lane.
#include "rotary.hpp"

namespace svhip {

constexpr int kNormThreads = 256;
constexpr int kNormTokens = 8;
constexpr int kNormAhead = 2;      // rows that a thread has in flight
constexpr int kMaxNormDim = 256;
constexpr int kNormGroups = 1024;  // workgroups of a gradient at most: each leaves its share of the weights' gradients

struct NormSide {
  const void *x, *dy, *w;
  void* out;      // y, or dx; null: not wanted
  int64_t sx_b, sx_h, sx_n, so_b, so_h, so_n, sd_b, sd_h, sd_n;
  int H;
};

struct NormArgs {
  NormSide side[2];
  const void* positions;
  const double* freq;
  int64_t B, N, sp_b, sp_n, tiles;  // tiles: groups of `tokens` tokens, of every window
  int D, half, turning, items, tokens;
  bool wide, interleaved, wide_weights;
  float eps, amplitude;
  float* partial;  // gradient: [workgroups][2][D], or null
};

// A lane's 16 elements of a row: 8 pairs, or 16 that are kept. Item e < turning has pairs 8 e ..
template <bool VEC>
struct Places {
  int first, second;  // of elements 0 .. 7 and 8 .. 15
  int n0, n1;         // how many of each there are (VEC: 0 or 8)
  int step;           // from element to element (1; interleaved pairs lie side by side like kept ones)
  int pair;           // first pair, or -1
  __device__ __forceinline__ Places(const NormArgs& a, int e) {
    if (e >= a.items) {
      first = second = n0 = n1 = 0;
      pair = -1;
      return;
    }
    const bool turns = e < a.turning;
    pair = turns ? 8 * e : -1;
    const int pairs = a.half - 8 * e < 8 ? a.half - 8 * e : 8;
    if (turns && !a.interleaved) {
      first = 8 * e;
      second = a.half + 8 * e;
      n0 = n1 = pairs;
    } else {
      first = turns ? 16 * e : 2 * a.half + 16 * (e - a.turning);
      second = first + 8;
      const int n = turns ? 2 * pairs : (a.D - first < 16 ? a.D - first : 16);
      n0 = n < 8 ? n : 8;
      n1 = n - n0;
    }
  }
};

template <typename T>
__device__ __forceinline__ void load_run(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    const float4 u = *reinterpret_cast<const float4*>(p), v = *reinterpret_cast<const float4*>(p + 4);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_row(const T* row, const Places<VEC>& at, float (&x)[16]) {
  if constexpr (VEC) {
    if (at.n0) load_run<T>(row + at.first, x);
    if (at.n1) load_run<T>(row + at.second, x + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < at.n0) x[i] = to_float<T>(row[at.first + i]);
      if (i < at.n1) x[8 + i] = to_float<T>(row[at.second + i]);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_one(T* p, float v) {
  if constexpr (sizeof(T) == 4) {
    *p = v;
  } else {
    *p = bf16_bits(v);
  }
}

template <typename T>
__device__ __forceinline__ void store_run(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(bf16_pack2(x[0], x[1]), bf16_pack2(x[2], x[3]), bf16_pack2(x[4], x[5]), bf16_pack2(x[6], x[7]));
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_row(T* row, const Places<VEC>& at, const float (&x)[16]) {
  if constexpr (VEC) {
    if (at.n0) store_run<T>(row + at.first, x);
    if (at.n1) store_run<T>(row + at.second, x + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < at.n0) store_one<T>(row + at.first + i, x[i]);
      if (i < at.n1) store_one<T>(row + at.second + i, x[8 + i]);
    }
  }
}

// Sum over the row's LPR lanes, in all of them.
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp_f<0xB1>(v);
  v += dpp_f<0x4E>(v);
  if constexpr (LPR >= 8) v += dpp_f<0x141>(v);
  if constexpr (LPR >= 16) v += dpp_f<0x140>(v);
  if constexpr (LPR >= 32) v += __shfl_xor(v, 16);
  return v;
}

// The lane's pairs turned by r = (cos, sin), sin by `sign`.
__device__ __forceinline__ void turn_pairs(const NormArgs& a, float (&x)[16], const float2* angle, int pairs, float sign) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float2 r = make_float2(1.f, 0.f);
    if (i < pairs) r = angle[i];
    r.y *= sign;
    if (a.interleaved) {
      rotary_turn(x[2 * i], x[2 * i + 1], r);
    } else {
      rotary_turn(x[i], x[8 + i], r);
    }
  }
}

// The weights of both sides into LDS as fp32 (ones where there are none).
__device__ __forceinline__ void load_weights(const NormArgs& a, float (*weights)[kMaxNormDim]) {
  for (int i = threadIdx.x; i < 2 * a.D; i += kNormThreads) {
    const int side = i >= a.D, d = i - side * a.D;
    const void* w = a.side[side].w;
    weights[side][d] = !w ? 1.f
                          : (a.wide_weights ? static_cast<const float*>(w)[d]
                                            : bf16_bits_to_float(static_cast<const uint16_t*>(w)[d]));
  }
}

// (cos, sin) of the tile's tokens.
__device__ __forceinline__ void load_angles(const NormArgs& a, float2* table, int64_t b, int64_t n0, int tokens) {
  for (int i = threadIdx.x; i < tokens * a.half; i += kNormThreads) {
    const int row = i / a.half, pr = i - row * a.half;
    table[i] = rotary_phase(rotary_position(a.positions, a.wide, b * a.sp_b + (n0 + row) * a.sp_n), a.freq[pr], a.amplitude);
  }
}

template <bool VEC>
__device__ __forceinline__ void weights_at(const float* weights, const Places<VEC>& at, float (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = i < at.n0 ? weights[at.first + i] : 0.f;
    w[8 + i] = i < at.n1 ? weights[at.second + i] : 0.f;
  }
}

template <typename T, bool VEC, int LPR>
__global__ __launch_bounds__(kNormThreads) void norm_rotary_kernel(NormArgs a, unsigned first_group) {
  __shared__ float2 table[kNormTokens * kMaxRotaryPairs];
  __shared__ float weights[2][kMaxNormDim];
  const unsigned per_window = static_cast<unsigned>((a.N + a.tokens - 1) / a.tokens);
  const unsigned group = first_group + blockIdx.x, window = group / per_window;
  const int64_t b = window, n0 = static_cast<int64_t>(group - window * per_window) * a.tokens;
  const int tokens = static_cast<int>(a.N - n0 < a.tokens ? a.N - n0 : a.tokens);
  const int e = static_cast<int>(threadIdx.x) % LPR, H0 = a.side[0].H, H = H0 + a.side[1].H;
  const Places<VEC> at(a, e);
  constexpr int kStep = kNormThreads / LPR;
  const int step_t = kStep / H, step_h = kStep - step_t * H;
  int t = static_cast<int>(threadIdx.x) / LPR / H, h = static_cast<int>(threadIdx.x) / LPR - t * H;
  struct Row {
    int t, h;
    float x[16];
  };
  Row rows[kNormAhead];
  auto load = [&](Row& r) __attribute__((always_inline)) {
    r.t = t;
    r.h = h;
#pragma unroll
    for (int i = 0; i < 16; ++i) r.x[i] = 0.f;
    if (t < tokens) {
      const NormSide& s = a.side[h < H0 ? 0 : 1];
      load_row<T, VEC>(static_cast<const T*>(s.x) + b * s.sx_b + (h < H0 ? h : h - H0) * s.sx_h + (n0 + t) * s.sx_n, at, r.x);
    }
    t += step_t;
    h += step_h;
    if (h >= H) {
      h -= H;
      ++t;
    }
  };
#pragma unroll
  for (int i = 0; i < kNormAhead; ++i) load(rows[i]);
  load_weights(a, weights);
  load_angles(a, table, b, n0, tokens);
  __syncthreads();
  const float per = 1.f / static_cast<float>(a.D);
  while (rows[0].t < tokens) {
#pragma unroll
    for (int i = 0; i < kNormAhead; ++i) {
      Row& r = rows[i];
      if (r.t >= tokens) break;  // (the same for the row's lanes)
      const int side = r.h < H0 ? 0 : 1;
      const NormSide& s = a.side[side];
      float sum = 0.f, w[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) sum = __builtin_fmaf(r.x[j], r.x[j], sum);
      const float unit = rsqrtf(__builtin_fmaf(lanes_sum<LPR>(sum), per, a.eps));
      weights_at<VEC>(weights[side], at, w);
#pragma unroll
      for (int j = 0; j < 16; ++j) r.x[j] = r.x[j] * unit * w[j];
      if (at.pair >= 0) turn_pairs(a, r.x, table + r.t * a.half + at.pair, a.half - at.pair, 1.f);
      store_row<T, VEC>(static_cast<T*>(s.out) + b * s.so_b + (side ? r.h - H0 : r.h) * s.so_h + (n0 + r.t) * s.so_n, at, r.x);
    }
#pragma unroll
    for (int i = 0; i < kNormAhead; ++i) load(rows[i]);
  }
}

template <typename T, bool VEC, int LPR>
__global__ __launch_bounds__(kNormThreads) void norm_rotary_grad_kernel(NormArgs a) {
  __shared__ float2 table[kNormTokens * kMaxRotaryPairs];
  __shared__ float weights[2][kMaxNormDim];
  __shared__ float sums[kNormThreads / 64][LPR][16];
  const unsigned per_window = static_cast<unsigned>((a.N + a.tokens - 1) / a.tokens);
  const int e = static_cast<int>(threadIdx.x) % LPR;
  const Places<VEC> at(a, e);
  constexpr int kStep = kNormThreads / LPR;
  const float per = 1.f / static_cast<float>(a.D);
  load_weights(a, weights);
  float dw[2][16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[0][i] = dw[1][i] = 0.f;
  for (unsigned group = blockIdx.x; group < static_cast<unsigned>(a.tiles); group += gridDim.x) {
    const unsigned window = group / per_window;
    const int64_t b = window, n0 = static_cast<int64_t>(group - window * per_window) * a.tokens;
    const int tokens = static_cast<int>(a.N - n0 < a.tokens ? a.N - n0 : a.tokens);
    __syncthreads();  // the angles are read until here
    load_angles(a, table, b, n0, tokens);
    __syncthreads();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const NormSide& s = a.side[side];
      const int H = s.H;
      if (H == 0) continue;
      float w[16];
      weights_at<VEC>(weights[side], at, w);
      const int step_t = kStep / H, step_h = kStep - step_t * H;
      int t = static_cast<int>(threadIdx.x) / LPR / H, h = static_cast<int>(threadIdx.x) / LPR - t * H;
      while (t < tokens) {
        float x[16], g[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = g[i] = 0.f;
        load_row<T, VEC>(static_cast<const T*>(s.x) + b * s.sx_b + h * s.sx_h + (n0 + t) * s.sx_n, at, x);
        load_row<T, VEC>(static_cast<const T*>(s.dy) + b * s.sd_b + h * s.sd_h + (n0 + t) * s.sd_n, at, g);
        float sum = 0.f, dot = 0.f;
        if (at.pair >= 0) turn_pairs(a, g, table + t * a.half + at.pair, a.half - at.pair, -1.f);
#pragma unroll
        for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(x[i], x[i], sum);
        const float unit = rsqrtf(__builtin_fmaf(lanes_sum<LPR>(sum), per, a.eps));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] *= unit;
          dw[side][i] = __builtin_fmaf(g[i], x[i], dw[side][i]);
          g[i] *= w[i];
          dot = __builtin_fmaf(g[i], x[i], dot);
        }
        dot = lanes_sum<LPR>(dot) * per;
        if (s.out) {
#pragma unroll
          for (int i = 0; i < 16; ++i) g[i] = unit * __builtin_fmaf(-x[i], dot, g[i]);
          store_row<T, VEC>(static_cast<T*>(s.out) + b * s.so_b + h * s.so_h + (n0 + t) * s.so_n, at, g);
        }
        t += step_t;
        h += step_h;
        if (h >= H) {
          h -= H;
          ++t;
        }
      }
    }
  }
  if (!a.partial) return;
  // The workgroup's sums: over a wave's rows, then over its waves, in order.
#pragma unroll
  for (int side = 0; side < 2; ++side) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int x = LPR; x < 64; x *= 2) dw[side][i] += __shfl_xor(dw[side][i], x);
    }
    __syncthreads();
    if ((threadIdx.x & 63) < LPR) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[threadIdx.x >> 6][e][i] = dw[side][i];
    }
    __syncthreads();
    if (threadIdx.x < LPR) {
      float* to = a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + side) * a.D;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = 0.f;
        for (int k = 0; k < kNormThreads / 64; ++k) v += sums[k][e][i];
        if (i < 8 ? i < at.n0 : i - 8 < at.n1) to[(i < 8 ? at.first : at.second - 8) + i] = v;
      }
    }
  }
}

// The workgroups' shares of the weights' gradients summed in order: workgroup = 32 elements of a side, 32 threads each.
__global__ __launch_bounds__(1024) void norm_weight_kernel(const float* partial, int groups, int D, int tiles, bool wide,
                                                           void* dq, void* dk) {
  __shared__ float sums[32][33];
  const int side = blockIdx.x / tiles, d = (blockIdx.x - side * tiles) * 32 + threadIdx.x % 32, part = threadIdx.x / 32;
  void* to = side ? dk : dq;
  if (!to) return;
  float v = 0.f;
  if (d < D) {
    const float* from = partial + static_cast<int64_t>(side) * D + d;
#pragma unroll 8
    for (int g = part; g < groups; g += 32) v += from[static_cast<int64_t>(g) * 2 * D];
  }
  sums[part][threadIdx.x % 32] = v;
  __syncthreads();
  if (part > 0 || d >= D) return;
  v = 0.f;
  for (int i = 0; i < 32; ++i) v += sums[i][threadIdx.x];
  if (wide) {
    static_cast<float*>(to)[d] = v;
  } else {
    static_cast<uint16_t*>(to)[d] = bf16_bits(v);
  }
}

template <typename T, bool VEC, int LPR>
void launch_norm(const NormArgs& a, int64_t grad_groups, hipStream_t s) {
  if (grad_groups > 0) {
    norm_rotary_grad_kernel<T, VEC, LPR><<<static_cast<unsigned>(grad_groups), kNormThreads, 0, s>>>(a);
  } else {
    in_launches(a.tiles, [&](unsigned first, unsigned grid) {
      norm_rotary_kernel<T, VEC, LPR><<<grid, kNormThreads, 0, s>>>(a, first);
    });
  }
}

template <typename T, bool VEC>
void launch_norm(const NormArgs& a, int64_t grad_groups, hipStream_t s) {
  if (a.items <= 4) {
    launch_norm<T, VEC, 4>(a, grad_groups, s);
  } else if (a.items <= 8) {
    launch_norm<T, VEC, 8>(a, grad_groups, s);
  } else if (a.items <= 16) {
    launch_norm<T, VEC, 16>(a, grad_groups, s);
  } else {
    launch_norm<T, VEC, 32>(a, grad_groups, s);
  }
}

int64_t norm_tokens(int64_t B, int64_t N) { return tokens_per_group(B * N, kNormTokens); }

int64_t norm_grad_groups(int64_t B, int64_t N) {
  const int64_t tiles = B * cdiv(N, norm_tokens(B, N));
  return tiles < kNormGroups ? tiles : kNormGroups;
}

int norm_rotary(const char* name, const svhip_norm_rotary_args* args, bool grad, void* stream) {
  clear_error();
  SVHIP_REQUIRE(args, "%s: null arguments", name);
  const svhip_norm_rotary_args& c = *args;
  SVHIP_REQUIRE(c.B >= 0 && c.B < (1ll << 31) && c.N >= 0 && c.N < (1ll << 31) && c.H >= 0 && c.Hk >= 0 && c.H <= 1 << 20 &&
                    c.Hk <= 1 << 20, "%s: bad sizes", name);
  SVHIP_REQUIRE(c.D >= 2 && c.D <= kMaxNormDim, "%s: head_dim %lld unsupported (2 to %d)", name, (long long)c.D, kMaxNormDim);
  SVHIP_REQUIRE((c.dtype == SVHIP_F32 || c.dtype == SVHIP_BF16) && (c.weight_dtype == SVHIP_F32 || c.weight_dtype == SVHIP_BF16),
                "%s: dtype %d of rows or %d of weights unsupported", name, (int)c.dtype, (int)c.weight_dtype);
  SVHIP_REQUIRE(c.layout == SVHIP_ROTARY_HALF || c.layout == SVHIP_ROTARY_INTERLEAVED, "%s: layout %d unsupported", name,
                (int)c.layout);
  SVHIP_REQUIRE(c.pairs >= 1 && c.pairs <= kMaxRotaryPairs && 2 * c.pairs <= c.D, "%s: %lld pairs do not fit head_dim %lld", name,
                (long long)c.pairs, (long long)c.D);
  SVHIP_REQUIRE(c.eps >= 0. && c.eps < INFINITY, "%s: eps must be 0 or more and finite", name);
  const bool weighed = grad && (c.dq_weight || c.dk_weight);
  const int64_t groups = c.B * c.N > 0 ? norm_grad_groups(c.B, c.N) : 0, bytes = groups * 2 * c.D * 4;
  if (c.B == 0 || c.N == 0 || c.H + c.Hk == 0) {
    // No rows: the weights' gradients are zeros.
    hipStream_t s = as_stream(stream);
    const int tiles = static_cast<int>(cdiv(c.D, 32));
    if (weighed) {
      norm_weight_kernel<<<2 * tiles, 1024, 0, s>>>(nullptr, 0, static_cast<int>(c.D), tiles, c.weight_dtype == SVHIP_F32,
                                                    c.dq_weight, c.dk_weight);
      SVHIP_LAUNCHED(name);
    }
    return SVHIP_OK;
  }
  SVHIP_REQUIRE((c.H == 0 || (c.q && (grad ? c.dq != nullptr : c.out_q != nullptr))) &&
                    (c.Hk == 0 || (c.k && (grad ? c.dk != nullptr : c.out_k != nullptr))) && c.positions && c.freq,
                "%s: null pointer", name);
  SVHIP_REQUIRE(!weighed || (c.workspace && c.workspace_bytes >= bytes && reinterpret_cast<uintptr_t>(c.workspace) % 4 == 0),
                "%s: workspace too small or misaligned (%lld < %lld bytes)", name, (long long)c.workspace_bytes,
                (long long)bytes);
  const int64_t tokens = norm_tokens(c.B, c.N), tiles = c.B * cdiv(c.N, tokens);
  SVHIP_REQUIRE(tiles < (1ll << 31), "%s: grid too large", name);
  const int half = static_cast<int>(c.pairs), D = static_cast<int>(c.D), turning = (half + 7) / 8;
  const NormArgs a{{{c.q, c.dq, c.q_weight, c.out_q, c.sq_b, c.sq_h, c.sq_n, c.soq_b, c.soq_h, c.soq_n, c.sdq_b, c.sdq_h, c.sdq_n,
                     static_cast<int>(c.H)},
                    {c.k, c.dk, c.k_weight, c.out_k, c.sk_b, c.sk_h, c.sk_n, c.sok_b, c.sok_h, c.sok_n, c.sdk_b, c.sdk_h, c.sdk_n,
                     static_cast<int>(c.Hk)}},
                   c.positions, c.freq, c.B, c.N, c.sp_b, c.sp_n, tiles, D, half, turning,
                   turning + (D - 2 * half + 15) / 16, static_cast<int>(tokens), c.positions_wide != 0,
                   c.layout == SVHIP_ROTARY_INTERLEAVED, c.weight_dtype == SVHIP_F32, static_cast<float>(c.eps),
                   static_cast<float>(c.amplitude), weighed ? static_cast<float*>(c.workspace) : nullptr};
  const int64_t run = c.dtype == SVHIP_F32 ? 4 : 8;
  bool vec = half % 8 == 0 && D % 8 == 0;
  for (const NormSide& s : a.side) {
    if (s.H == 0) continue;
    const auto on16 = [&](const void* p, int64_t b, int64_t h, int64_t n) {
      return reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
             (used_stride(c.B, b) | used_stride(s.H, h) | used_stride(c.N, n)) % run == 0;
    };
    vec = vec && on16(s.x, s.sx_b, s.sx_h, s.sx_n) && on16(s.out, s.so_b, s.so_h, s.so_n) &&
          (!grad || on16(s.dy, s.sd_b, s.sd_h, s.sd_n));
  }
  hipStream_t s = as_stream(stream);
  const int64_t launched = grad ? groups : 0;
  if (c.dtype == SVHIP_F32) {
    vec ? launch_norm<float, true>(a, launched, s) : launch_norm<float, false>(a, launched, s);
  } else {
    vec ? launch_norm<uint16_t, true>(a, launched, s) : launch_norm<uint16_t, false>(a, launched, s);
  }
  if (weighed) {
    const int blocks = static_cast<int>(cdiv(c.D, 32));
    norm_weight_kernel<<<2 * blocks, 1024, 0, s>>>(a.partial, static_cast<int>(groups), D, blocks, a.wide_weights, c.dq_weight,
                                                   c.dk_weight);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}

}  // namespace svhip

using namespace svhip;

extern "C" int svhip_norm_rotary(const svhip_norm_rotary_args* args, void* stream) {
  return norm_rotary("svhip_norm_rotary", args, false, stream);
}

extern "C" size_t svhip_norm_rotary_workspace_bytes(int64_t B, int64_t N, int64_t D) {
  if (B < 1 || B >= 1ll << 31 || N < 1 || N >= 1ll << 31 || D < 1 || D > kMaxNormDim) return 0;
  return static_cast<size_t>(norm_grad_groups(B, N) * 2 * D * 4);
}

extern "C" int svhip_norm_rotary_grad(const svhip_norm_rotary_args* args, void* stream) {
  return norm_rotary("svhip_norm_rotary_grad", args, true, stream);
}
