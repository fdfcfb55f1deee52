// svhip_norm_rotary: queries and keys normed for each head and turned by their rotary positions (rotary.hpp) in one pass, and
// its gradient.
//
// u = x / sqrt(mean x^2 + eps), y = R(p) (w u), R the rotation (times the amplitude) of the first 2 half elements. With g =
// R(p)^T dy and c = w g: dw = sum over rows of g u, dx = (c - u mean(c u)) / sqrt(mean x^2 + eps). Sums in fp32, results rounded
// once. The gradient forms u again from x: a pass over x is read anyway, and nothing is kept between the passes.
//
// Bound: HBM, every row read once and written once (gradient: x and dy read, dx written). Workgroup = some tokens of a
// window, all heads of the queries or of the keys; the tokens' (cos, sin) go to LDS once. A group of LPR lanes carries a
// row, a lane its pairs' 16 elements (two 8-element runs, half apart in the half layout), so that the row's sums are steps
// within the group, a pair turns within its lane, and a lane's weights stay in registers. A thread's first row is on its
// way before the angles are formed, and the next one while it computes. Measured: 32 768 tokens of 16 and 4 heads of 128 in
// bf16 (336 MB) 74 us, 4.5 TB/s of a copy's 5.1, their gradient (503 MB) 117, 4.3, and 4.7 for the weights' sums; 8192 of 12
// and 12 of 64 (50 MB) 13.0, gradient 22.6; 64 tokens 5.5; fp32 141 and 209 (4.8 TB/s), 23.8 and 36. Where pairs or rows are no whole runs
// of 8 (12 pairs of 96, 10 of 80) every element is read and written by itself, 8 or 16 apart from lane to lane: 199 and 273 us,
// 169 and 244, for 54 and 85 of 16 pairs of 96. Both sides in a workgroup, the weights in LDS: 50.9 us for the 50 MB, 873 for the
// 839 MB of a result and its gradient (197 now). Rows a thread: 2, 4, 8: 18.7, 14.5, 15.5 us for the 50 MB; workgroups of a
// gradient: 768 (three a CU at once), 1024, 2048: 204, 219, 208 us for the pair.
#include "rotary.hpp"

namespace svhip {

constexpr int kNormThreads = 256;
constexpr int kNormAngles = 2048;   // angles of a workgroup at most
constexpr int kMaxNormDim = 256;
constexpr int kNormGroups = 768;    // workgroups of a gradient at most: each leaves its share of a weight's gradient

struct NormSide {
  const void *x, *dy, *w;
  void* out;      // y, or dx; null: not wanted
  int64_t sx_b, sx_h, sx_n, so_b, so_h, so_n, sd_b, sd_h, sd_n;
  int H, tokens, per_window, tiles, groups;  // tokens: of a tile; tiles: of a window, of all; workgroups of the gradient
};

struct NormArgs {
  NormSide side[2];
  const void* positions;
  const double* freq;
  int64_t sp_b, sp_n;
  int N;
  RowItems row;
  bool wide, wide_weights;
  float eps, amplitude;
  float* partial;  // gradient: [workgroups][D], or null
};

// A lane's part of a row as it lies in memory.
template <typename T, bool VEC>
struct Part {
  static constexpr int kWords = sizeof(T) / 2;
  uint4 u[kWords], v[kWords];
  __device__ __forceinline__ void load(const T* row, const Places& at) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) u[i] = v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (at.n0) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) u[i] = reinterpret_cast<const uint4*>(row + at.first)[i];
    }
    if (at.n1) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) v[i] = reinterpret_cast<const uint4*>(row + at.second)[i];
    }
  }
  static __device__ __forceinline__ void words(const uint4 (&w)[kWords], float* x) {
    if constexpr (kWords == 2) {
      x[0] = __uint_as_float(w[0].x), x[1] = __uint_as_float(w[0].y), x[2] = __uint_as_float(w[0].z);
      x[3] = __uint_as_float(w[0].w), x[4] = __uint_as_float(w[1].x), x[5] = __uint_as_float(w[1].y);
      x[6] = __uint_as_float(w[1].z), x[7] = __uint_as_float(w[1].w);
    } else {
      x[0] = __uint_as_float(w[0].x << 16), x[1] = __uint_as_float(w[0].x & 0xffff0000u);
      x[2] = __uint_as_float(w[0].y << 16), x[3] = __uint_as_float(w[0].y & 0xffff0000u);
      x[4] = __uint_as_float(w[0].z << 16), x[5] = __uint_as_float(w[0].z & 0xffff0000u);
      x[6] = __uint_as_float(w[0].w << 16), x[7] = __uint_as_float(w[0].w & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void get(float (&x)[16]) const {
    words(u, x);
    words(v, x + 8);
  }
  static __device__ __forceinline__ void store_words(T* p, const float* x) {
    if constexpr (kWords == 2) {
      reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4*>(p) =
          make_uint4(bf16_pack2(x[0], x[1]), bf16_pack2(x[2], x[3]), bf16_pack2(x[4], x[5]), bf16_pack2(x[6], x[7]));
    }
  }
  static __device__ __forceinline__ void store(T* row, const Places& at, const float (&x)[16]) {
    if (at.n0) store_words(row + at.first, x);
    if (at.n1) store_words(row + at.second, x + 8);
  }
};

// The same element by element.
template <typename T>
struct Part<T, false> {
  float x0[16];
  __device__ __forceinline__ void load(const T* row, const Places& at) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x0[i] = i < at.n0 ? to_float<T>(row[at.first + i]) : 0.f;
      x0[8 + i] = i < at.n1 ? to_float<T>(row[at.second + i]) : 0.f;
    }
  }
  __device__ __forceinline__ void get(float (&x)[16]) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = x0[i];
  }
  static __device__ __forceinline__ void one(T* p, float v) {
    if constexpr (sizeof(T) == 4) {
      *p = v;
    } else {
      *p = bf16_bits(v);
    }
  }
  static __device__ __forceinline__ void store(T* row, const Places& at, const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < at.n0) one(row + at.first + i, x[i]);
      if (i < at.n1) one(row + at.second + i, x[8 + i]);
    }
  }
};

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

// The lane's pairs turned by `angle`'s (cos, sin), sin by `sign`.
template <bool VEC, bool INTER>
__device__ __forceinline__ void turn_pairs(float (&x)[16], const float2* angle, const Places& at, float sign) {
  if (at.pairs == 0) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!VEC && i >= at.pairs) break;
    const float2 r = make_float2(angle[i].x, sign * angle[i].y);
    rotary_turn(x[INTER ? 2 * i : i], x[INTER ? 2 * i + 1 : 8 + i], r);
  }
}

__device__ __forceinline__ void load_weights(const NormArgs& a, const void* w, const Places& at, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int d = (i < 8 ? at.first : at.second - 8) + i;
    const bool there = i < 8 ? i < at.n0 : i - 8 < at.n1;
    x[i] = !there ? 0.f
                  : (!w ? 1.f : (a.wide_weights ? static_cast<const float*>(w)[d]
                                                : bf16_bits_to_float(static_cast<const uint16_t*>(w)[d])));
  }
}

// (cos, sin) of a tile's tokens.
__device__ __forceinline__ void form_angles(const NormArgs& a, float2* table, int64_t b, int n0, int tokens) {
  for (int i = threadIdx.x; i < tokens * a.row.half; i += kNormThreads) {
    const int row = i / a.row.half, pr = i - row * a.row.half;
    table[i] = rotary_phase(rotary_position(a.positions, a.wide, b * a.sp_b + (n0 + row) * a.sp_n), a.freq[pr], a.amplitude);
  }
}

// The rows of a tile that a thread's group carries, one after the other: token t of the tile, head h.
template <int LPR>
struct Walk {
  int t, h, step_t, step_h, H;
  __device__ __forceinline__ explicit Walk(int heads) {
    constexpr int kStep = kNormThreads / LPR;
    const int at = static_cast<int>(threadIdx.x) / LPR;
    H = heads;
    t = at / H;
    h = at - t * H;
    step_t = kStep / H;
    step_h = kStep - step_t * H;
  }
  __device__ __forceinline__ void next() {
    t += step_t;
    h += step_h;
    if (h >= H) {
      h -= H;
      ++t;
    }
  }
};

template <typename T, bool VEC, bool INTER, int LPR>
__global__ __launch_bounds__(kNormThreads) void norm_rotary_kernel(NormArgs a, unsigned first_group) {
  __shared__ float2 table[kNormAngles];
  const int group = static_cast<int>(first_group + blockIdx.x);
  const bool keys = group >= a.side[0].tiles;
  const NormSide s = keys ? a.side[1] : a.side[0];
  const int tile = keys ? group - a.side[0].tiles : group;
  const int window = tile / s.per_window, n0 = (tile - window * s.per_window) * s.tokens;
  const int tokens = a.N - n0 < s.tokens ? a.N - n0 : s.tokens;
  const int64_t b = window;
  const Places at = places_of<INTER>(a.row, static_cast<int>(threadIdx.x) % LPR);
  const T* x = static_cast<const T*>(s.x) + b * s.sx_b + n0 * s.sx_n;
  T* out = static_cast<T*>(s.out) + b * s.so_b + n0 * s.so_n;
  Walk<LPR> walk(s.H);
  Part<T, VEC> part;
  auto load = [&]() __attribute__((always_inline)) {
    if (walk.t < tokens) part.load(x + walk.h * s.sx_h + walk.t * s.sx_n, at);
  };
  load();
  float w[16];
  load_weights(a, s.w, at, w);
  form_angles(a, table, b, n0, tokens);
  __syncthreads();
  const float per = 1.f / static_cast<float>(a.row.D);
  while (walk.t < tokens) {  // (the same for the row's lanes)
    const int t = walk.t, h = walk.h;
    float y[16], sum = 0.f;
    part.get(y);
    walk.next();
    load();
#pragma unroll
    for (int j = 0; j < 16; ++j) sum = __builtin_fmaf(y[j], y[j], sum);
    const float unit = rsqrtf(__builtin_fmaf(lanes_sum<LPR>(sum), per, a.eps));
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = y[j] * unit * w[j];
    turn_pairs<VEC, INTER>(y, table + t * a.row.half + at.pair, at, 1.f);
    Part<T, VEC>::store(out + h * s.so_h + t * s.so_n, at, y);
  }
}

template <typename T, bool VEC, bool INTER, int LPR>
__global__ __launch_bounds__(kNormThreads) void norm_rotary_grad_kernel(NormArgs a) {
  __shared__ float2 table[kNormAngles];
  __shared__ float sums[kNormThreads / 64][LPR][16];
  const int group = static_cast<int>(blockIdx.x);
  const bool keys = group >= a.side[0].groups;
  const NormSide s = keys ? a.side[1] : a.side[0];
  const Places at = places_of<INTER>(a.row, static_cast<int>(threadIdx.x) % LPR);
  const float per = 1.f / static_cast<float>(a.row.D);
  float w[16], dw[16];
  load_weights(a, s.w, at, w);
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.f;
  for (unsigned next = keys ? group - a.side[0].groups : group; next < static_cast<unsigned>(s.tiles); next += s.groups) {
    const int tile = static_cast<int>(next), window = tile / s.per_window, n0 = (tile - window * s.per_window) * s.tokens;
    const int tokens = a.N - n0 < s.tokens ? a.N - n0 : s.tokens;
    const int64_t b = window;
    const T* x = static_cast<const T*>(s.x) + b * s.sx_b + n0 * s.sx_n;
    const T* dy = static_cast<const T*>(s.dy) + b * s.sd_b + n0 * s.sd_n;
    T* dx = static_cast<T*>(s.out) + b * s.so_b + n0 * s.so_n;
    Walk<LPR> walk(s.H);
    int t, h;
    Part<T, VEC> xs, gs;
    auto load = [&]() __attribute__((always_inline)) {
      t = walk.t;
      h = walk.h;
      if (t < tokens) {
        xs.load(x + h * s.sx_h + t * s.sx_n, at);
        gs.load(dy + h * s.sd_h + t * s.sd_n, at);
      }
      walk.next();
    };
    load();
    __syncthreads();  // the angles are read until here
    form_angles(a, table, b, n0, tokens);
    __syncthreads();
    while (t < tokens) {
      float u[16], g[16];
      const int head = h, now = t;
      xs.get(u);
      gs.get(g);
      load();
      turn_pairs<VEC, INTER>(g, table + now * a.row.half + at.pair, at, -1.f);
      float sum = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(u[i], u[i], sum);
      const float unit = rsqrtf(__builtin_fmaf(lanes_sum<LPR>(sum), per, a.eps));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        u[i] *= unit;
        dw[i] = __builtin_fmaf(g[i], u[i], dw[i]);
        g[i] *= w[i];
        dot = __builtin_fmaf(g[i], u[i], dot);
      }
      if (s.out) {
        dot = lanes_sum<LPR>(dot) * per;
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = unit * __builtin_fmaf(-u[i], dot, g[i]);
        Part<T, VEC>::store(dx + head * s.so_h + now * s.so_n, at, g);
      }
    }
  }
  if (!a.partial) return;
  // The workgroup's sums: over a wave's rows, then over its waves, in order.
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int x = LPR; x < 64; x *= 2) dw[i] += __shfl_xor(dw[i], x);
  }
  if ((threadIdx.x & 63) < LPR) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sums[threadIdx.x >> 6][threadIdx.x & 63][i] = dw[i];
  }
  __syncthreads();
  if (threadIdx.x < LPR) {
    float* to = a.partial + static_cast<int64_t>(group) * a.row.D;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = 0.f;
      for (int k = 0; k < kNormThreads / 64; ++k) v += sums[k][threadIdx.x][i];
      if (i < 8 ? i < at.n0 : i - 8 < at.n1) to[(i < 8 ? at.first : at.second - 8) + i] = v;
    }
  }
}

// The workgroups' shares of the weights' gradients summed in order: workgroup = 32 elements of a side, 32 threads each.
__global__ __launch_bounds__(1024) void norm_weight_kernel(const float* partial, int q_groups, int k_groups, int D, int blocks,
                                                           bool wide, void* dq, void* dk) {
  __shared__ float sums[32][33];
  const int side = blockIdx.x / blocks, d = (blockIdx.x - side * blocks) * 32 + threadIdx.x % 32, part = threadIdx.x / 32;
  void* to = side ? dk : dq;
  if (!to) return;
  const int first = side ? q_groups : 0, groups = side ? k_groups : q_groups;
  float v = 0.f;
  if (d < D) {
    const float* from = partial + static_cast<int64_t>(first) * D + d;
#pragma unroll 8
    for (int g = part; g < groups; g += 32) v += from[static_cast<int64_t>(g) * D];
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

template <typename T, bool VEC, bool INTER, int LPR>
void launch_norm(const NormArgs& a, bool grad, hipStream_t s) {
  if (grad) {
    const int groups = a.side[0].groups + a.side[1].groups;
    norm_rotary_grad_kernel<T, VEC, INTER, LPR><<<static_cast<unsigned>(groups), kNormThreads, 0, s>>>(a);
  } else {
    in_launches(static_cast<int64_t>(a.side[0].tiles) + a.side[1].tiles, [&](unsigned first, unsigned grid) {
      norm_rotary_kernel<T, VEC, INTER, LPR><<<grid, kNormThreads, 0, s>>>(a, first);
    });
  }
}

template <typename T, bool VEC, bool INTER>
void launch_norm(const NormArgs& a, bool grad, hipStream_t s) {
  switch (row_lanes(a.row)) {
    case 4: return launch_norm<T, VEC, INTER, 4>(a, grad, s);
    case 8: return launch_norm<T, VEC, INTER, 8>(a, grad, s);
    case 16: return launch_norm<T, VEC, INTER, 16>(a, grad, s);
    default: return launch_norm<T, VEC, INTER, 32>(a, grad, s);
  }
}

template <typename T>
void launch_norm(const NormArgs& a, bool vec, bool interleaved, bool grad, hipStream_t s) {
  if (interleaved) {
    vec ? launch_norm<T, true, true>(a, grad, s) : launch_norm<T, false, true>(a, grad, s);
  } else {
    vec ? launch_norm<T, true, false>(a, grad, s) : launch_norm<T, false, false>(a, grad, s);
  }
}

// Tokens of a tile: as many as give every thread kNormRows rows, if that leaves two workgroups for every CU.
constexpr int64_t kNormRows = 4;
int64_t norm_tokens(int64_t B, int64_t H, int64_t N, int64_t lanes, int64_t half) {
  int64_t n = kNormRows * kNormThreads / lanes / (H > 0 ? H : 1);
  if (n > kNormAngles / half) n = kNormAngles / half;
  if (n > B * N / 512) n = B * N / 512;
  if (n > N) n = N;
  return n < 1 ? 1 : n;
}

// Workgroups of a side's gradient: its share of kNormGroups by its heads.
int64_t norm_groups(int64_t tiles, int64_t H, int64_t all) {
  const int64_t most = H * kNormGroups / all > 0 ? H * kNormGroups / all : 1;
  return H == 0 ? 0 : (tiles < most ? tiles : most);
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
  const int half = static_cast<int>(c.pairs), D = static_cast<int>(c.D);
  const int blocks = static_cast<int>(cdiv(D, 32));
  hipStream_t s = as_stream(stream);
  if (c.B == 0 || c.N == 0 || c.H + c.Hk == 0) {
    // No rows: the weights' gradients are zeros.
    if (weighed) {
      norm_weight_kernel<<<2 * blocks, 1024, 0, s>>>(nullptr, 0, 0, D, blocks, c.weight_dtype == SVHIP_F32, c.dq_weight,
                                                     c.dk_weight);
      SVHIP_LAUNCHED(name);
    }
    return SVHIP_OK;
  }
  SVHIP_REQUIRE((c.H == 0 || (c.q && (grad ? c.dq != nullptr : c.out_q != nullptr))) &&
                    (c.Hk == 0 || (c.k && (grad ? c.dk != nullptr : c.out_k != nullptr))) && c.positions && c.freq,
                "%s: null pointer", name);
  // (One that fp32 rounds to 0 would make a row of zeros NaN.)
  const float eps = c.eps > 0. && c.eps < 0x1p-149 ? 0x1p-149f : static_cast<float>(c.eps);
  NormArgs a{{{c.q, c.dq, c.q_weight, c.out_q, c.sq_b, c.sq_h, c.sq_n, c.soq_b, c.soq_h, c.soq_n, c.sdq_b, c.sdq_h, c.sdq_n,
               static_cast<int>(c.H), 1, 1, 0, 0},
              {c.k, c.dk, c.k_weight, c.out_k, c.sk_b, c.sk_h, c.sk_n, c.sok_b, c.sok_h, c.sok_n, c.sdk_b, c.sdk_h, c.sdk_n,
               static_cast<int>(c.Hk), 1, 1, 0, 0}},
             c.positions, c.freq, c.sp_b, c.sp_n, static_cast<int>(c.N), row_items(D, half),
             c.positions_wide != 0, c.weight_dtype == SVHIP_F32, eps, static_cast<float>(c.amplitude),
             weighed ? static_cast<float*>(c.workspace) : nullptr};
  const int64_t run = c.dtype == SVHIP_F32 ? 4 : 8;
  bool vec = half % 8 == 0 && D % 8 == 0;
  int64_t all = 0;
  for (NormSide& side : a.side) {
    if (side.H == 0) continue;
    const auto on16 = [&](const void* p, int64_t b, int64_t h, int64_t n) {
      return reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
             (used_stride(c.B, b) | used_stride(side.H, h) | used_stride(c.N, n)) % run == 0;
    };
    vec = vec && on16(side.x, side.sx_b, side.sx_h, side.sx_n) && on16(side.out, side.so_b, side.so_h, side.so_n) &&
          (!grad || on16(side.dy, side.sd_b, side.sd_h, side.sd_n));
    const int64_t tokens = norm_tokens(c.B, side.H, c.N, row_lanes(a.row), half), per_window = cdiv(c.N, tokens);
    const int64_t tiles = c.B * per_window;
    all += tiles;
    SVHIP_REQUIRE(all < (1ll << 31), "%s: grid too large", name);
    side.tokens = static_cast<int>(tokens);
    side.per_window = static_cast<int>(per_window);
    side.tiles = static_cast<int>(tiles);
    side.groups = static_cast<int>(norm_groups(tiles, side.H, c.H + c.Hk));
  }
  const int64_t bytes = (static_cast<int64_t>(a.side[0].groups) + a.side[1].groups) * D * 4;
  SVHIP_REQUIRE(!weighed || (c.workspace && c.workspace_bytes >= bytes && reinterpret_cast<uintptr_t>(c.workspace) % 4 == 0),
                "%s: workspace too small or misaligned (%lld < %lld bytes)", name, (long long)c.workspace_bytes,
                (long long)bytes);
  const bool interleaved = c.layout == SVHIP_ROTARY_INTERLEAVED;
  c.dtype == SVHIP_F32 ? launch_norm<float>(a, vec, interleaved, grad, s) : launch_norm<uint16_t>(a, vec, interleaved, grad, s);
  if (weighed) {
    norm_weight_kernel<<<2 * blocks, 1024, 0, s>>>(a.partial, a.side[0].groups, a.side[1].groups, D, blocks, a.wide_weights,
                                                   c.dq_weight, c.dk_weight);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}

}  // namespace svhip

using namespace svhip;

extern "C" int svhip_norm_rotary(const svhip_norm_rotary_args* args, void* stream) {
  return norm_rotary("svhip_norm_rotary", args, false, stream);
}

extern "C" size_t svhip_norm_rotary_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t D) {
  if (B < 1 || H < 0 || Hk < 0 || H + Hk < 1 || N < 1 || D < 1 || D > kMaxNormDim) return 0;
  // (A window of one token has a tile at least, and a side one workgroup.)
  const int64_t most = B < kNormGroups / N + 1 ? B * N + 1 : kNormGroups;
  return static_cast<size_t>(2 * (most < kNormGroups ? most : kNormGroups) * D * 4);
}

extern "C" int svhip_norm_rotary_grad(const svhip_norm_rotary_args* args, void* stream) {
  return norm_rotary("svhip_norm_rotary_grad", args, true, stream);
}
