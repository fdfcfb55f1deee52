// svhip_paged_append into int8 pools: whole numbers of at most 127 times one power of two for a block of 16, 32 or 64 rows
// and head (paged.hpp).
//
// A block's power of two is the least that holds its new rows, and not below the one it has if older rows of the window are in
// the block; those are halved with it where it grows. So a block is one piece of work, whichever of its rows are new: a
// wave takes the block of one head, of keys or of values, reads its new rows once, keeps them rotated in registers, finds
// the largest magnitude across its lanes and writes the codes. A workgroup looks at `per_group` consecutive tokens, takes
// the blocks whose first new token is among them, forms their (cos, sin) in LDS once for all heads, and its waves share
// out (head, keys or values) of its slice of the heads.
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

// 4 values times f, rounded to nearest even and cut to the codes' range, as bytes: added to 1.5 2^23, where the step is 1, a
// whole number stands in the low bits, two's complement.
__device__ __forceinline__ uint32_t int8_codes(float a, float b, float c, float d, float f) {
  const auto code = [&](float x) __attribute__((always_inline)) {
    return __float_as_uint(__builtin_amdgcn_fmed3f(x * f, -kInt8Most, kInt8Most) + 12582912.f);
  };
  const uint32_t lo = __builtin_amdgcn_perm(code(b), code(a), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(code(d), code(c), 0x04000c0cu);
  return lo | hi;
}

// A block that gets rows.
struct Block {
  int64_t first, src[2], page, pos;  // first token; its rows' places (key, value) and its position's
  int64_t key;                       // the first new key
  int rows, older, row;              // new rows, older ones in front of them, the block's first row in its page
};

// The wave's block of one head: SIDE 0 keys, 1 values.
template <int TURN, int LPR, int kBlock, int SIDE>
__device__ __forceinline__ void hold_block(const AppendArgs& a, const Block& blk, int h, const float2* table, int shift) {
  constexpr int kRowsAtOnce = 64 / LPR, kPasses = kBlock / kRowsAtOnce > 0 ? kBlock / kRowsAtOnce : 1;
  const int lane = static_cast<int>(threadIdx.x & 63), d0 = 8 * (lane % LPR), r0 = lane / LPR;
  const bool inside = d0 < a.D;
  const uint16_t* from = SIDE == 0 ? a.key + blk.src[0] + h * a.sk_h : a.value + blk.src[1] + h * a.sv_h;
  const int64_t step = SIDE == 0 ? a.sk_n : a.sv_n;
  constexpr bool turns = SIDE == 0 && TURN != kTurnNone;
  const int partner = turns && TURN == kTurnHalf && a.runs && d0 < 2 * a.half ? (d0 < a.half ? d0 + a.half : d0 - a.half) : d0;
  float x[kPasses][8];
  float most = 0.f;
  bool odd = false;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[p][e] = 0.f;
    const int r = r0 + kRowsAtOnce * p;
    if (r < blk.rows && inside) {
      const uint16_t* row = from + r * step;
      const uint4 raw = *reinterpret_cast<const uint4*>(row + d0);
      uint4 other = raw;
      if constexpr (turns && TURN == kTurnHalf) other = *reinterpret_cast<const uint4*>(row + partner);
      unpack_run(raw, x[p]);
      if constexpr (turns) turn_run<TURN>(a, x[p], other, row, table + r * a.half, d0);
    }
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      odd |= !(fabsf(x[p][e]) < INFINITY);
      x[p][e] = x[p][e] == x[p][e] ? x[p][e] : 0.f;
    }
    most = fmaxf(most, max_run(x[p]));
  }
  if (__builtin_amdgcn_ballot_w64(odd) != 0ull) set_bad(a.pages);
  int code = block_exponent(wave_max(most));
  uint8_t* exponent = SIDE == 0 ? a.ek + blk.page * a.sek_p + h * a.sek_h + (blk.row >> shift)
                                : a.ev + blk.page * a.sev_p + h * a.sev_h + (blk.row >> shift);
  uint8_t* rows = SIDE == 0 ? static_cast<uint8_t*>(a.ck) + blk.page * a.sck_p + h * a.sck_h + blk.row * a.sck_r
                            : static_cast<uint8_t*>(a.cv) + blk.page * a.scv_p + h * a.scv_h + blk.row * a.scv_r;
  const int64_t sr = SIDE == 0 ? a.sck_r : a.scv_r;
  if (blk.older > 0) {
    const int had = __builtin_amdgcn_readfirstlane(*exponent);
    if (had >= code) {
      code = had < kInt8Top ? had : kInt8Top;
    } else {
      // The codes that are there, by the power of two that the block's has grown by (127 2^-8 and less round to 0).
      const int grown = code - had < 30 ? code - had : 30;
      const float f = exponent_value(127 - grown);
      for (int r = r0; r < blk.older; r += kRowsAtOnce) {
        if (!inside) continue;
        uint2* at = reinterpret_cast<uint2*>(rows + r * sr + d0);
        const uint2 w = *at;
        float c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? w.x : w.y) >> 8 * (e & 3)));
        *at = make_uint2(int8_codes(c[0], c[1], c[2], c[3], f), int8_codes(c[4], c[5], c[6], c[7], f));
      }
    }
  }
  if (lane == 0) *exponent = static_cast<uint8_t>(code);
  const float f = exponent_value(254 - code);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int r = r0 + kRowsAtOnce * p;
    if (r < blk.rows && inside) {
      *reinterpret_cast<uint2*>(rows + (blk.older + r) * sr + d0) =
          make_uint2(int8_codes(x[p][0], x[p][1], x[p][2], x[p][3], f), int8_codes(x[p][4], x[p][5], x[p][6], x[p][7], f));
    }
  }
}

// LPR: lanes of a row (8: head_dim up to 64). blockIdx.y: the slice of `heads` heads.
template <int TURN, int LPR, int kBlock>
__global__ __launch_bounds__(kAppendThreads) void paged_append_int8_kernel(AppendArgs a, unsigned first_group, int heads) {
  __shared__ float2 table[TURN == kTurnNone ? 1 : kBlock * kMaxPagedDim / 2];
  __shared__ Block blocks[kLeadersMost];
  __shared__ int s_count;
  constexpr int shift = kBlock == 64 ? 6 : (kBlock == 32 ? 5 : 4);
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
      } else if (i == 0 || (j & (kBlock - 1)) == 0) {
        const int older = static_cast<int>(j & (kBlock - 1));
        blk.page = page_of(a.pages, b, j);
        leads = blk.page >= 0;
        blk.first = mine;
        // packed: the row's index alone places it
        blk.src[0] = (a.tokens.cu ? 0 : b * a.sk_b) + n * a.sk_n;
        blk.src[1] = (a.tokens.cu ? 0 : b * a.sv_b) + n * a.sv_n;
        blk.pos = a.positions ? (a.tokens.cu ? 0 : b * a.sp_b) + n * a.sp_n : j;
        blk.key = j;
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
  const int count = __builtin_amdgcn_readfirstlane(s_count);
  const int h0 = static_cast<int>(blockIdx.y) * heads, h1 = h0 + heads < a.H ? h0 + heads : a.H;
  for (int i = 0; i < count; ++i) {
    const Block blk = blocks[i];
    if constexpr (TURN != kTurnNone) {
      if (i > 0) __syncthreads();  // the table is read until here
      for (int e = tid; e < blk.rows * a.half; e += kAppendThreads) {
        const int r = e / a.half, pr = e - r * a.half;
        if constexpr (TURN == kTurnAxial) {
          const int per_axis = a.half / 3, axis = pr / per_axis;
          const float* pos = static_cast<const float*>(a.positions) + blk.pos + r * a.sp_n;
          const float phase = pos[axis] * static_cast<const float*>(a.freq)[pr - axis * per_axis];
          table[e] = make_float2(bf16_round1(cosf(phase)), bf16_round1(sinf(phase)));
        } else {
          const double at = a.positions ? rotary_position(a.positions, a.wide, blk.pos + r * a.sp_n)
                                        : static_cast<double>(blk.key + r);
          table[e] = rotary_phase(at, static_cast<const double*>(a.freq)[pr], a.amplitude);
        }
      }
      __syncthreads();
    }
    for (int u = wave; u < 2 * (h1 - h0); u += kAppendThreads / 64) {
      if (u & 1) {
        hold_block<TURN, LPR, kBlock, 1>(a, blk, h0 + (u >> 1), table, shift);
      } else {
        hold_block<TURN, LPR, kBlock, 0>(a, blk, h0 + (u >> 1), table, shift);
      }
    }
  }
}

template <int TURN, int LPR>
void launch_int8(const AppendArgs& a, int shift, dim3 grid, unsigned first, int heads, hipStream_t s) {
  switch (shift) {
    case 6: paged_append_int8_kernel<TURN, LPR, 64><<<grid, kAppendThreads, 0, s>>>(a, first, heads); break;
    case 5: paged_append_int8_kernel<TURN, LPR, 32><<<grid, kAppendThreads, 0, s>>>(a, first, heads); break;
    default: paged_append_int8_kernel<TURN, LPR, 16><<<grid, kAppendThreads, 0, s>>>(a, first, heads);
  }
}

template <int TURN>
void launch_int8(const AppendArgs& a, int shift, dim3 grid, unsigned first, int heads, hipStream_t s) {
  a.D <= 64 ? launch_int8<TURN, 8>(a, shift, grid, first, heads, s) : launch_int8<TURN, 16>(a, shift, grid, first, heads, s);
}

void launch_append_int8(const AppendArgs& args, int turn, int shift, hipStream_t s) {
  AppendArgs a = args;
  // A workgroup's tokens: a block's, or a window's where it has fewer (packed: as many as leave two workgroups for every CU,
  // since single tokens, each with a block of its own, may lie side by side).
  const int64_t block = 1ll << shift, N = a.tokens.N;
  a.per_group = static_cast<int>(a.tokens.cu ? tokens_per_group(a.total, 8) : (N < block ? N : block));
  const int64_t groups = cdiv(a.total, a.per_group), blocks = a.total / block + a.tokens.B;
  // Slices of heads where the blocks are few, two heads (four waves' work) at least.
  int64_t slices = cdiv(512, blocks);
  if (slices > (a.H + 1) / 2) slices = (a.H + 1) / 2;
  const int heads = static_cast<int>(cdiv(a.H, slices));
  slices = cdiv(a.H, heads);
  in_launches(groups, [&](unsigned first, unsigned count) {
    const dim3 grid(count, static_cast<unsigned>(slices));
    switch (turn) {
      case SVHIP_ROTARY_HALF: launch_int8<kTurnHalf>(a, shift, grid, first, heads, s); break;
      case SVHIP_ROTARY_INTERLEAVED: launch_int8<kTurnInterleaved>(a, shift, grid, first, heads, s); break;
      case SVHIP_ROTARY_AXIAL: launch_int8<kTurnAxial>(a, shift, grid, first, heads, s); break;
      default: launch_int8<kTurnNone>(a, shift, grid, first, heads, s);
    }
  });
}

}  // namespace svhip
