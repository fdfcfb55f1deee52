// svhip_paged_append: the new tokens' keys and values into their rows of a paged cache (paged.hpp), the keys rotated
// on the way: rotary positions (rotary.hpp, fp32, rounded once to the cache's type), or the three-axis rotation of
// svhip_axial_rope with its roundings (the phase one fp32 product; sin, cos, every product and sum rounded to bf16).
//
// Bound: HBM, the rows read once and written once. Workgroup = up to kAppendTokens tokens, all heads: where each
// token goes and its (cos, sin) are the same for every head and go to LDS once; a group of 8 or 16 lanes then carries
// a (token, head) row, 16 bytes of it a lane, so that an e4m3 row's largest magnitude is a reduction within the
// group. A thread's first rows are on their way before the chain length -> page -> positions -> table, which a launch
// of few tokens waits for. Measured: 32 ragged chunks of up to 1024 tokens, 8 x 128, into e4m3 pages of 16 (109 MB)
// 26.7 us, 4.1 TB/s (4 tokens a workgroup 31.9, 16: 26.5); 8480 tokens of 8 x 48 with three-axis positions (26 MB)
// 8.7 us (4: 9.9, 16: 9.6); 64 tokens of 16 x 64 4.1 us (eight in a workgroup 5.7). Element by element: 68, 22 and 19
// us. Pairs that lie across the 8 elements of a lane read their partners one by one: 8 x 1024 tokens of 12 x 64, 30
// pairs 13.9 us for 10.6 of 32 (31 interleaved 13.7 for 10.2, e4m3 13.4 for 11.4).
#include "paged_append.hpp"

namespace svhip {

__device__ __forceinline__ uint2 e4m3_run(const float (&x)[8], float f) {
  uint32_t w[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * g] * f, x[4 * g + 1] * f, 0, false);
    w[g] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * g + 2] * f, x[4 * g + 3] * f, lo, true));
  }
  return make_uint2(w[0], w[1]);
}

// LPR: lanes of a row (8: head_dim up to 64).
template <int TURN, bool FP8, int LPR>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(AppendArgs a, unsigned first_group) {
  __shared__ float2 table[kAppendTokens * kMaxPagedDim / 2];
  __shared__ int64_t s_src[kAppendTokens][2], s_page[kAppendTokens], s_pos[kAppendTokens];
  __shared__ int s_row[kAppendTokens];
  const int64_t t0 = static_cast<int64_t>(first_group + blockIdx.x) * a.per_group;
  const int tokens = static_cast<int>(a.total - t0 < a.per_group ? a.total - t0 : a.per_group);
  const int tid = static_cast<int>(threadIdx.x), H = a.H;
  const int64_t mine = t0 + tid;                     // threads below `tokens`: their token, its window and place there
  int64_t b = 0, n = mine;
  if (tid < tokens) {
    if (!a.tokens.cu) {
      b = static_cast<int>(mine) / static_cast<int>(a.tokens.N);
      n = mine - b * a.tokens.N;
    }
    s_src[tid][0] = b * a.sk_b + n * a.sk_n;         // packed: b is 0 here
    s_src[tid][1] = b * a.sv_b + n * a.sv_n;
  }
  __syncthreads();
  const int d0 = 8 * (tid % LPR), first = tid / LPR;
  const bool inside = d0 < a.D;
  const int partner = TURN == kTurnHalf && a.runs && d0 < 2 * a.half ? (d0 < a.half ? d0 + a.half : d0 - a.half) : d0;
  constexpr int kStep = kAppendThreads / LPR;
  const int step_t = kStep / H, step_h = kStep - step_t * H;
  int t = first / H, h = first - t * H;
  struct Row {
    int t, h;
    uint4 k, other, v;
  };
  Row rows[kAppendAhead];
  auto load = [&](Row& r) __attribute__((always_inline)) {
    r.t = t;
    r.h = h;
    if (t < tokens && inside) {
      const uint16_t* key = a.key + s_src[t][0] + h * a.sk_h;
      r.k = *reinterpret_cast<const uint4*>(key + d0);
      if constexpr (TURN == kTurnHalf) r.other = *reinterpret_cast<const uint4*>(key + partner);
      r.v = *reinterpret_cast<const uint4*>(a.value + s_src[t][1] + h * a.sv_h + d0);
    }
    t += step_t;
    h += step_h;
    if (h >= H) {
      h -= H;
      ++t;
    }
  };
#pragma unroll
  for (int i = 0; i < kAppendAhead; ++i) load(rows[i]);

  if (tid < tokens) {
    int64_t page = -1;
    if (a.tokens.cu) b = window_of(a.tokens, mine);
    if (b >= 0) {
      int64_t start, count;
      window_tokens(a.tokens, b, start, count);
      const int64_t j = a.pages.lengths[b] - a.before - count + (mine - start);
      if (j < 0 || j >= a.pages.max_pages << a.pages.shift) {
        set_bad(a.pages);
      } else {
        page = page_of(a.pages, b, j);
      }
      s_pos[tid] = a.positions ? (a.tokens.cu ? 0 : b * a.sp_b) + n * a.sp_n : j;
      s_row[tid] = static_cast<int>(j & ((1ll << a.pages.shift) - 1));
    }
    s_page[tid] = page;
  }
  __syncthreads();
  if constexpr (TURN != kTurnNone) {
    for (int i = tid; i < tokens * a.half; i += kAppendThreads) {
      const int at = i / a.half, pr = i - at * a.half;
      if (s_page[at] < 0) continue;
      if constexpr (TURN == kTurnAxial) {
        const int per_axis = a.half / 3, axis = pr / per_axis;
        const float* pos = static_cast<const float*>(a.positions) + s_pos[at];
        const float phase = pos[axis] * static_cast<const float*>(a.freq)[pr - axis * per_axis];
        table[i] = make_float2(bf16_round1(cosf(phase)), bf16_round1(sinf(phase)));
      } else {
        const double p = a.positions ? rotary_position(a.positions, a.wide, s_pos[at]) : static_cast<double>(s_pos[at]);
        table[i] = rotary_phase(p, static_cast<const double*>(a.freq)[pr], a.amplitude);
      }
    }
    __syncthreads();
  }
  while (rows[0].t < tokens) {
#pragma unroll
    for (int i = 0; i < kAppendAhead; ++i) {
      const Row& r = rows[i];
      if (r.t >= tokens) break;
      const int64_t page = s_page[r.t];
      if (page >= 0) {  // the same for all lanes of the row
        float k[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.f;
        if (inside) {
          unpack_run(r.k, k);
          unpack_run(r.v, v);
        }
        [[maybe_unused]] const float km = max_run(k), vm = max_run(v);
        if (inside) {
          turn_run<TURN>(a, k, r.other, a.key + s_src[r.t][0] + r.h * a.sk_h, table + r.t * a.half, d0);
        }
        const int64_t krow = page * a.sck_p + r.h * a.sck_h + s_row[r.t] * a.sck_r + d0;
        const int64_t vrow = page * a.scv_p + r.h * a.scv_h + s_row[r.t] * a.scv_r + d0;
        if constexpr (FP8) {
          const int ke = row_exponent(group_max<LPR>(km) * a.reach), ve = row_exponent(group_max<LPR>(vm));
          if (d0 == 0) {
            a.ek[page * a.sek_p + r.h * a.sek_h + s_row[r.t]] = static_cast<uint8_t>(ke);
            a.ev[page * a.sev_p + r.h * a.sev_h + s_row[r.t]] = static_cast<uint8_t>(ve);
          }
          if (inside) {
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.ck) + krow) = e4m3_run(k, exponent_value(254 - ke));
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.cv) + vrow) = e4m3_run(v, exponent_value(254 - ve));
          }
        } else if (inside) {
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.ck) + krow) =
              make_uint4(bf16_pack2(k[0], k[1]), bf16_pack2(k[2], k[3]), bf16_pack2(k[4], k[5]), bf16_pack2(k[6], k[7]));
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.cv) + vrow) = r.v;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAppendAhead; ++i) load(rows[i]);
  }
}

template <int TURN>
void launch_append(const AppendArgs& a, int64_t groups, bool fp8, hipStream_t s) {
  in_launches(groups, [&](unsigned first, unsigned grid) {
    if (a.D <= 64) {
      fp8 ? paged_append_kernel<TURN, true, 8><<<grid, kAppendThreads, 0, s>>>(a, first)
          : paged_append_kernel<TURN, false, 8><<<grid, kAppendThreads, 0, s>>>(a, first);
    } else {
      fp8 ? paged_append_kernel<TURN, true, 16><<<grid, kAppendThreads, 0, s>>>(a, first)
          : paged_append_kernel<TURN, false, 16><<<grid, kAppendThreads, 0, s>>>(a, first);
    }
  });
}

}  // namespace svhip

using namespace svhip;

extern "C" int svhip_paged_append(const svhip_paged_cache* cache, const svhip_paged_append_args* args, void* stream) {
  const char* name = "svhip_paged_append";
  clear_error();
  if (const int rc = check_cache(name, cache)) return rc;
  SVHIP_REQUIRE(args, "%s: null arguments", name);
  const svhip_paged_cache& p = *cache;
  const svhip_paged_append_args& c = *args;
  const int64_t D = p.head_dim;
  SVHIP_REQUIRE(c.N >= 0 && c.N < (1ll << 31) && c.before >= 0 && c.before < (1ll << 31), "%s: bad sizes", name);
  const bool turns = c.layout != SVHIP_ROTARY_NONE, axial = c.layout == SVHIP_ROTARY_AXIAL;
  SVHIP_REQUIRE(c.layout >= SVHIP_ROTARY_NONE && c.layout <= SVHIP_ROTARY_AXIAL, "%s: layout %d unsupported", name,
                (int)c.layout);
  SVHIP_REQUIRE(!turns || (c.pairs >= 1 && 2 * c.pairs <= D), "%s: %lld pairs do not fit head_dim %lld", name,
                (long long)c.pairs, (long long)D);
  SVHIP_REQUIRE(!axial || (2 * c.pairs == D && D % 6 == 0),
                "%s: the three-axis rotation takes the whole head, a multiple of 6", name);
  if (p.windows == 0 || p.heads == 0 || c.N == 0) return SVHIP_OK;
  if (const int rc = check_pool(name, p)) return rc;
  SVHIP_REQUIRE(c.key && c.value, "%s: null pointer", name);
  SVHIP_REQUIRE(!turns || c.freq, "%s: the rotation needs frequencies", name);
  SVHIP_REQUIRE(!axial || c.positions, "%s: the three-axis rotation needs positions", name);
  const int64_t even = c.cu_tokens ? 0 : p.windows;
  SVHIP_REQUIRE(rows_on(8, c.key, even, p.heads, c.N, c.sk_b, c.sk_h, c.sk_n) &&
                    rows_on(8, c.value, even, p.heads, c.N, c.sv_b, c.sv_h, c.sv_n),
                "%s: key and value rows must start on 16-byte boundaries", name);
  const int64_t total = c.cu_tokens ? c.N : p.windows * c.N;
  const int per_group = static_cast<int>(tokens_per_group(total, kAppendTokens));
  const int64_t groups = cdiv(total, per_group);
  SVHIP_REQUIRE(total < (1ll << 31), "%s: sizes too large", name);
  const float amplitude = static_cast<float>(c.amplitude), most = amplitude < 0.f ? -amplitude : amplitude;
  const bool fp8 = p.kv_dtype == SVHIP_FP8_E4M3;
  const AppendArgs a{static_cast<const uint16_t*>(c.key), static_cast<const uint16_t*>(c.value), c.sk_b, c.sk_h, c.sk_n,
                     c.sv_b, c.sv_h, c.sv_n, Tokens{c.cu_tokens, p.windows, c.N}, total, c.before,
                     static_cast<int>(p.heads), static_cast<int>(D), per_group, p.k_pages, p.v_pages, p.sk_p, p.sk_h, p.sk_r,
                     p.sv_p, p.sv_h, p.sv_r, p.k_exponents, p.v_exponents, p.sek_p, p.sek_h, p.sev_p, p.sev_h, pages_of(p),
                     c.positions, c.sp_b, c.sp_n, c.freq, turns ? static_cast<int>(c.pairs) : 0, c.positions_wide != 0,
                     c.pairs % (c.layout == SVHIP_ROTARY_HALF ? 8 : 4) == 0, amplitude,
                     turns ? 1.5f * (axial || most < 1.f ? 1.f : most) : 1.f};
  hipStream_t s = as_stream(stream);
  if (store_of(p.kv_dtype) == kInt8) {
    launch_append_int8(a, static_cast<int>(c.layout), block_shift(p.kv_dtype), s);
    SVHIP_LAUNCHED(name);
    return SVHIP_OK;
  }
  switch (c.layout) {
    case SVHIP_ROTARY_HALF: launch_append<kTurnHalf>(a, groups, fp8, s); break;
    case SVHIP_ROTARY_INTERLEAVED: launch_append<kTurnInterleaved>(a, groups, fp8, s); break;
    case SVHIP_ROTARY_AXIAL: launch_append<kTurnAxial>(a, groups, fp8, s); break;
    default: launch_append<kTurnNone>(a, groups, fp8, s);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
