// svhip_paged_append: the new tokens' keys and values into their rows of a paged cache (paged.hpp), the keys rotated on the
// way: rotary positions (rotary.hpp, fp32, rounded once to the cache's type), or the three-axis rotation of svhip_axial_rope
// with its roundings (the phase one fp32 product; sin, cos, every product and sum rounded to bf16).
//
// Bound: HBM, the rows read once and written once. Workgroup = kAppendTokens tokens, all heads: where each token goes and
// its (cos, sin) are the same for every head and go to LDS once; a group of 16 lanes then carries one (token, head) row,
// 8 elements a lane, so that an e4m3 row's largest magnitude is a reduction within the group.
#include "paged.hpp"
#include "rotary.hpp"

namespace svhip {

constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 8;
constexpr int kAppendLanes = 16;

enum AppendTurn { kTurnNone = 0, kTurnRotary = 1, kTurnAxial = 2 };

struct AppendArgs {
  const uint16_t *key, *value;
  int64_t sk_b, sk_h, sk_n, sv_b, sv_h, sv_n;
  Tokens tokens;
  int64_t before, H, D;
  void *ck, *cv;
  int64_t sck_p, sck_h, sck_r, scv_p, scv_h, scv_r;
  uint8_t *ek, *ev;
  int64_t sek_p, sek_h, sev_p, sev_h;
  Pages pages;
  const void* positions;
  int64_t sp_b, sp_n;
  const void* freq;
  int half;             // pairs that turn
  bool interleaved, wide;
  float amplitude, reach;  // reach: |turned| <= reach max |key|
};

// Element d of a key row turned; `row` is read again for the partner.
__device__ __forceinline__ float turned_element(const AppendArgs& a, int turn, const uint16_t* row, const float2* table,
                                                int d) {
  const float x = bf16_bits_to_float(row[d]);
  if (turn == kTurnNone || d >= 2 * a.half) return x;
  const bool second = a.interleaved ? (d & 1) : d >= a.half;
  const int pair = a.interleaved ? d >> 1 : (second ? d - a.half : d);
  const float y = bf16_bits_to_float(row[a.interleaved ? d ^ 1 : (second ? d - a.half : d + a.half)]);
  const float2 r = table[pair];
  if (turn == kTurnAxial) {
    const float p = bf16_round1(x * r.x), q = bf16_round1(y * r.y);
    return bf16_round1(second ? q + p : p - q);
  }
  return second ? __builtin_fmaf(x, r.x, y * r.y) : __builtin_fmaf(x, r.x, -(y * r.y));
}

template <int TURN, bool FP8>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(AppendArgs a) {
  __shared__ float2 table[kAppendTokens * kMaxPagedDim / 2];
  __shared__ int64_t s_src[kAppendTokens][2], s_page[kAppendTokens], s_pos[kAppendTokens];
  __shared__ int s_row[kAppendTokens];
  const int64_t total = a.tokens.cu ? a.tokens.N : a.tokens.B * a.tokens.N;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kAppendTokens;
  if (threadIdx.x < kAppendTokens) {
    const int64_t i = t0 + threadIdx.x;
    int64_t page = -1;
    if (i < total) {
      const int64_t b = a.tokens.cu ? window_of(a.tokens, i) : i / a.tokens.N;
      if (b >= 0) {
        int64_t first, count;
        window_tokens(a.tokens, b, first, count);
        const int64_t j = a.pages.lengths[b] - a.before - count + (i - first);
        if (j < 0 || j >= a.pages.max_pages << a.pages.shift) {
          set_bad(a.pages);
        } else {
          page = page_of(a.pages, b, j);
        }
        const int64_t n = a.tokens.cu ? i : i - first, bb = a.tokens.cu ? 0 : b;
        s_src[threadIdx.x][0] = bb * a.sk_b + n * a.sk_n;
        s_src[threadIdx.x][1] = bb * a.sv_b + n * a.sv_n;
        s_pos[threadIdx.x] = a.positions ? bb * a.sp_b + n * a.sp_n : j;
        s_row[threadIdx.x] = static_cast<int>(j & ((1ll << a.pages.shift) - 1));
      }
    }
    s_page[threadIdx.x] = page;
  }
  __syncthreads();
  if constexpr (TURN != kTurnNone) {
    for (int i = threadIdx.x; i < kAppendTokens * a.half; i += kAppendThreads) {
      const int t = i / a.half, pr = i - t * a.half;
      if (s_page[t] < 0) continue;
      if constexpr (TURN == kTurnAxial) {
        const int per_axis = a.half / 3, axis = pr / per_axis;
        const float phase =
            static_cast<const float*>(a.positions)[s_pos[t] + axis] * static_cast<const float*>(a.freq)[pr - axis * per_axis];
        table[i] = make_float2(bf16_round1(cosf(phase)), bf16_round1(sinf(phase)));
      } else {
        const double p = a.positions ? rotary_position(a.positions, a.wide, s_pos[t]) : static_cast<double>(s_pos[t]);
        table[i] = rotary_phase(p, static_cast<const double*>(a.freq)[pr], a.amplitude);
      }
    }
    __syncthreads();
  }
  const int lane = threadIdx.x % kAppendLanes, D = static_cast<int>(a.D), H = static_cast<int>(a.H);
  const int d0 = 8 * lane;
  for (int r = threadIdx.x / kAppendLanes; r < kAppendTokens * H; r += kAppendThreads / kAppendLanes) {
    const int t = r / H, h = r - t * H;
    const int64_t page = s_page[t];
    if (page < 0) continue;  // the same for the whole group
    const uint16_t* key = a.key + s_src[t][0] + h * a.sk_h;
    const uint16_t* value = a.value + s_src[t][1] + h * a.sv_h;
    float k[8], v[8], km = 0.f, vm = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      k[e] = v[e] = 0.f;
      if (d0 < D) {
        k[e] = turned_element(a, TURN, key, table + t * a.half, d0 + e);
        v[e] = bf16_bits_to_float(value[d0 + e]);
        km = fmaxf(km, fabsf(bf16_bits_to_float(key[d0 + e])));
        vm = fmaxf(vm, fabsf(v[e]));
      }
    }
    const int64_t krow = page * a.sck_p + h * a.sck_h + s_row[t] * a.sck_r + d0;
    const int64_t vrow = page * a.scv_p + h * a.scv_h + s_row[t] * a.scv_r + d0;
    if constexpr (FP8) {
      const int ke = row_exponent(row16_max(km) * a.reach), ve = row_exponent(row16_max(vm));
      const float ki = exponent_value(254 - ke), vi = exponent_value(254 - ve);
      if (lane == 0) {
        a.ek[page * a.sek_p + h * a.sek_h + s_row[t]] = static_cast<uint8_t>(ke);
        a.ev[page * a.sev_p + h * a.sev_h + s_row[t]] = static_cast<uint8_t>(ve);
      }
      if (d0 < D) {
        uint32_t kw[2], vw[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          int w = __builtin_amdgcn_cvt_pk_fp8_f32(k[4 * g] * ki, k[4 * g + 1] * ki, 0, false);
          kw[g] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(k[4 * g + 2] * ki, k[4 * g + 3] * ki, w, true));
          w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * g] * vi, v[4 * g + 1] * vi, 0, false);
          vw[g] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * g + 2] * vi, v[4 * g + 3] * vi, w, true));
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.ck) + krow) = make_uint2(kw[0], kw[1]);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.cv) + vrow) = make_uint2(vw[0], vw[1]);
      }
    } else if (d0 < D) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.ck) + krow) =
          make_uint4(bf16_pack2(k[0], k[1]), bf16_pack2(k[2], k[3]), bf16_pack2(k[4], k[5]), bf16_pack2(k[6], k[7]));
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.cv) + vrow) =
          make_uint4(bf16_pack2(v[0], v[1]), bf16_pack2(v[2], v[3]), bf16_pack2(v[4], v[5]), bf16_pack2(v[6], v[7]));
    }
  }
}

template <int TURN>
void launch_append(const AppendArgs& a, unsigned grid, bool fp8, hipStream_t s) {
  if (fp8) {
    paged_append_kernel<TURN, true><<<grid, kAppendThreads, 0, s>>>(a);
  } else {
    paged_append_kernel<TURN, false><<<grid, kAppendThreads, 0, s>>>(a);
  }
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
  SVHIP_REQUIRE(c.N >= 0 && c.before >= 0, "%s: bad sizes", name);
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
  SVHIP_REQUIRE(p.heads <= 1 << 20, "%s: sizes too large", name);
  SVHIP_REQUIRE(rows16(c.key, c.sk_b, c.sk_h, c.sk_n) && rows16(c.value, c.sv_b, c.sv_h, c.sv_n),
                "%s: key and value rows must start on 16-byte boundaries", name);
  const int64_t total = c.cu_tokens ? c.N : p.windows * c.N;
  const int64_t grid = cdiv(total, kAppendTokens);
  SVHIP_REQUIRE(grid < (1ll << 31), "%s: grid too large", name);
  const float amplitude = static_cast<float>(c.amplitude), most = amplitude < 0.f ? -amplitude : amplitude;
  const bool fp8 = p.kv_dtype == SVHIP_FP8_E4M3;
  const AppendArgs a{static_cast<const uint16_t*>(c.key), static_cast<const uint16_t*>(c.value), c.sk_b, c.sk_h, c.sk_n,
                     c.sv_b, c.sv_h, c.sv_n, Tokens{c.cu_tokens, p.windows, c.N}, c.before, p.heads, D, p.k_pages,
                     p.v_pages, p.sk_p, p.sk_h, p.sk_r, p.sv_p, p.sv_h, p.sv_r, p.k_exponents, p.v_exponents, p.sek_p,
                     p.sek_h, p.sev_p, p.sev_h, pages_of(p), c.positions, c.sp_b, c.sp_n, c.freq,
                     turns ? static_cast<int>(c.pairs) : 0, axial || c.layout == SVHIP_ROTARY_INTERLEAVED,
                     c.positions_wide != 0, amplitude, turns ? 1.5f * (axial || most < 1.f ? 1.f : most) : 1.f};
  hipStream_t s = as_stream(stream);
  if (axial) {
    launch_append<kTurnAxial>(a, static_cast<unsigned>(grid), fp8, s);
  } else if (turns) {
    launch_append<kTurnRotary>(a, static_cast<unsigned>(grid), fp8, s);
  } else {
    launch_append<kTurnNone>(a, static_cast<unsigned>(grid), fp8, s);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
