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
constexpr int kAppendMaxDim = 128;

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
  __shared__ float2 table[kAppendTokens * kAppendMaxDim / 2];
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

extern "C" int svhip_paged_append(const void* key, const void* value, int64_t sk_b, int64_t sk_h, int64_t sk_n,
                                  int64_t sv_b, int64_t sv_h, int64_t sv_n, int64_t B, int64_t H, int64_t N, int64_t D,
                                  const int32_t* cu_tokens, int64_t before, void* k_pages, void* v_pages,
                                  uint8_t* k_exponents, uint8_t* v_exponents, int kv_dtype, int64_t pages,
                                  int64_t page_size, int64_t sck_p, int64_t sck_h, int64_t sck_r, int64_t scv_p,
                                  int64_t scv_h, int64_t scv_r, int64_t sek_p, int64_t sek_h, int64_t sev_p,
                                  int64_t sev_h, const int32_t* page_table, int64_t st_b, int64_t max_pages,
                                  const int32_t* lengths, int layout, const void* positions, int positions_wide,
                                  int64_t sp_b, int64_t sp_n, const void* freq, int64_t pairs, float amplitude,
                                  int32_t* bad, void* stream) {
  const char* name = "svhip_paged_append";
  clear_error();
  SVHIP_REQUIRE(B >= 0 && H >= 0 && N >= 0 && before >= 0, "%s: bad sizes", name);
  SVHIP_REQUIRE(D >= 8 && D <= kAppendMaxDim && D % 8 == 0, "%s: head_dim %lld unsupported (a multiple of 8 up to %d)",
                name, (long long)D, kAppendMaxDim);
  SVHIP_REQUIRE(kv_dtype == SVHIP_BF16 || kv_dtype == SVHIP_FP8_E4M3, "%s: kv dtype %d unsupported", name, kv_dtype);
  SVHIP_REQUIRE(page_size >= kMinPage && page_size <= kMaxPage && (page_size & (page_size - 1)) == 0,
                "%s: page size %lld unsupported (a power of two, %d to %d)", name, (long long)page_size, kMinPage,
                kMaxPage);
  SVHIP_REQUIRE(pages >= 0 && pages < (1ll << 31) && max_pages >= 0 && max_pages < (1ll << 31), "%s: bad page counts", name);
  const bool turns = layout != SVHIP_ROTARY_NONE, axial = layout == SVHIP_ROTARY_AXIAL;
  SVHIP_REQUIRE(layout >= SVHIP_ROTARY_NONE && layout <= SVHIP_ROTARY_AXIAL, "%s: layout %d unsupported", name, layout);
  SVHIP_REQUIRE(!turns || (pairs >= 1 && 2 * pairs <= D), "%s: %lld pairs do not fit head_dim %lld", name, (long long)pairs,
                (long long)D);
  SVHIP_REQUIRE(!axial || (2 * pairs == D && D % 6 == 0),
                "%s: the three-axis rotation takes the whole head, a multiple of 6", name);
  const bool fp8 = kv_dtype == SVHIP_FP8_E4M3;
  if (B == 0 || H == 0 || N == 0) return SVHIP_OK;
  SVHIP_REQUIRE(key && value && k_pages && v_pages && page_table && lengths, "%s: null pointer", name);
  SVHIP_REQUIRE(!turns || freq, "%s: the rotation needs frequencies", name);
  SVHIP_REQUIRE(!axial || positions, "%s: the three-axis rotation needs positions", name);
  SVHIP_REQUIRE(!fp8 || (k_exponents && v_exponents), "%s: e4m3 pages need the rows' exponents", name);
  SVHIP_REQUIRE(H <= 1 << 20, "%s: sizes too large", name);
  auto runs = [](const void* p, int64_t x, int64_t y, int64_t z, uintptr_t bytes, int64_t elems) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && x % elems == 0 && y % elems == 0 && z % elems == 0;
  };
  SVHIP_REQUIRE(runs(key, sk_b, sk_h, sk_n, 16, 8) && runs(value, sv_b, sv_h, sv_n, 16, 8),
                "%s: key and value rows must start on 16-byte boundaries", name);
  SVHIP_REQUIRE(runs(k_pages, sck_p, sck_h, sck_r, fp8 ? 8 : 16, 8) && runs(v_pages, scv_p, scv_h, scv_r, fp8 ? 8 : 16, 8),
                "%s: rows of a page must start on %d-byte boundaries", name, fp8 ? 8 : 16);
  const int64_t total = cu_tokens ? N : B * N;
  const int64_t grid = cdiv(total, kAppendTokens);
  SVHIP_REQUIRE(grid < (1ll << 31), "%s: grid too large", name);
  const float most = amplitude < 0.f ? -amplitude : amplitude;
  const AppendArgs a{static_cast<const uint16_t*>(key), static_cast<const uint16_t*>(value), sk_b, sk_h, sk_n, sv_b, sv_h,
                     sv_n, Tokens{cu_tokens, B, N}, before, H, D, k_pages, v_pages, sck_p, sck_h, sck_r, scv_p, scv_h,
                     scv_r, k_exponents, v_exponents, sek_p, sek_h, sev_p, sev_h,
                     Pages{page_table, st_b, max_pages, pages, page_shift(page_size), lengths, bad}, positions, sp_b, sp_n,
                     freq, turns ? static_cast<int>(pairs) : 0, axial || layout == SVHIP_ROTARY_INTERLEAVED,
                     positions_wide != 0, amplitude, turns ? 1.5f * (axial || most < 1.f ? 1.f : most) : 1.f};
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
