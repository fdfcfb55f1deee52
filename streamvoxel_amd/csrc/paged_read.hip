// svhip_paged_read: keys and values out of a paged cache (paged.hpp) as bf16 rows, the inverse of the append.
//
// Bound: HBM, the rows read once and written once. Workgroup = up to kReadTokens keys, all heads: where each key lies is found
// once for all heads; a group of 8 or 16 lanes then carries a (key, head) row of keys and of values, 16 bytes out a lane,
// kReadAhead of them in flight. Measured: 8 contexts of up to 9744 keys of 12 x 64 in int8 (218 MB) on pools in turn 45 us, a
// copy's rate 43 (e4m3 48, bf16, 290 MB, 54; int8 53 where nothing is left in a cache, 36 on one pool, which the caches hold in
// part); 16 keys a workgroup 52 for 49, 2 and 8 in flight 50 and 47, at 8 x 128 56 and 63 for 60; 1552 keys (7 MB) 4.4 us, bf16 and e4m3 4.2.
#include "paged.hpp"
#include "rotary.hpp"

namespace svhip {

constexpr int kReadThreads = 256;
constexpr int kReadTokens = 8;
constexpr int kReadAhead = 4;

struct ReadArgs {
  uint16_t *key, *value;
  int64_t sk_b, sk_h, sk_n, sv_b, sv_h, sv_n;
  Tokens tokens;
  int64_t total, before;
  int H, D, per_group, block_shift;  // per_group: keys of a workgroup
  const char *ck, *cv;
  int64_t sck_p, sck_h, sck_r, scv_p, scv_h, scv_r;
  const uint8_t *ek, *ev;
  int64_t sek_p, sek_h, sev_p, sev_h;
  Pages pages;
};

// 8 elements of a row as bf16: in their storage, and decoded.
template <int ST>
struct Held {
  uint2 w;
  uint32_t e;
  __device__ __forceinline__ void load(const char* row, int d0, const uint8_t* exponent) {
    w = *reinterpret_cast<const uint2*>(row + d0);
    e = *exponent;
  }
  __device__ __forceinline__ uint4 get() const {
    if constexpr (ST == kInt8) return int8_values(w, int8_power(e));
    const float f = exponent_value(static_cast<int>(e));
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = i < 2 ? w.x : w.y;
      u[i] = __builtin_bit_cast(uint32_t, i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, f, true)
                                                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, f, false));
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <>
struct Held<kBf16> {
  uint4 w;
  __device__ __forceinline__ void load(const char* row, int d0, const uint8_t*) {
    w = *reinterpret_cast<const uint4*>(row + 2 * d0);
  }
  __device__ __forceinline__ uint4 get() const { return w; }
};

template <int ST, int LPR>
__global__ __launch_bounds__(kReadThreads) void paged_read_kernel(ReadArgs a, unsigned first_group) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ int64_t s_to[kReadTokens][2], s_page[kReadTokens];  // page: -1 zeros, -2 no window's row
  __shared__ int s_row[kReadTokens];
  const int64_t t0 = static_cast<int64_t>(first_group + blockIdx.x) * a.per_group;
  const int tokens = static_cast<int>(a.total - t0 < a.per_group ? a.total - t0 : a.per_group);
  const int tid = static_cast<int>(threadIdx.x), H = a.H;
  if (tid < tokens) {
    const int64_t mine = t0 + tid;
    int64_t b = -1, n = mine, page = -2;
    if (!a.tokens.cu) {
      b = static_cast<int>(mine) / static_cast<int>(a.tokens.N);
      n = mine - b * a.tokens.N;
    } else {
      b = window_of(a.tokens, mine);
    }
    if (b >= 0) {
      int64_t start, count;
      window_tokens(a.tokens, b, start, count);
      const int64_t j = a.pages.lengths[b] - a.before - count + (mine - start);
      page = -1;
      if (j >= a.pages.max_pages << a.pages.shift) {
        set_bad(a.pages);
      } else if (j >= 0) {
        page = page_of(a.pages, b, j);
      }
      s_row[tid] = static_cast<int>(j & ((1ll << a.pages.shift) - 1));
      s_to[tid][0] = (a.tokens.cu ? 0 : b * a.sk_b) + n * a.sk_n;
      s_to[tid][1] = (a.tokens.cu ? 0 : b * a.sv_b) + n * a.sv_n;
    }
    s_page[tid] = page;
  }
  __syncthreads();
  const int d0 = 8 * (tid % LPR), first = tid / LPR;
  if (d0 >= a.D) return;
  constexpr int kStep = kReadThreads / LPR;
  const int step_t = kStep / H, step_h = kStep - step_t * H;
  int t = first / H, h = first - t * H;
  while (t < tokens) {
    Held<ST> k[kReadAhead], v[kReadAhead];
    int at[kReadAhead], head[kReadAhead];
#pragma unroll
    for (int i = 0; i < kReadAhead; ++i) {
      at[i] = t;
      head[i] = h;
      if (t < tokens && s_page[t] >= 0) {
        const int64_t page = s_page[t], row = s_row[t], e = ST == kInt8 ? row >> a.block_shift : row;
        constexpr int ES = bytes_of(ST);
        k[i].load(a.ck + (page * a.sck_p + h * a.sck_h + row * a.sck_r) * ES, d0, a.ek + page * a.sek_p + h * a.sek_h + e);
        v[i].load(a.cv + (page * a.scv_p + h * a.scv_h + row * a.scv_r) * ES, d0, a.ev + page * a.sev_p + h * a.sev_h + e);
      }
      t += step_t;
      h += step_h;
      if (h >= H) {
        h -= H;
        ++t;
      }
    }
#pragma unroll
    for (int i = 0; i < kReadAhead; ++i) {
      if (at[i] >= tokens) break;
      const int64_t page = s_page[at[i]];
      if (page == -2) continue;
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(a.key + s_to[at[i]][0] + head[i] * a.sk_h + d0) = page >= 0 ? k[i].get() : zero;
      *reinterpret_cast<uint4*>(a.value + s_to[at[i]][1] + head[i] * a.sv_h + d0) = page >= 0 ? v[i].get() : zero;
    }
  }
#endif
}

template <int ST>
void launch_read(const ReadArgs& a, int64_t groups, hipStream_t s) {
  in_launches(groups, [&](unsigned first, unsigned grid) {
    a.D <= 64 ? paged_read_kernel<ST, 8><<<grid, kReadThreads, 0, s>>>(a, first)
              : paged_read_kernel<ST, 16><<<grid, kReadThreads, 0, s>>>(a, first);
  });
}

}  // namespace svhip

using namespace svhip;

extern "C" int svhip_paged_read(const svhip_paged_cache* cache, const svhip_paged_read_args* args, void* stream) {
  const char* name = "svhip_paged_read";
  clear_error();
  if (const int rc = check_cache(name, cache)) return rc;
  SVHIP_REQUIRE(args, "%s: null arguments", name);
  const svhip_paged_cache& p = *cache;
  const svhip_paged_read_args& c = *args;
  SVHIP_REQUIRE(c.N >= 0 && c.N < (1ll << 31) && c.before >= 0 && c.before < (1ll << 31), "%s: bad sizes", name);
  if (p.windows == 0 || p.heads == 0 || c.N == 0) return SVHIP_OK;
  if (const int rc = check_pool(name, p)) return rc;
  SVHIP_REQUIRE(c.key && c.value, "%s: null pointer", name);
  const int64_t even = c.cu_keys ? 0 : p.windows;
  SVHIP_REQUIRE(rows_on(8, c.key, even, p.heads, c.N, c.sk_b, c.sk_h, c.sk_n) &&
                    rows_on(8, c.value, even, p.heads, c.N, c.sv_b, c.sv_h, c.sv_n),
                "%s: key and value rows must start on 16-byte boundaries", name);
  const int64_t total = c.cu_keys ? c.N : p.windows * c.N;
  SVHIP_REQUIRE(total < (1ll << 31), "%s: sizes too large", name);
  const int per_group = static_cast<int>(tokens_per_group(total, kReadTokens));
  const ReadArgs a{static_cast<uint16_t*>(c.key), static_cast<uint16_t*>(c.value), c.sk_b, c.sk_h, c.sk_n, c.sv_b, c.sv_h,
                   c.sv_n, Tokens{c.cu_keys, p.windows, c.N}, total, c.before, static_cast<int>(p.heads),
                   static_cast<int>(p.head_dim), per_group, block_shift(p.kv_dtype), static_cast<const char*>(p.k_pages),
                   static_cast<const char*>(p.v_pages), p.sk_p, p.sk_h, p.sk_r, p.sv_p, p.sv_h, p.sv_r, p.k_exponents,
                   p.v_exponents, p.sek_p, p.sek_h, p.sev_p, p.sev_h, pages_of(p)};
  hipStream_t s = as_stream(stream);
  switch (store_of(p.kv_dtype)) {
    case kInt8: launch_read<kInt8>(a, cdiv(total, per_group), s); break;
    case kE4m3: launch_read<kE4m3>(a, cdiv(total, per_group), s); break;
    default: launch_read<kBf16>(a, cdiv(total, per_group), s);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
