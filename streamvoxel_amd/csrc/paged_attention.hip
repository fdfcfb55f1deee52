// svhip_paged_attention: attention of the windows' new tokens over their keys and values in a paged cache (paged.hpp).
//
// Simple form: one wave per (token, head) with the running maximum and sum of the softmax, 64 keys at a time: a lane scores
// one key, then holds head_dim elements of the output.
#include "paged.hpp"

namespace svhip {

constexpr int kPagedMaxDim = 128;
constexpr int kPagedThreads = 256;

struct PagedArgs {
  const uint16_t* q;
  const void *k, *v;
  const uint8_t *ek, *ev;
  uint16_t* o;
  Tokens tokens;
  Pages pages;
  int64_t H, G, D;  // G: heads of a key head
  int64_t sq_b, sq_h, sq_n, sk_p, sk_h, sk_r, sv_p, sv_h, sv_r, sek_p, sek_h, sev_p, sev_h, so_b, so_h, so_n;
  bool causal;
  float scale_log2;
};

template <bool FP8>
__device__ __forceinline__ float page_element(const void* p, int64_t i) {
  if constexpr (FP8) {
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(p)[i], 0);
  } else {
    return bf16_bits_to_float(static_cast<const uint16_t*>(p)[i]);
  }
}

template <bool FP8>
__global__ __launch_bounds__(kPagedThreads) void paged_simple_kernel(PagedArgs a) {
  __shared__ float s_q[4][kPagedMaxDim];
  __shared__ float s_p[4][64];
  __shared__ int64_t s_row[4][64];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, D = static_cast<int>(a.D);
  const int64_t total = (a.tokens.cu ? a.tokens.N : a.tokens.B * a.tokens.N) * a.H;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + w;
  int64_t b = -1, h = 0, n = 0, bb = 0, keys = 0;
  if (id < total) {
    const int64_t i = id / a.H;
    h = id - i * a.H;
    b = a.tokens.cu ? window_of(a.tokens, i) : i / a.tokens.N;
    if (b >= 0) {
      int64_t first, count;
      window_tokens(a.tokens, b, first, count);
      n = a.tokens.cu ? i : i - first;
      bb = a.tokens.cu ? 0 : b;
      keys = held_keys(a.pages, b);
      if (a.causal) keys = a.pages.lengths[b] - count + (i - first) + 1 < keys ? a.pages.lengths[b] - count + (i - first) + 1 : keys;
    }
  }
  if (b >= 0) {
    for (int d = lane; d < D; d += 64) s_q[w][d] = bf16_bits_to_float(a.q[bb * a.sq_b + h * a.sq_h + n * a.sq_n + d]);
  }
  __syncthreads();
  if (b < 0) return;
  const int64_t kvh = h / a.G;
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  for (int64_t j0 = 0; j0 < keys; j0 += 64) {
    const int64_t j = j0 + lane;
    float s = -INFINITY;
    int64_t row = -1;
    if (j < keys) {
      s = 0.f;
      const int64_t page = page_of(a.pages, b, j);
      const int64_t r = j & ((1ll << a.pages.shift) - 1);
      if (page >= 0) {
        const int64_t at = page * a.sk_p + kvh * a.sk_h + r * a.sk_r;
        for (int d = 0; d < D; ++d) s += s_q[w][d] * page_element<FP8>(a.k, at + d);
        if constexpr (FP8) s *= exponent_value(a.ek[page * a.sek_p + kvh * a.sek_h + r]);
        s *= a.scale_log2;
        row = (page << 16) | r;
      }
    }
    float mx = s;
    for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    const float mn = fmaxf(m, mx);
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    float p = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - mn);
    m = mn;
    s_p[w][lane] = p;
    s_row[w][lane] = row;
    for (int off = 32; off >= 1; off >>= 1) p += __shfl_xor(p, off);
    l = l * alpha + p;
    o[0] *= alpha;
    o[1] *= alpha;
    const int count = static_cast<int>(keys - j0 < 64 ? keys - j0 : 64);
    for (int t = 0; t < count; ++t) {
      const int64_t at = s_row[w][t];
      if (at < 0) continue;
      const int64_t page = at >> 16, r = at & 0xffff;
      const float x = FP8 ? s_p[w][t] * exponent_value(a.ev[page * a.sev_p + kvh * a.sev_h + r]) : s_p[w][t];
      const int64_t vat = page * a.sv_p + kvh * a.sv_h + r * a.sv_r;
      if (lane < D) o[0] += x * page_element<FP8>(a.v, vat + lane);
      if (lane + 64 < D) o[1] += x * page_element<FP8>(a.v, vat + lane + 64);
    }
  }
  uint16_t* out = a.o + bb * a.so_b + h * a.so_h + n * a.so_n;
  const float inv = keys > 0 ? 1.f / l : 0.f;
  if (lane < D) out[lane] = bf16_bits(o[0] * inv);
  if (lane + 64 < D) out[lane + 64] = bf16_bits(o[1] * inv);
}

}  // namespace svhip

using namespace svhip;

extern "C" size_t svhip_paged_attention_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t N, int packed,
                                                        int64_t D, int64_t max_keys) {
  return 0;
}

extern "C" int svhip_paged_attention(const void* q, const void* k_pages, const void* v_pages, const uint8_t* k_exponents,
                                     const uint8_t* v_exponents, void* out, int kv_dtype, int64_t B, int64_t H,
                                     int64_t Hkv, int64_t N, int64_t D, const int32_t* cu_queries, int64_t pages,
                                     int64_t page_size, const int32_t* page_table, int64_t st_b, int64_t max_pages,
                                     const int32_t* lengths, int64_t sq_b, int64_t sq_h, int64_t sq_n, int64_t sk_p,
                                     int64_t sk_h, int64_t sk_r, int64_t sv_p, int64_t sv_h, int64_t sv_r, int64_t sek_p,
                                     int64_t sek_h, int64_t sev_p, int64_t sev_h, int64_t so_b, int64_t so_h,
                                     int64_t so_n, int causal, float scale, int32_t* bad, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* name = "svhip_paged_attention";
  clear_error();
  SVHIP_REQUIRE(B >= 0 && H >= 0 && N >= 0, "%s: bad sizes", name);
  SVHIP_REQUIRE(D >= 8 && D <= kPagedMaxDim && D % 8 == 0, "%s: head_dim %lld unsupported (a multiple of 8 up to %d)",
                name, (long long)D, kPagedMaxDim);
  SVHIP_REQUIRE(Hkv >= 1 && H % Hkv == 0, "%s: %lld heads do not share %lld key heads evenly", name, (long long)H,
                (long long)Hkv);
  SVHIP_REQUIRE(kv_dtype == SVHIP_BF16 || kv_dtype == SVHIP_FP8_E4M3, "%s: kv dtype %d unsupported", name, kv_dtype);
  SVHIP_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", name);
  SVHIP_REQUIRE(page_size >= kMinPage && page_size <= kMaxPage && (page_size & (page_size - 1)) == 0,
                "%s: page size %lld unsupported (a power of two, %d to %d)", name, (long long)page_size, kMinPage,
                kMaxPage);
  SVHIP_REQUIRE(pages >= 0 && pages < (1ll << 31) && max_pages >= 0 && max_pages * page_size < (1ll << 31),
                "%s: bad page counts", name);
  const bool fp8 = kv_dtype == SVHIP_FP8_E4M3;
  if (B == 0 || H == 0 || N == 0) return SVHIP_OK;
  SVHIP_REQUIRE(q && out && lengths && (max_pages == 0 || page_table) && (pages == 0 || (k_pages && v_pages)),
                "%s: null pointer", name);
  SVHIP_REQUIRE(!fp8 || (k_exponents && v_exponents), "%s: e4m3 pages need the rows' exponents", name);
  auto runs = [](const void* p, int64_t x, int64_t y, int64_t z, uintptr_t bytes, int64_t elems) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && x % elems == 0 && y % elems == 0 && z % elems == 0;
  };
  SVHIP_REQUIRE(runs(q, sq_b, sq_h, sq_n, 16, 8), "%s: query rows must start on 16-byte boundaries", name);
  SVHIP_REQUIRE(runs(out, so_b, so_h, so_n, 8, 4), "%s: rows of out must start on 8-byte boundaries", name);
  SVHIP_REQUIRE(runs(k_pages, sk_p, sk_h, sk_r, fp8 ? 8 : 16, 8) && runs(v_pages, sv_p, sv_h, sv_r, fp8 ? 8 : 16, 8),
                "%s: rows of a page must start on %d-byte boundaries", name, fp8 ? 8 : 16);
  const PagedArgs a{static_cast<const uint16_t*>(q), k_pages, v_pages, k_exponents, v_exponents,
                    static_cast<uint16_t*>(out), Tokens{cu_queries, B, N},
                    Pages{page_table, st_b, max_pages, pages, page_shift(page_size), lengths, bad}, H, H / Hkv, D, sq_b,
                    sq_h, sq_n, sk_p, sk_h, sk_r, sv_p, sv_h, sv_r, sek_p, sek_h, sev_p, sev_h, so_b, so_h, so_n,
                    causal != 0, scale * kLog2e};
  const int64_t rows = (cu_queries ? N : B * N) * H;
  SVHIP_REQUIRE(cdiv(rows, 4) < (1ll << 31), "%s: grid too large", name);
  const unsigned grid = static_cast<unsigned>(cdiv(rows, 4));
  hipStream_t s = as_stream(stream);
  if (fp8) {
    paged_simple_kernel<true><<<grid, kPagedThreads, 0, s>>>(a);
  } else {
    paged_simple_kernel<false><<<grid, kPagedThreads, 0, s>>>(a);
  }
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
