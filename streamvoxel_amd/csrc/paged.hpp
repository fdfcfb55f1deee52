// A paged cache of keys and values: key j of window b is row j % S of page table[b][j / S] of a pool [pages, H, S,
// D], S a power of two. bf16 rows, or OCP e4m3fn rows with one power of two for each row and head, held as its
// exponent's byte (value = code 2^(byte - 127)): scaling by it is exact, so an e4m3 row decodes to bf16 without a
// second rounding and the row's scale takes part in neither product of the attention.
#pragma once

#include "common.hpp"

namespace svhip {

constexpr int kMinPage = 16;
constexpr int kMaxPage = 1024;
constexpr int kMaxPagedDim = 128;

struct Pages {
  const int32_t* table;   // [B, max_pages], rows st_b apart
  int64_t st_b, max_pages, pages;
  int shift;              // log2 of the page size
  const int32_t* lengths;
  int32_t* bad;           // set to 1 where a page lies outside the pool or a window outside its row of the table; or null
};

__host__ __device__ __forceinline__ void set_bad(const Pages& p) {
  if (p.bad) *p.bad = 1;
}

// Page of key j of window b, or -1 (and the flag) for a number outside the pool. j lies inside the table's row.
__device__ __forceinline__ int64_t page_of(const Pages& p, int64_t b, int64_t j) {
  const int32_t page = p.table[b * p.st_b + (j >> p.shift)];
  if (page >= 0 && page < p.pages) return page;
  set_bad(p);
  return -1;
}

// Keys of window b: its length, cut to what its row of the table can name.
__host__ __device__ __forceinline__ int64_t held_keys(const Pages& p, int64_t b) {
  const int64_t L = p.lengths[b], most = p.max_pages << p.shift;
  if (L > most) set_bad(p);
  return L < 0 ? 0 : (L > most ? most : L);
}

// The windows' new tokens: N of each, or packed [0, T) with the windows' borders.
struct Tokens {
  const int32_t* cu;  // [B + 1] or null
  int64_t B, N;       // N: tokens of a window, or T
};

// Border i of the packed windows, inside [0, T].
__host__ __device__ __forceinline__ int64_t border(const Tokens& t, int64_t i) {
  const int64_t c = t.cu[i];
  return c < 0 ? 0 : (c > t.N ? t.N : c);
}

// First token and count of window b.
__host__ __device__ __forceinline__ void window_tokens(const Tokens& t, int64_t b, int64_t& first, int64_t& count) {
  if (!t.cu) {
    first = b * t.N;
    count = t.N;
    return;
  }
  first = border(t, b);
  const int64_t end = border(t, b + 1);
  count = end > first ? end - first : 0;
}

// Window of packed token i (borders ascending), or -1 for one in front of the first border or behind the last.
__device__ __forceinline__ int64_t window_of(const Tokens& t, int64_t i) {
  if (i < t.cu[0] || i >= t.cu[t.B]) return -1;
  int64_t lo = 0, hi = t.B;  // cu[lo] <= i < cu[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    (t.cu[mid] <= i ? lo : hi) = mid;
  }
  return lo;
}

// Exponent byte of a row whose magnitudes are at most `bound`: of the least power of two with bound <= 448 2^e.
__device__ __forceinline__ int row_exponent(float bound) {
  const uint32_t u = __float_as_uint(bound);
  const int e = static_cast<int>(u >> 23) - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return e < 1 ? 1 : (e > 254 ? 254 : e);
}

__device__ __forceinline__ float exponent_value(int code) { return __uint_as_float(static_cast<uint32_t>(code) << 23); }

inline int page_shift(int64_t page) {
  int s = 0;
  while ((1ll << s) < page) ++s;
  return s;
}

// What both calls ask of a cache; the status of the first check that fails.
inline int check_cache(const char* name, const svhip_paged_cache* cache) {
  SVHIP_REQUIRE(cache, "%s: null cache", name);
  const svhip_paged_cache& c = *cache;
  SVHIP_REQUIRE(c.windows >= 0 && c.windows < (1ll << 31) && c.heads >= 0 && c.heads <= 1 << 20, "%s: bad sizes", name);
  SVHIP_REQUIRE(c.head_dim >= 8 && c.head_dim <= kMaxPagedDim && c.head_dim % 8 == 0,
                "%s: head_dim %lld unsupported (a multiple of 8 up to %d)", name, (long long)c.head_dim, kMaxPagedDim);
  SVHIP_REQUIRE(c.kv_dtype == SVHIP_BF16 || c.kv_dtype == SVHIP_FP8_E4M3, "%s: kv dtype %d unsupported", name,
                (int)c.kv_dtype);
  SVHIP_REQUIRE(c.page_size >= kMinPage && c.page_size <= kMaxPage && (c.page_size & (c.page_size - 1)) == 0,
                "%s: page size %lld unsupported (a power of two, %d to %d)", name, (long long)c.page_size, kMinPage,
                kMaxPage);
  SVHIP_REQUIRE(c.pages >= 0 && c.pages < (1ll << 31) && c.max_pages >= 0 && c.max_pages <= (1ll << 30) / c.page_size,
                "%s: bad page counts", name);  // (keys and a few blocks of them further on are counted in 32 bits)
  return SVHIP_OK;
}

// The checks of a cache that a call touches.
inline int check_pool(const char* name, const svhip_paged_cache& c) {
  const bool fp8 = c.kv_dtype == SVHIP_FP8_E4M3;
  SVHIP_REQUIRE(c.pages >= 1, "%s: a pool needs a page", name);
  SVHIP_REQUIRE(c.lengths && (c.max_pages == 0 || c.page_table) && c.k_pages && c.v_pages, "%s: null pointer", name);
  SVHIP_REQUIRE(!fp8 || (c.k_exponents && c.v_exponents), "%s: e4m3 pages need the rows' exponents", name);
  const uintptr_t bytes = fp8 ? 8 : 16;
  const int64_t sk_p = used_stride(c.pages, c.sk_p), sv_p = used_stride(c.pages, c.sv_p);
  const int64_t sk_h = used_stride(c.heads, c.sk_h), sv_h = used_stride(c.heads, c.sv_h);
  SVHIP_REQUIRE(reinterpret_cast<uintptr_t>(c.k_pages) % bytes == 0 && reinterpret_cast<uintptr_t>(c.v_pages) % bytes == 0 &&
                    (sk_p | sk_h | c.sk_r | sv_p | sv_h | c.sv_r) % 8 == 0,
                "%s: rows of a page must start on %d-byte boundaries", name, (int)bytes);
  // A head's rows of a page lie within 2^31 bytes, pages start less than 2^32 bytes apart.
  SVHIP_REQUIRE(c.sk_r >= 0 && c.sv_r >= 0 && c.sk_r < (1 << 29) / c.page_size && c.sv_r < (1 << 29) / c.page_size,
                "%s: rows of a page too far apart", name);
  const int64_t most = 1ll << 31;
  const int64_t sek_p = used_stride(c.pages, c.sek_p), sev_p = used_stride(c.pages, c.sev_p);
  SVHIP_REQUIRE(sk_p >= 0 && sk_p < most && sv_p >= 0 && sv_p < most && sek_p >= 0 && sek_p < most && sev_p >= 0 &&
                    sev_p < most,
                "%s: pages too far apart", name);
  return SVHIP_OK;
}

// Rows of bf16 values that start on boundaries of `values` values: strides of a window, a head and a token (windows 0:
// packed).
inline bool rows_on(int64_t values, const void* p, int64_t windows, int64_t heads, int64_t tokens, int64_t s_b, int64_t s_h,
                    int64_t s_n) {
  return reinterpret_cast<uintptr_t>(p) % (2 * values) == 0 &&
         (used_stride(windows, s_b) | used_stride(heads, s_h) | used_stride(tokens, s_n)) % values == 0;
}

inline Pages pages_of(const svhip_paged_cache& c) {
  return Pages{c.page_table, c.table_stride, c.max_pages, c.pages, page_shift(c.page_size), c.lengths, c.bad};
}

}  // namespace svhip
