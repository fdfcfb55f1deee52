// svhip_paged_attention: attention of the windows' new tokens over their keys and values in a paged cache (paged.hpp), bf16
// matrix cores, fp32 sums.
//
// A key head's queries are its G heads' rows of every token, row r = token r / G, head r % G; a wave takes 32 of them as the
// columns of S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_32x32x16_bf16), so that the softmax of a row stays in two lanes and
// P^T leaves the first product in the second one's operand layout (K rows lie in LDS under sigma_row; xattn_kernel.hpp). V
// rows lie as they come and are read transposed (ds_read_b64_tr_b16). Two forms of work:
//   * windows of more than kRows rows (tile): a workgroup takes 128 rows, 32 a wave; the 4 waves stage each block of 64 keys
//     together, the next one in flight while the current one is computed. Bound: the matrix cores and the exponentials.
//   * windows of up to kRows rows, single tokens among them (row): the 4 waves share the rows and split the keys, each
//     staging its own blocks of 32 keys in its own LDS; no barrier until the waves' sums are joined. Bound: HBM.
// Either form may cut a window's keys into parts for several workgroups; a part leaves O, its running maximum and its sum in
// fp32 and paged_join_kernel joins them in order.
//
// Staging: 16 keys lie in one page (pages are of 16 keys or more), so the wave's load of 8 rows has one base, a scalar buffer
// descriptor whose bound is the number of its keys that exist: keys past the window's end, bad pages and the chunks past
// head_dim read as zeros and nothing is read outside a page.
#include "paged.hpp"
#include "xattn_kernel.hpp"

namespace svhip {

constexpr int kPagedThreads = 256;
constexpr int kRows = 32;          // rows of a wave
constexpr int kTileRows = 128;     // rows of a tile workgroup
constexpr int kRowKeys = 32;       // keys of a row-form wave's block
constexpr int kTileTarget = 512;   // workgroups that a launch of tiles is cut into at least where its keys allow
constexpr int kRowTarget = 512;    // the same of the row form
constexpr int kRowLeast = 256;     // keys that a row-form part has a multiple of
constexpr int kTileLeast = 6;      // least key blocks of a tile part
constexpr float kNoMax = -3.0e38f; // running maximum before any key: finite, so that a row that sees nothing stays finite
[[maybe_unused]] constexpr uint32_t kOutside = 0x7ffffff0u;  // byte offset past every descriptor's bound

struct PagedArgs {
  const uint16_t* q;
  const void *k, *v;
  const uint8_t *ek, *ev;
  uint16_t* o;
  Tokens tokens;
  Pages pages;
  int64_t H, Hkv, G, D;  // G: heads of a key head
  int64_t sq_b, sq_h, sq_n, sk_p, sk_h, sk_r, sv_p, sv_h, sv_r, sek_p, sek_h, sev_p, sev_h, so_b, so_h, so_n;
  bool causal;
  float scale_log2;
  // The plan.
  int64_t q_tiles, tiles;  // tiles of a window (even windows), and of all (packed: at most)
  int parts;               // of a tile's keys, at most
  int64_t row_slots;       // row-form workgroups at most
  int slot_rows;           // rows of a row-form slot
  float *row_part, *tile_part;
  int4* plan;              // a window's first slot or tile, its parts (0: nothing to join), form and part length
};

// The window as a workgroup sees it.
struct Window {
  int64_t first, count;  // its tokens
  int64_t last;          // the last key that its first token sees (causal), or its last key
  int keys;              // keys that any of its tokens sees
};

__device__ __forceinline__ Window window_at(const PagedArgs& a, int64_t b) {
  Window w;
  window_tokens(a.tokens, b, w.first, w.count);
  const int64_t L = held_keys(a.pages, b);
  w.keys = static_cast<int>(L);
  w.last = a.causal ? a.pages.lengths[b] - w.count : L - 1;
  return w;
}

// Last key that token i sees (below 0: none).
__device__ __forceinline__ int last_key(const PagedArgs& a, const Window& w, int64_t i) {
  const int64_t j = a.causal ? w.last + i : w.last;
  return static_cast<int>(j < w.keys - 1 ? (j < -1 ? -1 : j) : w.keys - 1);
}

__device__ __forceinline__ bool row_form(const PagedArgs& a, int64_t count) { return count * a.G <= kRows; }

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Exclusive prefix over the wave's lanes; `total` the sum.
__device__ __forceinline__ int wave_prefix(int v, int& total) {
  int incl = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(incl, off, 64);
    if ((threadIdx.x & 63) >= off) incl += up;
  }
  total = __builtin_amdgcn_readlane(incl, 63);
  return incl - v;
}

// Page of the 16 keys at j (a multiple of 16) of the window whose table row this is, through the scalar cache; the number
// as it stands in the table (j may lie past the window's keys: its last entry then).
__device__ __forceinline__ int page_number(const PagedArgs& a, const int32_t* row, int j) {
  typedef const __attribute__((address_space(4))) int32_t* table_t;
  const int at = j >> a.pages.shift, last = static_cast<int>(a.pages.max_pages) - 1;
  return __builtin_amdgcn_readfirstlane(((table_t)row)[at < last ? at : last]);
}

#if defined(__HIP_DEVICE_COMPILE__)

// Descriptor of the rows of 16 keys, row in_page of `page` the first, from a head's part of a pool: `valid` of them, D
// elements of ES bytes each.
template <int ES>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const char* head, int page, int in_page, int64_t sp, int64_t sr,
                                                         int valid, int D) {
  const int row = static_cast<int>(sr) * ES;  // a page spans less than 2^31 bytes
  const char* base = head + static_cast<uint32_t>(page) * (sp * ES) + in_page * row;
  const uint32_t bytes = valid > 0 ? static_cast<uint32_t>((valid - 1) * row + D * ES) : 0u;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, bytes, kRsrcFlags);
}

// Keys of the 16 at j that exist: inside the window and on a page of the pool.
__device__ __forceinline__ int valid_keys(const PagedArgs& a, int keys, int j, int& page) {
  int valid = j + 16 <= keys ? 16 : (j < keys ? keys - j : 0);
  if (__builtin_expect(static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages.pages), 0)) {
    if (valid > 0) set_bad(a.pages);
    valid = 0;
    page = 0;
  }
  return valid;
}

// Head widths: KS steps of 16 head_dim elements in the score product, and output tiles of 32.
constexpr int tiles_of(int KS) { return (KS + 1) / 2; }

// A wave's 32 rows: the queries as B operands, O^T, running maximum (log2 units) and sum.
template <int KS>
struct Rows {
  bf16x8_t qf[KS];
  f32x16_t o[tiles_of(KS)];
  f32x4_t l;   // four equal entries: the lane's share of its row's sum
  float m;
  int last;    // last key that the lane's row sees
};

template <int KS>
__device__ __forceinline__ void load_rows(const PagedArgs& a, const Window& w, int64_t b, int64_t kvh, int64_t r,
                                          Rows<KS>& s) {
  const int hh = (threadIdx.x & 63) >> 5;
  const int64_t i = r / a.G, g = r - i * a.G;
  const bool ok = i < w.count;
  const uint16_t* q = a.q + (a.tokens.cu ? 0 : b * a.sq_b) + (kvh * a.G + g) * a.sq_h +
                      (a.tokens.cu ? w.first + i : i) * a.sq_n;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int d0 = 16 * k + 8 * hh;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (ok && d0 < a.D) raw = *reinterpret_cast<const uint4*>(q + d0);
    s.qf[k] = __builtin_bit_cast(bf16x8_t, raw);
  }
#pragma unroll
  for (int j = 0; j < tiles_of(KS); ++j) s.o[j] = f32x16_t{0};
  s.l = f32x4_t{0.f, 0.f, 0.f, 0.f};
  s.m = kNoMax;
  s.last = ok ? last_key(a, w, i) : -1;
}

// S^T of 32 keys: ka the K rows as A operands, row R of the tile key sigma_row(R).
template <int KS>
__device__ __forceinline__ f32x16_t scores(const Rows<KS>& s, const bf16x8_t (&ka)[KS]) {
  f32x16_t x;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[k], s.qf[k], k == 0 ? f32x16_t{0} : x, 0, 0, 0);
  }
  return x;
}

// The rest of 32 keys, `key0` the first, from their scores x: weights, sum, and O^T += V^T P^T with V rows staged at row 0 of
// vp (sub-tiles of 64 head_dim elements kSubBytes apart). The running maximum moves only for a score more than kMaxHigh
// above it (P then stays below 2^20, which fp32 sums and bf16 weights hold alike); the row's sum is taken over the bf16
// weights that the second product reads, by v_mfma_f32_4x4x4_16b_bf16 with ones in A, whose columns are single lanes: no
// row's NaN reaches another's sum.
template <int KS, int kSubBytes>
__device__ __forceinline__ void attend_half(Rows<KS>& s, f32x16_t x, const char* vp,
                                            const uint32_t (&rvt)[tiles_of(KS)], float sl2, bool masked, int key0) {
  constexpr int DT = tiles_of(KS);
  const int hh = (threadIdx.x & 63) >> 5;
  if (masked) {
    const int seen = s.last - key0 - 8 * hh;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if ((i < 8 ? i : i + 8) > seen) x[i] = -INFINITY;
    }
  }
  const auto max3 = [](float p, float q, float r) __attribute__((always_inline)) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(p, q), r);
  };
  const float mx = max3(max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[8])),
                        max3(x[9], x[10], x[11]), max3(max3(x[12], x[13], x[14]), x[15], x[15]));
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(__builtin_fmaf(mx, sl2, -s.m) > kMaxHigh) != 0ull, 0)) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_int(mx), __float_as_int(mx), false, false);
    const float top = fmaxf(__int_as_float(sw[0]), __int_as_float(sw[1]));
    const float cand = (top < kFltMax ? top : kFltMax) * sl2;
    const float mn = cand > s.m ? cand : s.m;
    const float alpha = __builtin_amdgcn_exp2f(s.m - mn);
    s.m = mn;
#pragma unroll
    for (int i = 0; i < 4; ++i) s.l[i] *= alpha;
#pragma unroll
    for (int j = 0; j < DT; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s.o[j][i] *= alpha;
    }
  }
  bf16x8_t pb[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const f32x2_t two = {__builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * ks + j], sl2, -s.m)),
                           __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * ks + j + 1], sl2, -s.m))};
      const bf16x2_t c = __builtin_convertvector(two, bf16x2_t);
      pb[ks][j] = c[0];
      pb[ks][j + 1] = c[1];
    }
  }
  typedef short i16x4_t __attribute__((ext_vector_type(4)));
  typedef short i16x8_t __attribute__((ext_vector_type(8)));
  const i16x4_t ones = {0x3F80, 0x3F80, 0x3F80, 0x3F80};
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const i16x8_t p8 = __builtin_bit_cast(i16x8_t, pb[ks]);
    s.l = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(ones, __builtin_shufflevector(p8, p8, 0, 1, 2, 3), s.l, 0, 0, 0);
    s.l = __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(ones, __builtin_shufflevector(p8, p8, 4, 5, 6, 7), s.l, 0, 0, 0);
  }
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    bf16x8_t va[DT];
#pragma unroll
    for (int j = 0; j < DT; ++j) {
      typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;
      char* at = const_cast<char*>(vp) + (j >> 1) * kSubBytes + rvt[j] + 16 * ks * kRow * 2;
      const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t*)(at));
      const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t*)(at + 4 * kRow * 2));
      va[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma unroll
    for (int j = 0; j < DT; ++j) s.o[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[j], pb[ks], s.o[j], 0, 0, 0);
  }
}

// Byte offsets of the reads of V rows, transposed: output tile j inside its sub-tile (xattn_kernel.hpp).
template <int DT>
__device__ __forceinline__ void v_offsets(uint32_t (&rvt)[DT]) {
  const int lane = threadIdx.x & 63, hh = lane >> 5;
  const int row = 8 * hh + ((lane & 15) >> 2), flip = (row >> 1) & 1;
  const int c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
  for (int j = 0; j < DT; ++j) {
    rvt[j] = static_cast<uint32_t>(row * kRow * 2 + 16 * (4 * ((j & 1) ^ flip) + c) + 8 * (lane & 1));
  }
}

// The lane's sum of its row, both lanes' shares.
__device__ __forceinline__ float row_sum(float l) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_int(l), __float_as_int(l), false, false);
  return __int_as_float(sw[0]) + __int_as_float(sw[1]);
}

// e4m3 rows on their way to LDS: a wave's kLoads loads of 8 rows, and the rows' exponents.
template <int DT, int kLoads>
struct Staged {
  uint2 w[kLoads * Width<DT>::kSubTiles];
  uint32_t e[kLoads];
};

// A lane's place in a load of 8 rows, the first or the second (odd) 8 of 16 keys: row lane / 8 and its chunk, K under
// sigma_row and swz, V under swzv.
struct Lane8 {
  uint32_t at[2];   // byte offset from the 16 keys' first row in each sub-tile, or kOutside past head_dim
  uint32_t key;     // the key's place among the 16
};

template <int ES>
__device__ __forceinline__ Lane8 lane_of_load(int64_t sr, int64_t D, int key, int chunk) {
  Lane8 n;
  n.key = static_cast<uint32_t>(key);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int d = 64 * u + 8 * chunk;
    n.at[u] = d < D ? static_cast<uint32_t>((key * sr + d) * ES) : kOutside;
  }
  return n;
}
template <int ES>
__device__ __forceinline__ Lane8 k_lane(const PagedArgs& a, int odd) {
  const int lane = threadIdx.x & 63, R = 8 * odd + (lane >> 3);
  return lane_of_load<ES>(a.sk_r, a.D, sigma_row(R), swz(R, lane & 7));
}
template <int ES>
__device__ __forceinline__ Lane8 v_lane(const PagedArgs& a, int odd) {
  const int lane = threadIdx.x & 63, R = 8 * odd + (lane >> 3);
  return lane_of_load<ES>(a.sv_r, a.D, R, swzv(R, lane & 7));
}

// One key head's part of a pool (of keys or of values).
struct Source {
  const char* rows;
  const uint8_t* exponents;
  int64_t sp, sr, se;  // elements from page to page and row to row, exponents from page to page
};
template <int ES>
__device__ __forceinline__ Source k_source(const PagedArgs& a, int64_t kvh) {
  return Source{static_cast<const char*>(a.k) + kvh * a.sk_h * ES, ES == 1 ? a.ek + kvh * a.sek_h : nullptr, a.sk_p,
                a.sk_r, a.sek_p};
}
template <int ES>
__device__ __forceinline__ Source v_source(const PagedArgs& a, int64_t kvh) {
  return Source{static_cast<const char*>(a.v) + kvh * a.sv_h * ES, ES == 1 ? a.ev + kvh * a.sev_h : nullptr, a.sv_p,
                a.sv_r, a.sev_p};
}

// Issues the loads of 8 of the 16 keys at row in_page of `page`, `valid` of which exist: bf16 straight into LDS at `to` (row 0
// of the 8 in sub-tile 0), e4m3 into registers at index i.
template <bool FP8, int DT, int kSubBytes, int kLoads>
__device__ __forceinline__ void stage_rows8(const Source& src, const Lane8& n, int page, int in_page, int valid, int D,
                                            int i, char* to, Staged<DT, kLoads>& st) {
  const auto r = rows_of<FP8 ? 1 : 2>(src.rows, page, in_page, src.sp, src.sr, valid, D);
#pragma unroll
  for (int u = 0; u < Width<DT>::kSubTiles; ++u) {
    if constexpr (FP8) {
      st.w[i * Width<DT>::kSubTiles + u] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, n.at[u], 0, 0));
    } else {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)(to + u * kSubBytes), 16, n.at[u], 0, 0, 0);
    }
  }
  if constexpr (FP8) {
    const auto er = rows_of<1>(reinterpret_cast<const char*>(src.exponents), page, in_page, src.se, 1, valid, 1);
    st.e[i] = __builtin_amdgcn_raw_buffer_load_b8(er, n.key, 0, 0);
  }
}

// 8 e4m3 codes times 2^(exponent - 127) as bf16, exact.
__device__ __forceinline__ uint4 decode8(uint2 w, uint32_t exponent) {
  const float f = exponent_value(static_cast<int>(exponent));
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, f, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, f, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, f, true);
  return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                    __builtin_bit_cast(uint32_t, d));
}

// e4m3: load i of `st` into its 8 rows at `to`.
template <int DT, int kSubBytes, int kLoads>
__device__ __forceinline__ void commit_rows8(const Staged<DT, kLoads>& st, int i, char* to) {
#pragma unroll
  for (int u = 0; u < Width<DT>::kSubTiles; ++u) {
    *reinterpret_cast<uint4*>(to + u * kSubBytes + 16 * (threadIdx.x & 63)) =
        decode8(st.w[i * Width<DT>::kSubTiles + u], st.e[i]);
  }
}

#endif  // __HIP_DEVICE_COMPILE__

// ------------------------------------------------------------------------------------------------------- tile form

template <bool FP8, int KS>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_tile_kernel(PagedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int DT = tiles_of(KS);
  constexpr int kSubBytes = kKB * kRow * 2, kTileBytes = Width<DT>::kSubTiles * kSubBytes;
  __shared__ __attribute__((aligned(16))) char sK0[kTileBytes], sK1[kTileBytes], sV0[kTileBytes], sV1[kTileBytes];
  // Workgroup -> (tile, key head, part): XCD id % 8 takes every 8th unit (window, key head, part) with all its tiles, so that
  // its L2 reads the unit's keys once.
  const int64_t seq = blockIdx.x >> 3;
  const int64_t q_tiles = a.tokens.cu ? 1 : a.q_tiles;
  int64_t qt = seq % q_tiles, unit = (seq / q_tiles) * kXcds + (blockIdx.x & 7);
  const int part = static_cast<int>(unit % a.parts);
  unit /= a.parts;
  const int64_t kvh = unit % a.Hkv;
  int64_t b = unit / a.Hkv, tile;
  if (a.tokens.cu) {
    // The window of tile number b, of the windows with more than kRows rows.
    tile = b;
    int64_t left = b;
    b = -1;
    for (int64_t b0 = 0; b0 < a.tokens.B; b0 += 64) {
      const int64_t c = b0 + (threadIdx.x & 63);
      int n = 0, total;
      if (c < a.tokens.B) {
        int64_t first, count;
        window_tokens(a.tokens, c, first, count);
        if (!row_form(a, count)) n = static_cast<int>(cdiv(count * a.G, kTileRows));
      }
      const int before = wave_prefix(n, total);
      if (left < total) {
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before <= left && left < before + n));
        b = b0 + at;
        qt = left - __builtin_amdgcn_readlane(before, at);
        break;
      }
      left -= total;
    }
    if (b < 0 || tile >= a.tiles) return;
  } else {
    if (b >= a.tokens.B) return;
    tile = b * a.q_tiles + qt;
  }
  b = __builtin_amdgcn_readfirstlane(static_cast<int>(b));
  qt = __builtin_amdgcn_readfirstlane(static_cast<int>(qt));
  const Window w = window_at(a, b);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
  const int64_t r0 = qt * kTileRows, r = r0 + wave * kRows + col;
  // Keys that the tile's last row sees, and this part's blocks of them.
  const int64_t rows = w.count * a.G;
  const int64_t r1 = r0 + kTileRows < rows ? r0 + kTileRows : rows;
  const int keys = __builtin_amdgcn_readfirstlane(last_key(a, w, (r1 - 1) / a.G) + 1);
  const int blocks = (keys + kKB - 1) / kKB;
  int each = (blocks + a.parts - 1) / a.parts;
  if (each < kTileLeast) each = kTileLeast;
  const int count = blocks > each ? (blocks + each - 1) / each : 1;
  if (part >= count) return;
  if (a.plan && part == 0 && kvh == 0 && qt == 0 && threadIdx.x == 0) a.plan[b] = make_int4(static_cast<int>(tile), 0, 1, 0);
  const int blk0 = part * each, blk1 = blk0 + each < blocks ? blk0 + each : blocks;

  Rows<KS> s;
  load_rows<KS>(a, w, b, kvh, r, s);
  // K rows: lane (col, hh) takes logical chunk 2 k + hh of rows col and 32 + col, which share their swizzle.
  uint32_t rd[4], rvt[DT];
#pragma unroll
  for (int k = 0; k < 4; ++k) rd[k] = static_cast<uint32_t>(col * kRow * 2 + swz(col, 2 * k + hh) * 16);
  v_offsets<DT>(rvt);
  constexpr int ES = FP8 ? 1 : 2;
  const Source ks = k_source<ES>(a, kvh), vs = v_source<ES>(a, kvh);
  const int32_t* row = a.pages.table + b * a.pages.st_b;
  // The wave's rows see every key up to `all` and none past `any`.
  const int64_t wr0 = r0 + wave * kRows, wr1 = wr0 + kRows < rows ? wr0 + kRows : rows;
  const int all = __builtin_amdgcn_readfirstlane(wr0 < rows ? last_key(a, w, wr0 / a.G) : -1);
  const int any = __builtin_amdgcn_readfirstlane(wr0 < rows ? last_key(a, w, (wr1 - 1) / a.G) : -1);

  // The wave stages rows 8 wave .. and 8 (wave + 4) .. of a block: 16 keys at 16 (wave / 2) and at 32 + 16 (wave / 2).
  Staged<DT, FP8 ? 2 : 1> kst, vst;
  const int g0 = 16 * (wave >> 1), in_mask = (1 << a.pages.shift) - 1, D = static_cast<int>(a.D);
  const Lane8 kl = k_lane<ES>(a, wave & 1), vl = v_lane<ES>(a, wave & 1);
  auto issue = [&](int kv0, int p0, int p1, char* sK, char* sV) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = kv0 + 32 * i + g0, to = (8 * wave + 32 * i) * kRow * 2;
      int page = i ? p1 : p0;
      const int valid = valid_keys(a, keys, j, page);
      stage_rows8<FP8, DT, kSubBytes>(ks, kl, page, j & in_mask, valid, D, i, sK + to, kst);
      stage_rows8<FP8, DT, kSubBytes>(vs, vl, page, j & in_mask, valid, D, i, sV + to, vst);
    }
  };
  auto commit = [&](char* sK, char* sV) __attribute__((always_inline)) {
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        commit_rows8<DT, kSubBytes>(kst, i, sK + (8 * wave + 32 * i) * kRow * 2);
        commit_rows8<DT, kSubBytes>(vst, i, sV + (8 * wave + 32 * i) * kRow * 2);
      }
    }
  };
  auto compute = [&](int kv0, const char* sK, const char* sV) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key0 = kv0 + 32 * t;
      if (key0 > any) break;
      bf16x8_t ka[KS];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        ka[k] = *reinterpret_cast<const bf16x8_t*>(sK + (k >> 2) * kSubBytes + rd[k & 3] + 32 * t * kRow * 2);
      }
      attend_half<KS, kSubBytes>(s, scores<KS>(s, ka), sV + 32 * t * kRow * 2, rvt, a.scale_log2, key0 + 31 > all, key0);
    }
  };
  if (blk0 < blk1) {
    int p0 = page_number(a, row, kKB * blk0 + g0), p1 = page_number(a, row, kKB * blk0 + 32 + g0);
    issue(kKB * blk0, p0, p1, sK0, sV0);
    p0 = page_number(a, row, kKB * (blk0 + 1) + g0);
    p1 = page_number(a, row, kKB * (blk0 + 1) + 32 + g0);
    commit(sK0, sV0);
    wait_vmem();
    __syncthreads();
    auto step = [&](int blk, char* cK, char* cV, char* nK, char* nV) __attribute__((always_inline)) {
      const bool more = blk + 1 < blk1;
      if (more) issue(kKB * (blk + 1), p0, p1, nK, nV);
      p0 = page_number(a, row, kKB * (blk + 2) + g0);
      p1 = page_number(a, row, kKB * (blk + 2) + 32 + g0);
      compute(kKB * blk, cK, cV);
      if (more) {
        commit(nK, nV);
        wait_vmem();
        __syncthreads();
      }
    };
    for (int blk = blk0; blk < blk1; blk += 2) {
      step(blk, sK0, sV0, sK1, sV1);
      if (blk + 1 < blk1) step(blk + 1, sK1, sV1, sK0, sV0);
    }
  }
  const float l = row_sum(s.l[0]);
  if (r >= rows) return;
  if (count > 1) {
    float* slot = a.tile_part + ((tile * a.Hkv + kvh) * a.parts + part) * (kTileRows * (a.D + 2)) +
                  (wave * kRows + col) * (a.D + 2);
#pragma unroll
    for (int j = 0; j < DT; ++j) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d0 = 32 * j + 8 * g + 4 * hh;
        if (d0 < a.D) {
          *reinterpret_cast<float2*>(slot + d0) = make_float2(s.o[j][4 * g], s.o[j][4 * g + 1]);
          *reinterpret_cast<float2*>(slot + d0 + 2) = make_float2(s.o[j][4 * g + 2], s.o[j][4 * g + 3]);
        }
      }
    }
    if (hh == 0) *reinterpret_cast<float2*>(slot + a.D) = make_float2(s.m, l);
    return;
  }
  const int64_t i = r / a.G, g0q = r - i * a.G;
  uint16_t* out = a.o + (a.tokens.cu ? 0 : b * a.so_b) + (kvh * a.G + g0q) * a.so_h + (a.tokens.cu ? w.first + i : i) * a.so_n;
  const float inv = s.last >= 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int j = 0; j < DT; ++j) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d0 = 32 * j + 8 * g + 4 * hh;
      if (d0 < a.D) {
        *reinterpret_cast<uint2*>(out + d0) = make_uint2(bf16_pack2(s.o[j][4 * g] * inv, s.o[j][4 * g + 1] * inv),
                                                         bf16_pack2(s.o[j][4 * g + 2] * inv, s.o[j][4 * g + 3] * inv));
      }
    }
  }
#endif
}

// -------------------------------------------------------------------------------------------------------- row form

// The windows' parts, a workgroup's worth each: an equal share of all keys for kRowTarget workgroups, a multiple of kRowLeast
// (4 waves' blocks). The lengths are on the device, so every workgroup forms the plan for itself.
__device__ __forceinline__ int row_part_keys(const PagedArgs& a) {
  int64_t sum = 0;
  for (int64_t c = threadIdx.x & 63; c < a.tokens.B; c += 64) {
    int64_t first, count;
    window_tokens(a.tokens, c, first, count);
    if (count > 0 && row_form(a, count)) sum += held_keys(a.pages, c);
  }
  const int64_t share = cdiv(wave_sum(sum) * a.Hkv, kRowTarget);
  const int64_t each = cdiv(share, kRowLeast) * kRowLeast;
  return static_cast<int>(each < kRowLeast ? kRowLeast : (each < (1 << 30) ? each : (1 << 30)));
}

// A wave takes every 4th block of 32 keys of its part (e4m3 up to head_dim 64: of 64 keys, as many bytes). K rows go straight from memory to the A operands, a lane its
// own key's chunks, the next block's while the current one's softmax and second product run; V rows go through the wave's LDS,
// since they are read transposed.
template <bool FP8, int KS>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_row_kernel(PagedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int DT = tiles_of(KS), ES = FP8 ? 1 : 2;
  constexpr int kHalves = FP8 && KS <= 4 ? 2 : 1, kKeys = kRowKeys * kHalves;  // of a wave's block
  constexpr int kSubBytes = kKeys * kRow * 2, kTileBytes = Width<DT>::kSubTiles * kSubBytes;
  // V of the four waves, bf16 two blocks of each; O of them at the end, 32 DT x 32 floats each.
  constexpr int kWaveO = 32 * DT * kRows, kFirst = FP8 ? 4 : 2;  // waves whose O goes to sV0
  constexpr int kBuffer = 4 * kTileBytes > kFirst * kWaveO * 4 ? 4 * kTileBytes : kFirst * kWaveO * 4;
  __shared__ __attribute__((aligned(16))) char sV0[kBuffer], sV1[FP8 ? 16 : kBuffer];
  __shared__ float s_ml[4][2][kRows];
  const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroup -> (window, part, key head).
  const int each = __builtin_amdgcn_readfirstlane(row_part_keys(a));
  const int id = static_cast<int>(blockIdx.x);
  int64_t b = -1;
  int part = 0, kvh = 0, parts = 0, before_b = 0;
  int left = id;
  for (int64_t b0 = 0; b0 < a.tokens.B; b0 += 64) {
    const int64_t c = b0 + lane;
    int n = 0, total;
    if (c < a.tokens.B) {
      int64_t first, count;
      window_tokens(a.tokens, c, first, count);
      if (count > 0 && row_form(a, count)) {
        const int64_t L = held_keys(a.pages, c);
        n = static_cast<int>(L > each ? cdiv(L, each) : 1) * static_cast<int>(a.Hkv);
      }
    }
    const int before = wave_prefix(n, total);
    if (left < total) {
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before <= left && left < before + n));
      b = b0 + at;
      const int in = left - __builtin_amdgcn_readlane(before, at);
      parts = __builtin_amdgcn_readlane(n, at) / static_cast<int>(a.Hkv);
      kvh = in / parts;
      part = in - kvh * parts;
      before_b = id - in;
      break;
    }
    left -= total;
  }
  if (b < 0) return;
  b = __builtin_amdgcn_readfirstlane(static_cast<int>(b));
  kvh = __builtin_amdgcn_readfirstlane(kvh);
  part = __builtin_amdgcn_readfirstlane(part);
  if (part == 0 && kvh == 0 && threadIdx.x == 0) a.plan[b] = make_int4(before_b, parts, 0, 0);
  const Window w = window_at(a, b);
  const int rows = static_cast<int>(w.count * a.G);
  const int keys = __builtin_amdgcn_readfirstlane(w.keys);
  const int k0 = part * each, k1 = k0 + each < keys ? k0 + each : keys;

  Rows<KS> s;
  load_rows<KS>(a, w, b, kvh, col, s);
  uint32_t rvt[DT];
  v_offsets<DT>(rvt);
  const Source ks = k_source<ES>(a, kvh), vs = v_source<ES>(a, kvh);
  const Lane8 vl[2] = {v_lane<ES>(a, 0), v_lane<ES>(a, 1)};
  const int32_t* row = a.pages.table + b * a.pages.st_b;
  const int all = __builtin_amdgcn_readfirstlane(last_key(a, w, 0));
  const int in_mask = (1 << a.pages.shift) - 1, D = static_cast<int>(a.D);
  // The lane's key among 16, and its offsets in a K row (the last step's chunk may lie past head_dim, where Q is zero: any
  // chunk of the row then).
  const int own = sigma_row(col) & 15;
  const int64_t k_own = (own * ks.sr + 8 * hh) * ES;
  const int k_last = 16 * (KS - 1) + 8 * hh < D ? 16 * (KS - 1) * ES : -8 * hh * ES;

  using KWord = typename std::conditional<FP8, uint2, uint4>::type;
  KWord kw[kHalves][KS];
  uint32_t ke[FP8 ? kHalves : 1];
  Staged<DT, FP8 ? 4 * kHalves : 1> vst;
  int page[2 * kHalves], valid[2 * kHalves];   // of the 16-key groups of the block to load
  bool broken = false;                         // the block in kw has keys on a bad page
  auto find = [&](int kv) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 2 * kHalves; ++g) page[g] = page_number(a, row, kv + 16 * g);
  };
  auto check = [&](int kv) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 2 * kHalves; ++g) valid[g] = valid_keys(a, k1, kv + 16 * g, page[g]);
  };
  auto load_v = [&](int kv, char* to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4 * kHalves; ++i) {
      stage_rows8<FP8, DT, kSubBytes>(vs, vl[i & 1], page[i >> 1], (kv + 8 * i) & in_mask & ~15, valid[i >> 1], D, i,
                                      to + 8 * i * kRow * 2, vst);
    }
  };
  // Keys that do not exist are never loaded (the block's first one is read instead, or page 0 where its page is bad; pools
  // have a page wherever a window has keys): their scores are masked, but for bad pages, which count as zeros.
  auto load_k = [&](int kv) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kHalves; ++t) {
      const bool second = col >= 16;
      const int g0 = 2 * t, in0 = (kv + 32 * t) & in_mask, in1 = (kv + 32 * t + 16) & in_mask;
      const char* b0 = ks.rows + (page[g0] * ks.sp + in0 * ks.sr) * ES;
      const char* b1 = ks.rows + (page[g0 + 1] * ks.sp + in1 * ks.sr) * ES;
      const uint8_t *e0 = ks.exponents + page[g0] * ks.se + in0, *e1 = ks.exponents + page[g0 + 1] * ks.se + in1;
      const bool here = own < (second ? valid[g0 + 1] : valid[g0]);
      const char* first = valid[0] > 0 ? ks.rows + (page[0] * ks.sp + (kv & in_mask) * ks.sr) * ES : ks.rows;
      const char* at = here ? (second ? b1 : b0) + k_own : first + 8 * hh * ES;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        kw[t][k] = *reinterpret_cast<const KWord*>(at + (k < KS - 1 ? 16 * k * ES : k_last));
      }
      if constexpr (FP8) ke[t] = *(here ? (second ? e1 : e0) + own : ks.exponents);
    }
    broken = false;
#pragma unroll
    for (int g = 0; g < 2 * kHalves; ++g) broken |= valid[g] == 0 && kv + 16 * g < k1;
  };
  const int stride = 4 * kKeys;
  int kv = k0 + wave * kKeys;
  char *c0 = sV0 + wave * kTileBytes, *c1 = FP8 ? c0 : sV1 + wave * kTileBytes;
  if (kv < k1) {
    find(kv);
    check(kv);
    load_v(kv, c0);
    load_k(kv);
    int kvn = kv + stride;
    find(kvn);
    auto step = [&](char* cur, char* next) __attribute__((always_inline)) {
      const bool more = kvn < k1;
      if constexpr (FP8) {
#pragma unroll
        for (int i = 0; i < 4 * kHalves; ++i) commit_rows8<DT, kSubBytes>(vst, i, cur + 8 * i * kRow * 2);
      }
      if (more) {
        check(kvn);
        load_v(kvn, next);
      }
      f32x16_t x[kHalves];
#pragma unroll
      for (int t = 0; t < kHalves; ++t) {
        bf16x8_t ka[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          if constexpr (FP8) {
            ka[k] = __builtin_bit_cast(bf16x8_t, decode8(kw[t][k], ke[t]));
          } else {
            ka[k] = __builtin_bit_cast(bf16x8_t, kw[t][k]);
          }
        }
        x[t] = scores<KS>(s, ka);
        if (broken) {
          // (The pages' numbers are the next block's by now: looked up again.)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int g = kv + 32 * t + (i < 8 ? 0 : 16);
            if (static_cast<uint32_t>(page_number(a, row, g)) >= static_cast<uint32_t>(a.pages.pages)) x[t][i] = 0.f;
          }
        }
      }
      if (more) {
        load_k(kvn);
        find(kvn + stride);
      } else {
        broken = false;
      }
      // V of this block was on its way before K of this block, which has arrived: at most the next block's loads are left.
      if constexpr (!FP8) {
        if (more) {
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * Width<DT>::kSubTiles + KS) : "memory");
        } else {
          wait_vmem();
        }
      }
#pragma unroll
      for (int t = 0; t < kHalves; ++t) {
        if (t == 0 || kv + 32 * t < k1) {
          attend_half<KS, kSubBytes>(s, x[t], cur + 32 * t * kRow * 2, rvt, a.scale_log2, kv + 32 * t + 31 > all,
                                     kv + 32 * t);
        }
      }
      kv = kvn;
      kvn += stride;
    };
    while (kv < k1) {
      step(c0, c1);
      if (!FP8 && kv < k1) step(c1, c0);
    }
  }
  // The waves' sums joined, in order: O of wave w [head_dim][row].
  const float l = row_sum(s.l[0]);
  __syncthreads();
  float* so = reinterpret_cast<float*>(wave < kFirst ? sV0 : sV1) + (wave % kFirst) * kWaveO;
  if (hh == 0) {
    s_ml[wave][0][col] = s.m;
    s_ml[wave][1][col] = l;
  }
#pragma unroll
  for (int j = 0; j < DT; ++j) {
#pragma unroll
    for (int e = 0; e < 16; ++e) so[(32 * j + 8 * (e >> 2) + 4 * hh + (e & 3)) * kRows + col] = s.o[j][e];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * (D / 2); e += kPagedThreads) {
    const int rr = e / (D / 2), d = 2 * (e - rr * (D / 2));
    float m = s_ml[0][0][rr];
#pragma unroll
    for (int x = 1; x < 4; ++x) m = fmaxf(m, s_ml[x][0][rr]);
    float sum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = __builtin_amdgcn_exp2f(s_ml[x][0][rr] - m);
      const float* from = reinterpret_cast<const float*>(x < kFirst ? sV0 : sV1) + (x % kFirst) * kWaveO;
      sum = __builtin_fmaf(s_ml[x][1][rr], f, sum);
      o0 = __builtin_fmaf(from[d * kRows + rr], f, o0);
      o1 = __builtin_fmaf(from[(d + 1) * kRows + rr], f, o1);
    }
    if (parts > 1) {
      float* slot = a.row_part + (static_cast<int64_t>(id) * a.slot_rows + rr) * (D + 2);
      *reinterpret_cast<float2*>(slot + d) = make_float2(o0, o1);
      if (d == 0) *reinterpret_cast<float2*>(slot + D) = make_float2(m, sum);
    } else {
      const int64_t i = rr / a.G, g = rr - i * a.G;
      uint16_t* out = a.o + (a.tokens.cu ? 0 : b * a.so_b) + (kvh * a.G + g) * a.so_h + (a.tokens.cu ? w.first + i : i) * a.so_n;
      const float inv = last_key(a, w, i) >= 0 ? 1.f / sum : 0.f;
      *reinterpret_cast<uint32_t*>(out + d) = bf16_pack2(o0 * inv, o1 * inv);
    }
  }
#endif
}

// The parts of a row joined in order. 32 lanes a row, 4 elements a lane, kAhead parts in flight.
constexpr int kAhead = 8;

__global__ __launch_bounds__(kPagedThreads) void paged_join_kernel(PagedArgs a) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kPagedThreads / 32) + threadIdx.x / 32;
  const int d0 = 4 * (threadIdx.x % 32);
  const int64_t total = (a.tokens.cu ? a.tokens.N : a.tokens.B * a.tokens.N);
  const int64_t token = id / a.H, h = id - token * a.H;
  if (token >= total || d0 >= a.D) return;
  const int64_t b = a.tokens.cu ? window_of(a.tokens, token) : token / a.tokens.N;
  if (b < 0) return;
  const Window w = window_at(a, b);
  if (w.count <= 0) return;
  const int64_t i = token - w.first, kvh = h / a.G, r = i * a.G + (h - kvh * a.G);
  const int4 plan = a.plan[b];
  const float* slot;
  int64_t step;
  int count;
  if (row_form(a, w.count)) {
    count = plan.y;
    if (plan.x < 0 || count < 0 || plan.x + a.Hkv * count > a.row_slots) return set_bad(a.pages);  // borders not ascending
    slot = a.row_part + ((plan.x + kvh * count) * a.slot_rows + r) * (a.D + 2);
    step = a.slot_rows * (a.D + 2);
  } else {
    const int64_t r0 = r / kTileRows * kTileRows, rows = w.count * a.G;
    const int64_t r1 = r0 + kTileRows < rows ? r0 + kTileRows : rows;
    const int blocks = (last_key(a, w, (r1 - 1) / a.G) + kKB) / kKB;
    int each = (blocks + a.parts - 1) / a.parts;
    if (each < kTileLeast) each = kTileLeast;
    count = blocks > each ? (blocks + each - 1) / each : 1;
    if (plan.x < 0 || plan.x + r / kTileRows >= a.tiles) return set_bad(a.pages);
    slot = a.tile_part + ((plan.x + r / kTileRows) * a.Hkv + kvh) * a.parts * (kTileRows * (a.D + 2)) + (r - r0) * (a.D + 2);
    step = kTileRows * (a.D + 2);
  }
  if (count < 2) return;
  float m = kNoMax, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < count; p0 += kAhead, slot += kAhead * step) {
    float2 ml[kAhead], oa[kAhead], ob[kAhead];
#pragma unroll
    for (int p = 0; p < kAhead; ++p) {  // the last part again behind the end: no branch around the loads
      const float* at = slot + (p0 + p < count ? p : count - 1 - p0) * step;
      ml[p] = *reinterpret_cast<const float2*>(at + a.D);
      oa[p] = *reinterpret_cast<const float2*>(at + d0);
      ob[p] = *reinterpret_cast<const float2*>(at + d0 + 2);
    }
#pragma unroll
    for (int p = 0; p < kAhead; ++p) {
      if (p0 + p >= count) break;
      const float mn = fmaxf(m, ml[p].x), x = __builtin_amdgcn_exp2f(m - mn), y = __builtin_amdgcn_exp2f(ml[p].x - mn);
      m = mn;
      l = join_value(l, ml[p].y, x, y);
      o[0] = join_value(o[0], oa[p].x, x, y);
      o[1] = join_value(o[1], oa[p].y, x, y);
      o[2] = join_value(o[2], ob[p].x, x, y);
      o[3] = join_value(o[3], ob[p].y, x, y);
    }
  }
  const float inv = last_key(a, w, i) >= 0 ? 1.f / l : 0.f;
  uint16_t* out = a.o + (a.tokens.cu ? 0 : b * a.so_b) + h * a.so_h + (a.tokens.cu ? token : i) * a.so_n;
  *reinterpret_cast<uint2*>(out + d0) = make_uint2(bf16_pack2(o[0] * inv, o[1] * inv), bf16_pack2(o[2] * inv, o[3] * inv));
}

// What a call launches, by its sizes alone.
struct PagedPlan {
  bool rows, tiles;        // the forms that its windows may take
  int64_t q_tiles, tile_count;
  int parts;
  int64_t row_slots;
  int slot_rows;
  int64_t row_floats, tile_floats, plan_windows;
  size_t bytes() const { return static_cast<size_t>(row_floats + tile_floats) * 4 + static_cast<size_t>(plan_windows) * 16; }
};

inline PagedPlan paged_plan(int64_t B, int64_t H, int64_t Hkv, int64_t N, bool packed, int64_t D, int64_t max_keys) {
  PagedPlan p{};
  const int64_t G = H / Hkv;
  p.rows = packed || N * G <= kRows;
  p.tiles = N * G > kRows;
  p.parts = 1;
  if (p.tiles) {
    p.q_tiles = packed ? 1 : cdiv(N * G, kTileRows);
    p.tile_count = packed ? N * G / kTileRows + (N * G / (kRows + 1) < B ? N * G / (kRows + 1) : B) : B * p.q_tiles;
    const int64_t most = cdiv(cdiv(max_keys, kKB), kTileLeast), want = kTileTarget / (p.tile_count * Hkv);
    p.parts = static_cast<int>(want < 1 ? 1 : (want < most ? want : (most < 1 ? 1 : most)));
    if (p.parts > 1) p.tile_floats = p.tile_count * Hkv * p.parts * kTileRows * (D + 2);
  }
  if (p.rows) {
    p.row_slots = kRowTarget + B * Hkv;
    p.slot_rows = static_cast<int>(packed ? (N * G < kRows ? N * G : kRows) : N * G);
    p.row_floats = p.row_slots * p.slot_rows * (D + 2);
    p.row_floats += p.row_floats & 1;
  }
  p.tile_floats = (p.tile_floats + 3) / 4 * 4;
  p.row_floats = (p.row_floats + 3) / 4 * 4;
  p.plan_windows = p.rows || p.parts > 1 ? B : 0;
  return p;
}

template <bool FP8, int KS>
void launch_paged(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  if (p.rows) {
    paged_row_kernel<FP8, KS><<<static_cast<unsigned>(p.row_slots), kPagedThreads, 0, s>>>(a);
  }
  if (p.tiles) {
    const int64_t units = p.tile_count / p.q_tiles * a.Hkv * p.parts;
    paged_tile_kernel<FP8, KS><<<static_cast<unsigned>(cdiv(units, kXcds) * kXcds * p.q_tiles), kPagedThreads, 0, s>>>(a);
  }
}

// By the steps that head_dim takes.
template <bool FP8>
void launch_width(const PagedArgs& a, const PagedPlan& p, hipStream_t s) {
  switch (static_cast<int>(cdiv(a.D, 16))) {
    case 8: return launch_paged<FP8, 8>(a, p, s);
    case 7: return launch_paged<FP8, 7>(a, p, s);
    case 6: return launch_paged<FP8, 6>(a, p, s);
    case 5: return launch_paged<FP8, 5>(a, p, s);
    case 4: return launch_paged<FP8, 4>(a, p, s);
    case 3: return launch_paged<FP8, 3>(a, p, s);
    case 2: return launch_paged<FP8, 2>(a, p, s);
    default: return launch_paged<FP8, 1>(a, p, s);
  }
}

}  // namespace svhip

using namespace svhip;

extern "C" size_t svhip_paged_attention_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t N, int packed,
                                                        int64_t D, int64_t max_keys) {
  if (B < 1 || H < 1 || Hkv < 1 || H % Hkv != 0 || N < 1 || D < 1 || max_keys < 0) return 0;
  return paged_plan(B, H, Hkv, N, packed != 0, D, max_keys).bytes();
}

extern "C" int svhip_paged_attention(const svhip_paged_cache* cache, const svhip_paged_attention_args* args,
                                     void* stream) {
  const char* name = "svhip_paged_attention";
  clear_error();
  if (const int rc = check_cache(name, cache)) return rc;
  SVHIP_REQUIRE(args, "%s: null arguments", name);
  const svhip_paged_cache& pc = *cache;
  const svhip_paged_attention_args& c = *args;
  const int64_t B = pc.windows, H = c.H, Hkv = pc.heads, N = c.N, D = pc.head_dim;
  SVHIP_REQUIRE(H >= 0 && N >= 0, "%s: bad sizes", name);
  SVHIP_REQUIRE(Hkv >= 1 && H % Hkv == 0, "%s: %lld heads do not share %lld key heads evenly", name, (long long)H,
                (long long)Hkv);
  const float scale = static_cast<float>(c.scale);
  SVHIP_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", name);
  if (B == 0 || H == 0 || N == 0) return SVHIP_OK;
  if (const int rc = check_pool(name, pc)) return rc;
  SVHIP_REQUIRE(c.q && c.out, "%s: null pointer", name);
  SVHIP_REQUIRE(rows16(c.q, c.sq_b, c.sq_h, c.sq_n), "%s: query rows must start on 16-byte boundaries", name);
  SVHIP_REQUIRE(reinterpret_cast<uintptr_t>(c.out) % 8 == 0 && (c.so_b | c.so_h | c.so_n) % 4 == 0,
                "%s: rows of out must start on 8-byte boundaries", name);
  const PagedPlan p = paged_plan(B, H, Hkv, N, c.cu_queries != nullptr, D, pc.max_pages * pc.page_size);
  SVHIP_REQUIRE(p.bytes() == 0 || (c.workspace && c.workspace_bytes >= static_cast<int64_t>(p.bytes()) &&
                                   reinterpret_cast<uintptr_t>(c.workspace) % 16 == 0),
                "%s: workspace too small or misaligned (%lld < %zu bytes)", name, (long long)c.workspace_bytes, p.bytes());
  const int64_t rows = (c.cu_queries ? N : B * N) * H, join = cdiv(rows, kPagedThreads / 32);
  SVHIP_REQUIRE(p.row_slots < (1ll << 31) && p.tile_count * Hkv * p.parts < (1ll << 30) && join < (1ll << 31),
                "%s: grid too large", name);
  float* const part = static_cast<float*>(c.workspace);
  const PagedArgs a{static_cast<const uint16_t*>(c.q), pc.k_pages, pc.v_pages, pc.k_exponents, pc.v_exponents,
                    static_cast<uint16_t*>(c.out), Tokens{c.cu_queries, B, N}, pages_of(pc), H, Hkv, H / Hkv, D, c.sq_b,
                    c.sq_h, c.sq_n, pc.sk_p, pc.sk_h, pc.sk_r, pc.sv_p, pc.sv_h, pc.sv_r, pc.sek_p, pc.sek_h, pc.sev_p,
                    pc.sev_h, c.so_b, c.so_h, c.so_n, c.causal != 0, scale * kLog2e, p.q_tiles, p.tile_count, p.parts,
                    p.row_slots, p.slot_rows, part, part + p.row_floats,
                    p.plan_windows ? reinterpret_cast<int4*>(part + p.row_floats + p.tile_floats) : nullptr};
  hipStream_t s = as_stream(stream);
  if (pc.kv_dtype == SVHIP_FP8_E4M3) {
    launch_width<true>(a, p, s);
  } else {
    launch_width<false>(a, p, s);
  }
  if (p.plan_windows) paged_join_kernel<<<static_cast<unsigned>(join), kPagedThreads, 0, s>>>(a);
  SVHIP_LAUNCHED(name);
  return SVHIP_OK;
}
