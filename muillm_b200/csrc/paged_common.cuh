// What the paged-cache kernels share: the device view of a paged cache and of the new tokens' layout, the search for a
// token's sequence, and the e4m3 helpers.
#pragma once

#include "common.cuh"

#define MUI_DEV_BAD_PAGE 6u  // a block-table entry outside [0, num_pages); detail: sequence index

// Sequences are packed: new token t of sequence b is row cu[b] + t of q / k / v / out (row b when cu == nullptr: one
// new token per sequence) and stands at cache position context_lens[b] + t.
struct PagedView {
  void *k_pages, *v_pages;      // [num_pages, kv_heads, page_size, head_dim], 16-bit elements or e4m3 bytes
  float *k_scales, *v_scales;   // [num_pages, kv_heads], e4m3 only
  const int32_t* block_table;   // [batch, table_stride]
  const int32_t* context_lens;  // [batch]
  const int32_t* cu;            // [batch + 1] or nullptr
  int num_pages, page_shift, kv_heads, batch, table_stride, total;
};

inline PagedView paged_view(const mui_paged_kv_t& c) {
  PagedView v;
  v.k_pages = c.k_pages;
  v.v_pages = c.v_pages;
  v.k_scales = c.k_scales;
  v.v_scales = c.v_scales;
  v.block_table = c.block_table;
  v.context_lens = c.context_lens;
  v.cu = c.cu_tokens;
  v.num_pages = c.num_pages;
  v.page_shift = __builtin_ctz(static_cast<unsigned>(c.page_size));
  v.kv_heads = c.kv_heads;
  v.batch = c.batch;
  v.table_stride = c.table_stride;
  v.total = c.total_tokens;
  return v;
}

// argument checks shared by the entry points; MUI_OK or a status with the error text set
inline mui_status_t paged_check(mui_dtype_t dtype, const mui_paged_kv_t* c) {
  MUI_REQUIRE(dtype == MUI_F16 || dtype == MUI_BF16, MUI_ERR_UNSUPPORTED, "dtype %d unsupported", (int)dtype);
  MUI_REQUIRE(c != nullptr, MUI_ERR_INVALID_ARG, "cache description must be non-null");
  MUI_REQUIRE(c->format == MUI_KV_16BIT || c->format == MUI_KV_E4M3, MUI_ERR_UNSUPPORTED, "cache format %d unsupported",
              (int)c->format);
  MUI_REQUIRE(c->head_dim == 64 || c->head_dim == 128, MUI_ERR_UNSUPPORTED, "head dim %d unsupported (64 or 128)",
              c->head_dim);
  MUI_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128,
              MUI_ERR_UNSUPPORTED, "page size %d unsupported (16, 32, 64 or 128)", c->page_size);
  MUI_REQUIRE(c->kv_heads >= 1 && c->num_pages >= 1 && c->batch >= 0 && c->total_tokens >= 0 && c->table_stride >= 1,
              MUI_ERR_INVALID_ARG, "bad sizes kv_heads=%d num_pages=%d batch=%d total_tokens=%d table_stride=%d",
              c->kv_heads, c->num_pages, c->batch, c->total_tokens, c->table_stride);
  MUI_REQUIRE(c->kv_heads <= 65535 && c->batch <= 65535, MUI_ERR_UNSUPPORTED, "kv_heads=%d or batch=%d above 65535",
              c->kv_heads, c->batch);
  MUI_REQUIRE(c->cu_tokens != nullptr || c->total_tokens == c->batch, MUI_ERR_INVALID_ARG,
              "total_tokens=%d must equal batch=%d without cu_tokens", c->total_tokens, c->batch);
  if (c->batch == 0 || c->total_tokens == 0) return MUI_OK;
  MUI_REQUIRE(c->k_pages && c->v_pages && c->block_table && c->context_lens, MUI_ERR_INVALID_ARG,
              "pages, block table and context lengths must be non-null");
  MUI_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_pages) | reinterpret_cast<uintptr_t>(c->v_pages)) & 15) == 0,
              MUI_ERR_INVALID_ARG, "pages must be 16-byte aligned");
  MUI_REQUIRE(c->format != MUI_KV_E4M3 || (c->k_scales && c->v_scales), MUI_ERR_INVALID_ARG,
              "e4m3 pages need k_scales and v_scales");
  return MUI_OK;
}

// How many of the `batch` non-decreasing values value(0), value(1), ... are <= x: with value(i) = the first unit of
// sequence i + 1 that is the sequence of unit x. Whole warp: the range is cut into 32 blocks whose last values the lanes look at,
// until a block has one value: one step for 32 sequences, two for 1024, four for 65535 (one after the other, 4096 sequences cost
// each token 128 round trips). Values that are not in order give a number within the range.
template <typename F>
__device__ __forceinline__ int warp_count_le(int batch, int x, F value) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = batch;  // the answer is in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32, i = lane * step + step - 1;
    const unsigned m = __ballot_sync(MUI_FULL_MASK, i < n && value(lo + i) <= x);
    const int whole = m == MUI_FULL_MASK ? 32 : __ffs(~m) - 1;  // blocks of which all values are <= x
    lo += whole * step;
    n = min(step - 1, n - whole * step);
  }
  return lo;
}

// new tokens of sequence b as [first row, count], clamped to the rows that exist
__device__ __forceinline__ void paged_new_tokens(const PagedView& v, int b, int& first, int& count) {
  if (v.cu == nullptr) {
    first = b;
    count = 1;
  } else {
    first = max(0, __ldcg(v.cu + b));
    count = max(0, min(v.total, __ldcg(v.cu + b + 1)) - first);
  }
}

// ---- e4m3 ----
// two fp32 values -> two e4m3 bytes (first one low), round to nearest even, beyond +-448 saturated, NaN kept
__device__ __forceinline__ uint32_t e4m3_pack2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// two e4m3 bytes -> two halves (exact)
__device__ __forceinline__ uint32_t e4m3_to_half2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
// Exponent e of the page scale 2^e: the smallest with amax <= 448 * 2^e, at least -100. With amax = m * 2^k, m in
// [1, 2), and 448 = 1.75 * 2^8 that is k - 8, or k - 7 where m > 1.75.
__device__ __forceinline__ int e4m3_scale_exp(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int k = static_cast<int>(bits >> 23) - 127;
  return max(-100, k - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
