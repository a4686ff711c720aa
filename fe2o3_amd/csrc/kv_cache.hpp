// kv_cache.hpp -- the paged key-value cache as its kernels see it: the
// division by a page's size, the quotients of the e4m3 write, the host's checks
// of the caller's record, and the form passed to kernels.
#pragma once

#include <stdint.h>

#include "../../include/fe2o3_mi355x.h"

#if defined(__HIPCC__)
#define FE2O3_KV_HD __host__ __device__ __forceinline__
#else
#define FE2O3_KV_HD inline
#endif

namespace kv_cache {

// n / d and n % d of n < 2^31 by a multiplication and a shift (Granlund and
// Montgomery's division by an invariant integer): with 2^l the
// least power of two >= d and m = ceil(2^(31+l) / d), n m / 2^(31+l) exceeds
// n / d by n e / (d 2^(31+l)) with e < d <= 2^l, which is less than 1 / d for
// n < 2^31, so the floors agree.  m fits 32 bits, since d > 2^(l-1) (for d = 1
// it is 2^31).
struct FastDiv {
  uint32_t mul, shift, divisor;
  static inline FastDiv of(uint32_t d) {
    uint32_t l = 0;
    while (l < 32u && (UINT64_C(1) << l) < d) ++l;
    // 31 + l <= 62 for d < 2^31
    const uint64_t m = ((UINT64_C(1) << (31u + l)) + d - 1u) / d;
    return FastDiv{(uint32_t)m, 31u + l, d};
  }
  FE2O3_KV_HD uint32_t div(uint32_t n) const {
    return (uint32_t)(((uint64_t)n * mul) >> shift);
  }
};

// A list of workgroups as a grid of rows of kGridWidth: number blockIdx.y * kGridWidth +
// blockIdx.x, those from n on in the last row with nothing to do.  A dimension of a grid
// holds fewer than 2^32 threads, and a workgroup has up to 1024.
constexpr uint32_t kGridWidth = 1u << 21;
struct Grid {
  uint32_t x, y;
  static inline Grid of(uint32_t n) {  // 1 <= n < 2^31
    return n < kGridWidth ? Grid{n, 1u} : Grid{kGridWidth, (n - 1u) / kGridWidth + 1u};
  }
};

// A row's scale and what divides by it.  x / scale is q = RN(x r) with r the rounded
// reciprocal, corrected once by its remainder: the correctly rounded quotient while
// the remainder is exact (r is at most half an ulp off, q less than one).  The remainder's
// last bit is at least 2^-46 of scale times q's binade; the codes need the quotients
// from 2^-11 up, so scales from 2^-92 up, whose remainders end at 2^-149 or above, give
// the division's code for every bf16 x up to the row's largest.  Smaller and infinite
// scales divide.  The remainder is taken as q scale - x, which is +0 where it is
// none, so that q keeps a zero's sign.  A host check goes through all largest values
// and x.  Three operations instead of the division's ten, with the hardware's packing
// of codes: 32768 tokens of 8 heads 79 us -> 44 (42 with nontemporal stores).
struct RowScale {
  float scale, r;
  bool usual;
  explicit FE2O3_KV_HD RowScale(float amax) {
    scale = (amax > 0x1p-126f ? amax : 0x1p-126f) / 448.0f;
    r = 1.0f / scale;
    usual = scale >= 0x1p-92f && scale <= 0x1.fffffep127f;
  }
  FE2O3_KV_HD float quotient(float x) const {
    const float q = x * r;
    return __builtin_fmaf(-__builtin_fmaf(q, scale, -x), r, q);
  }
};

// A cache's arrays and strides, in elements of its format.
struct View {
  uint8_t *k, *v;
  float *k_scale, *v_scale;  // E4M3: [pages, kv_heads, page_size]
  uint64_t page_stride, token_stride, head_stride;
  FastDiv page;  // of the slots in a page
  uint32_t pages, kv_heads, head_dim;
};

inline bool mul_ok(uint64_t a, uint64_t b, uint64_t* out) {
  return !__builtin_mul_overflow(a, b, out);
}
// (n - 1) * stride, n >= 1
inline bool reach(uint64_t n, uint64_t stride, uint64_t* total) {
  uint64_t add;
  return mul_ok(n - 1u, stride, &add) && !__builtin_add_overflow(*total, add, total);
}

// Rows of head_dim elements at (token, head) of a [tokens, heads, head_dim]
// array with these strides: FE2O3_ERR_STRIDE where two rows would share
// elements (one of the orders has to nest: heads within a token, or tokens
// within a head); otherwise the extent, FE2O3_ERR_OVERFLOW past 64 bits.
inline int32_t rows_extent(uint64_t tokens, uint64_t heads, uint64_t head_dim,
                           uint64_t token_stride, uint64_t head_stride, uint64_t* extent) {
  uint64_t token_reach = head_dim, head_reach = head_dim;
  if (!reach(heads, head_stride, &token_reach) || !reach(tokens, token_stride, &head_reach))
    return FE2O3_ERR_OVERFLOW;
  const bool heads_apart = heads == 1u || head_stride >= head_dim;
  const bool tokens_apart = tokens == 1u || token_stride >= head_dim;
  const bool nested = tokens == 1u || heads == 1u || token_stride >= token_reach ||
                      head_stride >= head_reach;
  if (!heads_apart || !tokens_apart || !nested) return FE2O3_ERR_STRIDE;
  *extent = token_reach;
  return reach(tokens, token_stride, extent) ? FE2O3_OK : FE2O3_ERR_OVERFLOW;
}

// The caller's record checked, in the order the header states.
inline int32_t check(const Fe2o3KvCacheV1* c, View* out) {
  if (c == nullptr) return FE2O3_ERR_NULL;
  if (c->format != FE2O3_KV_BF16 && c->format != FE2O3_KV_E4M3) return FE2O3_ERR_SHAPE;
  if (c->pages == 0u || c->page_size == 0u || c->kv_heads == 0u || c->head_dim == 0u)
    return FE2O3_ERR_SHAPE;
  const uint64_t slots = (uint64_t)c->pages * c->page_size;
  if (slots >= (UINT64_C(1) << 31) || c->head_dim >= (UINT32_C(1) << 31)) return FE2O3_ERR_SHAPE;
  uint64_t extent;
  const int32_t rc = rows_extent(c->page_size, c->kv_heads, c->head_dim, c->token_stride,
                                 c->head_stride, &extent);
  if (rc != FE2O3_OK) return rc;
  if (c->pages > 1u && c->page_stride < extent) return FE2O3_ERR_STRIDE;
  uint64_t bytes;
  if (!reach(c->pages, c->page_stride, &extent) || !mul_ok(extent, 2u, &bytes))
    return FE2O3_ERR_OVERFLOW;
  if (c->k_len < extent || c->v_len < extent) return FE2O3_ERR_LENGTH;
  const bool scaled = c->format == FE2O3_KV_E4M3;
  uint64_t scales = 0;
  if (scaled && !mul_ok(slots, c->kv_heads, &scales)) return FE2O3_ERR_OVERFLOW;
  if (c->k_scale_len != scales || c->v_scale_len != scales) return FE2O3_ERR_LENGTH;
  if (!c->k || !c->v || (scaled && (!c->k_scale || !c->v_scale))) return FE2O3_ERR_NULL;
  if (!scaled && (((uintptr_t)c->k | (uintptr_t)c->v) & 1u) != 0u) return FE2O3_ERR_ALIGNMENT;
  if (scaled && (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3u) != 0u)
    return FE2O3_ERR_ALIGNMENT;
  // the stride of a dimension of one says nothing
  *out = View{(uint8_t*)c->k,
              (uint8_t*)c->v,
              c->k_scale,
              c->v_scale,
              c->pages > 1u ? c->page_stride : 0u,
              c->page_size > 1u ? c->token_stride : 0u,
              c->kv_heads > 1u ? c->head_stride : 0u,
              FastDiv::of(c->page_size),
              c->pages,
              c->kv_heads,
              c->head_dim};
  return FE2O3_OK;
}

// Whether every row of the cache starts at a multiple of `bytes` (a power of two).
inline bool rows_aligned(const View& c, uint32_t format, uint64_t bytes) {
  const uint64_t strides = c.page_stride | c.token_stride | c.head_stride;
  const uint64_t all = (uint64_t)(uintptr_t)c.k | (uint64_t)(uintptr_t)c.v |
                       strides * (format == FE2O3_KV_BF16 ? 2u : 1u);
  return (all & (bytes - 1u)) == 0u;
}

}  // namespace kv_cache
