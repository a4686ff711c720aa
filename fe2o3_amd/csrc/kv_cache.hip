// kv_cache.hip -- a paged key-value cache on gfx950: new rows written into
// their slots, copied, quantised to e4m3 with a scale per token and head, or to
// microscaled 4-bit blocks of 32 (mxfp4.hpp); and cached rows of several
// sequences read back as packed bf16.
//
// Both are one pass over the rows, bound by memory: 32768 tokens of 8 heads, 128
// wide, bf16 51 us = 5.2 TB/s, e4m3 41 us = 5.0, 4-bit 28 us = 6.0; 16 sequences
// of 1 to 4097 read back from e4m3 34 us = 6.0, 8 of 4096 from 4-bit 28 us = 6.0.  A row (token, head) of K and the same of V belong
// to a group of `lanes` adjacent lanes, a power of two, 8 elements each: 16 bytes
// of bf16, 8 bytes of codes.  Adjacent groups take adjacent heads of a token, so
// that a wave reads and writes runs of whole cache lines wherever heads are
// dense.  gfx950's global accesses take any alignment, so odd strides need no
// other kernel; the last elements of a head_dim that is no multiple of 8 go one
// by one.
#include "common.hpp"
#include "internal.hpp"
#include "kv_cache.hpp"
#include "mxfp4.hpp"

namespace {

using namespace fe2o3;
using kv_cache::FastDiv;
using kv_cache::RowScale;
using kv_cache::View;

// a cache's format, FE2O3_KV_*
constexpr uint32_t kBf16 = FE2O3_KV_BF16, kE4m3 = FE2O3_KV_E4M3, kMxfp4 = FE2O3_KV_MXFP4;

constexpr int kThreads = 256;
constexpr uint32_t kMaxGrid = 1u << 20;  // workgroups

typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any_t __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_any_t __attribute__((aligned(1)));

// 8 bf16 values, the first `n` of them in memory (the others +0)
FE2O3_DEVICE u32x4_t load_bf16x8(const uint16_t* p, uint32_t n) {
  if (n >= 8u) return *reinterpret_cast<const u32x4_any_t*>(p);
  u32x4_t x = {0, 0, 0, 0};
#pragma unroll
  for (uint32_t i = 0; i < 7u; ++i)
    if (i < n) x[i / 2u] |= (uint32_t)p[i] << (16u * (i & 1u));
  return x;
}
FE2O3_DEVICE void store_bf16x8(uint16_t* p, u32x4_t x, uint32_t n) {
  if (n >= 8u) {
    __builtin_nontemporal_store(x, reinterpret_cast<u32x4_any_t*>(p));
    return;
  }
#pragma unroll
  for (uint32_t i = 0; i < 7u; ++i)
    if (i < n) p[i] = (uint16_t)(x[i / 2u] >> (16u * (i & 1u)));
}
FE2O3_DEVICE u32x2_t load_codes8(const uint8_t* p, uint32_t n) {
  if (n >= 8u) return *reinterpret_cast<const u32x2_any_t*>(p);
  u32x2_t x = {0, 0};
#pragma unroll
  for (uint32_t i = 0; i < 7u; ++i)
    if (i < n) x[i / 4u] |= (uint32_t)p[i] << (8u * (i & 3u));
  return x;
}
FE2O3_DEVICE void store_codes8(uint8_t* p, u32x2_t x, uint32_t n) {
  if (n >= 8u) {
    __builtin_nontemporal_store(x, reinterpret_cast<u32x2_any_t*>(p));
    return;
  }
#pragma unroll
  for (uint32_t i = 0; i < 7u; ++i)
    if (i < n) p[i] = (uint8_t)(x[i / 4u] >> (8u * (i & 3u)));
}

FE2O3_DEVICE float bf16_of(u32x4_t x, int i) {
  const uint32_t w = x[i / 2];
  return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
}

// max |x| of the 8; fmaxf leaves NaN out
FE2O3_DEVICE float amax8(u32x4_t x, float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(bf16_of(x, i)));
  return m;
}

FE2O3_DEVICE u32x2_t quantize8(u32x4_t x, const RowScale& s) {
  u32x2_t q;
  if (s.usual) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      // the quotients are at most 448 in magnitude: nothing to saturate
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(s.quotient(bf16_of(x, 4 * w)),
                                              s.quotient(bf16_of(x, 4 * w + 1)), 0, false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(s.quotient(bf16_of(x, 4 * w + 2)),
                                          s.quotient(bf16_of(x, 4 * w + 3)), c, true);
      q[w] = (uint32_t)c;
    }
  } else {
    q = u32x2_t{0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[i / 4] |= (uint32_t)e4m3_from_f32(bf16_of(x, i) / s.scale) << (8 * (i & 3));
  }
  return q;
}

// 8 codes times their row's scale: an f32 product, then bf16
FE2O3_DEVICE u32x4_t widen8(u32x2_t q, float scale) {
  u32x4_t x;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(q[w], false);
    const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8(q[w], true);
    x[2 * w] = pack_bf16x2(lo[0] * scale, lo[1] * scale);
    x[2 * w + 1] = pack_bf16x2(hi[0] * scale, hi[1] * scale);
  }
  return x;
}

// elements of chunk c (8 each) that a row of head_dim has
FE2O3_DEVICE uint32_t chunk_left(uint32_t head_dim, uint32_t c) {
  return min(head_dim - 8u * c, 8u);
}

struct WriteArgs {
  View cache;
  const uint16_t *k, *v;
  const uint32_t* slots;
  FastDiv heads;
  uint64_t token_stride, head_stride;
  uint32_t rows, lanes_log2;  // rows = tokens * kv_heads
};

// Rows of a group one after another, a whole grid's groups apart: a grid holds
// at most kMaxGrid workgroups, and only the largest calls take a second turn.
template <uint32_t F>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(WriteArgs a) {
  const uint32_t lanes = 1u << a.lanes_log2, c0 = threadIdx.x & (lanes - 1u);
  const uint32_t chunks = (a.cache.head_dim + 7u) / 8u;
  const uint32_t step = gridDim.x * ((uint32_t)kThreads >> a.lanes_log2);
  for (uint32_t row = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) >> a.lanes_log2;
       row < a.rows; row += step) {
    const uint32_t token = a.heads.div(row), head = row - token * a.heads.divisor;
    const uint32_t slot = a.slots[token];
    const uint64_t from = token * a.token_stride + head * a.head_stride;
    const uint16_t *k = a.k + from, *v = a.v + from;
    // the first chunk's loads need not wait for the slot
    u32x4_t kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
    if (c0 < chunks) {
      const uint32_t n = chunk_left(a.cache.head_dim, c0);
      kx = load_bf16x8(k + 8u * c0, n);
      vx = load_bf16x8(v + 8u * c0, n);
    }
    if (slot >= a.cache.pages * a.cache.page.divisor) continue;  // the whole group
    const uint32_t page = a.cache.page.div(slot), place = slot - page * a.cache.page.divisor;
    const uint64_t to = page * a.cache.page_stride + place * a.cache.token_stride +
                        head * a.cache.head_stride;
    if constexpr (F == kBf16) {
      uint16_t *ko = (uint16_t*)a.cache.k + to, *vo = (uint16_t*)a.cache.v + to;
      for (uint32_t c = c0; c < chunks; c += lanes) {
        const uint32_t n = chunk_left(a.cache.head_dim, c);
        if (c != c0) {
          kx = load_bf16x8(k + 8u * c, n);
          vx = load_bf16x8(v + 8u * c, n);
        }
        store_bf16x8(ko + 8u * c, kx, n);
        store_bf16x8(vo + 8u * c, vx, n);
      }
    } else if constexpr (F == kMxfp4) {
      // four lanes a block; a head_dim of whole blocks has whole chunks
      const uint64_t at = ((((uint64_t)page * a.cache.kv_heads + head) * a.cache.page.divisor) +
                           place) * (chunks / 4u);
      for (uint32_t c = c0; c < chunks; c += lanes) {
        if (c != c0) {
          kx = load_bf16x8(k + 8u * c, 8u);
          vx = load_bf16x8(v + 8u * c, 8u);
        }
        const uint32_t ks = mxfp4::scale_byte(mxfp4::quad_max(mxfp4::top8(kx)));
        const uint32_t vs = mxfp4::scale_byte(mxfp4::quad_max(mxfp4::top8(vx)));
        *reinterpret_cast<u32_any_t*>(a.cache.k + to + 4u * c) =
            mxfp4::encode8(kx, mxfp4::scale_float(ks));
        *reinterpret_cast<u32_any_t*>(a.cache.v + to + 4u * c) =
            mxfp4::encode8(vx, mxfp4::scale_float(vs));
        if (c % 4u == 0u) {
          a.cache.k_blocks()[at + c / 4u] = (uint8_t)ks;
          a.cache.v_blocks()[at + c / 4u] = (uint8_t)vs;
        }
      }
    } else {
      float km = amax8(kx, 0.0f), vm = amax8(vx, 0.0f);
      for (uint32_t c = c0 + lanes; c < chunks; c += lanes) {
        const uint32_t n = chunk_left(a.cache.head_dim, c);
        km = amax8(load_bf16x8(k + 8u * c, n), km);
        vm = amax8(load_bf16x8(v + 8u * c, n), vm);
      }
      for (uint32_t o = 1u; o < lanes; o <<= 1) {
        km = fmaxf(km, __shfl_xor(km, o, 64));
        vm = fmaxf(vm, __shfl_xor(vm, o, 64));
      }
      const RowScale ks(km), vs(vm);
      if (c0 == 0u) {
        const uint64_t at =
            ((uint64_t)page * a.cache.kv_heads + head) * a.cache.page.divisor + place;
        a.cache.k_scale[at] = ks.scale;
        a.cache.v_scale[at] = vs.scale;
      }
      for (uint32_t c = c0; c < chunks; c += lanes) {
        const uint32_t n = chunk_left(a.cache.head_dim, c);
        if (c != c0) {
          kx = load_bf16x8(k + 8u * c, n);
          vx = load_bf16x8(v + 8u * c, n);
        }
        store_codes8(a.cache.k + to + 8u * c, quantize8(kx, ks), n);
        store_codes8(a.cache.v + to + 8u * c, quantize8(vx, vs), n);
      }
    }
  }
}

// ---- reading back ---------------------------------------------------------------------------

constexpr uint32_t kReadTokens = 4;       // tokens per workgroup (8: one sequence's 2001 5.7 -> 6.7 us)
constexpr uint32_t kStagedStarts = 1024; // starts a workgroup searches in LDS

struct ReadArgs {
  View cache;
  const uint32_t *table, *starts;
  uint16_t *k, *v;
  FastDiv heads;
  uint64_t token_stride, head_stride;
  uint32_t seqs, table_cols, tokens, lanes_log2;
};

enum : uint32_t { kRowKept = 0u, kRowZero = 1u, kRowRead = 2u };

template <uint32_t F>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(ReadArgs a) {
  __shared__ uint32_t staged[kStagedStarts];
  __shared__ uint32_t kind[kReadTokens], page_of[kReadTokens], place_of[kReadTokens];
  const uint32_t first = (blockIdx.y * kMaxGrid + blockIdx.x) * kReadTokens;
  if (first >= a.tokens) return;  // the last row of a grid of two dimensions
  const uint32_t count = min(kReadTokens, a.tokens - first);
  const bool in_lds = a.seqs < kStagedStarts;
  if (in_lds) {
    for (uint32_t i = threadIdx.x; i <= a.seqs; i += kThreads) staged[i] = a.starts[i];
    __syncthreads();
  }
  if (threadIdx.x < count) {
    const uint32_t t = first + threadIdx.x;
    auto start = [&](uint32_t i) { return in_lds ? staged[i] : a.starts[i]; };
    // the last sequence that starts at or before t: lo - 1
    uint32_t lo = 0, hi = a.seqs + 1u;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2u;
      if (start(mid) <= t) lo = mid + 1u;
      else hi = mid;
    }
    uint32_t what = kRowKept, page = 0, place = 0;
    if (lo >= 1u && lo <= a.seqs) {
      const uint32_t at = t - start(lo - 1u), col = a.cache.page.div(at);
      what = kRowZero;
      if (col < a.table_cols) {
        page = a.table[(uint64_t)(lo - 1u) * a.table_cols + col];
        place = at - col * a.cache.page.divisor;
        if (page < a.cache.pages) what = kRowRead;
      }
    }
    kind[threadIdx.x] = what;
    page_of[threadIdx.x] = page;
    place_of[threadIdx.x] = place;
  }
  __syncthreads();
  const uint32_t lanes = 1u << a.lanes_log2, c0 = threadIdx.x & (lanes - 1u);
  const uint32_t chunks = (a.cache.head_dim + 7u) / 8u;
  const uint32_t rows = count * a.heads.divisor;
  for (uint32_t r = threadIdx.x >> a.lanes_log2; r < rows; r += (uint32_t)kThreads >> a.lanes_log2) {
    const uint32_t i = a.heads.div(r), head = r - i * a.heads.divisor;
    if (kind[i] == kRowKept) continue;
    const bool read = kind[i] == kRowRead;
    const uint64_t from = page_of[i] * a.cache.page_stride + place_of[i] * a.cache.token_stride +
                          head * a.cache.head_stride;
    const uint64_t to = (uint64_t)(first + i) * a.token_stride + head * a.head_stride;
    float ks = 0.0f, vs = 0.0f;
    if (F == kE4m3 && read) {
      const uint64_t at =
          ((uint64_t)page_of[i] * a.cache.kv_heads + head) * a.cache.page.divisor + place_of[i];
      ks = a.cache.k_scale[at];
      vs = a.cache.v_scale[at];
    }
    for (uint32_t c = c0; c < chunks; c += lanes) {
      const uint32_t n = chunk_left(a.cache.head_dim, c);
      u32x4_t kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
      if (read) {
        if constexpr (F == kMxfp4) {
          const uint64_t at = (((uint64_t)page_of[i] * a.cache.kv_heads + head) *
                                   a.cache.page.divisor + place_of[i]) * (chunks / 4u) + c / 4u;
          kx = mxfp4::decode8_bf16(*reinterpret_cast<const u32_any_t*>(a.cache.k + from + 4u * c),
                                   mxfp4::scale_float(a.cache.k_blocks()[at]));
          vx = mxfp4::decode8_bf16(*reinterpret_cast<const u32_any_t*>(a.cache.v + from + 4u * c),
                                   mxfp4::scale_float(a.cache.v_blocks()[at]));
        } else if constexpr (F == kE4m3) {
          kx = widen8(load_codes8(a.cache.k + from + 8u * c, n), ks);
          vx = widen8(load_codes8(a.cache.v + from + 8u * c, n), vs);
        } else {
          kx = load_bf16x8((const uint16_t*)a.cache.k + from + 8u * c, n);
          vx = load_bf16x8((const uint16_t*)a.cache.v + from + 8u * c, n);
        }
      }
      store_bf16x8(a.k + to + 8u * c, kx, n);
      store_bf16x8(a.v + to + 8u * c, vx, n);
    }
  }
}

// lanes per row: the least power of two that holds its chunks, one wave at most
uint32_t row_lanes_log2(uint32_t head_dim) {
  uint32_t log2 = 0;
  while (log2 < 6u && (8u << log2) < head_dim) ++log2;
  return log2;
}

#define FE2O3_KV_KERNELS(F, NAME) \
  fe2o3_host::KernelRegistrar({"fe2o3_kv_cache_write", "kv_write_kernel<" NAME ">", (const void*)kv_write_kernel<F>, kThreads, 0}), \
  fe2o3_host::KernelRegistrar({"fe2o3_kv_cache_read", "kv_read_kernel<" NAME ">", (const void*)kv_read_kernel<F>, kThreads, 0})
const fe2o3_host::KernelRegistrar kRegistered[] = {FE2O3_KV_KERNELS(kBf16, "bf16"),
                                                   FE2O3_KV_KERNELS(kE4m3, "e4m3"),
                                                   FE2O3_KV_KERNELS(kMxfp4, "mxfp4")};
#undef FE2O3_KV_KERNELS

}  // namespace

extern "C" {

int32_t fe2o3_kv_cache_write(const Fe2o3KvCacheV1* cache, const uint16_t* k, uint64_t k_len,
                             const uint16_t* v, uint64_t v_len, const uint32_t* slots,
                             uint64_t slots_len, uint32_t tokens, uint64_t token_stride,
                             uint64_t head_stride, void* stream) {
  FE2O3_ENTRY("fe2o3_kv_cache_write");
  WriteArgs a;
  int32_t rc = kv_cache::check(cache, &a.cache);
  if (rc != FE2O3_OK) return rc;
  const uint64_t rows = (uint64_t)tokens * cache->kv_heads;
  if (rows >= (UINT64_C(1) << 31)) return FE2O3_ERR_SHAPE;
  if (slots_len != tokens) return FE2O3_ERR_LENGTH;
  if (tokens == 0u) return FE2O3_OK;
  uint64_t extent;
  rc = kv_cache::rows_extent(tokens, cache->kv_heads, cache->head_dim, token_stride, head_stride,
                             &extent);
  if (rc != FE2O3_OK) return rc;
  if (k_len < extent || v_len < extent) return FE2O3_ERR_LENGTH;
  if (!k || !v || !slots) return FE2O3_ERR_NULL;
  if ((((uintptr_t)k | (uintptr_t)v) & 1u) != 0u || ((uintptr_t)slots & 3u) != 0u)
    return FE2O3_ERR_ALIGNMENT;
  a.k = k;
  a.v = v;
  a.slots = slots;
  a.heads = FastDiv::of(cache->kv_heads);
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.rows = (uint32_t)rows;
  a.lanes_log2 = row_lanes_log2(cache->head_dim);
  const uint64_t wgs = ((rows << a.lanes_log2) + kThreads - 1u) / kThreads;
  const uint32_t grid = (uint32_t)(wgs < kMaxGrid ? wgs : kMaxGrid);
  hipStream_t s = (hipStream_t)stream;
  if (cache->format == kE4m3) kv_write_kernel<kE4m3><<<grid, kThreads, 0, s>>>(a);
  else if (cache->format == kMxfp4) kv_write_kernel<kMxfp4><<<grid, kThreads, 0, s>>>(a);
  else kv_write_kernel<kBf16><<<grid, kThreads, 0, s>>>(a);
  return fe2o3_host::after_launch();
}

int32_t fe2o3_kv_cache_read(const Fe2o3KvCacheV1* cache, const uint32_t* block_table,
                            uint64_t table_len, const uint32_t* starts, uint64_t starts_len,
                            uint16_t* k, uint64_t k_len, uint16_t* v, uint64_t v_len,
                            uint32_t seqs, uint32_t table_cols, uint32_t tokens,
                            uint64_t token_stride, uint64_t head_stride, void* stream) {
  FE2O3_ENTRY("fe2o3_kv_cache_read");
  ReadArgs a;
  int32_t rc = kv_cache::check(cache, &a.cache);
  if (rc != FE2O3_OK) return rc;
  if ((uint64_t)tokens * cache->kv_heads >= (UINT64_C(1) << 31) || seqs >= (1u << 31))
    return FE2O3_ERR_SHAPE;
  if (table_len != (uint64_t)seqs * table_cols || starts_len != (uint64_t)seqs + 1u)
    return FE2O3_ERR_LENGTH;
  if (tokens == 0u || seqs == 0u) return FE2O3_OK;
  uint64_t extent;
  rc = kv_cache::rows_extent(tokens, cache->kv_heads, cache->head_dim, token_stride, head_stride,
                             &extent);
  if (rc != FE2O3_OK) return rc;
  if (k_len < extent || v_len < extent) return FE2O3_ERR_LENGTH;
  if (!k || !v || !starts || (table_len != 0u && !block_table)) return FE2O3_ERR_NULL;
  if ((((uintptr_t)k | (uintptr_t)v) & 1u) != 0u ||
      (((uintptr_t)starts | (uintptr_t)block_table) & 3u) != 0u)
    return FE2O3_ERR_ALIGNMENT;
  a.table = block_table;
  a.starts = starts;
  a.k = k;
  a.v = v;
  a.heads = FastDiv::of(cache->kv_heads);
  a.token_stride = token_stride;
  a.head_stride = head_stride;
  a.seqs = seqs;
  a.table_cols = table_cols;
  a.tokens = tokens;
  a.lanes_log2 = row_lanes_log2(cache->head_dim);
  const uint32_t wgs = (tokens - 1u) / kReadTokens + 1u;
  const dim3 grid(wgs < kMaxGrid ? wgs : kMaxGrid, (wgs - 1u) / kMaxGrid + 1u);
  hipStream_t s = (hipStream_t)stream;
  if (cache->format == kE4m3) kv_read_kernel<kE4m3><<<grid, kThreads, 0, s>>>(a);
  else if (cache->format == kMxfp4) kv_read_kernel<kMxfp4><<<grid, kThreads, 0, s>>>(a);
  else kv_read_kernel<kBf16><<<grid, kThreads, 0, s>>>(a);
  return fe2o3_host::after_launch();
}

}  // extern "C"
