// mxfp4.hip -- matrices into the packed microscaled 4-bit form (mxfp4.hpp) and back.
//
// Both are one pass, bound by memory: a piece is a row's panel of 256 columns, 32 lanes
// of eight columns, four lanes to a block of 32.  A workgroup takes 8 or 16 rows of
// one panel, so that the scales of neighbouring rows, which lie beside each other, come
// from one workgroup; a wave's accesses of x are runs of 512 bytes (bf16).
//
// Measured: 14336 x 4096 of f32 into 4 bits 46 us = 5.8 TB/s, back 38 us = 7.0 (part of the
// codes cached); 16384 x 4096 of bf16 28 us = 6.1 and 25 us = 6.9; 33 x 4096 2.1 each, as
// any launch.
#include "common.hpp"
#include "internal.hpp"
#include "kv_cache.hpp"
#include "mxfp4.hpp"

#include <type_traits>

namespace {

using namespace fe2o3;
using kv_cache::FastDiv;

constexpr int kThreads = 256;
constexpr uint32_t kPass = kThreads / 32;  // rows of one pass
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));

struct Args {
  const void* x;  // quantize
  void* out;      // dequantize
  uint8_t *q, *scales;
  uint64_t stride;  // elements from a row of x (or out) to the next
  uint64_t scale_panel;  // bytes of a panel of scales
  FastDiv panels;
  uint32_t rows, cols;
};

// Eight elements of type T from p, the first n of them in memory (the others +0).
template <class T>
struct Eight;
template <>
struct Eight<uint16_t> {
  u32x4_t v;
  FE2O3_DEVICE void load(const uint16_t* p, uint32_t n) {
    if (n >= 8u) {
      v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any_t*>(p));
      return;
    }
    v = u32x4_t{0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 7u; ++i)
      if (i < n) v[i / 2u] |= (uint32_t)p[i] << (16u * (i & 1u));
  }
};
template <>
struct Eight<float> {
  float v[8];
  FE2O3_DEVICE void load(const float* p, uint32_t n) {
    if (n >= 8u) {
      const f32x4_t a = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any_t*>(p));
      const f32x4_t b = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any_t*>(p + 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
      return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) v[i] = i < n ? p[i] : 0.0f;
  }
};

// A workgroup's panel, first row, and the lane's first column and columns left.
struct Place {
  uint32_t panel, row, lane, col, left;
  FE2O3_DEVICE Place(const Args& a, uint32_t rows_per_wg) {
    const uint32_t id = blockIdx.y * kv_cache::kGridWidth + blockIdx.x;
    const uint32_t group = a.panels.div(id);
    panel = id - group * a.panels.divisor;
    lane = threadIdx.x & 31u;
    row = group * rows_per_wg + (threadIdx.x >> 5);
    col = panel * mxfp4::kPanel + 8u * lane;
    left = col < a.cols ? a.cols - col : 0u;
  }
};

// Rows of a workgroup: 32 bytes of x a thread in flight.  Of bf16 half or twice that takes
// longer, of f32 twice (16384 x 4096 bf16: 30.8 | 28.1 | 28.4 us; 14336 x 4096 f32: 46.0 |
// 49.7); only of few rows less (33 x 4096 bf16: 2.1 | 2.2).
template <class T>
constexpr uint32_t quantize_rows() {
  return kPass * 4u / sizeof(T);
}

template <class T>
__global__ void __launch_bounds__(kThreads) mxfp4_quantize_kernel(Args a) {
  constexpr uint32_t kRows = quantize_rows<T>(), kEach = kRows / kPass;
  const Place at(a, kRows);
  Eight<T> x[kEach];
#pragma unroll
  for (uint32_t u = 0; u < kEach; ++u) {
    const uint32_t row = at.row + u * kPass;
    x[u].load((const T*)a.x + (row < a.rows ? row : 0u) * a.stride + at.col,
              row < a.rows ? at.left : 0u);
  }
#pragma unroll
  for (uint32_t u = 0; u < kEach; ++u) {
    const uint32_t row = at.row + u * kPass;
    const uint32_t byte = mxfp4::scale_byte(mxfp4::quad_max(mxfp4::top8(x[u].v)));
    const uint32_t q = mxfp4::encode8(x[u].v, mxfp4::scale_float(byte));
    if (row >= a.rows) return;
    *reinterpret_cast<uint32_t*>(a.q + ((uint64_t)row * a.panels.divisor + at.panel) *
                                           mxfp4::kRowBytes + 4u * at.lane) = q;
    if (at.lane % 4u == 0u)
      a.scales[at.panel * a.scale_panel + (uint64_t)row * 8u + at.lane / 4u] = (uint8_t)byte;
  }
}

// A store covers whole lines: 16 bytes a lane of neighbouring columns, eight of bf16, four of
// f32 in either half of the panel (eight of f32 a lane, two stores 32 bytes apart: 14336 x
// 4096 88 us).  8 rows a workgroup (16, 32 rows: 38.1, 38.2, 40.7).
template <class T>
__global__ void __launch_bounds__(kThreads) mxfp4_dequantize_kernel(Args a) {
  constexpr uint32_t kParts = sizeof(T) / 2u, kEach = 8u / kParts;  // stores, columns of one
  using Codes = std::conditional_t<kParts == 1u, uint32_t, uint16_t>;
  const Place at(a, kPass);
  if (at.row >= a.rows) return;
  const uint8_t* codes =
      a.q + ((uint64_t)at.row * a.panels.divisor + at.panel) * mxfp4::kRowBytes;
  const uint8_t* scales = a.scales + at.panel * a.scale_panel + (uint64_t)at.row * 8u;
  uint32_t q[kParts], byte[kParts];
#pragma unroll
  for (uint32_t h = 0; h < kParts; ++h) {
    const uint32_t first = 128u * h + kEach * at.lane;
    q[h] = *reinterpret_cast<const Codes*>(codes + first / 2u);
    byte[h] = scales[first / mxfp4::kBlock];
  }
#pragma unroll
  for (uint32_t h = 0; h < kParts; ++h) {
    const uint32_t col = at.panel * mxfp4::kPanel + 128u * h + kEach * at.lane;
    const uint32_t n = col < a.cols ? min(a.cols - col, kEach) : 0u;
    T* out = (T*)a.out + at.row * a.stride + col;
    const float scale = mxfp4::scale_float(byte[h]);
    if constexpr (kParts == 1u) {
      const u32x4_t v = mxfp4::decode8_bf16(q[h], scale);
      if (n == kEach) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any_t*>(out));
      else
#pragma unroll
        for (uint32_t i = 0; i < kEach - 1u; ++i)
          if (i < n) out[i] = (T)(v[i / 2u] >> (16u * (i & 1u)));
    } else {
      float v[4];
      mxfp4::decode4_f32(q[h], scale, v);
      if (n == kEach)
        __builtin_nontemporal_store(f32x4_t{v[0], v[1], v[2], v[3]},
                                    reinterpret_cast<f32x4_any_t*>(out));
      else
#pragma unroll
        for (uint32_t i = 0; i < kEach - 1u; ++i)
          if (i < n) out[i] = v[i];
    }
  }
}

template <class T>
void launch(bool quantize, const Args& a, hipStream_t s) {
  const uint32_t rows = quantize ? quantize_rows<T>() : kPass;
  const kv_cache::Grid g =
      kv_cache::Grid::of((uint32_t)(((uint64_t)a.rows + rows - 1u) / rows) * a.panels.divisor);
  const dim3 grid(g.x, g.y);
  if (quantize) mxfp4_quantize_kernel<T><<<grid, kThreads, 0, s>>>(a);
  else mxfp4_dequantize_kernel<T><<<grid, kThreads, 0, s>>>(a);
}

int32_t run(bool quantize, const void* x, void* out, uint64_t x_len, uint32_t dtype, uint8_t* q,
            uint64_t q_len, uint8_t* scales, uint64_t scales_len, uint32_t rows, uint32_t cols,
            uint64_t stride, hipStream_t s) {
  if (dtype > 1u) return FE2O3_ERR_SHAPE;
  const mxfp4::Packed p = mxfp4::Packed::of(rows, cols);
  const uint64_t groups = ((uint64_t)rows + kPass - 1u) / kPass * p.panels;
  if (p.panels > mxfp4::kMaxPanels || groups >= (UINT64_C(1) << 31)) return FE2O3_ERR_SHAPE;
  if (rows > 1u && stride < cols) return FE2O3_ERR_STRIDE;
  uint64_t extent = cols, bytes;
  if (rows == 0u || cols == 0u) extent = 0;
  else if (!kv_cache::reach(rows, stride, &extent) || !kv_cache::mul_ok(extent, 4u, &bytes))
    return FE2O3_ERR_OVERFLOW;
  if (x_len < extent || q_len != p.codes || scales_len != p.scales) return FE2O3_ERR_LENGTH;
  if (extent == 0u) return FE2O3_OK;
  const void* dense = quantize ? x : out;
  if (!dense || !q || !scales) return FE2O3_ERR_NULL;
  if (((uintptr_t)dense & (dtype == 0u ? 3u : 1u)) != 0u ||
      (((uintptr_t)q | (uintptr_t)scales) & 15u) != 0u)
    return FE2O3_ERR_ALIGNMENT;
  Args a;
  a.x = x;
  a.out = out;
  a.q = q;
  a.scales = scales;
  a.stride = stride;
  a.scale_panel = p.scale_rows * (mxfp4::kPanel / mxfp4::kBlock);
  a.panels = FastDiv::of(p.panels);
  a.rows = rows;
  a.cols = cols;
  if (dtype == 0u) launch<float>(quantize, a, s);
  else launch<uint16_t>(quantize, a, s);
  return fe2o3_host::after_launch();
}

#define FE2O3_MX(ENTRY, K) \
  fe2o3_host::KernelRegistrar({ENTRY, #K "<f32>", (const void*)K<float>, kThreads, 0}), \
  fe2o3_host::KernelRegistrar({ENTRY, #K "<bf16>", (const void*)K<uint16_t>, kThreads, 0})
const fe2o3_host::KernelRegistrar kRegistered[] = {
    FE2O3_MX("fe2o3_quantize_mxfp4", mxfp4_quantize_kernel),
    FE2O3_MX("fe2o3_dequantize_mxfp4", mxfp4_dequantize_kernel)};
#undef FE2O3_MX

}  // namespace

extern "C" {

int32_t fe2o3_quantize_mxfp4(const void* x, uint64_t x_len, uint32_t dtype, uint8_t* q,
                             uint64_t q_len, uint8_t* scales, uint64_t scales_len, uint32_t rows,
                             uint32_t cols, uint64_t row_stride, void* stream) {
  FE2O3_ENTRY("fe2o3_quantize_mxfp4");
  return run(true, x, nullptr, x_len, dtype, q, q_len, scales, scales_len, rows, cols, row_stride,
             (hipStream_t)stream);
}

int32_t fe2o3_dequantize_mxfp4(const uint8_t* q, uint64_t q_len, const uint8_t* scales,
                               uint64_t scales_len, void* x, uint64_t x_len, uint32_t dtype,
                               uint32_t rows, uint32_t cols, uint64_t row_stride, void* stream) {
  FE2O3_ENTRY("fe2o3_dequantize_mxfp4");
  return run(false, nullptr, x, x_len, dtype, const_cast<uint8_t*>(q), q_len,
             const_cast<uint8_t*>(scales), scales_len, rows, cols, row_stride,
             (hipStream_t)stream);
}

}  // extern "C"
