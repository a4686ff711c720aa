// rotary.hip -- rotary positions of Q and K, and their gradient, for gfx950.
//
//   (a, b) -> m (a cos t - b sin t, b cos t + a sin t),  t = position * freq_i
//
// for the pairs i of a head's first rotary_dim elements: (i, i + rotary_dim / 2), or
// (2 i, 2 i + 1) interleaved; the rest of the head is copied.  The inverse turns by -t:
// with the same m it is the transposed map, which takes a gradient back.
//
// An angle reaches 10^6 radians, where 32 bits are off by 0.06, so it is taken in turns:
// position * (freq / 2 pi) in 64 bits, less its nearest whole number, is off by 2^-52 of
// the turns (2^-34 of one at 10^6 radians).  Sine and cosine of what is left, times the
// scale, are f32: a few units of 2^-24 off, far below a bf16 output's rounding.  f32 outputs
// are off by 6e-8 (rms, of 64 bits), where the rounding alone would be 2.5e-8, and by 1.8e-7
// of their pair's magnitudes at the most (three ranges of positions up to 10^6).
//
// Bound by memory: x is read once and written once.  A workgroup takes a few tokens, each
// pair's sine and cosine is computed once for all heads and kept in LDS, and a lane turns
// eight pairs, 16 bytes of bf16 on each side.  Measured: 16384 tokens of 32 + 8 heads of
// 128, bf16, into other rows 59 us = 5.7 TB/s; 32 tokens 2.9, the chain of position,
// frequency, sine, table and rows.  18 pairs of such a head, which end in a part of eight, 94.
#include "common.hpp"
#include "internal.hpp"
#include "kv_cache.hpp"

#include <type_traits>

namespace {

using namespace fe2o3;
using kv_cache::FastDiv;

constexpr int kThreads = 256;
constexpr uint32_t kMaxPairs = 2048;
constexpr uint32_t kTable = 2048;  // sines and cosines in LDS, 8 bytes each
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any_t __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_any_t __attribute__((aligned(2)));

// Rows of one of the two arrays, strides in elements.
struct Rows {
  const void* x;
  void* out;
  uint64_t token_stride, head_stride, out_token_stride, out_head_stride;
  uint32_t heads;
};

struct Args {
  Rows rows[2];
  const uint32_t* positions;
  const double* freq;
  FastDiv heads;   // of both arrays
  FastDiv chunks;  // of a head: eight pairs each, then 16 copied elements each
  FastDiv pairs;
  FastDiv parts;   // workgroups that share a token's tasks
  uint32_t tokens, per_wg, part_tasks, head_dim, turned;  // turned: chunks of pairs
  float cos_scale, sin_scale;  // the inverse has another sign of the sine
};

// N elements (a power of two to 8) at any alignment of theirs, as 32-bit words; a single bf16
// in the low half of one.
template <class T, uint32_t N>
struct Piece {
  static constexpr uint32_t kBytes = N * sizeof(T), kWords = (kBytes + 3u) / 4u;
  uint32_t w[kWords];
  FE2O3_DEVICE void load(const T* p) {
    if constexpr (kBytes == 2u) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else if constexpr (kBytes == 4u) {
      w[0] = *reinterpret_cast<const u32_any_t*>(p);
    } else if constexpr (kBytes == 8u) {
      const u32x2_t x = *reinterpret_cast<const u32x2_any_t*>(p);
      w[0] = x[0];
      w[1] = x[1];
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kWords; i += 4u) {
        const u32x4_t x = reinterpret_cast<const u32x4_any_t*>(p)[i / 4u];
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) w[i + e] = x[e];
      }
    }
  }
  FE2O3_DEVICE void store(T* p) const {
    if constexpr (kBytes == 2u) {
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    } else if constexpr (kBytes == 4u) {
      *reinterpret_cast<u32_any_t*>(p) = w[0];
    } else if constexpr (kBytes == 8u) {
      *reinterpret_cast<u32x2_any_t*>(p) = u32x2_t{w[0], w[1]};
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kWords; i += 4u)
        reinterpret_cast<u32x4_any_t*>(p)[i / 4u] = u32x4_t{w[i], w[i + 1], w[i + 2], w[i + 3]};
    }
  }
};
template <uint32_t N, class T>
FE2O3_DEVICE void load(const T* p, float* v) {
  Piece<T, N> x;
  x.load(p);
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    if constexpr (sizeof(T) == 4u) v[i] = __uint_as_float(x.w[i]);
    else v[i] = __uint_as_float(i & 1u ? x.w[i / 2u] & 0xffff0000u : x.w[i / 2u] << 16);
  }
}
template <uint32_t N, class T>
FE2O3_DEVICE void store(T* p, const float* v) {
  Piece<T, N> x;
#pragma unroll
  for (uint32_t i = 0; i < Piece<T, N>::kWords; ++i) {
    if constexpr (sizeof(T) == 4u) x.w[i] = __float_as_uint(v[i]);
    else if constexpr (N == 1u) x.w[i] = bf16_bits_from_f32(v[0]);
    else x.w[i] = pack_bf16x2(v[2u * i], v[2u * i + 1u]);
  }
  x.store(p);
}
template <uint32_t N, class T>
FE2O3_DEVICE void copy(const T* p, T* out) {  // the bits, those of a NaN too
  Piece<T, N> x;
  x.load(p);
  x.store(out);
}

// What a task calls for n of eight pairs, or elements: at<N>(place, first) for a piece of N
// from the `first` one on, which are places place .. of eight; a part of eight goes in
// pieces of four, two and one, in fixed registers.
template <class At>
FE2O3_DEVICE void pieces(uint32_t n, At at) {
  using std::integral_constant;
  if (n >= 8u) {
    at(integral_constant<uint32_t, 8>{}, integral_constant<uint32_t, 0>{}, 0u);
    return;
  }
  if ((n & 4u) != 0u) at(integral_constant<uint32_t, 4>{}, integral_constant<uint32_t, 0>{}, 0u);
  if ((n & 2u) != 0u) at(integral_constant<uint32_t, 2>{}, integral_constant<uint32_t, 4>{}, n & 4u);
  if ((n & 1u) != 0u) at(integral_constant<uint32_t, 1>{}, integral_constant<uint32_t, 6>{}, n & 6u);
}

template <class T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) float2 table[kTable];
  __shared__ uint32_t skipped[kThreads];
  const uint32_t id = blockIdx.y * kv_cache::kGridWidth + blockIdx.x;
  const uint32_t group = a.parts.div(id), part = id - group * a.parts.divisor;
  const uint32_t first = group * a.per_wg;
  if (first >= a.tokens) return;  // the last row of a grid of two dimensions
  const uint32_t count = min(a.per_wg, a.tokens - first);
  const uint32_t pairs = a.pairs.divisor;
  for (uint32_t i = threadIdx.x; i < count * pairs; i += kThreads) {
    const uint32_t t = a.pairs.div(i), pair = i - t * pairs;
    const uint32_t position = a.positions[first + t];
    const double turns = (double)position * (a.freq[pair] * 0.15915494309189533577);
    const float rest = (float)(turns - __builtin_rint(turns));
    float s, c;
    sincospif(2.0f * rest, &s, &c);
    table[i] = float2{c * a.cos_scale, s * a.sin_scale};
    if (pair == 0u) skipped[t] = position == FE2O3_KV_NO_SLOT;
  }
  __syncthreads();
  const uint32_t heads = a.heads.divisor, chunks = a.chunks.divisor;
  const uint32_t end = min(count * heads * chunks, (part + 1u) * a.part_tasks);
  for (uint32_t i = part * a.part_tasks + threadIdx.x; i < end; i += kThreads) {
    const uint32_t row = a.chunks.div(i), chunk = i - row * chunks;
    const uint32_t t = a.heads.div(row), h = row - t * heads;
    if (skipped[t]) continue;
    const bool second = h >= a.rows[0].heads;
    const Rows& r = a.rows[second ? 1 : 0];
    const uint32_t head = second ? h - a.rows[0].heads : h;
    const T* x = (const T*)r.x + (first + t) * r.token_stride + head * r.head_stride;
    T* out = (T*)r.out + (first + t) * r.out_token_stride + head * r.out_head_stride;
    if (chunk < a.turned) {
      const uint32_t p0 = 8u * chunk;
      auto turn = [&](auto number) {
        const uint32_t n = number;
        // the pairs' elements: of the halves eight each, or interleaved
        float x_in[16] = {}, x_out[16];
        pieces(n, [&](auto size, auto place, uint32_t from) {
          constexpr uint32_t N = decltype(size)::value, P = decltype(place)::value;
          if constexpr (INTERLEAVED && N == 8u) {
            load<8>(x + 2u * p0, x_in);
            load<8>(x + 2u * p0 + 8u, x_in + 8);
          } else if constexpr (INTERLEAVED) {
            load<2u * N>(x + 2u * (p0 + from), x_in + 2u * P);
          } else {
            load<N>(x + p0 + from, x_in + P);
            load<N>(x + pairs + p0 + from, x_in + 8u + P);
          }
          // keeps the pieces apart: merged, their registers would become an array in memory
          asm volatile("; %0" : : "n"(N));
        });
        // the pair at place 4, and at 6
        const uint32_t four = n >= 8u ? 4u : n & 4u, six = n >= 8u ? 6u : n & 6u;
        const float2* turns = table + t * pairs + p0;
#pragma unroll
        for (uint32_t j = 0; j < 8u; ++j) {
          const uint32_t pair = min(j < 4u ? j : j < 6u ? four + j - 4u : six + j - 6u, n - 1u);
          const float2 cs = turns[pair];
          const uint32_t i0 = INTERLEAVED ? 2u * j : j, i1 = INTERLEAVED ? 2u * j + 1u : 8u + j;
          const float p = x_in[i0], q = x_in[i1];
          x_out[i0] = p * cs.x - q * cs.y;
          x_out[i1] = q * cs.x + p * cs.y;
        }
        pieces(n, [&](auto size, auto place, uint32_t from) {
          constexpr uint32_t N = decltype(size)::value, P = decltype(place)::value;
          if constexpr (INTERLEAVED && N == 8u) {
            store<8>(out + 2u * p0, x_out);
            store<8>(out + 2u * p0 + 8u, x_out + 8);
          } else if constexpr (INTERLEAVED) {
            store<2u * N>(out + 2u * (p0 + from), x_out + 2u * P);
          } else {
            store<N>(out + p0 + from, x_out + P);
            store<N>(out + pairs + p0 + from, x_out + 8u + P);
          }
        });
      };
      if (pairs - p0 >= 8u) turn(std::integral_constant<uint32_t, 8>{});
      else turn(pairs - p0);
    } else if (x != out) {
      const uint32_t at = 2u * pairs + 16u * (chunk - a.turned), n = min(a.head_dim - at, 16u);
#pragma unroll
      for (uint32_t h = 0; h < 16u; h += 8u)
        pieces(n > h ? min(n - h, 8u) : 0u, [&](auto size, auto, uint32_t from) {
          constexpr uint32_t N = decltype(size)::value;
          copy<N>(x + at + h + from, out + at + h + from);
        });
    }
  }
}

const fe2o3_host::KernelRegistrar kRegistered[] = {
    fe2o3_host::KernelRegistrar({"fe2o3_rotary", "rotary_kernel<bf16>", (const void*)rotary_kernel<uint16_t, false>, kThreads, 0}),
    fe2o3_host::KernelRegistrar({"fe2o3_rotary", "rotary_kernel<bf16,interleaved>", (const void*)rotary_kernel<uint16_t, true>, kThreads, 0}),
    fe2o3_host::KernelRegistrar({"fe2o3_rotary", "rotary_kernel<f32>", (const void*)rotary_kernel<float, false>, kThreads, 0}),
    fe2o3_host::KernelRegistrar({"fe2o3_rotary", "rotary_kernel<f32,interleaved>", (const void*)rotary_kernel<float, true>, kThreads, 0})};

// The caller's record, its strides and lengths, for `tokens` rows.
int32_t check_rows(const Fe2o3RotaryRowsV1* r, uint32_t tokens, uint32_t head_dim, Rows* out) {
  uint64_t extent, out_extent, bytes;
  int32_t rc = kv_cache::rows_extent(tokens, r->heads, head_dim, r->token_stride, r->head_stride,
                                     &extent);
  if (rc == FE2O3_OK)
    rc = kv_cache::rows_extent(tokens, r->heads, head_dim, r->out_token_stride, r->out_head_stride,
                               &out_extent);
  if (rc != FE2O3_OK) return rc;
  if (!kv_cache::mul_ok(extent, 4u, &bytes) || !kv_cache::mul_ok(out_extent, 4u, &bytes))
    return FE2O3_ERR_OVERFLOW;
  if (r->x_len < extent || r->out_len < out_extent) return FE2O3_ERR_LENGTH;
  *out = Rows{r->x, r->out, r->token_stride, r->head_stride, r->out_token_stride,
              r->out_head_stride, r->heads};
  return FE2O3_OK;
}

}  // namespace

extern "C" int32_t fe2o3_rotary(const Fe2o3RotaryRowsV1* q, const Fe2o3RotaryRowsV1* k,
                                const uint32_t* positions, uint64_t positions_len,
                                const double* freq, uint64_t freq_len, uint32_t dtype,
                                uint32_t tokens, uint32_t head_dim, uint32_t rotary_dim,
                                uint32_t flags, float scale, void* stream) {
  FE2O3_ENTRY("fe2o3_rotary");
  if (q == nullptr) return FE2O3_ERR_NULL;
  const uint64_t heads = (uint64_t)q->heads + (k ? k->heads : 0u);
  const uint32_t pairs = rotary_dim / 2u;
  if (dtype > 1u || flags > 3u || rotary_dim == 0u || rotary_dim % 2u != 0u ||
      rotary_dim > head_dim || pairs > kMaxPairs || !__builtin_isfinite(scale))
    return FE2O3_ERR_SHAPE;
  if (q->heads == 0u || (k && k->heads == 0u)) return FE2O3_ERR_SHAPE;
  const uint32_t turned = (pairs + 7u) / 8u;
  const uint64_t chunks = FE2O3_ROTARY_PIECES(1u, head_dim, rotary_dim);
  const uint64_t tasks = heads * chunks;  // of one token: below 2^33 times 2^29
  if (tasks >= (UINT64_C(1) << 22) || tokens >= (1u << 31)) return FE2O3_ERR_SHAPE;
  if (positions_len != tokens || freq_len != pairs) return FE2O3_ERR_LENGTH;
  if (tokens == 0u) return FE2O3_OK;
  Args a{};
  int32_t rc = check_rows(q, tokens, head_dim, &a.rows[0]);
  if (rc == FE2O3_OK && k) rc = check_rows(k, tokens, head_dim, &a.rows[1]);
  if (rc != FE2O3_OK) return rc;
  if (!q->x || !q->out || (k && (!k->x || !k->out)) || !positions || !freq) return FE2O3_ERR_NULL;
  uintptr_t any = (uintptr_t)q->x | (uintptr_t)q->out;
  if (k) any |= (uintptr_t)k->x | (uintptr_t)k->out;
  if ((any & (dtype == 0u ? 3u : 1u)) != 0u || ((uintptr_t)positions & 3u) != 0u ||
      ((uintptr_t)freq & 7u) != 0u)
    return FE2O3_ERR_ALIGNMENT;
  a.positions = positions;
  a.freq = freq;
  a.heads = FastDiv::of((uint32_t)heads);
  a.chunks = FastDiv::of((uint32_t)chunks);
  a.pairs = FastDiv::of(pairs);
  a.tokens = tokens;
  a.head_dim = head_dim;
  a.turned = turned;
  a.cos_scale = scale;
  a.sin_scale = (flags & FE2O3_ROTARY_INVERSE) != 0u ? -scale : scale;
  // Tokens of a workgroup: two tasks for every thread, as far as a pair each and the device
  // filled twice allow (us, a token | this | as many as have a pair for every thread):
  //   2048 tokens of 32 + 8 heads, d 128 7.8 | 7.8 | 8.7   16384 of them 59.0 | 59.3 | 62.0
  //   16384 of 8 + 1, d 64, 32 turned 16.4 | 9.4 | 9.7     16384 of 16 + 2, d 64 17.5 | 13.3 | 13.4
  tile_plan::Topology topo;
  rc = fe2o3_host::device_topology(&topo);
  if (rc != FE2O3_OK) return rc;
  const uint32_t most[] = {kThreads / pairs, 2u * kThreads / (uint32_t)tasks,
                           tokens / (2u * topo.cus)};
  uint32_t per_wg = most[0];
  for (const uint32_t n : most) per_wg = n < per_wg ? n : per_wg;
  a.per_wg = per_wg = per_wg > 1u ? per_wg : 1u;
  // few tokens: their heads over as many workgroups as have tasks for all threads (us, one a
  // token and this: 1 token of 160 heads, d 128 17.1, 3.5; 32 of 40 4.1, 2.9; 111 of 256
  // 13.3, 5.0)
  uint32_t parts = 2u * topo.cus / tokens;
  const uint32_t most_parts = ((uint32_t)tasks - 1u) / kThreads + 1u;
  parts = parts < most_parts ? parts : most_parts;
  parts = parts > 1u ? parts : 1u;
  a.parts = FastDiv::of(parts);
  a.part_tasks = parts > 1u ? ((uint32_t)tasks - 1u) / parts + 1u : ~0u;
  const kv_cache::Grid g = kv_cache::Grid::of(((tokens - 1u) / per_wg + 1u) * parts);
  const dim3 grid(g.x, g.y);
  hipStream_t s = (hipStream_t)stream;
  if ((flags & FE2O3_ROTARY_INTERLEAVED) != 0u) {
    if (dtype == 0u) rotary_kernel<float, true><<<grid, kThreads, 0, s>>>(a);
    else rotary_kernel<uint16_t, true><<<grid, kThreads, 0, s>>>(a);
  } else {
    if (dtype == 0u) rotary_kernel<float, false><<<grid, kThreads, 0, s>>>(a);
    else rotary_kernel<uint16_t, false><<<grid, kThreads, 0, s>>>(a);
  }
  return fe2o3_host::after_launch();
}
