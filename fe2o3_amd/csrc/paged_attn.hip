// paged_attn.hip -- attention of one new token per sequence over a paged
// key-value cache, for gfx950.
//
//   s_j = scale q.k_j,  o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
//
// over a sequence's keys, for the `group` query heads that share a KV head at
// once: K and V are read once for all of them.  With group <= 16 that is 2
// group flops a byte of bf16 cache, so the bound is memory and the MFMAs'
// unused rows cost nothing.
//
// A wave works on tiles of 32 keys of its own, with no barrier among waves:
//   * K and V rows come to registers with 16-byte nontemporal loads, adjacent
//     lanes on adjacent pieces of a row, one tile ahead of their use.  Lane l
//     looks up the page of key l % 32; its offset reaches the lanes that load the
//     row by a lane permutation, so pages of any size and place cost the same.
//   * They pass through LDS of the wave's own, chunks XOR-permuted per row, into
//     the MFMAs' layouts; e4m3 codes are widened to bf16, exactly, on the way out.
//   * S^T = K Q^T with v_mfma_f32_16x16x32_bf16: row m of key block b is key
//     8 (m / 4) + 4 b + m % 4, so that lane l holds query row l % 16 and the
//     eight keys 8 (l / 16) .. + 7, and the probabilities, in two bf16 parts, are the
//     second operand of O^T += V^T P^T where they stand; V^T comes by transposing LDS
//     reads.  The softmax is the prompt kernel's: exponentials against a
//     running reference that is raised only when a tile exceeds it by 2^8.
//   * An e4m3 cache's K scales multiply the scores, its V scales the
//     probabilities before these are split for the MFMA.
// With a multiple of four KV heads (and group <= 16) a workgroup's four waves
// have a head each in large calls: they read neighbouring rows, and nothing is added
// in LDS.
// Otherwise they take every fourth tile of one head and add their sums; of a group
// above 32 four teams of three or four waves, a wave for every 16 query rows, do so.
//
// The tiles of all sequences and heads, one behind another, are dealt in equal
// runs to as many workgroups as the device holds, so that one long sequence
// fills it as well as many, and mixed lengths leave no tail (Plan).  Each
// workgroup finds its run from the lengths.  A head that takes more than one run
// has its sums in the workspace; paged_join_kernel adds them in the order of the
// keys.  Short calls run one workgroup a head instead (launch).
//
// Measured, of a repeated call, bytes of K and V read once (a kernel that only
// reads them: 6.4-6.9 TB/s): 8 sequences of 4096 keys, 32 heads, bf16: 80-82 us =
// 6.6 TB/s, and 4.6 of the join; 130001 keys of one sequence, 8 heads: 82 us and
// 6; 64 sequences of 2 to 8190 keys, 8 heads, e4m3: 88 us = 6.3 TB/s, 4.8; 500
// keys of one: 7.7 us.  48 query heads on one KV head, 48 sequences of 100 to 6000
// keys: 21 us and 4.0, half of it starting, adding and ending.  4-bit rows (DecodeBlocks):
// 64 sequences of 2 to 8190 keys, 32 heads on 8: 54 us = 5.2 TB/s, 5.0 (65 and 6 over caches
// that the last call did not read); 500 keys of one: 6.7 us; 40 windows of 1024, 64 wide, 24
// heads on 8: 10.6 us.
#include "common.hpp"
#include "internal.hpp"
#include "kv_cache.hpp"
#include "mxfp4.hpp"

#include <type_traits>

namespace {

using namespace fe2o3;
using kv_cache::View;

// a cache's format, FE2O3_KV_*
constexpr uint32_t kBf16 = FE2O3_KV_BF16, kE4m3 = FE2O3_KV_E4M3, kMxfp4 = FE2O3_KV_MXFP4;
constexpr uint32_t kWaves = 4, kThreads = kWaves * 64;  // of a workgroup, if not said otherwise
constexpr uint32_t kKeys = 32;              // keys per tile
constexpr uint32_t kBlockKeys = 64;         // of 4-bit codes, where a wave has one row tile
constexpr float kLazyBound = 256.0f;        // p may reach 2^8 before a rescale
constexpr uint32_t kMaxWorkgroups = FE2O3_PAGED_ATTENTION_MAX_WORKGROUPS;
constexpr uint32_t kWholeTiles = 40;        // of a call without a join
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));
constexpr uint32_t kBlockRows = 64;         // query heads that one pass over K and V serves

struct Args {
  View cache;
  const uint16_t* q;
  const uint32_t *table, *lengths;
  uint16_t* o;
  float* lse;
  float* stats;  // workspace: reference and sum, [workgroup][2][rows][2],
  float* sums;   // and weighted V, [workgroup][2][rows][head_dim]
  uint64_t q_stride;
  uint32_t seqs, q_heads, group, blocks_per_head, rows;  // rows: per block, at most kBlockRows
  uint32_t table_cols, max_length, window, workgroups, xcds;
  float scale_log2;
};

// keys [first, end) of a sequence and its tiles, one at least
struct Span {
  uint32_t first, end, tile0, tiles;
};
template <uint32_t KEYS>
FE2O3_DEVICE Span span_of(const Args& a, uint32_t length) {
  Span s;
  s.end = min(length, a.max_length);
  s.first = a.window != 0u && s.end > a.window ? s.end - a.window : 0u;
  s.tile0 = s.first / KEYS;
  s.tiles = max((s.end + KEYS - 1u) / KEYS - s.tile0, 1u);
  return s;
}

// The same of a sequence that the whole wave works on, in scalar registers, so
// that what follows from it branches as a whole.
FE2O3_DEVICE uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
template <uint32_t KEYS>
FE2O3_DEVICE Span uniform_span_of(const Args& a, uint32_t seq) {
  const Span s = span_of<KEYS>(a, a.lengths[seq]);
  return Span{uniform(s.first), uniform(s.end), uniform(s.tile0), uniform(s.tiles)};
}

FE2O3_DEVICE uint64_t shfl64(uint64_t v, uint32_t lane) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)v, (int)lane, 64);
  const uint32_t hi = (uint32_t)__shfl((int)(uint32_t)(v >> 32), (int)lane, 64);
  return lo | (uint64_t)hi << 32;
}

// Inclusive sums over the lanes of a wave, within rows of 16 by lane shifts, then
// over the rows: DPP moves, which take no trip through LDS.
FE2O3_DEVICE uint32_t wave_scan(uint32_t v) {
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);  // row_shr:1
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
  // lane 15 of a row to the next one (rows 1 and 3), lane 31 to rows 2 and 3
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
  return v;
}
FE2O3_DEVICE uint32_t at_lane(uint32_t v, uint32_t lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane);
}

// max / sum over the four lanes of a query row (l, l ^ 16, l ^ 32, l ^ 48)
FE2O3_DEVICE float row_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
FE2O3_DEVICE float row_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

FE2O3_DEVICE u32x4_t widen_codes8(uint32_t lo, uint32_t hi) {
  u32x4_t x;
  x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
  x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
  x[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
  x[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  return x;
}

// A tile in a wave's LDS: the K rows, then the V rows, as the cache holds them.
// 16-byte chunk c of row r lies at chunk c ^ swz(r), so that the lanes that are
// served at once reach all banks:
//   K, 8 rows (r % 4 and bit 3 apart) of two neighbouring chunks;
//   V, half a wave's transposing read: bf16 4 rows of two chunks for each of two
//   lane groups, whose rows differ in bit 3; e4m3 8 rows of one chunk for each.
template <int D, uint32_t F>
struct Tile {
  static constexpr uint32_t kRowBytes = F == kBf16 ? 2 * D : F == kE4m3 ? D : D / 2;
  static constexpr uint32_t kRowLanes = kRowBytes / 16u;  // lanes that load a row
  static constexpr uint32_t kRowsPerLoad = 64u / kRowLanes;
  static constexpr int kLoads = kKeys / kRowsPerLoad;     // of K, and of V
  static constexpr uint32_t kBytes = kKeys * kRowBytes;   // of K, and of V
  static FE2O3_DEVICE constexpr uint32_t swz(uint32_t r) {
    if constexpr (F == kE4m3)
      return D == 128 ? (r >> 2 & 1u) | (r & 2u) | (r >> 1 & 4u) : (r >> 2 & 1u) | (r >> 2 & 2u);
    else
      return D == 128 ? 2u * ((r & 3u) | (r >> 1 & 4u)) : 2u * ((r >> 1 & 1u) | (r >> 2 & 2u));
  }
  // the sums of 16 query rows take the tile's place at the end of a run
  static constexpr uint32_t kSumStride = D + 4u;  // floats
  static constexpr uint32_t kSumBytes = 16u * kSumStride * 4u;
};

// How RT tiles of 16 query rows are dealt: row_tiles to a wave, so that sharers waves
// share each tile of keys; and the waves of a workgroup.  One wave's chain of products
// and exponentials over three or four tiles of rows is longer than the loads of the
// next keys, so they have a wave each (a KV head's 64 rows, 48 sequences of 24000 keys:
// 118 us in one wave, 96 shared; 48 sequences of 100 to 6000 with 48 rows: 25 us, 21).
// Two keep up, and a wave of their own reads LDS and widens codes once for both (48
// sequences of 24000 keys, e4m3: 32 rows 61 us, shared 107; 20 rows 59, 103; bf16: 32 rows
// 101 either way, 20 rows 98, 100).
constexpr int row_tiles(int rt) { return rt == 2 ? 2 : 1; }
constexpr uint32_t sharers(int rt) { return (uint32_t)(rt / row_tiles(rt)); }
constexpr uint32_t waves(int rt) { return kWaves * sharers(rt); }

// LDS of a workgroup of W waves: their tiles, or two places for tiles that S waves
// share, which the sums of 16 query rows of each wave take at the end of a run; their
// tiles' scales; their reference and sum of each query row.
template <int D, uint32_t F, uint32_t S, uint32_t W, bool BLOCKS = false>
struct Lds {
  using T = Tile<D, F == kE4m3 && S == 1 ? kE4m3 : kBf16>;
  // of S waves; BLOCKS (DecodeBlocks): V rows of 64 D bytes and 8 D of scales
  static constexpr uint32_t kTiles = BLOCKS ? 68u * D : (S == 1 ? 2u : 4u) * T::kBytes;
  static constexpr uint32_t kSums = S == 1 && kTiles > T::kSumBytes ? kTiles : T::kSumBytes;
  static constexpr uint32_t kOwn = S == 1 ? kSums : kTiles;  // from S waves' to the next
  static constexpr uint32_t kScales = W / S * kOwn > W * kSums ? W / S * kOwn : W * kSums;
  static constexpr uint32_t kStats = kScales + (F == kE4m3 ? W * 2u * kKeys * 4u : 0u);
  static constexpr uint32_t kBytes = kStats + W * 16u * 8u;
  static_assert(kOwn % 256u == 0u, "chunks are chosen by exclusive or");
};

// Workgroups per CU: as many as registers and LDS allow, but two of the widest of one
// row tile (three of them, e4m3, 64 sequences of 4096 keys: 98.5 -> 105.5 us).
template <int D, uint32_t F, int RT, int C>
constexpr int per_cu() {
  if (RT == 1) return D == 64 || (F == kMxfp4 && C == 2) ? 3 : 2;
  return RT == 2 && (D == 64 || F != kBf16) ? 2 : 1;
}

// D: head_dim.  RW: tiles of 16 query rows of a wave.  S waves, a team, share a tile of
// keys, or each has its own (1).  WH: KV heads that a workgroup works on at once, of its
// W waves W / WH on each.
template <int D, uint32_t F, int RW, uint32_t S, int WH, uint32_t W, bool BLOCKS = false>
struct Decode {
  // Codes lie in LDS as they are and are widened on the way out, but waves that share
  // a tile would all widen it: they do on the way in, a part each.
  // 4-bit codes are widened on the way in too, with their scales, so that what follows
  // is a bf16 cache's.
  static constexpr bool E4M3 = F == kE4m3, kCodes = E4M3 && S == 1;
  using R = Tile<D, F>;                       // as loaded
  using T = Tile<D, kCodes ? kE4m3 : kBf16>;  // in LDS
  using L = Lds<D, F, S, W, BLOCKS>;
  static constexpr uint32_t kWiden = T::kRowBytes / R::kRowBytes;  // chunks from one loaded
  static_assert(S == 1 || WH == 1, "waves share a tile of one head");
  static constexpr uint32_t kStep = W / S / WH;  // tiles of a head per round
  static constexpr int kDb = D / 16;     // V^T row blocks
  static constexpr int kFrags = D / 32;  // 16-byte pieces of a query operand per lane
  static constexpr uint32_t kMine = (2u * R::kLoads + S - 1u) / S;  // a wave's loads of a tile

  struct Stage {
    u32x4_t x[kMine];  // the wave's loads i (mine) of a tile: below kLoads K, then V
    float scale;       // E4M3: lanes below 32 the K scale of key l, the others the V scale
    uint32_t blocks;   // MXFP4: the same of a row's scale bytes
    uint32_t valid;    // bit per key
  };
  struct Query {
    u32x4_t f[kFrags];
  };

  const Args& a;
  uint8_t* smem;
  const uint32_t wave, team, member;
  uint32_t buffer;  // S > 1: where the next tile goes, 0 or the offset of the second place

  FE2O3_DEVICE Decode(const Args& args, uint8_t* lds)
      : a(args), smem(lds), wave(uniform(threadIdx.x >> 6)), team(wave / S),
        member(wave % S), buffer(0u) {}

  // The thread's number, as a value that the compiler cannot follow: what is
  // derived from it is then made where it is used, not kept in registers over
  // every run of a workgroup.
  static FE2O3_DEVICE uint32_t thread() {
    uint32_t t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
  }
  // nontemporal, but for 4-bit rows, which share their lines with other heads'
  static FE2O3_DEVICE u32x4_t load(const uint8_t* p) {
    const u32x4_t* row = reinterpret_cast<const u32x4_t*>(p);
    if constexpr (F == kMxfp4) return *row;
    else return __builtin_nontemporal_load(row);
  }
  FE2O3_DEVICE float* scales(uint32_t w) const {
    return (float*)(smem + L::kScales + w * (2u * kKeys * 4u));
  }
  FE2O3_DEVICE float2* stat(uint32_t w) const {
    return (float2*)(smem + L::kStats + w * (16u * 8u));
  }

  // number j of the wave's loads of a tile
  FE2O3_DEVICE uint32_t mine(uint32_t j) const {
    return S == 1 ? j / 2u + j % 2u * R::kLoads : j * S + member;
  }

  // The query operand of lane (lr, g) for row `row` of `rows` (others 0): piece f
  // has the d that the lane's piece of K has (compute): bf16 32 f + 8 g .. + 7;
  // e4m3, where a lane reads 16 codes at once, halves of 16 g .. + 15 and, 128
  // wide, of 64 more.
  FE2O3_DEVICE Query query(const uint16_t* q, uint32_t row, uint32_t rows, uint32_t g) const {
    Query r;
    const bool has = row < rows;
    const uint16_t* from = q + (has ? row : 0u) * D + g * (kCodes ? 16u : 8u);
#pragma unroll
    for (int f = 0; f < kFrags; ++f) {
      r.f[f] = *reinterpret_cast<const u32x4_t*>(from + (kCodes ? (f >> 1) * 64 + (f & 1) * 8
                                                                : f * 32));
      if (!has) r.f[f] = u32x4_t{0, 0, 0, 0};
    }
    return r;
  }

  // Keys of tiles [tile, tile + n) of sequence `seq` for blocks hb0 .. hb0 + WH - 1
  // of the KV heads' query rows.  Place `slot` of this workgroup's workspace
  // takes the sums unless they are the span's every tile.
  FE2O3_DEVICE void run(uint32_t seq, uint32_t hb0, const Span& sp, uint32_t tile, uint32_t n,
                        uint32_t slot) {
    const uint32_t tid = thread(), lane = tid & 63u, lr = lane & 15u, g = lane >> 4;
    const uint32_t head = WH > 1 ? hb0 + team / kStep : hb0 / a.blocks_per_head;
    const uint32_t row0 = WH > 1 ? 0u : (hb0 - head * a.blocks_per_head) * kBlockRows;
    const uint32_t rows = min(a.group - row0, (uint32_t)kBlockRows);
    const uint32_t q_head = head * a.group + row0;
    const uint32_t* table = a.table + (uint64_t)seq * a.table_cols;
    const uint64_t head_at = head * a.cache.head_stride * (F == kBf16 ? 2u : 1u);
    const uint32_t pr = lane / R::kRowLanes, pc = lane % R::kRowLanes;  // as loaded: row, piece
    const uint8_t* kb = a.cache.k + head_at + pc * 16u;
    const uint8_t* vb = a.cache.v + head_at + pc * 16u;
    const float* sb = (lane < 32u ? a.cache.k_scale : a.cache.v_scale);

    const uint32_t end = sp.tile0 + tile + n;
    uint32_t t = sp.tile0 + tile + team % kStep;
    // the table's entry for this lane's key of tile t; none past the run
    auto entry = [&](uint32_t at) {
      const uint32_t key = at * kKeys + (lane & 31u);
      return at < end && key >= sp.first && key < sp.end ? table[a.cache.page.div(key)]
                                                         : 0xffffffffu;
    };
    Stage st;
    auto issue = [&](uint32_t at, uint32_t page) {
      const uint32_t key = at * kKeys + (lane & 31u);
      const uint32_t place = key - a.cache.page.div(key) * a.cache.page.divisor;
      const bool ok = page < a.cache.pages;
      st.valid = uniform((uint32_t)__ballot(ok));
      // a key that is left out reads slot 0, which every cache has
      uint64_t off = ok ? page * a.cache.page_stride + place * a.cache.token_stride : 0u;
      if constexpr (E4M3) {
        const uint64_t at_scale =
            ((uint64_t)(ok ? page : 0u) * a.cache.kv_heads + head) * a.cache.page.divisor +
            (ok ? place : 0u);
        st.scale = sb[at_scale];
      } else if constexpr (F == kMxfp4) {
        const uint64_t row =
            ((uint64_t)(ok ? page : 0u) * a.cache.kv_heads + head) * a.cache.page.divisor +
            (ok ? place : 0u);
        // a key that is left out: a scale that is no NaN, for its V of +0
        if constexpr (D == 128) st.blocks = ok ? ((const uint32_t*)sb)[row] : 0u;
        else st.blocks = ok ? (uint32_t)((const uint16_t*)sb)[row] : 0u;
      } else {
        off *= 2u;
      }
      // nontemporal: 16384 tokens of 8 heads run at 6.4 TB/s, at 5.7 without
#pragma unroll
      for (uint32_t i = 0; i < R::kLoads; ++i) {
        if constexpr (S == 1) {
          const uint64_t row = shfl64(off, i * R::kRowsPerLoad + pr);
          st.x[2u * i] = load(kb + row);
          st.x[2u * i + 1u] = load(vb + row);
        } else if (i < kMine && mine(i) < 2u * R::kLoads) {
          const uint64_t row = shfl64(off, mine(i) % R::kLoads * R::kRowsPerLoad + pr);
          st.x[i] = load((mine(i) < R::kLoads ? kb : vb) + row);
        }
      }
    };

    uint32_t page = entry(t);
    const uint16_t* q = a.q + seq * a.q_stride + (uint64_t)q_head * D;
    Query qf[RW];
    f32x4_t acc[RW][kDb];
    // as in the prompt kernel: the lowest finite value, against which scores of -inf
    // alone have exponentials of 0
    float m_ref[RW], l_run[RW];
#pragma unroll
    for (int rt = 0; rt < RW; ++rt) {
      qf[rt] = query(q, (member * RW + rt) * 16u + lr, rows, g);
      m_ref[rt] = -__FLT_MAX__;
      l_run[rt] = 0.0f;
#pragma unroll
      for (int db = 0; db < kDb; ++db) acc[rt][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    if (t < end) {
      issue(t, page);
      page = entry(t + kStep);
    }

    // LDS addresses.  The wave's tile is aligned to 256 bytes and the swizzle
    // moves chunk bits alone, so another chunk of a row is an exclusive or, and
    // another row an offset and the exclusive or of its swizzle.  Row m of key
    // block b is key 8 (m / 4) + 4 b + m % 4.
    const uint32_t own_at = team * L::kOwn;
    const uint32_t k_row = 8u * (lr >> 2) + (lr & 3u);
    const uint32_t v_row = 8u * g + (kCodes ? lr >> 1 : lr >> 2);
    uint32_t put_at = own_at + pr * T::kRowBytes + ((kWiden * pc ^ T::swz(pr)) << 4);
    uint32_t k_at = own_at + k_row * T::kRowBytes +
                    ((g ^ T::swz(k_row)) << 4);
    uint32_t v_at = own_at + T::kBytes + v_row * T::kRowBytes +
                    ((((kCodes ? 0u : (lr & 3u) >> 1)) ^ T::swz(v_row)) << 4) + (lr & 1u) * 8u;

    // the stage's tile into the wave's LDS.  Keys that are left out have scores
    // of -inf whatever K holds, but 0 times their V must be 0: V becomes +0.
    auto put = [&] {
      asm volatile("" : "+v"(put_at));
      if (st.valid != 0xffffffffu) {
#pragma unroll
        for (uint32_t j = 0; j < kMine; ++j) {
          const uint32_t i = mine(j), r = i % R::kLoads * R::kRowsPerLoad;
          if (i >= R::kLoads && (st.valid >> (r + pr) & 1u) == 0u) st.x[j] = u32x4_t{0, 0, 0, 0};
        }
        asm volatile("");  // a branch, not a select in every tile
      }
#pragma unroll
      for (uint32_t j = 0; j < kMine; ++j) {
        const uint32_t i = mine(j), r = i % R::kLoads * R::kRowsPerLoad;
        if (S > 1 && i >= 2u * R::kLoads) break;
        // the swizzle of row r + pr (r a multiple of a power of two above pr) is that
        // of both
        const uint32_t at = ((put_at + buffer) ^ T::swz(r) << 4) + r * T::kRowBytes +
                            (i < R::kLoads ? 0u : T::kBytes);
        if constexpr (kWiden == 1u) {
          *reinterpret_cast<u32x4_t*>(smem + at) = st.x[j];
        } else if constexpr (F == kMxfp4) {
          const uint32_t bytes =
              (uint32_t)__shfl((int)st.blocks, (int)(r + pr + (i < R::kLoads ? 0u : 32u)), 64);
          const float scale = mxfp4::scale_float(bytes >> (8u * pc) & 255u);
#pragma unroll
          for (uint32_t c = 0; c < 4u; ++c)
            *reinterpret_cast<u32x4_t*>(smem + (at ^ c << 4)) =
                mxfp4::decode8_bf16(st.x[j][c], scale);
        } else {  // swizzles of bf16 rows are even: the two chunks stay together
          *reinterpret_cast<u32x4_t*>(smem + at) = widen_codes8(st.x[j][0], st.x[j][1]);
          *reinterpret_cast<u32x4_t*>(smem + at + 16u) = widen_codes8(st.x[j][2], st.x[j][3]);
        }
      }
      if constexpr (E4M3)
        scales(wave)[lane] = (st.valid >> (lane & 31u) & 1u) != 0u
                                 ? st.scale * (lane < 32u ? a.scale_log2 : 1.0f)
                                 : 0.0f;
    };

    auto compute = [&](uint32_t valid) {
      // the addresses of the pieces are made here, tile by tile: kept over the
      // loop they would take the registers of a stage
      asm volatile("" : "+v"(k_at), "+v"(v_at));
      const uint32_t k_from = k_at + buffer, v_from = v_at + buffer;
      f32x4_t sc[RW][2];
      // Codes are widened to bf16, exactly, where the MFMA takes them.  The fp8 MFMA
      // would take them as they are (and a query as the sum of two e4m3), but
      // drops what is 2^-15 of its largest product: lse was off by 6e-5.
#pragma unroll
      for (int f = 0; f < kFrags; f += kCodes ? 2 : 1) {
        bf16x8_t kf[2][kCodes ? 2 : 1];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const u32x4_t x = *reinterpret_cast<const u32x4_t*>(
              smem + (k_from ^ (kCodes ? 32u : 64u) * f ^ T::swz(4u * b) << 4) +
              4u * T::kRowBytes * b);
          if constexpr (kCodes) {
            kf[b][0] = __builtin_bit_cast(bf16x8_t, widen_codes8(x[0], x[1]));
            kf[b][1] = __builtin_bit_cast(bf16x8_t, widen_codes8(x[2], x[3]));
          } else {
            kf[b][0] = __builtin_bit_cast(bf16x8_t, x);
          }
        }
#pragma unroll
        for (int rt = 0; rt < RW; ++rt)
#pragma unroll
          for (int h = 0; h < (kCodes ? 2 : 1); ++h)
#pragma unroll
            for (int b = 0; b < 2; ++b)
              sc[rt][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  kf[b][h], __builtin_bit_cast(bf16x8_t, qf[rt].f[f + h]),
                  f + h == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : sc[rt][b], 0, 0, 0);
      }
      // lane's key j (0..7) is 8 g + j
      float ks[8], vs[8];
      if constexpr (E4M3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4_t x = *reinterpret_cast<const f32x4_t*>(scales(wave) + 8u * g + 4 * h);
          const f32x4_t y = *reinterpret_cast<const f32x4_t*>(scales(wave) + 32u + 8u * g + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ks[4 * h + e] = x[e];
            vs[4 * h + e] = y[e];
          }
        }
      }
      // scores in the log2 domain (bf16 cache: before its scale), then probabilities
      // of all query rows, so that one branch serves them
      float x[RW][8], p[RW][8], psum[RW];
#pragma unroll
      for (int rt = 0; rt < RW; ++rt)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[rt][j] = sc[rt][j >> 2][j & 3] * (E4M3 ? ks[j] : 1.0f);
      if (valid != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool keep = (valid >> (8u * g + j) & 1u) != 0u;
#pragma unroll
          for (int rt = 0; rt < RW; ++rt) x[rt][j] = keep ? x[rt][j] : -INFINITY;
        }
        asm volatile("");
      }
      auto probabilities = [&] {
        bool small = true;
#pragma unroll
        for (int rt = 0; rt < RW; ++rt) {
          psum[rt] = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            p[rt][j] = __builtin_amdgcn_exp2f(
                E4M3 ? x[rt][j] - m_ref[rt] : __builtin_fmaf(x[rt][j], a.scale_log2, -m_ref[rt]));
            psum[rt] += p[rt][j];
          }
          small = small && psum[rt] <= kLazyBound;
        }
        return small;
      };
      if (__any(!probabilities())) {
#pragma unroll
        for (int rt = 0; rt < RW; ++rt) {
          float top = x[rt][0];
#pragma unroll
          for (int j = 1; j < 8; ++j) top = fmaxf(top, x[rt][j]);
          if (!E4M3) top *= a.scale_log2;  // positive
          const float m_new = fmaxf(m_ref[rt], row_max(top));
          const float alpha = __builtin_amdgcn_exp2f(m_ref[rt] - m_new);
          m_ref[rt] = m_new;
          l_run[rt] *= alpha;
#pragma unroll
          for (int db = 0; db < kDb; ++db)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[rt][db][e] *= alpha;
        }
        (void)probabilities();
      }
      // Two bf16 parts: the second MFMA takes what the first one leaves, to half a step
      // of its own rounding, 2^-16 of the probability, for 1% more time.  The first part of a
      // probability is the next bf16 below it, so that both are positive and an infinite
      // V row's products do not cancel (rounded to nearest, the second may be 0 or
      // negative).  Codes hold no infinity, and a V scale may have any sign.
      bf16x8_t pf[RW], pl[RW];
#pragma unroll
      for (int rt = 0; rt < RW; ++rt) {
        l_run[rt] += psum[rt];
        u32x4_t below;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (E4M3) {
            const float y = p[rt][j] * vs[j];
            pf[rt][j] = (__bf16)y;
            pl[rt][j] = (__bf16)(y - (float)pf[rt][j]);
          } else {  // +0 stays +0
            const uint32_t part =
                __builtin_elementwise_sub_sat(__float_as_uint(p[rt][j]), 1u) & 0xffff0000u;
            below[j / 2] = j % 2 == 0 ? part >> 16 : below[j / 2] | part;
            pl[rt][j] = (__bf16)(p[rt][j] - __uint_as_float(part));
          }
        }
        if constexpr (!E4M3) pf[rt] = __builtin_bit_cast(bf16x8_t, below);
      }
      // O^T += V^T P^T: lane i of group g receives d 16 db + i of keys 8 g .. + 7.
      // Two blocks of d at a time, so that no MFMA waits for the one before it.
#pragma unroll
      for (int d2 = 0; d2 < kDb; d2 += 2) {
        bf16x8_t vf[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int db = d2 + i;
          if constexpr (kCodes) {
            const i32x2_t c = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (lds_i32x2_t*)(smem + (v_from ^ (16u * db))));
            vf[i] = __builtin_bit_cast(bf16x8_t, widen_codes8((uint32_t)c[0], (uint32_t)c[1]));
          } else {
            bf16x4_t half[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
              half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                  (lds_bf16x4_t*)(smem + (v_from ^ (32u * db)) + 4u * T::kRowBytes * h));
            vf[i] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
          }
        }
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int rt = 0; rt < RW; ++rt)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              acc[rt][d2 + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  vf[i], part == 0 ? pf[rt] : pl[rt], acc[rt][d2 + i], 0, 0, 0);
      }
    };

    // A wave's LDS operations run in order, so a tile's reads see its writes and
    // the next tile's writes wait for them; the fences keep the compiler from
    // reordering them (it sees one lane's addresses).  One tile is in flight while
    // another is computed: two were no faster where a CU's waves have 128 KiB in flight
    // so (8 x 32 heads x 4096: 87, 97 us).
    // A tile that waves share goes to the other place than the one before it, which
    // a wave that is behind may still read; the barrier leaves none two behind.
    if constexpr (S == 1) {
      for (; t < end; t += kStep) {
        put();
        const uint32_t valid = st.valid;
        asm volatile("" ::: "memory");
        if (t + kStep < end) {
          issue(t + kStep, page);
          page = entry(t + 2u * kStep);
        }
        compute(valid);
        asm volatile("" ::: "memory");
      }
    } else {
      for (uint32_t round = sp.tile0 + tile; round < end; round += kStep, t += kStep) {
        if (t < end) put();
        const uint32_t valid = st.valid;
        __syncthreads();
        if (t + kStep < end) {
          issue(t + kStep, page);
          page = entry(t + 2u * kStep);
        }
        if (t < end) compute(valid);
        buffer ^= 2u * T::kBytes;
      }
      __syncthreads();
    }
    finish(seq, WH > 1 ? q_head - team / kStep * a.group : q_head, rows, n == sp.tiles, slot, acc,
           m_ref, l_run);
  }

  // The sums of a run's waves added for each head in wave order, 16 query rows of each
  // wave at a time.  q_head: the first head's first.
  FE2O3_DEVICE void finish(uint32_t seq, uint32_t q_head, uint32_t rows, bool whole, uint32_t slot,
                           const f32x4_t (&acc)[RW][kDb], const float (&m_ref)[RW],
                           const float (&l_run)[RW]) {
    const uint32_t tid = thread(), lr = tid & 15u, g = tid >> 4 & 3u;
    const uint64_t part = ((uint64_t)blockIdx.x * 2u + slot) * WH * a.rows;
#pragma unroll
    for (int rt = 0; rt < RW; ++rt) {
      if (rt * 16u >= rows) break;
      const float sum = row_sum(l_run[rt]);
      if (g == 0u) stat(wave)[lr] = float2{m_ref[rt], sum};
      float* own = (float*)(smem + wave * L::kSums) + lr * T::kSumStride + 4u * g;
#pragma unroll
      for (int db = 0; db < kDb; ++db) *reinterpret_cast<f32x4_t*>(own + 16 * db) = acc[rt][db];
      __syncthreads();
      // this turn's rows: of one head behind another's, or of every sharer
      const uint32_t turn_rows = S > 1 ? 16u * S : min(rows - rt * 16u, 16u);
      for (uint32_t i = tid; i < WH * turn_rows * (D / 4u); i += W * 64u) {
        const uint32_t at = i / (D / 4u), d = 4u * (i % (D / 4u));
        const uint32_t wh = WH > 1 ? at / turn_rows : 0u, r = at - wh * turn_rows;
        const uint32_t first = S == 1 ? wh * kStep : r / 16u, tile_row = r % 16u;
        const uint32_t row = S == 1 ? rt * 16u + r : (first * RW + rt) * 16u + tile_row;
        if (S > 1 && row >= rows) continue;
        float2 s[kStep];
        float m = -__FLT_MAX__, l = 0.0f;
#pragma unroll
        for (uint32_t x = 0; x < kStep; ++x) {
          s[x] = stat(first + x * S)[tile_row];
          m = fmaxf(m, s[x].x);
        }
        f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t x = 0; x < kStep; ++x) {
          const float weight = __builtin_amdgcn_exp2f(s[x].x - m);
          l += weight * s[x].y;
          y += weight * *reinterpret_cast<const f32x4_t*>(
                            (const float*)(smem + (first + x * S) * L::kSums) +
                            tile_row * T::kSumStride + d);
        }
        if (whole) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key: +0
          const uint64_t out = (uint64_t)seq * a.q_heads + q_head + wh * a.group + row;
          *reinterpret_cast<u32x2_t*>(a.o + out * D + d) =
              u32x2_t{pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv)};
          if (a.lse != nullptr && d == 0u)
            a.lse[out] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
        } else {
          const uint64_t p = part + wh * a.rows + row;
          *reinterpret_cast<f32x4_t*>(a.sums + p * D + d) = y;
          if (d == 0u) *reinterpret_cast<float2*>(a.stats + p * 2u) = float2{m, l};
        }
      }
      __syncthreads();
    }
  }
};

// A 4-bit cache, 16 query heads a KV head at the most.  A tile is 64 keys, a key a lane
// where their pages are looked up, in two subtiles of 32:
//   * K codes are loaded as the product wants them: lane (l % 16, l / 16) a quarter of a
//     key's row, widened with its block's scale; the query operand has the same
//     quarter's d.  Loads of which adjacent lanes take different rows run at a quarter of
//     the rate, which 4-bit rows leave room for.
//   * V codes are widened with their scales on the way into LDS, a subtile at a time,
//     whose registers then take the next tile's.
//   * With few query heads most lanes of a product hold no query: with at most eight
//     (C = 2) the scores of both subtiles are moved side by side for the softmax and the
//     probabilities' two bf16 parts, and these moved back for each product with V.
//   * A key that is left out reads slot 0, which every cache has, with scales of 2^-127: its
//     score is set to -inf all the same, its probability is 0 and its V finite.
// No branch but the rescale's and that of the keys left out, so that products, conversions
// and LDS accesses overlap.  Loads go by the caches: a head's row is half of a line of 128
// bytes, whose other half another wave wants (64 sequences of 2 to 8190 keys, 8 heads in
// token order: 54 us; nontemporal 71, with 1.36 times the bytes).  Three workgroups a CU
// with tiles of 64 keys; 128 keys, twice the registers and two workgroups: 59 us.
template <int D, int C, int WH, uint32_t W>
struct DecodeBlocks : Decode<D, kMxfp4, 1, 1, WH, W, true> {
  using Base = Decode<D, kMxfp4, 1, 1, WH, W, true>;
  using Base::a;
  using Base::smem;
  using Base::wave;
  static constexpr uint32_t kStep = Base::kStep;
  static constexpr int kDb = Base::kDb, kFrags = Base::kFrags;
  static constexpr uint32_t kRowBytes = D / 2, kRowLanes = kRowBytes / 16u;
  static constexpr uint32_t kRowsPerLoad = 64u / kRowLanes;  // 16 or 32
  static constexpr int kLoads = kBlockKeys / kRowsPerLoad;   // of K, and of V
  static constexpr int kSub = kBlockKeys / 32, kSubLoads = kLoads / kSub;  // subtiles, and their V's loads
  static constexpr int kSets = kSub / C;                     // softmax registers, 8 each
  // LDS: V rows of a subtile, K's scales, V's
  static constexpr uint32_t kVRow = 2u * D;
  static constexpr uint32_t kScaleAt = kKeys * kVRow, kScaleRow = D / 32u;
  static constexpr uint32_t kScales = kBlockKeys * kScaleRow;
  static_assert(kScaleAt + 2u * kScales == 68u * D, "as Lds has it");
  using ScaleT = std::conditional_t<D == 128, uint32_t, uint16_t>;  // a row's
  using Quarter = std::conditional_t<D == 128, u32x4_t, u32x2_t>;   // of a row of K

  FE2O3_DEVICE DecodeBlocks(const Args& args, uint8_t* lds) : Base(args, lds) {}

  // V: chunk c of row r lies at c ^ v_swz(r).  The transposing reads take pairs of chunks
  // of rows 0-3 and 8-11, the writes chunk 4 piece + c of rows 0, 1, 4 and 5 (64 wide:
  // 0-3 and 8-11).
  static FE2O3_DEVICE constexpr uint32_t v_swz(uint32_t r) {
    return D == 128 ? 2u * ((r & 3u) | (r >> 1 & 4u)) | (r >> 2 & 1u)
                    : 2u * ((r >> 1 & 1u) | (r >> 2 & 2u)) | (r >> 3 & 1u);
  }

  // C = 2: the upper eight lanes of each row of 16 take v of the lower ones
  static FE2O3_DEVICE float beside(float low, float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
        (int)__float_as_uint(low), (int)__float_as_uint(v), 0x118, 0xf, 0xc, false));  // row_shr:8
  }
  // and back: the lower ones take v of the upper
  static FE2O3_DEVICE u32x4_t from_beside(u32x4_t v) {
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i)  // row_shl:8
      r[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v[i], 0x108, 0xf, 0xf, true);
    return r;
  }
  // over the lanes of a query in both subtiles
  static FE2O3_DEVICE float sets_max(float v) {
    return C == 2 ? fmaxf(v, __shfl_xor(v, 8, 64)) : v;
  }
  static FE2O3_DEVICE float sets_sum(float v) { return C == 2 ? v + __shfl_xor(v, 8, 64) : v; }

  FE2O3_DEVICE void run(uint32_t seq, uint32_t hb0, const Span& sp, uint32_t tile, uint32_t n,
                        uint32_t slot) {
    const uint32_t tid = Base::thread(), lane = tid & 63u, lr = lane & 15u, g = lane >> 4;
    const uint32_t head = WH > 1 ? hb0 + wave / kStep : hb0, rows = a.group;
    const uint32_t q_head = head * a.group;
    const uint32_t* table = a.table + (uint64_t)seq * a.table_cols;
    const uint64_t head_at = head * a.cache.head_stride;
    const uint32_t pr = lane / kRowLanes, pc = lane % kRowLanes;  // V as loaded: row, piece
    const uint32_t k_row = 8u * (lr >> 2) + (lr & 3u);            // K, + 32 j + 4 b
    const uint8_t* kb = a.cache.k + head_at + g * (kRowBytes / 4u);
    const uint8_t* vb = a.cache.v + head_at + pc * 16u;
    const ScaleT* kscales = (const ScaleT*)a.cache.k_blocks();
    const ScaleT* vscales = (const ScaleT*)a.cache.v_blocks();

    const uint32_t end = sp.tile0 + tile + n;
    uint32_t t = sp.tile0 + tile + wave % kStep;
    // of the tile whose loads are in flight, lane l's key l
    uint32_t page, place, k_scale, v_scale;
    uint64_t valid;
    // the loads' rows, in 16 bytes from the head's first
    uint32_t k16[2 * kSub], v16[kLoads];
    Quarter kx[2 * kSub];  // rows 32 j + 4 b + k_row at 2 j + b
    u32x4_t vx[kLoads];
    // the table's entry for this lane's key of tile `at`; none past the run
    auto entry = [&](uint32_t at) {
      const uint32_t key = at * kBlockKeys + lane, col = a.cache.page.div(key);
      place = key - col * a.cache.page.divisor;
      page = at < end && key >= sp.first && key < sp.end ? table[col] : 0xffffffffu;
    };
    // rows in 32 bits: the host has seen to it
    const uint32_t page16 = (uint32_t)(a.cache.page_stride >> 4);
    const uint32_t token16 = (uint32_t)(a.cache.token_stride >> 4);
    const uint32_t page_rows = a.cache.kv_heads * a.cache.page.divisor;
    const uint32_t head_rows = head * a.cache.page.divisor;
    auto locate = [&] {
      const bool ok = page < a.cache.pages;
      if (!ok) page = place = 0u;
      valid = __ballot(ok);
      const uint32_t row16 = page * page16 + place * token16;
      const uint32_t row = page * page_rows + head_rows + place;
      k_scale = (uint32_t)kscales[row];
      v_scale = (uint32_t)vscales[row];
      if (!ok) k_scale = v_scale = 0u;
#pragma unroll
      for (uint32_t i = 0; i < 2u * kSub; ++i)
        k16[i] = (uint32_t)__shfl((int)row16, (int)(16u * i - 12u * (i % 2u) + k_row), 64);
#pragma unroll
      for (uint32_t i = 0; i < (uint32_t)kLoads; ++i)
        v16[i] = (uint32_t)__shfl((int)row16, (int)(i * kRowsPerLoad + pr), 64);
    };
    auto load_k = [&](uint32_t i) {
      kx[i] = *reinterpret_cast<const Quarter*>(kb + ((uint64_t)k16[i] << 4));
    };
    auto load_v = [&](uint32_t i) {
      vx[i] = *reinterpret_cast<const u32x4_t*>(vb + ((uint64_t)v16[i] << 4));
    };

    entry(t);
    // the lane's quarter of a row: d D / 4 g + 8 f .. + 7
    const uint16_t* q = a.q + seq * a.q_stride + (uint64_t)q_head * D +
                        (lr < rows ? lr : 0u) * D + g * (D / 4u);
    u32x4_t qf[kFrags];
    f32x4_t acc[1][kDb];
    float m_ref[1] = {-__FLT_MAX__}, l_run[1] = {0.0f};
#pragma unroll
    for (int f = 0; f < kFrags; ++f) {
      qf[f] = *reinterpret_cast<const u32x4_t*>(q + 8 * f);
      if (lr >= rows) qf[f] = u32x4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int db = 0; db < kDb; ++db) acc[0][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (t < end) {
      locate();
      entry(t + kStep);
#pragma unroll
      for (uint32_t i = 0; i < 2u * kSub; ++i) load_k(i);
#pragma unroll
      for (uint32_t i = 0; i < (uint32_t)kLoads; ++i) load_v(i);
    }

    uint8_t* own = smem + wave * Base::L::kOwn;
    const uint32_t v_row = 8u * g + (lr >> 2);
    // V's row r + 32 j lies a constant further on, and r + 4 also where its swizzle says
    uint32_t v_put = pr * kVRow + ((4u * pc ^ v_swz(pr)) << 4);
    uint32_t v_at = v_row * kVRow + ((((lr & 3u) >> 1) ^ v_swz(v_row)) << 4) + (lr & 1u) * 8u;
    uint32_t ks_at = kScaleAt + k_row * kScaleRow + (D == 128 ? g : g >> 1);
    uint32_t vs_at = kScaleAt + kScales + pr * kScaleRow + pc;

    for (; t < end; t += kStep) {
      // other addresses are made from these tile by tile: kept over the loop they would
      // take the registers of a stage
      asm volatile("" : "+v"(v_put), "+v"(v_at), "+v"(ks_at), "+v"(vs_at));
      // the scales to LDS; a wave's LDS operations run in order
      ScaleT* to = reinterpret_cast<ScaleT*>(own + kScaleAt) + lane;
      to[0] = (ScaleT)k_scale;
      to[kBlockKeys] = (ScaleT)v_scale;
      asm volatile("" ::: "memory");
      const uint64_t kept = valid;
      // behind the run's last tile, slot 0 once more
      locate();
      entry(t + 2u * kStep);
      // scores: lane's key e (0..7) of subtile j is 32 j + 8 g + e.  Barriers keep the
      // compiler from reading further ahead than the registers go.
      float x[kSub][8];
      uint32_t byte[2 * kSub];
#pragma unroll
      for (uint32_t i = 0; i < 2u * kSub; ++i)
        byte[i] = own[ks_at + (16u * i - 12u * (i % 2u)) * kScaleRow];
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        f32x4_t s[2] = {};
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
#pragma unroll
          for (int b = 0; b < 2; ++b)
            s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t,
                                   mxfp4::decode8_bf16(kx[2 * j + b][f],
                                                       mxfp4::scale_float(byte[2 * j + b]))),
                __builtin_bit_cast(bf16x8_t, qf[f]), s[b], 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] = s[e / 4][e % 4];
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (C == 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[0][e] = beside(x[0][e], x[1][e]);
      }
      if (kept != ~UINT64_C(0)) {
        uint32_t mine = lr, shift = 8u * g;
        asm volatile("" : "+v"(mine), "+v"(shift));  // no masks kept over the loop
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
          // the lane's subtile of set s
          const uint32_t low = (uint32_t)kept, high = (uint32_t)(kept >> 32);
          const uint32_t word = (C == 2 ? (mine >= 8u ? high : low) : s == 0 ? low : high) >> shift;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((word >> e & 1u) == 0u) x[s][e] = -INFINITY;
        }
      }
      // the next tile's K: its registers are not needed before
#pragma unroll
      for (uint32_t i = 0; i < 2u * kSub; ++i) load_k(i);
      // as Decode's: against a running reference, the same in all sets
      float p[kSets][8], psum;
      auto probabilities = [&] {
        psum = 0.0f;
#pragma unroll
        for (int s = 0; s < kSets; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[s][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[s][e], a.scale_log2, -m_ref[0]));
            psum += p[s][e];
          }
        return psum <= kLazyBound;
      };
      if (__any(!probabilities())) {
        float top = x[0][0];
#pragma unroll
        for (int s = 0; s < kSets; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, x[s][e]);
        const float m_new = fmaxf(m_ref[0], sets_max(row_max(top * a.scale_log2)));
        const float alpha = __builtin_amdgcn_exp2f(m_ref[0] - m_new);
        m_ref[0] = m_new;
        l_run[0] *= alpha;
#pragma unroll
        for (int db = 0; db < kDb; ++db)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[0][db][e] *= alpha;
        (void)probabilities();
      }
      l_run[0] += psum;
      u32x4_t hi, lo;
      // V codes of subtile j widened into LDS, its registers to the next tile's
      auto put_v = [&](auto number) {
        constexpr int j = decltype(number)::value;
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)kSubLoads; ++i) {
          const uint32_t r = i * kRowsPerLoad;  // of the subtile, with pr
          const u32x4_t codes = vx[j * kSubLoads + i];
          const float scale = mxfp4::scale_float(
              own[vs_at + (32u * j + r) * kScaleRow]);
#pragma unroll
          for (uint32_t c = 0; c < 4u; ++c)
            *reinterpret_cast<u32x4_t*>(own + (v_put ^ c << 4) + r * kVRow) =
                mxfp4::decode8_bf16(codes[c], scale);
          load_v(j * kSubLoads + i);
        }
      };
      auto subtile = [&](auto number) {
        constexpr int j = decltype(number)::value;
        if constexpr (j % C == 0) {
          // two bf16 parts, as Decode's, to the nearest: the write makes no infinite value
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float first = p[j / C][2 * e], second = p[j / C][2 * e + 1];
            const uint32_t w = pack_bf16x2(first, second);
            hi[e] = w;
            lo[e] = pack_bf16x2(first - __uint_as_float(w << 16),
                                second - __uint_as_float(w & 0xffff0000u));
          }
        }
        constexpr bool kBeside = j % C != 0;
        const u32x4_t parts[2] = {kBeside ? from_beside(hi) : hi, kBeside ? from_beside(lo) : lo};
        // lane i of group g receives d 16 db + i of keys 8 g .. + 7; half of the d at a time
#pragma unroll
        for (int d0 = 0; d0 < kDb; d0 += kDb / 2) {
          bf16x8_t vf[kDb / 2];
#pragma unroll
          for (int i = 0; i < kDb / 2; ++i) {
            bf16x4_t half[2];
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h)
              half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                  (lds_bf16x4_t*)(own + (v_at ^ 32u * (d0 + i) ^ v_swz(4u * h) << 4) +
                                  4u * kVRow * h));
            vf[i] = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
          }
          __builtin_amdgcn_sched_barrier(0);
          // the next subtile's conversions and writes run beside these products
          if constexpr (j + 1 < kSub)
            if (d0 != 0) put_v(std::integral_constant<int, j + 1>{});
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int i = 0; i < kDb / 2; ++i)
              acc[0][d0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  vf[i], __builtin_bit_cast(bf16x8_t, parts[part]), acc[0][d0 + i], 0, 0, 0);
          if (d0 != 0) __builtin_amdgcn_sched_barrier(0);
        }
      };
      __builtin_amdgcn_sched_barrier(0);
      put_v(std::integral_constant<int, 0>{});
      __builtin_amdgcn_sched_barrier(0);
      subtile(std::integral_constant<int, 0>{});
      subtile(std::integral_constant<int, 1>{});
      asm volatile("" ::: "memory");
    }
    l_run[0] = sets_sum(l_run[0]);
    Base::finish(seq, WH > 1 ? q_head - wave / kStep * a.group : q_head, rows, n == sp.tiles, slot,
                 acc, m_ref, l_run);
  }
};

// How a form works on its tiles: 4-bit codes of one row tile by DecodeBlocks, C subtiles'
// scores side by side.  More query heads go the way of a bf16 cache, widened into LDS, one KV
// head a workgroup: of heads in token order it takes whole lines of 128 bytes for rows that
// are half of one, or 64 wide a quarter (64 sequences of 2 to 8190 keys, 8 KV heads: 560 MB
// for 290, or 147).  Times with the join over caches that alternate, by query heads a KV head,
// 128 wide and 64: 8 78 and 46 us, 16 84 and 48, 17 106 and 88, 32 110 and 89, 48 137 and 104,
// 64 154 and 108 (there the conversions count as well, VALU 62-66%).
template <uint32_t F, int RT>
constexpr uint32_t keys_of() {
  return F == kMxfp4 && RT == 1 ? kBlockKeys : kKeys;
}
template <int D, uint32_t F, int RT, uint32_t W>
using LdsOf = Lds<D, F, sharers(RT), W, F == kMxfp4 && RT == 1>;
template <int D, uint32_t F, int RT, int C, int WH, uint32_t W>
using DecodeOf = std::conditional_t<F == kMxfp4 && RT == 1, DecodeBlocks<D, C, WH, W>,
                                    Decode<D, F, row_tiles(RT), sharers(RT), WH, W>>;

// One workgroup of W waves per sequence and block of query rows, for calls whose
// sequences are too short to be worth a join.
template <int D, uint32_t F, int RT, int C, uint32_t W>
__global__ void __launch_bounds__(W * 64, (W == waves(RT) ? per_cu<D, F, RT, C>() * sharers(RT) : 2)) paged_whole_kernel(Args a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t blocks = a.cache.kv_heads * a.blocks_per_head;
  uint32_t id = blockIdx.y * kv_cache::kGridWidth + blockIdx.x;
  // 4-bit rows of neighbouring heads share their lines: such workgroups on one XCD, which
  // workgroups are dealt to in turn (64 x 500 keys, 8 heads: 11.0 us, in turn 15.7; 64 x
  // 2000: 28.8, 45.9)
  if constexpr (F == kMxfp4) {
    const uint32_t total = a.seqs * blocks;
    if (total % a.xcds == 0u && id < total) id = id % a.xcds * (total / a.xcds) + id / a.xcds;
  }
  const uint32_t seq = id / blocks, hb = id - seq * blocks;
  if (seq >= a.seqs) return;  // the last row of a grid of two dimensions
  const Span sp = uniform_span_of<keys_of<F, RT>()>(a, seq);
  DecodeOf<D, F, RT, C, 1, W>(a, smem).run(seq, hb, sp, 0u, sp.tiles, 0u);
}

// The list of all work: sequence, then block of query rows (or WH KV heads), then
// round, a round being a tile for each wave.  What starting on a head costs (its
// pages, queries and first loads, and the sums at the end) counts as kSetup
// rounds before its first.  Workgroup i takes rounds i run .. + run - 1.
//
// Every wave counts the list by itself: lane l the sequences chunk l .. + chunk - 1,
// four lengths a load, then one scan over the lanes; a place is found among the
// lanes, then in a chunk.  4096 sequences of 1 to 300 keys, 2 heads: 127 us so, 134
// by single lengths, 154 with a scan for every 64 sequences.
template <int RT, int WH, uint32_t KEYS>
struct Plan {
  static constexpr uint32_t kStep = kWaves / WH, kSetup = RT == 1 ? 1u : 2u;
  const Args& a;
  uint32_t lane, blocks, chunk;
  uint32_t first_length;  // of sequence `lane`, if a chunk is one
  uint32_t chunk_scan;    // rounds of a block of lanes 0 .. lane's chunks
  uint32_t total, run;

  static FE2O3_DEVICE uint32_t rounds(const Span& sp) {
    return (sp.tiles + kStep - 1u) / kStep + kSetup;
  }
  FE2O3_DEVICE explicit Plan(const Args& args)
      : a(args), lane(threadIdx.x & 63u), blocks(a.cache.kv_heads * a.blocks_per_head / WH),
        chunk(a.seqs <= 64u ? 1u : ((a.seqs - 1u) / 256u + 1u) * 4u), first_length(0u) {
    uint32_t sum = 0;
    if (chunk == 1u) {
      first_length = lane < a.seqs ? a.lengths[lane] : 0u;
      sum = lane < a.seqs ? rounds(span_of<KEYS>(a, first_length)) : 0u;
    } else {
#pragma unroll 4
      for (uint32_t i = 0; i < chunk; i += 4u) {
        const uint32_t s = lane * chunk + i, from = min(s, a.seqs - 4u);
        const u32x4_any_t x = *reinterpret_cast<const u32x4_any_t*>(a.lengths + from);
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) sum += from + e >= s ? rounds(span_of<KEYS>(a, x[e])) : 0u;
      }
    }
    chunk_scan = wave_scan(sum);
    total = at_lane(chunk_scan, 63u) * blocks;
    run = uniform((total - 1u) / a.workgroups + 1u);
  }
  // rounds of a block of sequences base .. base + lane, those below limit
  FE2O3_DEVICE uint32_t scan(uint32_t base, uint32_t limit) const {
    const uint32_t s = base + lane;
    return wave_scan(s < limit ? rounds(span_of<KEYS>(a, a.lengths[s])) : 0u);
  }
  FE2O3_DEVICE Span span(uint32_t seq) const {
    return span_of<KEYS>(a, chunk == 1u ? at_lane(first_length, seq) : uniform(a.lengths[seq]));
  }
  // the sequence that round `at` (below total) falls into, and the rounds of a
  // block before it
  FE2O3_DEVICE uint32_t find(uint32_t at, uint32_t* before) const {
    const uint32_t c = (uint32_t)__popcll(__ballot(chunk_scan * blocks <= at));
    uint32_t skipped = c != 0u ? at_lane(chunk_scan, c - 1u) : 0u, seq = c * chunk;
    if (chunk != 1u) {
      const uint32_t limit = min(seq + chunk, a.seqs);
      while (true) {
        const uint32_t sums = scan(seq, limit);
        const uint32_t n = (uint32_t)__popcll(
            __ballot(seq + lane < limit && (skipped + sums) * blocks <= at));
        if (n < 64u) {
          if (n != 0u) skipped += at_lane(sums, n - 1u);
          seq += n;
          break;
        }
        skipped += at_lane(sums, 63u);
        seq += 64u;
      }
    }
    *before = skipped;
    return seq;
  }
  // the rounds of a block before sequence seq
  FE2O3_DEVICE uint32_t before(uint32_t seq) const {
    const uint32_t c = chunk == 1u ? seq : uniform(seq / chunk);
    uint32_t skipped = c != 0u ? at_lane(chunk_scan, c - 1u) : 0u;
    if (chunk != 1u)
      for (uint32_t base = c * chunk; base < seq; base += 64u)
        skipped += at_lane(scan(base, seq), 63u);
    return skipped;
  }
};

template <int D, uint32_t F, int RT, int C, int WH>
__global__ void __launch_bounds__(waves(RT) * 64, (per_cu<D, F, RT, C>() * sharers(RT))) paged_split_kernel(Args a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  using P = Plan<RT, WH, keys_of<F, RT>()>;
  const P plan(a);
  uint32_t at = blockIdx.x * plan.run;  // below total + grid: the host keeps it in 32 bits
  const uint32_t end = min(at + plan.run, plan.total);
  if (at >= plan.total) return;
  uint32_t before;
  uint32_t seq = plan.find(at, &before);
  const uint32_t rest = at - before * plan.blocks;
  Span sp = plan.span(seq);
  uint32_t length = P::rounds(sp);
  uint32_t hb = uniform(rest / length), pos = rest - hb * length;
  DecodeOf<D, F, RT, C, WH, waves(RT)> decode(a, smem);
  while (true) {
    const uint32_t stop = min(length, pos + (end - at));
    const uint32_t tile = P::kStep * (max(pos, P::kSetup) - P::kSetup);
    const uint32_t tile_end = min(sp.tiles, P::kStep * (max(stop, P::kSetup) - P::kSetup));
    // begun before this run: place 0; begun in it and going on: place 1
    if (tile < tile_end)
      decode.run(seq, hb * WH, sp, tile, tile_end - tile, tile == 0u ? 1u : 0u);
    at += stop - pos;
    if (at >= end) return;
    pos = 0u;
    if (++hb == plan.blocks) {
      hb = 0u;
      sp = plan.span(++seq);
      length = P::rounds(sp);
    }
  }
}

// Query rows blockIdx.y * ROWS .. of a sequence and block (or WH heads): the sums
// that the runs over it left, if it took more than one: place 1 of the run that
// began it and place 0 of the runs that follow, in order.  D / 4 threads cover a
// row; the threads that ROWS rows leave over take every kWays-th part.  blockIdx.x
// is the head, or with by_runs the run that began it: of more heads than runs,
// most lie within one (4096 sequences of 1 to 200 keys, 8 heads: 12 us; 213 over
// the heads, counted 64 by 64).  Bound by latency: the lengths, then the parts (4.6 us after 64
// sequences, 6 us for the 256 parts of one).
template <int D, int RT, int WH, uint32_t KEYS, int ROWS, int THREADS>
__global__ void __launch_bounds__(THREADS) paged_join_kernel(Args a, bool by_runs) {
  using P = Plan<RT, WH, KEYS>;
  constexpr uint32_t kQuads = D / 4u, kWays = THREADS / (kQuads * ROWS);
  constexpr uint32_t kShared = kWays > 1u ? THREADS / 64u * kQuads * ROWS : 1u;
  __shared__ f32x4_t part_sum[kShared];
  __shared__ float2 part_stat[kShared];
  const P plan(a);
  const uint32_t quad = threadIdx.x % kQuads, d = 4u * quad;
  const uint32_t r = threadIdx.x / kQuads % ROWS, way = threadIdx.x / (kQuads * ROWS);
  const uint32_t row = blockIdx.y * ROWS + r;  // one head's behind another's
  // by_runs: the head that the next run starts in
  const uint32_t next = (blockIdx.x + 1u) * plan.run;
  if (by_runs && next >= plan.total) return;
  uint32_t before, seq;
  if (by_runs) seq = plan.find(next, &before);
  else before = plan.before(seq = uniform(blockIdx.x / plan.blocks));
  const uint32_t length = P::rounds(plan.span(seq));
  const uint32_t hb = by_runs ? uniform((next - before * plan.blocks) / length)
                              : blockIdx.x - seq * plan.blocks;
  const uint32_t start = before * plan.blocks + hb * length;
  const uint32_t first = uniform((start + P::kSetup) / plan.run);
  const uint32_t parts = uniform((start + length - 1u) / plan.run) - first + 1u;
  if (parts == 1u || (by_runs && first != blockIdx.x)) return;
  float m = -__FLT_MAX__, l = 0.0f;
  f32x4_t y = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float2 s, f32x4_t x) {
    const float top = fmaxf(m, s.x);
    const float old = __builtin_amdgcn_exp2f(m - top);
    const float weight = __builtin_amdgcn_exp2f(s.x - top);
    m = top;
    l = l * old + weight * s.y;
    y = y * old + weight * x;
  };
#pragma unroll 4
  for (uint32_t i = way; i < parts; i += kWays) {
    const uint64_t p = ((uint64_t)(first + i) * 2u + (i == 0u ? 1u : 0u)) * WH * a.rows +
                       min(row, WH * a.rows - 1u);
    add(*reinterpret_cast<const float2*>(a.stats + p * 2u),
        *reinterpret_cast<const f32x4_t*>(a.sums + p * D + d));
  }
  if constexpr (kWays > 1u) {
    // a wave's ways by lane exchanges, then the waves' sums: largest first, so that
    // no addition waits for another's exponential
    constexpr uint32_t kRowLanes = kQuads * ROWS, kAll = THREADS / 64;
#pragma unroll
    for (uint32_t o = kRowLanes; o < 64u; o <<= 1) {
      const float2 s = {__shfl_xor(m, o, 64), __shfl_xor(l, o, 64)};
      f32x4_t x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __shfl_xor(y[e], o, 64);
      add(s, x);
    }
    const uint32_t lane = threadIdx.x & 63u;
    if (lane < kRowLanes) {
      part_sum[threadIdx.x / 64u * kRowLanes + lane] = y;
      part_stat[threadIdx.x / 64u * kRowLanes + lane] = float2{m, l};
    }
    __syncthreads();
    if (way == 0u) {
#pragma unroll
      for (uint32_t w = 1; w < kAll; ++w) m = fmaxf(m, part_stat[w * kRowLanes + lane].x);
      l = 0.0f;
      y = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (uint32_t w = 0; w < kAll; ++w) {
        const float2 s = part_stat[w * kRowLanes + lane];
        const float weight = __builtin_amdgcn_exp2f(s.x - m);
        l += weight * s.y;
        y += weight * part_sum[w * kRowLanes + lane];
      }
    }
  }
  uint32_t q_head;
  bool has = way == 0u && row < WH * a.rows;
  if constexpr (WH > 1) {  // a.rows is the group
    q_head = hb * WH * a.group + row;
  } else {
    const uint32_t head = hb / a.blocks_per_head, block = hb - head * a.blocks_per_head;
    has = has && block * kBlockRows + row < a.group;
    q_head = head * a.group + block * kBlockRows + row;
  }
  if (!has) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const uint64_t out = (uint64_t)seq * a.q_heads + q_head;
  *reinterpret_cast<u32x2_t*>(a.o + out * D + d) =
      u32x2_t{pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv)};
  if (a.lse != nullptr && d == 0u)
    a.lse[out] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
}

template <int D, uint32_t F, int RT, int C, int WH>
int32_t launch_split(Args a, uint64_t tiles, uint32_t cus, hipStream_t s) {
  constexpr uint32_t kSmem = LdsOf<D, F, RT, waves(RT)>::kBytes;
  constexpr uint32_t kTileKeys = keys_of<F, RT>();
  using P = Plan<RT, WH, kTileKeys>;
  const auto fn = paged_split_kernel<D, F, RT, C, WH>;
  static const int32_t lds_rc = fe2o3_host::set_dynamic_lds({(const void*)fn}, (int)kSmem);
  if (lds_rc != FE2O3_OK) return lds_rc;
  // as many workgroups as are resident at once, and work for each wave
  const uint32_t heads = a.seqs * a.cache.kv_heads * a.blocks_per_head / WH;
  const uint64_t most = heads * ((tiles + P::kStep - 1u) / P::kStep + P::kSetup);
  uint32_t workgroups = per_cu<D, F, RT, C>() * cus;
  if (workgroups > kMaxWorkgroups) workgroups = kMaxWorkgroups;
  if (workgroups > most) workgroups = (uint32_t)most;
  a.workgroups = workgroups;
  fn<<<workgroups, waves(RT) * 64u, kSmem, s>>>(a);
  const int32_t rc = fe2o3_host::after_launch();
  if (rc != FE2O3_OK) return rc;
  // Many heads have few parts each, and rows share the threads; few have many,
  // which a row's threads share.  us of the join with 512 workgroups; rows share from
  // 64 heads on, 1024 threads take a row below 8 (rows sharing, 256, 1024 threads a row):
  //   2 heads, 16 rows 28, 6.0, 5.8     2 x 64 rows 31, 7.2, 6.2    6 x 16 12, 4.6, 4.6
  //   8 x 16            9.0, 4.6, 4.5   16 x 64      7.0, 5.7, 8.6  32 x 64 4.9, 5.4, 13
  //   60 x 64           5.2, 7.7, 21    128 x 16     4.5, 6.2, 17   256 x 16 4.5, 9.8, 31
  constexpr int kRows = kThreads / (D / 4);
  const uint32_t rows = WH * a.rows;
  const bool by_runs = heads > workgroups;
  const uint32_t grid = by_runs ? workgroups : heads;
  if (heads >= workgroups / 8u)
    paged_join_kernel<D, RT, WH, kTileKeys, kRows, kThreads>
        <<<dim3(grid, (rows - 1u) / kRows + 1u), kThreads, 0, s>>>(a, by_runs);
  else if (heads >= workgroups / 64u)
    paged_join_kernel<D, RT, WH, kTileKeys, 1, kThreads>
        <<<dim3(grid, rows), kThreads, 0, s>>>(a, by_runs);
  else
    paged_join_kernel<D, RT, WH, kTileKeys, 1, 1024><<<dim3(grid, rows), 1024, 0, s>>>(a, by_runs);
  return fe2o3_host::after_launch();
}

template <int D, uint32_t F, int RT, int C, uint32_t W>
int32_t launch_whole(const Args& a, hipStream_t s) {
  constexpr uint32_t kSmem = LdsOf<D, F, RT, W>::kBytes;
  const auto fn = paged_whole_kernel<D, F, RT, C, W>;
  static const int32_t lds_rc = fe2o3_host::set_dynamic_lds({(const void*)fn}, (int)kSmem);
  if (lds_rc != FE2O3_OK) return lds_rc;
  const uint32_t heads = a.seqs * a.cache.kv_heads * a.blocks_per_head;
  const kv_cache::Grid grid = kv_cache::Grid::of(heads);
  fn<<<dim3(grid.x, grid.y), W * 64u, kSmem, s>>>(a);
  return fe2o3_host::after_launch();
}

// Tiles of the longest span that a call may have.
uint64_t most_tiles(const Args& a, uint32_t keys) {
  if (a.window != 0u && a.window < a.max_length) return ((uint64_t)a.window + keys - 1u) / keys + 1u;
  return ((uint64_t)a.max_length + keys - 1u) / keys;
}

template <int D, uint32_t F, int RT, int C>
int32_t launch(const Args& a, uint32_t cus, hipStream_t s) {
  const uint64_t tiles = most_tiles(a, keys_of<F, RT>());
  const uint64_t heads = (uint64_t)a.seqs * a.cache.kv_heads * a.blocks_per_head;
  // Whether one workgroup a head is enough, without a plan and a join: rounds of
  // tiles on the busiest wave, against an even share of them plus two rounds for
  // the join, for heads of few tiles (us, even shares against one a head; 8 KV
  // heads of 128, bf16):
  //   1 x 500  9.4,  7.7    16 x 500  16.0, 10.8    30 x 500  18.9, 13.4
  //   64 x 500 29.6, 23.5   200 x 500 75.7, 68.6    64 x 1..1000 28.8 (one a head)
  //   1 x 1000 9.7, 14.8    4 x 1000  12.1, 15.7    16 x 1000 20.8, 17.7
  //   64 x 1..2000 48.1, 55.2   30 x 1..2000 27.4, 30.1   40 windows of 1024
  //   (64 wide, e4m3) 16.8, 13.0
  // Past 40 tiles one a head would be up to 7% faster for equal lengths, but up to 20%
  // slower where they differ, which max_length does not tell:
  //   64 x 1300 59.4, 55.8    64 x 1600 72.0, 67.0    16 x 1300 22.4, 22.6
  //   64 x 1..1300 34.9, 37.0   64 x 1..2000 47.8, 55.0   64 x 1..3000 68.5, 81.3
  // Few heads take eight waves each.  More than one tile of query rows has more to
  // join, and a head its own rounds at least (48 rows, one KV head):
  //   48 x 170 14.0, 9.5    48 x 1000 16.4, 21.9    8 x 500   13.6, 13.1
  //   64 x 500 16.0, 14.2   200 x 500 24.6, 15.9    300 x 500 32.5, 29.0
  // 4-bit rows, tiles of 64 keys, in the same rounds (8 KV heads of 128 in token order):
  //   1 x 500   8.5,  6.5   1 x 2000   8.7, 13.6    4 x 2000  10.2, 13.7
  //   16 x 2000 17.7, 14.7  64 x 500  18.1, 11.0    64 x 2000 35.3, 28.8
  //   200 x 500 32.6, 25.5  64 x 1..2000 24.4, 22.6 30 x 1..2000 18.0, 14.6
  //   8 x 3000  17.0, 18.3  64 x 1..4000 36.3, 38.6 64 x 1000 (64 wide) 16.9, 10.7
  const uint32_t resident = (per_cu<D, F, RT, C>() == 1 ? 1u : 2u) * cus;
  const bool wide = RT == 1 && heads <= cus;
  const uint64_t rounds_whole =
      wide ? (tiles + 7u) / 8u : ((tiles + 3u) / 4u * heads + resident - 1u) / resident;
  const uint64_t rounds_split = (heads * tiles + 4u * resident - 1u) / (4u * resident);
  const uint64_t least = RT == 1 ? 0u : (tiles + 3u) / 4u;  // of one head
  if (tiles <= kWholeTiles && (rounds_whole > least ? rounds_whole : least) <=
                                  rounds_split + (RT == 1 ? 2u : 4u)) {
    if constexpr (RT == 1)
      if (wide && tiles > kWaves) return launch_whole<D, F, RT, C, 8>(a, s);
    return launch_whole<D, F, RT, C, waves(RT)>(a, s);
  }
  // Four heads a workgroup read neighbouring rows, but every part that the join adds
  // has the rows of four: worth it where a workgroup has six rounds at least (1 x 130001
  // 91.8, 88.7 with four; 4 x 16000 49.6, 47.7; 1 x 40000 34.5, 35.4; 8 x 1200..2400,
  // group 7: 17.7, 20.0; 1 x 17313 of 4 KV heads, group 16, e4m3: 15.5, 19.4).  4-bit rows
  // of four heads in token order are two lines, which single heads read twice: from two
  // rounds on (1 x 40000 23.8, 21.8; 4 x 16000 30.9, 24.2; 64 x 2000 50.3, 36.0; but 4 x
  // 2000 10.3, 11.3; 8 x 1200..2400, group 7: 13.5, 15.2).
  if constexpr (RT == 1)
    if (a.cache.kv_heads % kWaves == 0u &&
        heads / kWaves * tiles >= (F == kMxfp4 ? 2u : 6u) * resident)
      return launch_split<D, F, RT, C, kWaves>(a, tiles, cus, s);
  return launch_split<D, F, RT, C, 1>(a, tiles, cus, s);
}

template <int D, uint32_t F>
int32_t launch_rows(const Args& a, uint32_t cus, hipStream_t s) {
  if constexpr (F == kMxfp4) {
    if (a.rows <= 8u) return launch<D, F, 1, 2>(a, cus, s);
  }
  if (a.rows <= 16u) return launch<D, F, 1, 1>(a, cus, s);
  if (a.rows <= 32u) return launch<D, F, 2, 1>(a, cus, s);
  if (a.rows <= 48u) return launch<D, F, 3, 1>(a, cus, s);
  return launch<D, F, 4, 1>(a, cus, s);
}

#define FE2O3_KERNEL(NAME, FN, THREADS, LDS) \
  fe2o3_host::KernelRegistrar({"fe2o3_paged_attention_decode", NAME, (const void*)FN, THREADS, LDS})
#define FE2O3_SPLIT(D, F, RT, C, WH) \
  FE2O3_KERNEL("paged_split_kernel<" #D "," #F "," #RT "," #C "," #WH ">", (paged_split_kernel<D, F, RT, C, WH>), waves(RT) * 64u, (LdsOf<D, F, RT, waves(RT)>::kBytes))
#define FE2O3_WHOLE(D, F, RT, C, W) \
  FE2O3_KERNEL("paged_whole_kernel<" #D "," #F "," #RT "," #C "," #W ">", (paged_whole_kernel<D, F, RT, C, W>), (W) * 64u, (LdsOf<D, F, RT, W>::kBytes))
#define FE2O3_PAGED_ONE(D, F, C)                                                                \
  FE2O3_SPLIT(D, F, 1, C, 1), FE2O3_SPLIT(D, F, 1, C, 4), FE2O3_WHOLE(D, F, 1, C, 4),           \
  FE2O3_WHOLE(D, F, 1, C, 8)
#define FE2O3_PAGED_ALL(D, F)                                                                   \
  FE2O3_PAGED_ONE(D, F, 1), FE2O3_SPLIT(D, F, 2, 1, 1), FE2O3_SPLIT(D, F, 3, 1, 1),             \
  FE2O3_SPLIT(D, F, 4, 1, 1), FE2O3_WHOLE(D, F, 2, 1, waves(2)),                                \
  FE2O3_WHOLE(D, F, 3, 1, waves(3)), FE2O3_WHOLE(D, F, 4, 1, waves(4))
#define FE2O3_JOIN_OF(D, RT, WH, KEYS, ROWS, THREADS)                                           \
  fe2o3_host::KernelRegistrar({"fe2o3_paged_attention_decode", "paged_join_kernel<" #D "," #RT "," #WH "," #KEYS "," #ROWS ">", (const void*)paged_join_kernel<D, RT, WH, KEYS, ROWS, THREADS>, THREADS, 0})
#define FE2O3_JOIN(D, RT, WH, KEYS, ROWS) \
  FE2O3_JOIN_OF(D, RT, WH, KEYS, ROWS, kThreads), FE2O3_JOIN_OF(D, RT, WH, KEYS, 1, kThreads), \
  FE2O3_JOIN_OF(D, RT, WH, KEYS, 1, 1024)
#define FE2O3_JOIN_ALL(D, ROWS) \
  FE2O3_JOIN(D, 1, 1, 32, ROWS), FE2O3_JOIN(D, 1, 4, 32, ROWS), FE2O3_JOIN(D, 2, 1, 32, ROWS), \
  FE2O3_JOIN(D, 3, 1, 32, ROWS), FE2O3_JOIN(D, 4, 1, 32, ROWS), FE2O3_JOIN(D, 1, 1, 64, ROWS), \
  FE2O3_JOIN(D, 1, 4, 64, ROWS)
const fe2o3_host::KernelRegistrar kRegistered[] = {
    FE2O3_PAGED_ALL(64, kBf16),       FE2O3_PAGED_ALL(64, kE4m3),
    FE2O3_PAGED_ALL(64, kMxfp4),      FE2O3_PAGED_ONE(64, kMxfp4, 2),
    FE2O3_PAGED_ALL(128, kBf16),
    FE2O3_PAGED_ALL(128, kE4m3),      FE2O3_PAGED_ALL(128, kMxfp4),
    FE2O3_PAGED_ONE(128, kMxfp4, 2),
    FE2O3_JOIN_ALL(64, 16),           FE2O3_JOIN_ALL(128, 8)};
#undef FE2O3_KERNEL
#undef FE2O3_SPLIT
#undef FE2O3_PAGED_ALL
#undef FE2O3_PAGED_ONE
#undef FE2O3_WHOLE
#undef FE2O3_JOIN
#undef FE2O3_JOIN_OF
#undef FE2O3_JOIN_ALL

}  // namespace

extern "C" int32_t fe2o3_paged_attention_decode(
    const Fe2o3KvCacheV1* cache, const uint16_t* q, uint64_t q_len, const uint32_t* block_table,
    uint64_t table_len, const uint32_t* lengths, uint64_t lengths_len, uint16_t* o, uint64_t o_len,
    float* lse, uint64_t lse_len, void* workspace, uint64_t workspace_bytes, uint32_t seqs,
    uint32_t q_heads, uint32_t table_cols, uint32_t max_length, uint64_t q_stride,
    uint32_t window, float scale, void* stream) {
  FE2O3_ENTRY("fe2o3_paged_attention_decode");
  Args a;
  int32_t rc = kv_cache::check(cache, &a.cache);
  if (rc != FE2O3_OK) return rc;
  const uint32_t d = cache->head_dim, kv_heads = cache->kv_heads;
  if (d != 64u && d != 128u) return FE2O3_ERR_SHAPE;
  if (q_heads == 0u || q_heads % kv_heads != 0u) return FE2O3_ERR_SHAPE;
  if (max_length >= (1u << 31) || max_length > (uint64_t)table_cols * cache->page_size)
    return FE2O3_ERR_SHAPE;
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(scale > 0.0f) || !__builtin_isfinite(scale_log2)) return FE2O3_ERR_SHAPE;
  const uint32_t group = q_heads / kv_heads;
  const uint32_t blocks_per_head = (group - 1u) / kBlockRows + 1u;
  const uint64_t row = (uint64_t)q_heads * d;
  // every product below is of factors that keep it under 2^64
  const uint64_t blocks = (uint64_t)kv_heads * blocks_per_head;  // at most q_heads
  uint64_t tiles = ((uint64_t)max_length + kKeys - 1u) / kKeys;
  if (window != 0u && window < max_length) tiles = ((uint64_t)window + kKeys - 1u) / kKeys + 1u;
  // rounds of the plan, a head's start among them, and what a grid adds
  const uint64_t most = blocks * (tiles + 2u * kWaves);
  if (most >= (UINT64_C(1) << 31) || seqs * most >= (UINT64_C(1) << 31)) return FE2O3_ERR_SHAPE;
  if (seqs > 1u && q_stride < row) return FE2O3_ERR_STRIDE;
  if (seqs == 0u) return FE2O3_OK;
  uint64_t extent = row, bytes;
  if (!kv_cache::reach(seqs, q_stride, &extent) || !kv_cache::mul_ok(extent, 2u, &bytes))
    return FE2O3_ERR_OVERFLOW;
  const uint64_t heads = (uint64_t)seqs * q_heads;
  uint64_t o_need;
  if (!kv_cache::mul_ok(heads, d, &o_need)) return FE2O3_ERR_OVERFLOW;
  if (q_len < extent || table_len != (uint64_t)seqs * table_cols || lengths_len != seqs ||
      o_len != o_need || (lse != nullptr && lse_len != heads))
    return FE2O3_ERR_LENGTH;
  if (!q || (table_len != 0u && !block_table) || !lengths || !o || !workspace)
    return FE2O3_ERR_NULL;
  if (!kv_cache::rows_aligned(a.cache, cache->format, 16u) ||
      (((uintptr_t)q | (uintptr_t)o | (uintptr_t)workspace) & 15u) != 0u ||
      (seqs > 1u && q_stride % 8u != 0u) ||
      (((uintptr_t)lse | (uintptr_t)block_table | (uintptr_t)lengths) & 3u) != 0u)
    return FE2O3_ERR_ALIGNMENT;
  // DecodeBlocks has rows' numbers, and their places in 16 bytes, in 32 bits
  if (cache->format == kMxfp4) {
    uint64_t last = 0, n;
    if (!kv_cache::reach(a.cache.pages, a.cache.page_stride, &last) ||
        !kv_cache::reach(cache->page_size, a.cache.token_stride, &last) ||
        last >= (UINT64_C(1) << 36) ||
        !kv_cache::mul_ok((uint64_t)cache->pages * cache->page_size, kv_heads, &n) ||
        n >= (UINT64_C(1) << 32))
      return FE2O3_ERR_SHAPE;
  }
  if (workspace_bytes < FE2O3_PAGED_ATTENTION_WORKSPACE_BYTES(q_heads, kv_heads, d))
    return FE2O3_ERR_WORKSPACE;
  tile_plan::Topology topo;
  rc = fe2o3_host::device_topology(&topo);
  if (rc != FE2O3_OK) return rc;
  a.q = q;
  a.table = block_table;
  a.lengths = lengths;
  a.o = o;
  a.lse = lse;
  a.rows = group < kBlockRows ? group : kBlockRows;
  const uint32_t part_rows = FE2O3_PAGED_ATTENTION_PART_ROWS(q_heads, kv_heads);
  a.sums = (float*)workspace;
  a.stats = a.sums + (uint64_t)kMaxWorkgroups * 2u * part_rows * d;
  a.q_stride = q_stride;
  a.seqs = seqs;
  a.q_heads = q_heads;
  a.group = group;
  a.blocks_per_head = blocks_per_head;
  a.table_cols = table_cols;
  a.max_length = max_length;
  a.window = window;
  a.scale_log2 = scale_log2;
  a.xcds = topo.xcds ? topo.xcds : 1u;
  hipStream_t s = (hipStream_t)stream;
  switch (cache->format) {
    case kE4m3:
      return d == 64u ? launch_rows<64, kE4m3>(a, topo.cus, s)
                      : launch_rows<128, kE4m3>(a, topo.cus, s);
    case kMxfp4:
      return d == 64u ? launch_rows<64, kMxfp4>(a, topo.cus, s)
                      : launch_rows<128, kMxfp4>(a, topo.cus, s);
    default:
      return d == 64u ? launch_rows<64, kBf16>(a, topo.cus, s)
                      : launch_rows<128, kBf16>(a, topo.cus, s);
  }
}
