// gemm_mxfp4.hip -- C (bf16) = A B^T of two packed microscaled 4-bit matrices
// (mxfp4.hpp), with fp32 accumulation, for gfx950.
//
// One v_mfma_scale_f32_16x16x128_f8f6f4 takes 128 k of e2m1 codes of 16 rows of each
// operand, four blocks a row, with their scales: lane l holds the 32 codes of block l / 16
// of row l % 16, and a byte of its scale register is that block's scale.  The matrix
// core multiplies by both scales, so the epilogue only rounds.
//
// The tile is the bf16 GEMM's (gemm_pipe.hpp): a panel of 256 k is 128 bytes a row, the
// bytes of 64 bf16, and an MFMA takes the same 16 bytes a lane, so that the copies into
// LDS, their swizzle and the fragment reads are its, with four times the work in each
// MFMA.  What is added is the scales: a stage's are 8 bytes a row, contiguous for the
// tile's rows (2 KiB for 256), copied behind the stage's codes.  A lane reads a row's
// eight with one ds_read_b64 and keeps its block's of both substeps in one register.
//
// Measured: 8192 x 8192 x 8192 210-237 us in calls and replays = 4.6-5.2 PFLOP/s, by the card
// and its power (median of a traced run 242).  The instruction alone, from registers, sustains
// 6.3-7.4 by the card on codes of normal values, where power limits it, and 9.6 on zeros, on
// which this kernel takes 169-176 us: three quarters of it in the loop
// either way (8192 k more take 198 us of 149, on zeros 151 of 114), and 4 us a round of tiles
// besides.  The loop waits for its copies: waves spend 19% of their time at the wait and the
// barrier for the next stage, of which LDS holds two (68 KiB each), and 25% waiting to issue.
// LDS is no limit: busy 21%, no conflicts, and without the reads of scales 207-209 us for 213.
// 16 x 14336 x 4096 9.0 us with the weights from memory (3.5 TB/s), 5.6 from the caches;
// 4096 x 4096 x 4096 33-38.
//
// A tile's steps follow one another, so that few tiles take the steps' time whatever their
// number: 128 and 256 rows by 8192 x 8192 24 us (64 and 128 workgroups of 32 steps of 0.58 us,
// 0.2 of it products), from the caches 18; 512 rows 25 (0.8 a step).
#include "common.hpp"
#include "gemm_core.hpp"
#include "gemm_direct.hpp"
#include "gemm_pipe.hpp"
#include "internal.hpp"
#include "mxfp4.hpp"

#include <type_traits>

namespace {

using namespace fe2o3;
using gemm_pipe::Acc16T;
using gemm_pipe::CopyOrder;
using gemm_pipe::Geo;
using gemm_pipe::Spread;

constexpr int kRow = 128;            // bytes of a row's codes in a stage
constexpr uint32_t kK16 = kRow / 2;  // 16-bit units
using G = Geo<kRow>;

// The scales of an operand's tile rows: 8 bytes a row of a panel, panels `step` bytes
// apart, `bytes` of them in the tile's rows.  Rows past them load zeros (2^-127); their
// products reach no stored output.
struct ScaleRows {
  const uint8_t* base;
  uint64_t step;
  uint32_t bytes;
};

// Stage t of a tile: where the codes of its rows begin, and the scales that this wave copies.
struct From {
  const uint8_t *a, *b, *scales;
  uint32_t t;
  FE2O3_DEVICE From stage(uint32_t to) const {
    return From{a, b, scales, (uint32_t)__builtin_amdgcn_readfirstlane(to)};
  }
};

// A tile of 32 RB rows of A by 32 CB rows of B: four waves, 2 x 2, of RB x CB MFMA tiles.
// EVEN: no row is clamped, so that a wave's copies lie 32 rows apart.
template <int RB, int CB, int STAGES, bool EVEN = false>
struct Tile {
  static constexpr int kMfma = RB * CB;  // per substep of 128 k
  static constexpr int kARows = 32 * RB, kBRows = 32 * CB;
  static constexpr int NA = G::insts(kARows), NB = G::insts(kBRows);
  static constexpr int NC = NA + NB + 1;  // copies per stage and wave: codes, then scales
  using L = gemm_pipe::Lay<kRow, STAGES, kARows, kBRows * kRow>;
  static constexpr uint32_t kScaleTile = (kARows + kBRows) * 8u;
  static constexpr uint32_t kScaleRegion = L::b_region + STAGES * kBRows * kRow;
  static constexpr uint32_t kSmem = kScaleRegion + STAGES * kScaleTile;
  static_assert(RB == CB, "a wave copies a quarter of the scales, of one operand");
  using RowsT = gemm_pipe::Rows<kRow, NA>;
  using Acc = Acc16T<RB, CB>;

  struct Frags {
    i32x4_t a[RB], b[CB];
  };
  // byte h: the scale of the lane's block in substep h
  struct Scales {
    uint32_t a[RB], b[CB];
  };
  struct Lanes {
    uint32_t a[2], b[2];  // per substep; a row's swizzle repeats every 8 rows
    uint32_t sa, sb;
    uint32_t pick;
  };

  const RowsT& ar;
  const RowsT& br;
  const ScaleRows own;  // of the operand that this wave copies
  uint8_t* smem;
  const uint32_t wave, steps;
  Lanes ln;

  FE2O3_DEVICE Tile(const RowsT& a, const RowsT& b, const ScaleRows& sa, const ScaleRows& sb,
                    uint32_t panels, uint8_t* lds)
      : ar(a), br(b), own(gemm_pipe::wave_id() < 2u ? sa : sb), smem(lds),
        wave(gemm_pipe::wave_id()), steps(panels) {
    const uint32_t lane = threadIdx.x & 63u, lr = lane & 15u, g = lane >> 4;
    const uint32_t ra = (wave >> 1) * 16u * RB + lr, rb = (wave & 1u) * 16u * CB + lr;
#pragma unroll
    for (uint32_t s = 0; s < 2u; ++s) {
      ln.a[s] = ra * kRow + (((4u * s + g) ^ G::swz(ra)) << 4);
      ln.b[s] = L::b_region + rb * kRow + (((4u * s + g) ^ G::swz(rb)) << 4);
    }
    ln.sa = kScaleRegion + ra * 8u;
    ln.sb = kScaleRegion + (kARows + rb) * 8u;
    ln.pick = 0x0c0c0400u + g * 0x0101u;  // bytes g and 4 + g, zeros above
  }

  FE2O3_DEVICE From tile() const {  // the one that the rows were made for
    return From{(const uint8_t*)ar.base[0], (const uint8_t*)br.base[0], own.base, 0u};
  }
  FE2O3_DEVICE From at(const From& from, uint32_t t) const {  // clamped to the last
    return from.stage(t < steps ? t : steps - 1u);
  }

  template <int J>
  FE2O3_DEVICE uint32_t at_row(const From& from) const {
    return from.t * (uint32_t)kRow + (EVEN ? J * 32u * kRow * steps : 0u);
  }
  // copy C of a stage into buffer buf: B's codes, the scales, then A's codes
  template <int C>
  FE2O3_DEVICE void copy(const From& from, int buf) const {
    if constexpr (C < NB) {
      gemm_pipe::b2l_b128(gemm_pipe::rsrc(from.b, br.bytes),
                          smem + L::b_region + L::b(buf) + (4u * C + wave) * 1024u,
                          br.voff[EVEN ? 0 : C], at_row<C>(from));
    } else if constexpr (C == NB) {
      // a quarter of the tile's scales, 16 bytes a lane
      constexpr uint32_t kPart = kScaleTile / 4u;
      const uint32_t lane = threadIdx.x & 63u;
      if (kPart == 1024u || lane < kPart / 16u)
        gemm_pipe::b2l_b128(gemm_pipe::rsrc(from.scales + from.t * own.step, own.bytes),
                            smem + kScaleRegion + buf * kScaleTile + wave * kPart,
                            (wave & 1u) * kPart + lane * 16u, 0u);
    } else {
      constexpr int j = C - NB - 1;
      gemm_pipe::b2l_b128(gemm_pipe::rsrc(from.a, ar.bytes),
                          smem + L::a(buf) + (4u * j + wave) * 1024u, ar.voff[EVEN ? 0 : j],
                          at_row<j>(from));
    }
  }

  // read unit R of substep S in buffer P, in the order the MFMAs use them
  static constexpr int kReads = RB + CB;
  template <int P, int S, int R>
  FE2O3_DEVICE void read(Frags& f) const {
    if constexpr (R >= 1 && R <= CB) {
      constexpr int j = R - 1;
      f.b[j] = *reinterpret_cast<const i32x4_t*>(smem + ln.b[S] + (L::b(P) + j * 16u * kRow));
    } else {
      constexpr int i = R == 0 ? 0 : R - CB;
      f.a[i] = *reinterpret_cast<const i32x4_t*>(smem + ln.a[S] + (L::a(P) + i * 16u * kRow));
    }
  }
  // A row's eight scales of buffer P, then the lane's two of them: apart, so that no
  // permute waits for its read.
  template <int P, int R>
  FE2O3_DEVICE void read_scale(u32x2_t (&raw)[kReads]) const {
    constexpr bool is_b = R >= 1 && R <= CB;
    constexpr int block = is_b ? R - 1 : R == 0 ? 0 : R - CB;
    raw[R] = *reinterpret_cast<const u32x2_t*>(smem + (is_b ? ln.sb : ln.sa) +
                                               (P * kScaleTile + block * 128u));
  }
  template <int R>
  FE2O3_DEVICE void pick_scale(const u32x2_t (&raw)[kReads], Scales& s) const {
    uint32_t& to = R >= 1 && R <= CB ? s.b[R - 1] : s.a[R == 0 ? 0 : R - CB];
    to = __builtin_amdgcn_perm(raw[R][1], raw[R][0], ln.pick);
    asm volatile("" : "+v"(to));  // here: moved to its use, it would be too near (mfma)
  }

  // Inline asm with the accumulator tied to the destination, as gemm_pipe::Bf16Mma's, and
  // for its reason.  What the compiler then does not provide: the accumulators are
  // zeroed before the first copies are waited for, scale registers are written at least
  // two MFMAs before their first use, and finish() waits before the epilogue reads.
  template <int S, int I, bool ZERO>
  static FE2O3_DEVICE void mfma(Acc& acc, const Frags& f, const Scales& s) {
    constexpr int i = I / CB, j = I % CB;
    if constexpr (ZERO && S == 0)  // a sum's first
      asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 "
                   "op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                   : "=a"(acc.v[i][j]) : "v"(f.b[j]), "v"(f.a[i]), "v"(s.b[j]), "v"(s.a[i]));
    else if constexpr (S == 0)
      asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 "
                   "op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                   : "+a"(acc.v[i][j]) : "v"(f.b[j]), "v"(f.a[i]), "v"(s.b[j]), "v"(s.a[i]));
    else
      asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 "
                   "op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                   : "+a"(acc.v[i][j]) : "v"(f.b[j]), "v"(f.a[i]), "v"(s.b[j]), "v"(s.a[i]));
  }
  static FE2O3_DEVICE void pin(Acc& acc) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) asm volatile("" : "+a"(acc.v[i][j]));
  }

  // Slot I of substep S of step t, held in buffer P (gemm_pipe's schedule): substep 0
  // reads its substep 1's fragments and copies the rest of stage t + STAGES - 1;
  // substep 1 waits for stage t + 1 halfway, then reads its first fragments and scales,
  // and starts the first copies of stage t + STAGES into buffer P.
  static constexpr int kEarly = NB + 1, kLate = NA;
  static constexpr int kBarrier = kMfma / 2;
  static constexpr int kPickFrom = kBarrier + kMfma / 8;
  // KIND, of tiles one after another (run_all): a tile's first step finds stage 1 copied
  // before the last tile's stores, which it does not wait for, and starts the sums; its last
  // step copies all of the next tile's stage 1.
  static constexpr int kFirst = 1, kLast = 2;
  static constexpr int kStores = RB * CB / 2;  // at least, of a wave's outputs, 16 bytes a lane
  template <int P, int S, int KIND, int I = 0>
  FE2O3_DEVICE void slots(const From& next, const From& next2, Frags (&f)[2], const Scales& now,
                          Scales& then, u32x2_t (&raw)[kReads], Acc& acc) const {
    if constexpr (I < kMfma) {
      if constexpr (S == 1 && I == kBarrier) {
        __builtin_amdgcn_s_waitcnt(
            gemm_pipe::waitcnt_imm((KIND & kFirst) != 0 ? kStores : (STAGES - 2) * NC, 0));
        __builtin_amdgcn_s_barrier();
      }
      mfma<S, I, (KIND & kFirst) != 0>(acc, f[S], now);
      if constexpr (S == 1) {
        Spread<(KIND & kLast) != 0 ? NC : kEarly, kBarrier, kMfma>::template at<I>(
            [&](auto n) { copy<decltype(n)::value>(next2, P); });
        Spread<kReads, kBarrier, kMfma>::template at<I>([&](auto n) {
          constexpr int PN = (P + 1) % STAGES;
          read_scale<PN, decltype(n)::value>(raw);
          read<PN, 0, decltype(n)::value>(f[0]);
        });
        Spread<kReads, kPickFrom, kMfma>::template at<I>(
            [&](auto n) { pick_scale<decltype(n)::value>(raw, then); });
      } else {
        if constexpr ((KIND & kFirst) == 0)
          Spread<kLate, 0, kMfma>::template at<I>([&](auto n) {
            copy<kEarly + decltype(n)::value>(next, (P + STAGES - 1) % STAGES);
          });
        Spread<kReads, kMfma / 8, kMfma - kMfma / 8>::template at<I>(
            [&](auto n) { read<P, 1, decltype(n)::value>(f[1]); });
      }
      __builtin_amdgcn_sched_barrier(0);
      slots<P, S, KIND, I + 1>(next, next2, f, now, then, raw, acc);
    }
  }
  // Steps t .. of a round, U of kRound: buffers and the two sets of scale registers
  // alternate by U, so that no register is copied.
  static constexpr int kRound = STAGES % 2 == 0 ? STAGES : 2 * STAGES;
  template <int U, bool TAIL>
  FE2O3_DEVICE void step(const From& from, uint32_t t, Frags (&f)[2], Scales (&s)[2],
                         Acc& acc) const {
    if (TAIL && t >= steps) return;
    const From next = at(from, t + STAGES - 1), next2 = at(from, t + STAGES);
    u32x2_t raw[kReads];
    __builtin_amdgcn_sched_barrier(0);
    slots<U % STAGES, 0, 0>(next, next2, f, s[U & 1], s[~U & 1], raw, acc);
    slots<U % STAGES, 1, 0>(next, next2, f, s[U & 1], s[~U & 1], raw, acc);
    if constexpr (U + 1 < kRound) step<U + 1, TAIL>(from, t + 1u, f, s, acc);
  }
  // Steps t and t + 1 of a tile with two stages, `then` being the next one (or it).
  template <int KIND>
  FE2O3_DEVICE void pair(const From& from, const From& then, uint32_t t, Frags (&f)[2],
                         Scales (&s)[2], Acc& acc) const {
    static_assert(STAGES == 2, "a buffer a step");
    constexpr bool kEnd = (KIND & kLast) != 0;
    const From one = from.stage(t + 1u);
    const From two = kEnd ? then.stage(0u) : from.stage(t + 2u);
    const From three = kEnd ? then.stage(1u) : from.stage(t + 3u);
    u32x2_t raw[kReads];
    __builtin_amdgcn_sched_barrier(0);
    slots<0, 0, KIND & kFirst>(one, two, f, s[0], s[1], raw, acc);
    slots<0, 1, KIND & kFirst>(one, two, f, s[0], s[1], raw, acc);
    slots<1, 0, KIND & kLast>(two, three, f, s[1], s[0], raw, acc);
    slots<1, 1, KIND & kLast>(two, three, f, s[1], s[0], raw, acc);
  }
  template <int C, int END>
  FE2O3_DEVICE void copies(const From& from, int buf) const {
    if constexpr (C < END) {
      copy<C>(from, buf);
      copies<C + 1, END>(from, buf);
    }
  }

  // step 0's fragments and scales; the copies of stage 0 have landed
  FE2O3_DEVICE void read_first(Frags (&f)[2], Scales (&s)[2]) const {
    u32x2_t raw[kReads];
    Spread<kReads, 0, 1>::template at<0>([&](auto n) { read_scale<0, decltype(n)::value>(raw); });
    Spread<kReads, 0, 1>::template at<0>([&](auto n) { pick_scale<decltype(n)::value>(raw, s[0]); });
    __builtin_amdgcn_sched_barrier(0);
    Spread<kReads, 0, 1>::template at<0>([&](auto n) { read<0, 0, decltype(n)::value>(f[0]); });
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
  // the last MFMA's result is written before the epilogue reads it
  FE2O3_DEVICE void finish(Acc& acc) const {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
    pin(acc);
    __builtin_amdgcn_sched_barrier(0);
  }

  FE2O3_DEVICE void run(Acc& acc) const {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) acc.v[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    pin(acc);
    const From from = tile();
#pragma unroll
    for (int st = 0; st + 1 < STAGES; ++st) copies<0, NC>(at(from, st), st);
    copies<0, kEarly>(at(from, STAGES - 1), STAGES - 1);
    __builtin_amdgcn_s_waitcnt(gemm_pipe::waitcnt_imm((STAGES - 2) * NC + kEarly, 0));
    __builtin_amdgcn_s_barrier();
    Frags f[2];
    Scales s[2];
    read_first(f, s);
    uint32_t t = 0;
    for (; t + kRound <= steps; t += kRound) step<0, false>(from, t, f, s, acc);
    if (t < steps) step<0, true>(from, t, f, s, acc);
    __builtin_amdgcn_sched_barrier(0);
    // copies past the last stage land before the workgroup's LDS is another's
    __builtin_amdgcn_s_waitcnt(gemm_pipe::kWaitVm0Lgkm0);
    finish(acc);
  }
  // Tiles one after another, of an even number of steps each: a tile's last steps copy the
  // first two stages of the next, which is under way while the sums are stored.
  // next(&from): whether there is one; store(acc): a tile's sums, kStores stores at least.
  template <class Next, class Store>
  FE2O3_DEVICE void run_all(From from, Next next, Store store) const {
    copies<0, NC>(from.stage(0u), 0);
    copies<0, NC>(from.stage(1u), 1);
    // all of both: the first step counts on stores behind them, of which there are none yet
    __builtin_amdgcn_s_waitcnt(gemm_pipe::kWaitVm0Lgkm0);
    __builtin_amdgcn_s_barrier();
    Frags f[2];
    Scales s[2];
    read_first(f, s);
    while (true) {
      From then = from;
      const bool more = next(&then);
      Acc acc;
      if (steps == 2u) {
        pair<kFirst | kLast>(from, then, 0u, f, s, acc);
      } else {
        pair<kFirst>(from, then, 0u, f, s, acc);
        for (uint32_t t = 2u; t + 2u < steps; t += 2u) pair<0>(from, then, t, f, s, acc);
        pair<kLast>(from, then, steps - 2u, f, s, acc);
      }
      finish(acc);
      store(acc);
      if (!more) break;
      from = then;
    }
    // copies of the tile that `then` was at the end
    __builtin_amdgcn_s_waitcnt(gemm_pipe::kWaitVm0Lgkm0);
  }
};

struct Operand {
  const uint8_t *codes, *scales;
  uint64_t scale_rows;
};

// Rows row0 .. row0 + valid - 1 of an operand for a tile of ROWS.
template <int ROWS>
FE2O3_DEVICE auto code_rows(const Operand& o, uint32_t row0, uint32_t valid, uint32_t panels) {
  const uint32_t k16 = panels * kK16;
  return gemm_pipe::dense_rows<kRow, ROWS>(
      reinterpret_cast<const uint16_t*>(o.codes + (uint64_t)row0 * panels * kRow), k16, valid, k16);
}
template <int ROWS>
FE2O3_DEVICE ScaleRows scale_rows(const Operand& o, uint32_t row0) {
  const uint64_t left = o.scale_rows - row0;
  return ScaleRows{o.scales + (uint64_t)row0 * 8u, o.scale_rows * 8u,
                   left < ROWS ? (uint32_t)left * 8u : ROWS * 8u};
}

using Big = Tile<8, 8, 2>;
template <int STAGES>
using Small = Tile<4, 4, STAGES>;

// 256 x 256 tiles.  STAGED and EDGE as the fp8 GEMM's (fp8.hip).
template <bool STAGED, bool EDGE>
__global__ void __launch_bounds__(256, 1) gemm_mxfp4_kernel(Operand a, Operand b,
                                                            uint16_t* __restrict__ c, uint32_t m,
                                                            uint32_t n, uint32_t panels,
                                                            uint32_t xcds) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  uint32_t tm, tn;
  gemm_core::xcd_tile_order(blockIdx.x, (m + 255u) / 256u, (n + 255u) / 256u, xcds, &tm, &tn);
  const uint32_t rows_a = EDGE ? min(256u, m - tm * 256u) : 256u;
  const uint32_t rows_b = EDGE ? min(256u, n - tn * 256u) : 256u;
  const auto ar = code_rows<256>(a, tm * 256u, rows_a, panels);
  const auto br = code_rows<256>(b, tn * 256u, rows_b, panels);
  const Big tile(ar, br, scale_rows<256>(a, tm * 256u), scale_rows<256>(b, tn * 256u), panels,
                 smem);
  const uint32_t wave = gemm_pipe::wave_id();
  Big::Acc acc;
  tile.run(acc);
  uint16_t* c_tile = c + (uint64_t)tm * 256 * n + (uint64_t)tn * 256;
  if constexpr (EDGE) gemm_pipe::store_bf16_edge(acc, c_tile, n, rows_a, rows_b, wave);
  else if constexpr (STAGED) gemm_pipe::store_bf16_staged(acc, smem, c_tile, n, wave);
  else gemm_pipe::store_bf16(acc, c_tile, n, wave);
}

// 256 x 256 tiles of the list entries blockIdx.x + i gridDim.x, one workgroup a CU.  A tile
// of its own costs 8 us besides its products: its start, its first loads from memory, its
// stores, which all tiles begin together, and the next workgroup's start.  Here the first
// stages of a tile arrive while the one before is stored, and the stores drain during the
// first steps (us, a workgroup a tile against this):
//   8192 x 8192 x 512 44.4, 38.0    x 1024 61.5, 51.5   x 2048 84.3, 75.6   x 4096 131.2, 123.0
//   x 8192 231.0, 221.9   x 16384 430.4, 418.9   5120 x 5120 x 4096 60.4, 59.1
//   4096 x 8192 x 4096 68.6, 63.7   16384 x 16384 x 4096 548, 520   6144 x 6144 x 1024 40.8, 38.8
// But where the stores go through LDS (staged_epilogue) they cannot overlap, and that is
// worth more: 1024 x 57344 x 8192 220, 226; 4096 x 57344 x 8192 786, 801.
// Whole tiles, an even number of panels.
__global__ void __launch_bounds__(256, 1) gemm_mxfp4_rounds_kernel(Operand a, Operand b,
                                                                   uint16_t* __restrict__ c,
                                                                   uint32_t m, uint32_t n,
                                                                   uint32_t panels, uint32_t xcds,
                                                                   uint32_t tiles) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t wave = gemm_pipe::wave_id();
  const Operand& own = wave < 2u ? a : b;
  uint32_t id = blockIdx.x, tm, tn;
  auto place = [&](From* from) {
    gemm_core::xcd_tile_order(id, m / 256u, n / 256u, xcds, &tm, &tn);
    const uint64_t row_a = tm * 256u, row_b = tn * 256u;
    from->a = a.codes + row_a * panels * kRow;
    from->b = b.codes + row_b * panels * kRow;
    from->scales = own.scales + (wave < 2u ? row_a : row_b) * 8u;
  };
  From from{};
  place(&from);
  const auto ar = code_rows<256>(a, 0u, 256u, panels), br = code_rows<256>(b, 0u, 256u, panels);
  const Tile<8, 8, 2, true> tile(ar, br, scale_rows<256>(a, 0u), scale_rows<256>(b, 0u), panels,
                                 smem);
  uint16_t* c_tile = c + (uint64_t)tm * 256u * n + (uint64_t)tn * 256u;
  tile.run_all(
      from,
      [&](From* to) {
        id += gridDim.x;
        if (id >= tiles) return false;
        place(to);
        return true;
      },
      [&](const Big::Acc& acc) {
        uint32_t ld = n;
        asm volatile("" : "+s"(ld));  // no addresses kept over the loop
        gemm_pipe::store_bf16(acc, c_tile, ld, wave);
        c_tile = c + (uint64_t)tm * 256u * n + (uint64_t)tn * 256u;
      });
}

// 128 x 128 tiles: small grids, and (TAIL) the quarters of a last round (tile_plan.hpp).
// Every output has the MFMAs of the 256 x 256 tile in its order, and its bits.
template <int STAGES, bool WHOLE, bool TAIL>
__global__ void __launch_bounds__(256, STAGES == 2 ? 2 : 1) gemm_mxfp4_128_kernel(
    Operand a, Operand b, uint16_t* __restrict__ c, uint32_t m, uint32_t n, uint32_t panels,
    uint32_t xcds, uint32_t first_big) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  uint32_t tm, tn;
  if constexpr (TAIL) {
    if (!gemm_core::tail_quarter(blockIdx.x, first_big, m, n, xcds, &tm, &tn)) return;
  } else {
    gemm_core::xcd_tile_order(blockIdx.x, (m + 127u) / 128u, (n + 127u) / 128u, xcds, &tm, &tn);
  }
  const uint32_t rows_a = WHOLE ? 128u : min(128u, m - tm * 128u);
  const uint32_t rows_b = WHOLE ? 128u : min(128u, n - tn * 128u);
  const auto ar = code_rows<128>(a, tm * 128u, rows_a, panels);
  const auto br = code_rows<128>(b, tn * 128u, rows_b, panels);
  using T = Small<STAGES>;
  const T tile(ar, br, scale_rows<128>(a, tm * 128u), scale_rows<128>(b, tn * 128u), panels, smem);
  typename T::Acc acc;
  tile.run(acc);
  gemm_pipe::store_bf16_128<WHOLE>(acc, c + (uint64_t)tm * 128 * n + (uint64_t)tn * 128, n,
                                   rows_a, rows_b);
}

// Few output tiles (gemm_direct.hpp): the outputs' partial sums over a workgroup's waves.
template <bool WIDE>
__global__ void __launch_bounds__(gemm_direct::kThreads, WIDE ? 2 : 4) gemm_mxfp4_direct_kernel(
    int form, Operand a, Operand b, uint16_t* __restrict__ c, uint32_t m, uint32_t n,
    uint32_t panels, uint32_t xcds) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const gemm_direct::BlockScales s{a.scales, b.scales, a.scale_rows, b.scale_rows};
  gemm_direct::run_form<gemm_direct::Mxfp4, WIDE>(form, a.codes, b.codes, c, m, n,
                                                  panels * (uint32_t)kRow, 1.0f, xcds, smem, s);
}

// Whether the direct kernel takes a product: by the rule of the other types, and few rows (of
// k from eight units on) also whatever k is, once what they stream is more than a round of
// tiles (us, the streamed operand from memory, tile against direct):
//   16 x 40000 x 2048 18.4, 14.8    16 x 65536 x 2048 23.3, 22.7   x 4096 40.3, 35.2
//   16 x 128256 x 2048 43.8, 37.7   x 4096 77.0, 62.9   1 x 128256 x 4096 73.8, 58.9
//   32 x 128256 x 4096 75.6, 70.6   65536 x 16 x 4096 43.8, 33.7
// The other types' rule (gemm_direct::prefer) on 4-bit operands, so measured, by cost:
//   2  1 x 4096 x 4096 11.1, 4.5    4  64 x 4096 x 1024 6.1, 4.1    x 4096 11.4, 5.9
//   4  32 x 8192 x 8192 19.8, 11.5  4  64 x 4096 x 16384 35.2, 15.1
//   5  16 x 14336 x 4096 14.1, 10.0 6  64 x 8192 x 1024 6.3, 4.8    x 8192 20.6, 14.9
//   6  256 x 2048 x 4096 11.6, 7.2  6  128 x 4096 x 16384 40.7, 20.0
//   9  16 x 20000 x 512 5.5, 5.2    x 4096 15.2, 12.0
//   10 16 x 28672 x 4096 17.1, 17.5 x 1024 7.3, 8.8 (goes to direct)
//   12 128 x 8192 x 1024 6.9, 7.3   x 4096 14.6, 15.1   x 16384 42.5, 37.0 (goes to the tile)
//   12 32 x 20000 x 4096 15.3, 17.0 32 x 28672 x 1024 7.2, 8.9   x 4096 17.1, 19.3
//   12 64 x 14336 x 4096 14.5, 16.4 512 x 2048 x 4096 11.8, 12.2   8192 x 128 x 4096 14.4, 17.3
bool prefer_direct(uint32_t m, uint32_t n, uint32_t kbytes, uint32_t cus) {
  const uint32_t rows = m > n ? m : n, few = m > n ? n : m;
  return gemm_direct::prefer(m, n, kbytes, 1u, cus) ||
         (few <= 32u && kbytes >= gemm_direct::kWaves * gemm_direct::kUnit &&
          ((uint64_t)rows + 127u) / 128u > cus);
}

// The forms for any K leave C as it is for this type: every k has to fit the others.
static_assert(gemm_direct::k_fits(mxfp4::kMaxPanels * (uint32_t)kRow, 1u),
              "more panels would plan a form that this type lacks");

int32_t launch_direct(const gemm_direct::Launch& l, const Operand& a, const Operand& b,
                      uint16_t* c, uint32_t m, uint32_t n, uint32_t panels,
                      const tile_plan::Topology& topo, hipStream_t s) {
  static const int32_t lds_rc = fe2o3_host::set_dynamic_lds(
      {(const void*)gemm_mxfp4_direct_kernel<true>, (const void*)gemm_mxfp4_direct_kernel<false>},
      gemm_direct::kWideSmem);
  if (lds_rc != FE2O3_OK) return lds_rc;
  if (l.grid > 0x7fffffffu) return FE2O3_ERR_SHAPE;
  const dim3 grid = gemm_direct::list_grid(l.grid);
  if (l.wide)
    gemm_mxfp4_direct_kernel<true><<<grid, gemm_direct::kThreads, l.smem, s>>>(
        l.form, a, b, c, m, n, panels, topo.xcds);
  else
    gemm_mxfp4_direct_kernel<false><<<grid, gemm_direct::kThreads, l.smem, s>>>(
        l.form, a, b, c, m, n, panels, topo.xcds);
  return fe2o3_host::after_launch();
}

int32_t set_tile_lds() {
  static const int32_t rc = [] {
    int32_t r = fe2o3_host::set_dynamic_lds(
        {(const void*)gemm_mxfp4_kernel<false, false>, (const void*)gemm_mxfp4_kernel<true, false>,
         (const void*)gemm_mxfp4_kernel<false, true>, (const void*)gemm_mxfp4_rounds_kernel},
        (int)Big::kSmem);
    if (r == FE2O3_OK)
      r = fe2o3_host::set_dynamic_lds({(const void*)gemm_mxfp4_128_kernel<2, true, false>,
                                       (const void*)gemm_mxfp4_128_kernel<2, false, false>,
                                       (const void*)gemm_mxfp4_128_kernel<2, true, true>,
                                       (const void*)gemm_mxfp4_128_kernel<2, false, true>},
                                      (int)Small<2>::kSmem);
    if (r == FE2O3_OK)
      r = fe2o3_host::set_dynamic_lds({(const void*)gemm_mxfp4_128_kernel<3, true, false>,
                                       (const void*)gemm_mxfp4_128_kernel<3, false, false>,
                                       (const void*)gemm_mxfp4_128_kernel<3, true, true>,
                                       (const void*)gemm_mxfp4_128_kernel<3, false, true>},
                                      (int)Small<3>::kSmem);
    return r;
  }();
  return rc;
}

int32_t launch_tiles(const Operand& a, const Operand& b, uint16_t* c, uint32_t m, uint32_t n,
                     uint32_t panels, const tile_plan::Topology& topo, hipStream_t s) {
  // The plan's lines on 4-bit operands (us, all in tiles of 128, in tiles of 256 in rounds, and
  // as planned where that is neither):
  //   2048 x 2048 x 4096 15.5, 27.7   2816 x 2816 x 1024 11.2, 15.2   x 8192 39.9, 50.1
  //   1024 x 8192 x 8192 46, 52       1024 x 9216 x 8192 72, 55
  //   3328 x 2816 x 1024 15.1, 15.3   x 4096 35.4, 31.4   4096 x 2560 x 4096 35.3, 31.4
  //   4352 x 4096 x 1024 21.5, 24.1, a round and quarters 22.0   x 4096 54.4, 56.2, 46.9
  const tile_plan::Plan plan = tile_plan::plan(m, n, topo);
  if (plan.grid > 0x7fffffffu || plan.tail_grid > 0x7fffffffu) return FE2O3_ERR_SHAPE;
  const int32_t lds_rc = set_tile_lds();
  if (lds_rc != FE2O3_OK) return lds_rc;
  const bool aligned = ((uintptr_t)c & 15u) == 0u;
  const bool whole = m % 256u == 0u && n % 256u == 0u && aligned;
  const bool whole128 = m % 128u == 0u && n % 128u == 0u && aligned;
  auto small = [&](auto stages, auto tail, uint64_t grid, uint32_t first) {
    constexpr int S = decltype(stages)::value;
    constexpr bool T = decltype(tail)::value;
    if (whole128)
      gemm_mxfp4_128_kernel<S, true, T><<<(unsigned)grid, 256, Small<S>::kSmem, s>>>(
          a, b, c, m, n, panels, topo.xcds, first);
    else
      gemm_mxfp4_128_kernel<S, false, T><<<(unsigned)grid, 256, Small<S>::kSmem, s>>>(
          a, b, c, m, n, panels, topo.xcds, first);
    return fe2o3_host::after_launch();
  };
  using Two = std::integral_constant<int, 2>;
  using Three = std::integral_constant<int, 3>;
  if (plan.small)
    return plan.stages == 2 ? small(Two{}, std::false_type{}, plan.grid, 0u)
                            : small(Three{}, std::false_type{}, plan.grid, 0u);
  const unsigned big = (unsigned)plan.grid;
  const bool staged = gemm_core::staged_epilogue(((uint64_t)m + n) * panels * kRow);
  if (whole && !staged && panels % 2u == 0u && big > topo.cus)
    gemm_mxfp4_rounds_kernel<<<topo.cus, 256, Big::kSmem, s>>>(a, b, c, m, n, panels, topo.xcds, big);
  else if (!whole)
    gemm_mxfp4_kernel<false, true><<<big, 256, Big::kSmem, s>>>(a, b, c, m, n, panels, topo.xcds);
  else if (staged)
    gemm_mxfp4_kernel<true, false><<<big, 256, Big::kSmem, s>>>(a, b, c, m, n, panels, topo.xcds);
  else
    gemm_mxfp4_kernel<false, false><<<big, 256, Big::kSmem, s>>>(a, b, c, m, n, panels, topo.xcds);
  const int32_t rc = fe2o3_host::after_launch();
  if (rc != FE2O3_OK || !plan.tail) return rc;
  return plan.tail_stages == 2 ? small(Two{}, std::true_type{}, plan.tail_grid, plan.first_big)
                               : small(Three{}, std::true_type{}, plan.tail_grid, plan.first_big);
}

#define FE2O3_MX(NAME, FN, THREADS, LDS) \
  fe2o3_host::KernelRegistrar({"fe2o3_gemm_mxfp4_nt", NAME, (const void*)FN, THREADS, LDS})
#define FE2O3_MX_128(S, W, T) \
  FE2O3_MX("gemm_mxfp4_128_kernel<" #S "," #W "," #T ">", (gemm_mxfp4_128_kernel<S, W, T>), 256, Small<S>::kSmem)
const fe2o3_host::KernelRegistrar kRegistered[] = {
    FE2O3_MX("gemm_mxfp4_kernel", (gemm_mxfp4_kernel<false, false>), 256, Big::kSmem),
    FE2O3_MX("gemm_mxfp4_kernel<staged>", (gemm_mxfp4_kernel<true, false>), 256, Big::kSmem),
    FE2O3_MX("gemm_mxfp4_rounds_kernel", gemm_mxfp4_rounds_kernel, 256, Big::kSmem),
    FE2O3_MX("gemm_mxfp4_kernel<edge>", (gemm_mxfp4_kernel<false, true>), 256, Big::kSmem),
    FE2O3_MX_128(2, true, false), FE2O3_MX_128(2, false, false), FE2O3_MX_128(2, true, true),
    FE2O3_MX_128(2, false, true), FE2O3_MX_128(3, true, false), FE2O3_MX_128(3, false, false),
    FE2O3_MX_128(3, true, true), FE2O3_MX_128(3, false, true),
    FE2O3_MX("gemm_mxfp4_direct_kernel", gemm_mxfp4_direct_kernel<false>, gemm_direct::kThreads, gemm_direct::kLightSmem),
    FE2O3_MX("gemm_mxfp4_direct_kernel<wide>", gemm_mxfp4_direct_kernel<true>, gemm_direct::kThreads, gemm_direct::kWideSmem)};
#undef FE2O3_MX
#undef FE2O3_MX_128

}  // namespace

extern "C" int32_t fe2o3_gemm_mxfp4_nt(const uint8_t* a, uint64_t a_len, const uint8_t* a_scales,
                                       uint64_t a_scales_len, const uint8_t* b, uint64_t b_len,
                                       const uint8_t* b_scales, uint64_t b_scales_len,
                                       uint16_t* c, uint64_t c_len, uint32_t m, uint32_t n,
                                       uint32_t k, void* stream) {
  FE2O3_ENTRY("fe2o3_gemm_mxfp4_nt");
  const mxfp4::Packed pa = mxfp4::Packed::of(m, k), pb = mxfp4::Packed::of(n, k);
  if (pa.panels > mxfp4::kMaxPanels) return FE2O3_ERR_SHAPE;
  if (a_len != pa.codes || a_scales_len != pa.scales || b_len != pb.codes ||
      b_scales_len != pb.scales || c_len != (uint64_t)m * n)
    return FE2O3_ERR_LENGTH;
  if (c_len == 0u) return FE2O3_OK;
  if (!c || (k != 0u && (!a || !a_scales || !b || !b_scales))) return FE2O3_ERR_NULL;
  if ((((uintptr_t)a | (uintptr_t)a_scales | (uintptr_t)b | (uintptr_t)b_scales) & 15u) != 0u ||
      ((uintptr_t)c & 1u) != 0u)
    return FE2O3_ERR_ALIGNMENT;
  tile_plan::Topology topo;
  const int32_t rc = fe2o3_host::device_topology(&topo);
  if (rc != FE2O3_OK) return rc;
  hipStream_t s = (hipStream_t)stream;
  const Operand oa{a, a_scales, pa.scale_rows}, ob{b, b_scales, pb.scale_rows};
  if (k == 0u) return launch_direct(gemm_direct::plan_fill(c_len), oa, ob, c, m, n, 0u, topo, s);
  const uint32_t kbytes = pa.panels * (uint32_t)kRow;
  if (prefer_direct(m, n, kbytes, topo.cus))
    return launch_direct(gemm_direct::plan(m, n, kbytes, 1u, topo.cus), oa, ob, c, m, n, pa.panels,
                         topo, s);
  return launch_tiles(oa, ob, c, m, n, pa.panels, topo, s);
}
