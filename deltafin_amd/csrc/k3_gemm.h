// Tiled matrix-core products D[m, n] = sum_k W(n, k) X(m, k) for many positions:
// the device core of the dense layers (k3_dense.hip).  Both operands are BF16 planes
// in memory (an fp32 operand is several planes, see below; int8 weights are widened
// in registers), sums are fp32.
//
// Segments.  A product is a list of up to six segments, each a pair of planes over the
// same K: the three BF16 terms of an fp32 activation against one matrix, the six
// leading term pairs of two fp32 operands, or the gate and the up half of a gradient.
// All segments of an output meet in the same accumulators, so an fp32 product costs
// three (or six) BF16 products and no pass over the output in between.
//
// Tile.  A workgroup of eight waves, one to a CU, computes BN x BM outputs in K steps of 64
// from three weight tiles and two position tiles in LDS: while one step is multiplied the
// next ones come from memory straight into the others (global_load_lds, 16 bytes per lane,
// no registers held).  One instruction of a wave fills 1 KB of LDS in lane order, so the
// layout in LDS is chosen by which 16 bytes of memory each lane asks for:
//   KMAJOR  rows of 64 k (128 bytes), 16-byte chunk c of row r at slot c ^ kmajor_swizzle(r);
//   INT8    rows of 64 k (64 bytes), chunk c at slot c ^ int8_swizzle(r);
//   NMAJOR  (the operand's k runs over memory rows) 64 k rows of BN (BM) values,
//           32-byte chunk c of row k at slot c ^ nmajor_swizzle(k), read back through
//           ds_read_b64_tr_b16, which hands 16 lanes the columns of 4 rows x 16 values.
// The exclusive-ors spread each read of a wave over all banks (no conflict is counted).
//
// A step is two halves of 32 k; each half's fragments are read while the other half is
// multiplied, and one barrier per step stands between two halves' products.
//
// Rate.  4096 x 4096 x 7168 (a gated block's two projections, three BF16 outputs) takes
// 181 us, 1.33 PFLOP/s; 4096 x 7168 x 6144 with bias and residual 288, 1.25.  The matrix
// cores are busy 67-74 % of the cycles, at 1.65 GHz: power bounds it (without its loads
// from memory the first took 155 us, without waiting for them 183).
//
// The k of an operand element is 16 g + 8 kk + e in a step (lane group g = lane / 16,
// half kk, element e) instead of the matrix instruction's 32 kk + 8 g + e: any order
// serves as long as both operands use it, and this one lets an int8 lane read its 16
// values of both halves at once.
//
// The weight operand is the instruction's first, so a lane's four results are four
// consecutive n of one m: 8 or 16 bytes of a row-major output.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "k3_device.h"

namespace k3 {
namespace gemm {

enum { L_KMAJOR = 0, L_INT8 = 1, L_NMAJOR = 2 };

constexpr int kStep = 64;      // k of a step
constexpr int kMaxSegments = 6;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct GemmArgs {
  const uint8_t* w[kMaxSegments];   // weight-side planes
  const uint8_t* w2[kMaxSegments];  // GLU: the up matrix's (w is the gate's)
  const uint8_t* x[kMaxSegments];   // position-side planes
  int segments;
  int n, m, k;         // n: of one matrix (GLU: outputs); k per segment
  int kw, kx;          // k held by a KMAJOR / INT8 row in memory, whole chunks (>= k)
  uint32_t ldw, ldx;   // bytes between rows
  int tiles_n, tiles_m;
  int splits, per;     // whole steps [z * per, ...) of all segments' for grid z
};

__device__ const u32x4 g_zero_chunk = {0u, 0u, 0u, 0u};

// 16 bytes per lane from memory to LDS at `lds` + 16 lane (wave-uniform, as is `base`).  In
// assembly for its address form, a scalar base and a 32-bit lane offset: through the
// builtin every load took a 64-bit lane address of its own, whose sums and register pairs
// cost the large tile its spare registers.  It writes no register but m0, which the
// compiler holds nothing in (it sets m0 right ahead of what reads it); vmcnt ends it.
__device__ __forceinline__ void load_lds(const uint8_t* base, uint32_t offset, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
      :
      : "s"(lds), "v"(offset), "s"(base)
      : "memory");
}
__device__ __forceinline__ void load_lds(const uint8_t* lane_address, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(lane_address)
               : "memory");
}
// All but the last N of this wave's loads have landed, then everybody's.
template <int N>
__device__ __forceinline__ void landed() {
  static_assert(N < 16, "the counter's low bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | N);
  __syncthreads();
}

// A 16-byte read of a wave runs as four passes of 16 lanes, lanes 0-3, 12-15 and 20-27
// the first: 16 different rows of the 16, eight of them in one lane group's chunk and
// eight in the next one's.  These orders put such a pass on all 64 banks (counted: with
// c ^ (r % 8) or c ^ (r / 2 % 8) every read took twice its cycles).
__device__ __forceinline__ int kmajor_swizzle(int r) {
  const int q = (r >> 1) & 7;
  return q ^ ((q & 2) << 1);
}
__device__ __forceinline__ int int8_swizzle(int r) {
  const int t = (r >> 2) & 3;
  return (t >> 1) | (((t ^ (t >> 1)) & 1) << 1);
}

template <int R>
__device__ __forceinline__ int nmajor_swizzle(int k) {
  return ((k & 3) | ((k >> 4 & 1) << 2)) & (R / 16 - 1);
}

// An operand's tile of R rows (n or m) x 64 k.
template <int R, int L, int WAVES, bool kPairs>
struct Tile {
  static constexpr int kBytes = R * kStep * (L == L_INT8 ? 1 : 2);
  static constexpr int kLoads = kBytes / 1024;                      // wave instructions
  static constexpr int kPer = kLoads / WAVES;                       // of one wave
  static constexpr int kChunkK = L == L_INT8 ? 16 : 8;              // k of a 16-byte chunk
  static constexpr int kRowLoads = R / 8;                           // NMAJOR: chunks of a k row
  static_assert(kLoads * 1024 == kBytes, "whole instructions");

  uint32_t off[kPer];  // lane offsets from the segment's (matrix's) base at k = 0

  // rows: of the operand (n or m); r0: the tile's first.  With kPairs the tile's
  // blocks of 16 rows alternate between the gate and the up matrix.
  __device__ __forceinline__ void init(int wave, int lane, int r0, int rows, uint32_t ld) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = wave * kPer + i;
      if constexpr (L == L_NMAJOR) {
        const int kr = j * (64 / kRowLoads) + lane / kRowLoads;
        const int pos = lane % kRowLoads;
        const int c = (pos >> 1) ^ nmajor_swizzle<R>(kr);
        // rows past the last chunk repeat the tile's first (never stored)
        const int r = c * 16 + (pos & 1) * 8;
        off[i] = (uint32_t)kr * ld + (uint32_t)(r0 + r < rows ? r : 0) * 2u;
      } else {
        const int per = L == L_INT8 ? 16 : 8;  // rows of an instruction
        const int rl = j * per + lane / (64 / per);
        const int r = kPairs ? (rl >> 5) * 16 + (rl & 15) : rl;
        const int slot = lane % (64 / per);
        const int c = L == L_INT8 ? slot ^ int8_swizzle(rl) : slot ^ kmajor_swizzle(rl);
        off[i] = (uint32_t)min(r, rows - 1 - r0) * ld + 16u * c;
      }
    }
  }

  // Load i of this wave of the whole step at base (the operand's row r0, k = k0; NMAJOR:
  // k = k0, column r0; base2 in the up matrix) to lds.
  __device__ __forceinline__ void load(int i, const uint8_t* base, const uint8_t* base2, int wave,
                                       uint32_t lds) const {
    const int j = wave * kPer + i;
    load_lds(kPairs && (j / (L == L_INT8 ? 1 : 2)) % 2 ? base2 : base, off[i], lds + 1024 * j);
  }

  // The whole share of a step of which `left` < 64 k exist in memory: zeros past them.
  __device__ __forceinline__ void load_tail(const uint8_t* base, const uint8_t* base2, int wave,
                                            int lane, int left, uint32_t lds) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = wave * kPer + i;
      int k;
      if constexpr (L == L_NMAJOR) {
        k = j * (64 / kRowLoads) + lane / kRowLoads;
      } else {
        const int per = L == L_INT8 ? 16 : 8;
        const int rl = j * per + lane / (64 / per);
        const int slot = lane % (64 / per);
        k = kChunkK * (L == L_INT8 ? slot ^ int8_swizzle(rl) : slot ^ kmajor_swizzle(rl));
      }
      const uint8_t* b = kPairs && (j / (L == L_INT8 ? 1 : 2)) % 2 ? base2 : base;
      uint32_t o = off[i];
      asm volatile("" : "+v"(o));  // its 64-bit form lives here, not across the main loop
      load_lds(k < left ? b + o : reinterpret_cast<const uint8_t*>(&g_zero_chunk),
               lds + 1024 * j);
    }
  }
};

__device__ __forceinline__ bf16x8 widen8(uint32_t a, uint32_t b) {
  uint32_t p[4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t v = e ? b : a;
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __float_as_uint((float)((int32_t)(v << (24 - 8 * i)) >> 24));
    p[2 * e] = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
    p[2 * e + 1] = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
  }
  return __builtin_bit_cast(bf16x8, u32x4{p[0], p[1], p[2], p[3]});
}

// Operand fragments: F blocks of 16 rows from row16 * 16 of the tile, both halves.  int8
// values are read with the first half and widened by widen() ahead of each half's use.
template <int R, int L, int F>
struct Frags {
  bf16x8 v[2][F];
  u32x4 raw[L == L_INT8 ? F : 1];  // both halves' int8 values as read

  // Where this lane reads in half kk, formed anew for each: block row16 of the tile, or
  // (NMAJOR) block 0, whose chunk number another block's number is exclusive-or'ed into.
  template <int kk>
  __device__ static __forceinline__ uint32_t place(int row16, int lane) {
    const int i16 = lane & 15, g = lane >> 4;
    uint32_t at;
    if constexpr (L == L_KMAJOR) {
      at = row16 * 2048 + i16 * 128 + (((2 * g + kk) ^ kmajor_swizzle(i16)) << 4);
    } else if constexpr (L == L_INT8) {
      at = row16 * 1024 + i16 * 64 + ((g ^ int8_swizzle(i16)) << 4);
    } else {
      const int kr = 16 * g + 8 * kk + (i16 >> 2);  // and kr + 4: the same swizzle
      at = kr * (2 * R) + (i16 & 3) * 8 + (nmajor_swizzle<R>(kr) << 5);  // of block 0
    }
    return at;
  }

  // Block f from row16 on of half kk, `at` being place<kk>.  int8 blocks come whole with the
  // first half.
  template <int kk>
  __device__ __forceinline__ void read(int f, const uint8_t* tile, uint32_t at, int row16) {
    if constexpr (L == L_KMAJOR) {
      v[kk][f] = *reinterpret_cast<const bf16x8*>(tile + at + 2048 * f);
    } else if constexpr (L == L_INT8) {
      if constexpr (kk == 0) raw[f] = *reinterpret_cast<const u32x4*>(tile + at + 1024 * f);
    } else {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const uint8_t* q = tile + (at ^ ((uint32_t)(row16 + f) << 5));
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)q);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(q + 8 * R));
      const bf16x4 a = __builtin_bit_cast(bf16x4, lo), b = __builtin_bit_cast(bf16x4, hi);
      v[kk][f] = bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }

  template <int kk>
  __device__ __forceinline__ void widen() {
    if constexpr (L == L_INT8) {
#pragma unroll
      for (int f = 0; f < F; ++f) v[kk][f] = widen8(raw[f][2 * kk], raw[f][2 * kk + 1]);
    }
  }
};

// Workgroup of tile t: the eight XCDs take contiguous runs of tiles, so that one L2
// holds the panels that its workgroups share, and within the order a band of kBand
// row panels is walked before the next column panel (81 % of requests hit; bands of 2, 8
// and 16 were within 2 %, no runs 5 % slower for fp32 gate/up at 2048 positions).
constexpr int kXcds = 8;
constexpr int kBand = 4;
__device__ __forceinline__ void tile_of(int b, int tiles_n, int tiles_m, int* tn, int* tm) {
  const int total = tiles_n * tiles_m;
  const int q = total / kXcds, r = total % kXcds, x = b % kXcds;
  const int t = x * q + min(x, r) + b / kXcds;
  const int band = t / (kBand * tiles_n);
  const int m0 = band * kBand, mh = min(kBand, tiles_m - m0);
  const int in = t - m0 * tiles_n;
  *tm = m0 + in % mh;
  *tn = in / mh;
}

// The tile's sums: acc[fn][fm] of a wave, n = n0 + 16 fn + 4 (lane / 16) + i,
// m = m0 + 16 fm + lane % 16 with the wave's n0, m0 below.
template <int BN, int BM, int NWN, int NWM, int WL, int XL, bool kPairs>
struct Core {
  static constexpr int kWaves = NWN * NWM;
  static constexpr int FN = BN / 16 / NWN, FM = BM / 16 / NWM;
  // rows that the weight side's tile has in LDS: a power of two
  static constexpr int kRowsW = BN <= 128 ? 128 : 256;
  typedef Tile<kRowsW, WL, kWaves, kPairs> TW;
  typedef Tile<BM, XL, kWaves, false> TX;
  static_assert(TW::kLoads % kWaves == 0 && TX::kLoads % kWaves == 0, "equal shares of loads");
  // Three tiles of the weight side and two of the other: 160 KB, all of a CU's LDS, at 256 x
  // 256 BF16.  Half of a step's loads are issued two steps ahead, the others, the first
  // after the barrier that frees their tile, one.
  static constexpr int kSlotX = 3 * TW::kBytes;  // offset of the second operand's tiles
  static constexpr int kLds = kSlotX + 2 * TX::kBytes;

  __device__ static __forceinline__ void run(const GemmArgs& a, uint8_t* lds, int tn, int tm,
                                             int split, f32x4 (&acc)[FN][FM]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave % NWN, wm = wave / NWN;
    const int rn = tn * (kPairs ? BN / 2 : BN), rm = tm * BM;
    TW tw;
    TX tx;
    tw.init(wave, lane, rn, a.n, a.ldw);
    tx.init(wave, lane, rm, a.m, a.ldx);
    const uint64_t w0 = WL == L_NMAJOR ? (uint64_t)rn * 2 : (uint64_t)rn * a.ldw;
    const uint64_t x0 = XL == L_NMAJOR ? (uint64_t)rm * 2 : (uint64_t)rm * a.ldx;
    // whole steps of every segment, then each segment's rest in the last split
    const int steps = a.k / kStep;
    const int s0 = min(split * a.per, steps * a.segments);
    const int s1 = min(s0 + a.per, steps * a.segments);

#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // where the next step comes from: pointers that advance, read anew per segment
    const uint64_t dw = WL == L_NMAJOR ? (uint64_t)kStep * a.ldw : kStep * (WL == L_INT8 ? 1 : 2);
    const uint64_t dx = XL == L_NMAJOR ? (uint64_t)kStep * a.ldx : kStep * 2;
    const uint8_t *pw = nullptr, *pu = nullptr, *px = nullptr;
    int segw = 0, leftw = 0, segx = 0, leftx = 0;  // steps of the segment from the next one on
    auto open_w = [&](int step) {
      pw = a.w[segw] + w0 + step * dw;
      if constexpr (kPairs) pu = a.w2[segw] + w0 + step * dw;
      leftw = steps - step;
    };
    auto open_x = [&](int step) {
      px = a.x[segx] + x0 + step * dx;
      leftx = steps - step;
    };
    auto advance_w = [&] {
      pw += dw;
      if constexpr (kPairs) pu += dw;
      if (--leftw == 0 && ++segw < a.segments) open_w(0);
    };
    auto advance_x = [&] {
      px += dx;
      if (--leftx == 0 && ++segx < a.segments) open_x(0);
    };
    typedef Frags<kRowsW, WL, FN> FW;
    typedef Frags<BM, XL, FM> FX;
    FW fw;
    FX fx;
    // block b of the FN + FM that a half step needs
    auto read = [&](auto half, int b, const uint8_t* tw_at, const uint8_t* tx_at, uint32_t at_w,
                    uint32_t at_x) {
      constexpr int kk = decltype(half)::value;
      if (b < FN)
        fw.template read<kk>(b, tw_at, at_w, wn * FN);
      else
        fx.template read<kk>(b - FN, tx_at, at_x, wm * FM);
    };
    // Half kk's products, a column of FN at a time; between the columns go the loads of
    // later steps, then the reads of the other half, few at a time: 64 loads of 1 KB issued
    // together keep the waves from their products for the 1000 cycles that the address
    // units take over them.
    constexpr int kReads = (FN + FM + FM - 2) / (FM - 1);  // per column, none behind the last
    constexpr int kLoadsPer = (TW::kPer + TX::kPer + FM - 1) / FM;
    auto half = [&](auto kk_, auto reads_, auto load_x, auto load_w, const uint8_t* tw_at,
                    const uint8_t* tx_at, uint32_t to_x, uint32_t to_w) {
      constexpr int kk = decltype(kk_)::value;
      constexpr bool lx = decltype(load_x)::value, lw = decltype(load_w)::value;
      std::integral_constant<int, 1 - kk> other;
      const uint32_t at_w = FW::template place<1 - kk>(wn * FN, lane);
      const uint32_t at_x = FX::template place<1 - kk>(wm * FM, lane);
      fw.template widen<kk>();
#pragma unroll
      for (int j = 0; j < FM; ++j) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
          acc[i][j] =
              __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw.v[kk][i], fx.v[kk][j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = j * kLoadsPer; i < (j + 1) * kLoadsPer; ++i) {
          if (lx && i < TX::kPer) tx.load(i, px, nullptr, wave, to_x);
          if (lw && i >= TX::kPer && i < TX::kPer + TW::kPer)
            tw.load(i - TX::kPer, pw, pu, wave, to_w);
        }
        if constexpr (decltype(reads_)::value) {
#pragma unroll
          for (int b = j * kReads; b < (j + 1) * kReads; ++b)
            if (b < FN + FM) read(other, b, tw_at, tx_at, at_w, at_x);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (lx) advance_x();
      if constexpr (lw) advance_w();
    };
    const std::integral_constant<int, 0> h0;
    const std::integral_constant<int, 1> h1;
    const std::true_type yes;
    const std::false_type no;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    auto first_half = [&](const uint8_t* tw_at, const uint8_t* tx_at) {
      const uint32_t at_w = FW::template place<0>(wn * FN, lane);
      const uint32_t at_x = FX::template place<0>(wm * FM, lane);
#pragma unroll
      for (int b = 0; b < FN + FM; ++b) read(h0, b, tw_at, tx_at, at_w, at_x);
    };
    auto blocks_there = [] {
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): issued a half step ago
      __builtin_amdgcn_sched_barrier(0);
    };
    if (s0 < s1) {
      auto all_w = [&](uint32_t to) {
#pragma unroll
        for (int i = 0; i < TW::kPer; ++i) tw.load(i, pw, pu, wave, to);
        advance_w();
      };
      auto all_x = [&](uint32_t to) {
#pragma unroll
        for (int i = 0; i < TX::kPer; ++i) tx.load(i, px, nullptr, wave, to);
        advance_x();
      };
      const int n = s1 - s0;
      segw = segx = s0 / steps;
      open_w(s0 - segw * steps);
      open_x(s0 - segx * steps);
      all_w(lds0);
      all_x(lds0 + kSlotX);
      landed<0>();
      if (n > 1) {
        all_w(lds0 + TW::kBytes);
        all_x(lds0 + kSlotX + TX::kBytes);
      }
      if (n > 2) all_w(lds0 + 2 * TW::kBytes);
      first_half(lds, lds + kSlotX);
      uint32_t w_at = 0, x_at = kSlotX;  // the step's tiles
      auto next_w = [&] { return w_at == 2 * TW::kBytes ? 0u : w_at + (uint32_t)TW::kBytes; };
      auto next_x = [&] { return 2 * kSlotX + TX::kBytes - x_at; };
      // A step: its first half, the barrier behind which the next step's tiles are there and
      // its own are free, its second half.
      auto step = [&](auto wait, auto reads, auto load_x, auto load_w) {
        blocks_there();
        half(h0, yes, no, no, lds + w_at, lds + x_at, 0, 0);
        if constexpr (decltype(reads)::value) {
          landed<decltype(wait)::value>();
          __builtin_amdgcn_sched_barrier(0);
        }
        half(h1, reads, load_x, load_w, lds + next_w(), lds + next_x(), lds0 + x_at, lds0 + w_at);
        w_at = next_w();
        x_at = next_x();
      };
      const std::integral_constant<int, TW::kPer> ahead;  // loads of the tile two steps on
      for (int s = 0; s < n - 3; ++s) step(ahead, yes, yes, yes);
      if (n > 2) step(ahead, yes, yes, no);
      if (n > 1) step(h0, yes, no, no);
      step(h0, no, no, no);
    }
    const int rest = a.k - steps * kStep;
    if (rest > 0 && split == a.splits - 1) {
      // the segments' rests in turn through two slots, the next one's loads under way
      auto load_rest = [&](int segment) {
        segw = segx = segment;
        open_w(steps);
        open_x(steps);
        tw.load_tail(pw, pu, wave, lane, a.kw - steps * kStep, lds0 + (segment & 1) * TW::kBytes);
        tx.load_tail(px, nullptr, wave, lane, a.kx - steps * kStep,
                     lds0 + kSlotX + (segment & 1) * TX::kBytes);
      };
      __syncthreads();  // the tiles are no longer read
      load_rest(0);
      for (int i = 0; i < a.segments; ++i) {
        if (i + 1 < a.segments) {
          load_rest(i + 1);
          landed<TW::kPer + TX::kPer>();
        } else {
          landed<0>();
        }
        const uint8_t* tw_at = lds + (i & 1) * TW::kBytes;
        const uint8_t* tx_at = lds + kSlotX + (i & 1) * TX::kBytes;
        first_half(tw_at, tx_at);
        half(h0, yes, no, no, tw_at, tx_at, 0, 0);
        half(h1, no, no, no, tw_at, tx_at, 0, 0);
        __syncthreads();  // before the load behind the next one
      }
    }
  }
};

}  // namespace gemm
}  // namespace k3
