// Matrix products on the 16-bit matrix pipe, as a device function for one output tile:  OUT[j][i] = sum_k I(i, k) J(j, k).
//
// Operand storage: rows of `ldb` bytes (16-byte aligned).
//   plain  bf16 elements
//   split  fp32 values as two fp16 planes, x = hi + lo (22 bits), in groups of 32 columns: [32 x hi][32 x lo], 128 bytes a group
// and one of two orientations:
//   KC     a row of the tile axis per stored row, k contiguous          (k-step: 128 bytes of each row)
//   KS     a row of k per stored row, the tile axis contiguous          (k-step: 64 rows, split 32)
// so a k-step moves the same number of bytes in every form: 128 per row of the tile, 64 k (plain) or 32 k (split).
//
// Split products are hi*hi + hi*lo + lo*hi in fp32 accumulators: what is dropped (lo*lo and the 23rd bit) is 2^-22 of a product, below the
// rounding of an fp32 sum, for three passes of the fp16 pipe -- whose rate is 16 times the fp32 pipe's.
// The matrix instruction aligns its products and the accumulator to the largest of them and drops what lies 2 bits below that one's last place (16
// products of 1/16 ulp of the accumulator add nothing), so a long sum of one sign drifts: 1e-5 of a sum of 3456 squares, 4e-5 of 9408.  Split
// products therefore add the accumulators up in fp32 every 128 k and start again from zero: 3e-7 at any length, less than plain fp32 sums lose
// (every 32 k: 1e-7, and 10 % slower on the 128 x 128 tile).
// bf16 products need none of it: sums of up to 2^22 of them of one sign show no drift (mean relative error below 3e-4, the noise of their operands'
// rounding; the cut above would have made it 2e-2), and their results are rounded to 2^-8.
//
// v_mfma_f32_16x16x32 rather than 32x32x16: the chip is bound by power under such products, and the smaller shape sustains 1656 TFLOP/s from registers where
// the larger one does 1510 (random operands).  8192^3, bf16, 256 x 256 tiles: 1330 TFLOP/s in all three operand orientations (1260 with 32x32x16).
//
// Tiles go from global memory to LDS with direct loads (16 bytes a lane, no register stop), double buffered, one barrier a k-step.
// Such a load writes lane l to base + 16 l, so the bank swizzle is applied to the SOURCE address: in a KC tile the 16-byte chunk c of
// row r sits at slot c ^ ((r >> 1) & 7) (16 consecutive rows read the same c from 16 different bank groups); in a KS tile the 64-byte unit u of
// k-row r sits at u ^ (r & 3), rows of two units: u ^ (r >> 1 & 1) (the transposing read ds_read_b64_tr_b16 takes 4 k-rows of one unit at a time).
#pragma once
#include "mr3d_common.h"

namespace gemm16 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

// one operand of one tile: `base` points at the tile's first row / column and first k; `left` bytes may be read from there (loads
// behind it give zeros); `step` bytes advance one k-step
struct Side {
  const char *base;
  long long left, step;
  unsigned ldb;
};

template <int BI_, int BJ_, int NWI_, int NWJ_, bool IKS_, bool JKS_, bool SPLIT_, int STAGES_> struct Tile {
  static constexpr int BI = BI_, BJ = BJ_, NWI = NWI_, NWJ = NWJ_, NW = NWI * NWJ, THREADS = NW * 64;
  static constexpr bool IKS = IKS_, JKS = JKS_, SPLIT = SPLIT_;
  static constexpr int RB = 128, STAGES = STAGES_;                          // bytes of a KC row per k-step, tiles in LDS
  static constexpr int TI = BI / NWI / 16, TJ = BJ / NWJ / 16;              // 16 x 16 blocks of a wave
  static constexpr int IBYTES = BI * RB, JBYTES = BJ * RB, STAGE = IBYTES + JBYTES, LDS_BYTES = STAGES * STAGE;
  static constexpr int KK = SPLIT ? RB / 4 : RB / 2;                        // k of a k-step
  static constexpr int NLI = IBYTES / 1024 / NW, NLJ = JBYTES / 1024 / NW;  // 1 KB loads of a wave per k-step
  static constexpr int RESTART = SPLIT ? 128 / KK : 0;                     // k-steps between two restarts of the accumulators (0: never)
  static_assert(!SPLIT || TI * TJ <= 16, "accumulators and their sums fit the registers");
  static_assert(IBYTES % (1024 * NW) == 0 && JBYTES % (1024 * NW) == 0, "whole 1 KB loads per wave");
  static_assert(KK % 32 == 0, "whole matrix instructions");
};

// KC: rows [row0, rows) of `row_bytes` bytes (padding to the k-step included), from k-step kstep0 on
template <class T>
__device__ __forceinline__ Side side_kc(const void *p, long long ldb, long long rows, long long row_bytes, long long row0, long long kstep0) {
  const long long off = row0 * ldb + kstep0 * T::RB;
  return {(const char *)p + off, (rows - 1) * ldb + row_bytes - off, T::RB, (unsigned)ldb};
}
// KS: k rows [kstep0 * KK, krows), columns from byte `col_bytes` on
template <class T>
__device__ __forceinline__ Side side_ks(const void *p, long long ldb, long long krows, long long row_bytes, long long col_bytes, long long kstep0) {
  const long long off = kstep0 * T::KK * ldb + col_bytes;
  return {(const char *)p + off, (krows - 1) * ldb + row_bytes - off, T::KK * ldb, (unsigned)ldb};
}

// the same for the 16-byte chunk c of k-row kr in a KS tile with rows of ROWB bytes: four k-rows of a 64-byte unit lie in four different bank
// groups, and k-rows 8 apart in the two halves of one
template <int ROWB> __device__ __forceinline__ int place(int kr, int c) {
  const int u = ROWB >= 256 ? kr & 3 : (kr >> 1) & 1;
  return c ^ (u << 2) ^ (((kr >> 3) & 1) << 1);
}
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// source byte offset of this lane in load q of the wave (BT = tile extent, NL loads per wave)
template <class T, int BT, int NL, bool KS>
__device__ __forceinline__ unsigned source_offset(int wave, int lane, int q, unsigned ldb) {
  const int pos = (wave * NL + q) * 64 + lane;                              // 16-byte slot of the tile
  if constexpr (!KS) {
    constexpr int CPR = T::RB / 16;
    const int row = pos / CPR;
    return row * ldb + (((pos % CPR) ^ swizzle(row)) << 4);
  } else {
    constexpr int ROWB = BT * (T::SPLIT ? 4 : 2), CPR = ROWB / 16;
    const int kr = pos / CPR, c = pos % CPR;
    return kr * ldb + (place<ROWB>(kr, c) << 4);
  }
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

// 64 lanes x 16 bytes to LDS bytes [lds, lds + 1024) in lane order.  In assembly, because the compiler puts a wait for ALL such loads in front of every
// transposing LDS read (it cannot tell the tiles apart); the waits are run()'s own.  M0 holds the LDS address and needs one state in between
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"            // m0 is reserved: the clobber is meant all the same
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop

template <int NL>
__device__ __forceinline__ void stage_load(const Side &s, const unsigned (&off)[NL], unsigned lds) {
  const long long l = s.left;
  const int records = (int)(l < 0 ? 0 : (l > 0x7ffffff0 ? 0x7ffffff0 : l));
  const uint64_t base = (uint64_t)s.base;
  // a raw buffer: no stride, byte offsets checked against `records`; every word is wave-uniform
  const i32x4 rsrc = {__builtin_amdgcn_readfirstlane((int)(uint32_t)base), __builtin_amdgcn_readfirstlane((int)(uint32_t)(base >> 32) & 0xffff),
                      __builtin_amdgcn_readfirstlane(records), 0x00020000};
#pragma unroll
  for (int q = 0; q < NL; ++q) load_to_lds(rsrc, off[q], lds + q * 1024);
}

// fragment of 16 rows (block `b` of the tile) x 32 k (substep ks, plane p): lane l holds row l % 16, k = 8 (l / 16) + 0..7
template <class T, int BT, bool KS>
__device__ __forceinline__ i16x8 fragment(const char *lds, int b, int ks, int p, int lane) {
  if constexpr (!KS) {
    const int row = b * 16 + (lane & 15), chunk = (T::SPLIT ? p * 4 : 0) + ks * 4 + (lane >> 4);
    return *reinterpret_cast<const i16x8 *>(lds + row * T::RB + ((chunk ^ swizzle(row)) << 4));
  } else {
    constexpr int ROWB = BT * (T::SPLIT ? 4 : 2);
    const int s = lane & 15, kr = ks * 32 + (lane >> 4) * 8 + (s >> 2);
    // 16 columns: half a unit; split: the unit pairs of a group of 32 columns are its hi and its lo
    const int chunk = (T::SPLIT ? (b >> 1) * 8 + p * 4 : (b >> 1) * 4) + (b & 1) * 2 + ((s & 3) >> 1);
    const char *a = lds + kr * ROWB + (s & 1) * 8;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(a + (place<ROWB>(kr, chunk) << 4)));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(a + 4 * ROWB + (place<ROWB>(kr + 4, chunk) << 4)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

template <bool SPLIT>
__device__ __forceinline__ f32x4 mfma(i16x8 a, i16x8 b, f32x4 c) {
  if constexpr (SPLIT) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// acc[ti][tj][e] of wave (wi, wj), lane l:  i = (wi TI + ti) 16 + 4 (l / 16) + e,  j = (wj TJ + tj) 16 + l % 16
//
// STAGES - 1 k-steps are on their way while one is multiplied (a trip to L2 or HBM is longer than a k-step of 0.3 - 0.9 us).  Loads past the
// last k-step are issued with an empty range (zeros into a tile nobody reads), so that the count of outstanding loads is the same in every step.
// A wave keeps the J fragments of the current 32 k and the next in registers and passes its I fragments by, AHEAD of them read in advance,
// across the barrier of a k-step too; the reads go between the products (a wave that queues LDS reads issues nothing else).
//
// `weight(part, b)`: a tile that restarts its accumulators may weight what each part (RESTART k-steps) adds to the sums of this lane's j of block b
struct Unweighted {
  __device__ float operator()(int, int) const { return 1.f; }
};
template <class T, class W = Unweighted>
__device__ __forceinline__ void run(char *lds, Side si, Side sj, int nsteps, f32x4 (&acc)[T::TI][T::TJ], W weight = W()) {
  constexpr bool WEIGHTED = !__is_same(W, Unweighted);
  static_assert(!WEIGHTED || T::RESTART, "");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave % T::NWI, wj = wave / T::NWI;
  unsigned oi[T::NLI], oj[T::NLJ];
#pragma unroll
  for (int q = 0; q < T::NLI; ++q) oi[q] = source_offset<T, T::BI, T::NLI, T::IKS>(wave, lane, q, si.ldb);
#pragma unroll
  for (int q = 0; q < T::NLJ; ++q) oj[q] = source_offset<T, T::BJ, T::NLJ, T::JKS>(wave, lane, q, sj.ldb);
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int a = 0; a < T::TI; ++a)
#pragma unroll
    for (int b = 0; b < T::TJ; ++b) acc[a][b] = zero;
  if (nsteps <= 0) return;
  int to_load = nsteps;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane((int)(uintptr_t)(__attribute__((address_space(3))) char *)lds);
  auto load = [&](int buf) {
    if (to_load-- <= 0) si.left = sj.left = 0;
    stage_load<T::NLI>(si, oi, lds0 + buf * T::STAGE + wave * (T::NLI * 1024));
    stage_load<T::NLJ>(sj, oj, lds0 + buf * T::STAGE + T::IBYTES + wave * (T::NLJ * 1024));
    si.base += si.step; si.left -= si.step;
    sj.base += sj.step; sj.left -= sj.step;
  };
  constexpr int NP = T::SPLIT ? 2 : 1, KS = T::KK / 32, POS = KS * T::TI;   // positions of a k-step: (substep, I block)
  constexpr int AHEAD = T::TI < 3 ? T::TI : 3;
  i16x8 fi[AHEAD + 1][NP], fj[2][T::TJ][NP];
  auto fetch_i = [&](int slot, int buf, int pos) {
#pragma unroll
    for (int p = 0; p < NP; ++p) fi[slot][p] = fragment<T, T::BI, T::IKS>(lds + buf * T::STAGE, wi * T::TI + pos % T::TI, pos / T::TI, p, lane);
  };
  auto fetch_j = [&](int which, int buf, int ks, int b) {
#pragma unroll
    for (int p = 0; p < NP; ++p) fj[which][b][p] = fragment<T, T::BJ, T::JKS>(lds + buf * T::STAGE + T::IBYTES, wj * T::TJ + b, ks, p, lane);
  };
#pragma unroll
  for (int k = 0; k < T::STAGES - 1; ++k) load(k);
  // outstanding loads that may remain when stage s + 1 is needed: those of stages s + 2 .. s + STAGES - 1
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((T::STAGES - 2) * (T::NLI + T::NLJ)) : "memory");
  __builtin_amdgcn_s_barrier();
  load(T::STAGES - 1);
#pragma unroll
  for (int b = 0; b < T::TJ; ++b) fetch_j(0, 0, 0, b);
#pragma unroll
  for (int x = 0; x < AHEAD; ++x) fetch_i(x, 0, x);
  int buf = 0;
  f32x4 sum[T::TI][T::TJ];
  if constexpr (T::RESTART) {
#pragma unroll
    for (int a = 0; a < T::TI; ++a)
#pragma unroll
      for (int b = 0; b < T::TJ; ++b) sum[a][b] = zero;
  }
  // registers have no index: a k-step is unrolled as often as it takes for its fragments to sit in the same registers again
  constexpr int RING = POS % (AHEAD + 1) == 0 ? 1 : (2 * POS) % (AHEAD + 1) == 0 ? 2 : AHEAD + 1;
  constexpr int UNR = RING * KS % 2 == 0 ? RING : 2 * RING;
  for (int s0 = 0; s0 < nsteps; s0 += UNR) {
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      if (UNR > 1 && s0 + u >= nsteps) break;
      const int next = buf + 1 == T::STAGES ? 0 : buf + 1;
#pragma unroll
      for (int pos = 0; pos < POS; ++pos) {
        const int g = u * POS + pos, ahead = pos + AHEAD, ks = pos / T::TI, a = pos % T::TI, w = (u * KS + ks) & 1, slot = g % (AHEAD + 1);
        if (ahead == POS) {
          // this wave's last fragments of the step are in registers and its loads of the next stage have landed: behind the barrier both hold for
          // every wave, the step's tile is free
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((T::STAGES - 2) * (T::NLI + T::NLJ)) : "memory");
          __builtin_amdgcn_s_barrier();
          load(buf);
        }
        const bool over = ahead >= POS;
        fetch_i((g + AHEAD) % (AHEAD + 1), over ? next : buf, over ? ahead - POS : ahead);
        // the J fragments of the next substep, a share per position; those of the next k-step behind the barrier
        const bool last_ks = ks == KS - 1;
        const int from = last_ks ? T::TI - AHEAD : 0, share = (T::TJ + T::TI - from - 1) / (T::TI - from);
        if (a >= from) {
#pragma unroll
          for (int b = 0; b < T::TJ; ++b)
            if (b / share == a - from) fetch_j(w ^ 1, last_ks ? next : buf, last_ks ? 0 : ks + 1, b);
        }
#pragma unroll
        for (int b = 0; b < T::TJ; ++b) {
          f32x4 t = acc[a][b];
          if constexpr (T::SPLIT) {                        // small terms first: one rounding at the size of the result instead of three
            t = mfma<true>(fi[slot][0], fj[w][b][1], t);
            t = mfma<true>(fi[slot][1], fj[w][b][0], t);
          }
          t = mfma<T::SPLIT>(fi[slot][0], fj[w][b][0], t);
          acc[a][b] = t;
        }
        constexpr int M = T::TJ * (T::SPLIT ? 3 : 1);
#pragma unroll
        for (int m = 0; m < M; ++m) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      buf = next;
      if constexpr (T::RESTART) {
        if ((s0 + u + 1) % T::RESTART == 0) {
#pragma unroll
          for (int b = 0; b < T::TJ; ++b) {
            const float f = weight((s0 + u) / T::RESTART, b);
#pragma unroll
            for (int a = 0; a < T::TI; ++a) {
              sum[a][b] += WEIGHTED ? acc[a][b] * f : acc[a][b];
              acc[a][b] = zero;
            }
          }
        }
      }
    }
  }
  if constexpr (T::RESTART) {
#pragma unroll
    for (int b = 0; b < T::TJ; ++b) {
      const float f = WEIGHTED && nsteps % T::RESTART ? weight(nsteps / T::RESTART, b) : 1.f;      // no such part: acc is zero
#pragma unroll
      for (int a = 0; a < T::TI; ++a) acc[a][b] = (WEIGHTED ? acc[a][b] * f : acc[a][b]) + sum[a][b];
    }
  }
  // the fragments read last belong to no k-step; the loads of empty ranges must not land in what LDS holds next
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
}

// x = hi + lo in fp16 (x already scaled into fp16's range)
__device__ __forceinline__ void split16(float x, _Float16 &hi, _Float16 &lo) {
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

// Workgroup -> tile order.  Consecutive workgroups go to the 8 XCDs in turn and each XCD has its own L2: give an XCD a contiguous run
// of the order, and let the order walk bands of 8 tiles of one axis so that a run's operand rows stay in that L2
__device__ __forceinline__ void tile_of(int bid, int total, int ti, int tj, int &i, int &j) {
  const int per = total / 8, rest = total % 8, x = bid % 8;
  int t = (x < rest ? x * (per + 1) : rest * (per + 1) + (x - rest) * per) + bid / 8;
  constexpr int BAND = 8;
  const int band = t / (BAND * ti), j0 = band * BAND, w = tj - j0 < BAND ? tj - j0 : BAND;
  t -= band * BAND * ti;
  j = j0 + t % w;
  i = t / w;
}

}  // namespace gemm16
