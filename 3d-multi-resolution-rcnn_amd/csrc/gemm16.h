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
//
// Tiles go from global memory to LDS with direct loads (16 bytes a lane, no register stop), double buffered, one barrier a k-step.
// Such a load writes lane l to base + 16 l, so the bank swizzle is applied to the SOURCE address: in a KC tile the 16-byte chunk c of
// row r sits at slot c ^ ((r >> 1) & 7) (16 consecutive rows read the same c from 16 different bank groups); in a KS tile the 64-byte unit u of
// k-row r sits at u ^ (r & 3) (the transposing read ds_read_b64_tr_b16 takes 4 k-rows of one unit at a time).
#pragma once
#include "mr3d_common.h"

namespace gemm16 {

typedef float f32x16 __attribute__((ext_vector_type(16)));
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

// KC: rows [row0, rows), k-steps from k0 on.  `row_bytes`: bytes of a row that are data (padding to 128 included)
__device__ __forceinline__ Side side_kc(const void *p, long long ldb, long long rows, long long row_bytes, long long row0, long long kstep0) {
  const long long off = row0 * ldb + kstep0 * 128;
  return {(const char *)p + off, (rows - 1) * ldb + row_bytes - off, 128, (unsigned)ldb};
}
// KS: k rows [kstep0 * KR, krows), columns from byte `col_bytes` on
template <bool SPLIT>
__device__ __forceinline__ Side side_ks(const void *p, long long ldb, long long krows, long long row_bytes, long long col_bytes, long long kstep0) {
  constexpr int KR = SPLIT ? 32 : 64;
  const long long off = kstep0 * KR * ldb + col_bytes;
  return {(const char *)p + off, (krows - 1) * ldb + row_bytes - off, KR * ldb, (unsigned)ldb};
}

template <int BI_, int BJ_, int NWI_, int NWJ_, bool IKS_, bool JKS_, bool SPLIT_> struct Tile {
  static constexpr int BI = BI_, BJ = BJ_, NWI = NWI_, NWJ = NWJ_, NW = NWI * NWJ, THREADS = NW * 64;
  static constexpr bool IKS = IKS_, JKS = JKS_, SPLIT = SPLIT_;
  static constexpr int TI = BI / NWI / 32, TJ = BJ / NWJ / 32;              // 32 x 32 blocks of a wave
  static constexpr int IBYTES = BI * 128, JBYTES = BJ * 128, STAGE = IBYTES + JBYTES, LDS_BYTES = 2 * STAGE;
  static constexpr int KK = SPLIT ? 32 : 64;                                // k of a k-step
  static_assert(BI % (8 * NW) == 0 && BJ % (8 * NW) == 0, "whole 1 KB loads per wave");
};

// source byte offset of this lane in load q of the wave (BT = tile extent, NL loads per wave)
template <int BT, int NW, bool KS, bool SPLIT>
__device__ __forceinline__ unsigned source_offset(int wave, int lane, int q, unsigned ldb) {
  constexpr int NL = BT / 8 / NW;
  const int piece = wave * NL + q;
  if constexpr (!KS) {
    const int row = piece * 8 + (lane >> 3);
    return row * ldb + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  } else {
    constexpr int CPR = BT * (SPLIT ? 4 : 2) / 16;                          // 16-byte chunks of a k-row
    const int pos = piece * 64 + lane, kr = pos / CPR, c = pos % CPR;
    return kr * ldb + ((((c >> 2) ^ (kr & 3)) << 6) | ((c & 3) << 4));
  }
}

template <int BT, int NW>
__device__ __forceinline__ void stage_load(const Side &s, const unsigned (&off)[BT / 8 / NW], char *lds, int wave) {
  constexpr int NL = BT / 8 / NW;
  const long long l = s.left;
  const int records = (int)(l < 0 ? 0 : (l > 0x7ffffff0 ? 0x7ffffff0 : l));
  __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(s.base), 0, records, 0x00020000);
#pragma unroll
  for (int q = 0; q < NL; ++q)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(lds + (wave * NL + q) * 1024), 16, (int)off[q], 0, 0, 0);
}

// fragment of 32 rows (block `b` of the tile) x 16 k (substep ks, plane p): lane l holds row l % 32, k = 8 (l / 32) + 0..7
template <int BT, bool KS, bool SPLIT>
__device__ __forceinline__ i16x8 fragment(const char *lds, int b, int ks, int p, int lane) {
  if constexpr (!KS) {
    const int row = lane & 31, chunk = (SPLIT ? p * 4 : 0) + ks * 2 + (lane >> 5);
    return *reinterpret_cast<const i16x8 *>(lds + b * 4096 + row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4));
  } else {
    constexpr int ROWB = BT * (SPLIT ? 4 : 2);
    const int s = lane & 15, j = s >> 2, unit = SPLIT ? b * 2 + p : b;
    const char *a = lds + (ks * 16 + (lane >> 5) * 8 + j) * ROWB + ((unit ^ j) << 6) + ((lane >> 4) & 1) * 32 + (s & 3) * 8;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)a);
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(a + 4 * ROWB));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

template <bool SPLIT>
__device__ __forceinline__ f32x16 mfma(i16x8 a, i16x8 b, f32x16 c) {
  if constexpr (SPLIT) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// acc[ti][tj][e] of wave (wi, wj), lane l:  i = (wi TI + ti) 32 + 8 (e / 4) + 4 (l / 32) + e % 4,  j = (wj TJ + tj) 32 + l % 32
template <class T>
__device__ __forceinline__ void run(char *lds, Side si, Side sj, int nsteps, f32x16 (&acc)[T::TI][T::TJ]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave % T::NWI, wj = wave / T::NWI;
  constexpr int NLI = T::BI / 8 / T::NW, NLJ = T::BJ / 8 / T::NW;
  unsigned oi[NLI], oj[NLJ];
#pragma unroll
  for (int q = 0; q < NLI; ++q) oi[q] = source_offset<T::BI, T::NW, T::IKS, T::SPLIT>(wave, lane, q, si.ldb);
#pragma unroll
  for (int q = 0; q < NLJ; ++q) oj[q] = source_offset<T::BJ, T::NW, T::JKS, T::SPLIT>(wave, lane, q, sj.ldb);
#pragma unroll
  for (int a = 0; a < T::TI; ++a)
#pragma unroll
    for (int b = 0; b < T::TJ; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
  if (nsteps <= 0) return;
  auto load = [&](int buf) {
    stage_load<T::BI, T::NW>(si, oi, lds + buf * T::STAGE, wave);
    stage_load<T::BJ, T::NW>(sj, oj, lds + buf * T::STAGE + T::IBYTES, wave);
    si.base += si.step; si.left -= si.step;
    sj.base += sj.step; sj.left -= sj.step;
  };
  load(0);
  for (int s = 0; s < nsteps; ++s) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // this wave's part of stage s has landed
    __syncthreads();                                       // everyone's has, and the other buffer is free
    if (s + 1 < nsteps) load((s + 1) & 1);
    const char *li = lds + (s & 1) * T::STAGE, *lj = li + T::IBYTES;
#pragma unroll
    for (int ks = 0; ks < T::KK / 16; ++ks) {
      constexpr int NP = T::SPLIT ? 2 : 1;
      i16x8 fi[T::TI][NP], fj[T::TJ][NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
#pragma unroll
        for (int b = 0; b < T::TJ; ++b) fj[b][p] = fragment<T::BJ, T::JKS, T::SPLIT>(lj, wj * T::TJ + b, ks, p, lane);
#pragma unroll
        for (int a = 0; a < T::TI; ++a) fi[a][p] = fragment<T::BI, T::IKS, T::SPLIT>(li, wi * T::TI + a, ks, p, lane);
      }
#pragma unroll
      for (int a = 0; a < T::TI; ++a)
#pragma unroll
        for (int b = 0; b < T::TJ; ++b) {
          if constexpr (T::SPLIT) {                        // small terms first: one rounding at the size of the result instead of three
            acc[a][b] = mfma<true>(fi[a][0], fj[b][1], acc[a][b]);
            acc[a][b] = mfma<true>(fi[a][1], fj[b][0], acc[a][b]);
          }
          acc[a][b] = mfma<T::SPLIT>(fi[a][0], fj[b][0], acc[a][b]);
        }
    }
  }
  __syncthreads();                                         // LDS is the caller's again
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
