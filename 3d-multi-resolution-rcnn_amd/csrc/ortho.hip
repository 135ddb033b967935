// Orthogonalised updates: Newton-Schulz products of a LIST of matrices, all of them in one launch per stage.
//   X = G / (|G|_F + eps), wide (m <= n; a tall G is read transposed);  steps times:  A = X X^T,  P = a I + b A + c A A,  X = P X
//
// Up to 64 rows (small path): three launches.  The iteration is a function of A alone, X = Q(A) G, so A is formed once in DOUBLE, all steps run
// on the m x m matrices in one workgroup's LDS (A <- P A P, Q <- P Q: polynomials of A commute, products of them are symmetric), and Q is applied
// once.  Double, because the noise of A is amplified by a^2 a step where singular values are small: fp32 loses 1e-5 .. 1e-4 over five steps.
// It also gives |G|_F = sqrt(trace A) without overflow.
//
// Larger ones: every factor is kept as two fp16 planes (gemm16.h, split storage), scaled by powers of two into fp16's range: 22 bits (of X down to
// steps of 2^-36 |G|_F, of A and P 2^-36 and 2^-34), three passes of the 16-bit matrix pipe, fp32 accumulators.  Plain bf16 or fp16 factors would lose 2e-2 / 2e-3 of the result over five steps (p's slope at 0
// is a = 3.4: rounding errors of the first steps are amplified a few hundred times).  Symmetric results: only the tiles on and below the diagonal are
// computed and stored twice.  Iterating on A here too, in rounds of two or three steps between looks at X, was measured: 1.6 to 2.4 times fewer
// products at n = 9 m, but no less time for the 64 matrices of a detector (the m x m products are short), and A's noise, amplified,
// takes the result from 1.0e-6 to 2.5e-6 (two steps) or 5e-6 (three) where plain fp32 loses 1.6e-6.
// In bf16 lists the last two steps with the hi planes alone were measured too: 4096 x 4096 3.92 -> 3.52 ms (such tiles wait for their loads: half of every
// cache line is unused), the error against 64 bits 1.12 times that of rounding the result: not taken.
// MFMA-bound on large matrices; on small ones the dependent launches are what counts, hence the list and the small path.
// Measured: 64 x 1728 70 us (A 9, the iteration 46: 17 products of 1.3 us of the double matrix pipe each and their barriers; Q G 12), 777 x 2311 and
// 333 x 1301 277 us (15 products of 13 to 22 us), the 64 matrices of a detector (179 GFLOP) 0.96 ms, 4096 x 4096 bf16 3.8 to 3.9 ms (1.06 PFLOP/s of passes).
#include "gemm16.h"
#include <new>

using namespace gemm16;

namespace {

// powers of two that bring X, A and P into fp16's range: |X| < 16, |A| < 16, |P| < 64
constexpr float kSX = 4096.f, kSA = 4096.f, kSP = 1024.f;
constexpr int kSmall = 64;                                  // rows of the small path
constexpr int kThreads = 256;

// 128 x 128 with two tiles in LDS, two workgroups a CU, or 64 x 64 with three and as many workgroups
template <int BT, bool APPLY> struct Pick { typedef Tile<BT, BT, 2, 2, APPLY, false, true, BT == 128 ? 2 : 3> T; };

enum Stage { kNorm, kPack, kGram, kGramJoin, kSquare, kSquareJoin, kApply, kApplyJoin, kSmallGram, kSmallPoly, kSmallApply, kStages };
enum Buf { kA, kP, kX0, kX1, kBufs };

// tiles [0, whole) are computed by one workgroup each, the others by z workgroups with a share of the k-steps; their parts are joined afterwards
struct Split { int tiles, whole, z; };

struct Mat {
  long long in, out;                                        // places: bytes from the workspace (also the caller's matrices)
  long long in_i, in_j, out_i, out_j;                       // element strides along n (i) and m (j)
  long long buf[kBufs];                                     // planes
  long long part;                                           // parts of split tiles, [tile - whole][z][BT * BT] floats
  long long norm;                                           // doubles; small path: parts of A, [z][mp][64], then Q
  int m, n, ldx, lda;                                       // ld in bytes
  int bf16, norm_blocks;
  Split gram, square, apply;
  int first[kStages];                                       // first workgroup of this matrix in each stage
};
static_assert(sizeof(Mat) <= 240, "fifteen of them, and the maps, are kernel arguments (4 KB)");

struct Plan {
  int blocks[kStages];
  int bt_square, bt_gram, bt_apply;
  size_t bytes, mats_off, map_off[kStages];
};

constexpr int kBatch = 15;
struct MatBatch { Mat m[kBatch]; };

// Places are stored as distances from the workspace, a kernel argument: a pointer read from the table would count as generic, and generic (flat)
// accesses wait for LDS and memory alike, one after the other
template <class T> __device__ __forceinline__ T *at(char *ws, long long place) { return reinterpret_cast<T *>(ws + place); }

__device__ __forceinline__ int triangle(int t, int &ti) {
  int tj = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while ((tj + 1) * (tj + 2) / 2 <= t) ++tj;
  while (tj * (tj + 1) / 2 > t) --tj;
  ti = t - tj * (tj + 1) / 2;
  return tj;
}

// The table in memory and, per stage, workgroup -> matrix.  A launch takes a batch of matrices as arguments and fills in both for its own: workgroups
// from its first matrix's first one to `end`
struct Maps { int *map[kStages]; int end[kStages]; };
__global__ __launch_bounds__(256) void ortho_table_kernel(MatBatch batch, int count, int at, Mat *__restrict__ mats, Maps maps) {
  const int s = blockIdx.y;
  if (s == 0 && blockIdx.x == 0 && (int)threadIdx.x < count) mats[at + threadIdx.x] = batch.m[threadIdx.x];
  for (int b = batch.m[0].first[s] + blockIdx.x * 256 + threadIdx.x; b < maps.end[s]; b += gridDim.x * 256) {
    int k = 0;                                              // the last matrix whose first workgroup is <= b
    for (int i = 1; i < count; ++i) k = batch.m[i].first[s] <= b ? i : k;
    maps.map[s][b] = at + k;
  }
}

__device__ __forceinline__ float read_in(char *ws, const Mat &p, long long off) {
  return p.bf16 ? (float)at<const __bf16>(ws, p.in)[off] : at<const float>(ws, p.in)[off];
}

// squares of the input in double: fp32 squares would overflow from 2^64 on
__global__ __launch_bounds__(256) void ortho_norm_kernel(char *ws, const Mat *__restrict__ mats, const int *__restrict__ map) {
  const Mat p = mats[map[blockIdx.x]];
  const int chunk = blockIdx.x - p.first[kNorm];
  const bool wide = p.in_i == 1;                            // walk the contiguous axis with the threads
  const int inner = wide ? p.n : p.m, outer = wide ? p.m : p.n;
  const long long si = wide ? 1 : p.in_j, so = wide ? p.in_j : p.in_i;
  const long long total = (long long)inner * outer;
  double s = 0;
  long long e = (long long)chunk * 256 + threadIdx.x;
  const long long stride = (long long)p.norm_blocks * 256;
  if (si == 1 && so == inner && ((uintptr_t)(ws + p.in) & 15) == 0) {            // packed: 16 bytes a load
    const int per = p.bf16 ? 8 : 4;
    const long long groups = total / per;
#pragma unroll 2
    for (; e < groups; e += stride) {
      float v[8];
      if (p.bf16) {
        const bf16x8 t = at<const bf16x8>(ws, p.in)[e];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)t[k];
      } else {
        const float4 t = at<const float4>(ws, p.in)[e];
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        v[4] = v[5] = v[6] = v[7] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s += (double)v[k] * (double)v[k];
    }
    for (e = groups * per + (long long)chunk * 256 + threadIdx.x; e < total; e += stride) {
      const double v = (double)read_in(ws, p, e);
      s += v * v;
    }
  } else {
    for (; e < total; e += stride) {
      const int o = (int)(e / inner), i = (int)(e - (long long)o * inner);
      const double v = (double)read_in(ws, p, o * so + i * si);
      s += v * v;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  __shared__ double w[4];
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) at<double>(ws, p.norm)[chunk] = w[0] + w[1] + w[2] + w[3];
}

constexpr int kChunk = 64;                                  // columns of X in LDS

// rows [0, 64) x columns [i0, i0 + 64) of the wide matrix, zeros outside -> t[row][col]; read along the contiguous axis, 16 loads a thread in flight
__device__ __forceinline__ void load_tile(char *ws, const Mat *__restrict__ p, int i0, int j0, float (*t)[kChunk + 1]) {
  const long long si = p->in_i, sj = p->in_j;
  const bool wide = si == 1;
  const int fast = threadIdx.x & 63, slow = threadIdx.x >> 6, m = p->m - j0, n = p->n - i0;
  const long long base = i0 * si + j0 * sj;
  float v[16];
  auto each = [&](auto *in) {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int q = wide ? fast : slow + 4 * k, r = wide ? slow + 4 * k : fast;
      v[k] = q < n && r < m ? (float)in[base + q * si + r * sj] : 0.f;
    }
  };
  if (p->bf16) each(at<const __bf16>(ws, p->in));
  else each(at<const float>(ws, p->in));
#pragma unroll
  for (int k = 0; k < 16; ++k) t[wide ? slow + 4 * k : fast][wide ? fast : slow + 4 * k] = v[k];
}

// 64 x 64 of the input -> planes of X; the tile goes through LDS so that a tall input is read along its rows too
__global__ __launch_bounds__(256) void ortho_pack_kernel(char *ws, const Mat *__restrict__ mats, const int *__restrict__ map, float eps) {
  __shared__ float t[64][65];
  __shared__ double w[4];
  const Mat p = mats[map[blockIdx.x]];
  const int tile = blockIdx.x - p.first[kPack], tn = (p.n + 63) / 64;
  const int j0 = tile / tn * 64, i0 = tile % tn * 64;
  double s = 0;
  for (int k = threadIdx.x; k < p.norm_blocks; k += 256) s += at<double>(ws, p.norm)[k];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  load_tile(ws, mats + map[blockIdx.x], i0, j0, t);
  __syncthreads();
  const double scale = (double)kSX / (sqrt(w[0] + w[1] + w[2] + w[3]) + (double)eps);      // may leave fp32's range where G does not
  const int np = (p.n + 31) / 32 * 32;
  for (int k = threadIdx.x; k < 64 * 16; k += 256) {
    const int j = k >> 4, i = (k & 15) * 4;
    if (j0 + j >= p.m || i0 + i >= np) continue;
    _Float16 h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split16((float)((double)t[j][i + e] * scale), h[e], l[e]);
    char *d = ws + p.buf[kX0] + (long long)(j0 + j) * p.ldx + (i0 + i) / 32 * 128 + (i & 31) * 2;
    *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<uint2 *>(h);
    *reinterpret_cast<uint2 *>(d + 64) = *reinterpret_cast<uint2 *>(l);
  }
}

// four consecutive columns of a row, as planes
__device__ __forceinline__ void store_planes(char *row, int i, const float (&v)[4]) {
  _Float16 h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) split16(v[e], h[e], l[e]);
  char *d = row + (i >> 5) * 128 + (i & 31) * 2;
  *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<uint2 *>(h);
  *reinterpret_cast<uint2 *>(d + 64) = *reinterpret_cast<uint2 *>(l);
}
__device__ __forceinline__ void load_planes(const char *row, int i, float (&v)[4]) {
  const char *d = row + (i >> 5) * 128 + (i & 31) * 2;
  const uint2 h = *reinterpret_cast<const uint2 *>(d), l = *reinterpret_cast<const uint2 *>(d + 64);
  const _Float16 *hh = reinterpret_cast<const _Float16 *>(&h), *ll = reinterpret_cast<const _Float16 *>(&l);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)hh[e] + (float)ll[e];
}

// The three products of a step.  kind 0: A = X X^T.  1: P = a I + b A + c A A (symmetric too; alpha acc + beta A + gamma I in raw plane values).
// 2: alpha P X, to planes or (last) to the caller's matrix
struct Op {
  int x;                                                    // buffer of X
  float alpha, beta, gamma;
  int last;
};

// 16 x 16 block (bi, bj) of tile (ti, tj), one accumulator of a wave
template <int KIND, int BT>
__device__ __forceinline__ void finish_block(char *ws, const Mat *__restrict__ mat, const Op &op, int ti, int tj, int bi, int bj, const f32x4 &acc) {
  const int lane = threadIdx.x & 63, m = mat->m;
  const int j = tj * BT + bj * 16 + (lane & 15), i = ti * BT + bi * 16 + (lane >> 4) * 4;
  float v[4];
  if constexpr (KIND < 2) {
    const int mp = (m + 31) / 32 * 32, lda = mat->lda;
    char *dst = ws + mat->buf[KIND == 0 ? kA : kP];
    if constexpr (KIND == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = op.alpha * acc[e];
    } else {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (j < m && i < mp) load_planes(ws + mat->buf[kA] + (long long)j * lda, i, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = op.alpha * acc[e] + op.beta * f[e] + (i + e == j ? op.gamma : 0.f);
    }
    if (j < m && i < mp) store_planes(dst + (long long)j * lda, i, v);
    if (ti != tj && j < mp) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < m) {
          _Float16 h, l;
          split16(v[e], h, l);
          _Float16 *d = reinterpret_cast<_Float16 *>(dst + (long long)(i + e) * lda + (j >> 5) * 128) + (j & 31);
          d[0] = h;
          d[32] = l;
        }
    }
  } else {
    if (j >= m) return;
    const int n = mat->n, np = (n + 31) / 32 * 32;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = acc[e] * op.alpha;
    if (!op.last) {
      if (i < np) store_planes(ws + mat->buf[op.x == kX0 ? kX1 : kX0] + (long long)j * mat->ldx, i, v);
    } else {
      const long long oj = mat->out_j, oi = mat->out_i;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) {
          const long long k = j * oj + (i + e) * oi;
          if (mat->bf16) at<__bf16>(ws, mat->out)[k] = (__bf16)v[e];
          else at<float>(ws, mat->out)[k] = v[e];
        }
    }
  }
}

template <int KIND> __device__ __forceinline__ Split split_of(const Mat *__restrict__ m) { return KIND == 0 ? m->gram : KIND == 1 ? m->square : m->apply; }

template <int KIND, int BT>
__device__ __forceinline__ void tile_at(const Mat *__restrict__ mat, int t, int &ti, int &tj) {
  if constexpr (KIND < 2) {
    tj = triangle(t, ti);
  } else {
    const int tm = (mat->m + BT - 1) / BT;
    tj = t % tm;
    ti = t / tm;
  }
}

template <int KIND, int BT>
__global__ __launch_bounds__(kThreads, 2) void ortho_product_kernel(char *ws, const Mat *__restrict__ mats, const int *__restrict__ map, Op op) {
  typedef typename Pick<BT, KIND == 2>::T T;
  constexpr int kFirst = KIND == 0 ? kGram : KIND == 1 ? kSquare : kApply;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int b = blockIdx.x;
  const Mat *__restrict__ mat = mats + map[b];
  const Split sp = split_of<KIND>(mat);
  const int local = b - mat->first[kFirst], m = mat->m;
  int t = local, zi = 0, z = 1;
  if (local >= sp.whole) {
    z = sp.z;
    t = sp.whole + (local - sp.whole) / z;
    zi = (local - sp.whole) % z;
  }
  int ti, tj;
  tile_at<KIND, BT>(mat, t, ti, tj);
  const int total = ((KIND == 0 ? mat->n : m) + 31) / 32;
  const int s0 = (int)((long long)total * zi / z), s1 = (int)((long long)total * (zi + 1) / z);
  const int ldl = KIND == 1 ? mat->lda : mat->ldx, ldr = KIND == 0 ? mat->ldx : mat->lda;
  const char *l = ws + mat->buf[KIND == 1 ? kA : op.x], *r = ws + mat->buf[KIND == 0 ? op.x : KIND == 1 ? kA : kP];
  f32x4 acc[T::TI][T::TJ];
  if constexpr (KIND == 2) run<T>(lds, side_ks<T>(l, ldl, m, ldl, (long long)ti * BT * 4, s0), side_kc<T>(r, ldr, m, ldr, tj * BT, s0), s1 - s0, acc);
  else run<T>(lds, side_kc<T>(l, ldl, m, ldl, ti * BT, s0), side_kc<T>(r, ldr, m, ldr, tj * BT, s0), s1 - s0, acc);
  const int wave = threadIdx.x >> 6, wi = wave % T::NWI, wj = wave / T::NWI;
  if (z == 1) {
#pragma unroll
    for (int x = 0; x < T::TI; ++x)
#pragma unroll
      for (int y = 0; y < T::TJ; ++y) finish_block<KIND, BT>(ws, mat, op, ti, tj, wi * T::TI + x, wj * T::TJ + y, acc[x][y]);
  } else {
    f32x4 *d = at<f32x4>(ws, mat->part) + ((long long)(t - sp.whole) * z + zi) * (BT * BT / 4) + threadIdx.x;
#pragma unroll
    for (int x = 0; x < T::TI; ++x)
#pragma unroll
      for (int y = 0; y < T::TJ; ++y) d[(x * T::TJ + y) * kThreads] = acc[x][y];
  }
}

// the parts of split tiles, added in a fixed order; a workgroup takes four 16 x 16 blocks of every wave
template <int KIND, int BT>
__global__ __launch_bounds__(kThreads) void ortho_join_kernel(char *ws, const Mat *__restrict__ mats, const int *__restrict__ map, Op op) {
  typedef typename Pick<BT, KIND == 2>::T T;
  constexpr int kFirst = KIND == 0 ? kGramJoin : KIND == 1 ? kSquareJoin : kApplyJoin, Q = T::TI * T::TJ / 4;
  const int b = blockIdx.x;
  const Mat *__restrict__ mat = mats + map[b];
  const Split sp = split_of<KIND>(mat);
  const int local = b - mat->first[kFirst], u = local / Q, q = local % Q;
  int ti, tj;
  tile_at<KIND, BT>(mat, sp.whole + u, ti, tj);
  const f32x4 *s = at<const f32x4>(ws, mat->part) + (long long)u * sp.z * (BT * BT / 4) + q * 4 * kThreads + threadIdx.x;
  f32x4 acc[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) acc[k] = s[k * kThreads];
  for (int zi = 1; zi < sp.z; zi += 2) {                    // 8 loads of 16 bytes in flight
    const f32x4 *s1 = s + (long long)zi * (BT * BT / 4);
    const bool two = zi + 1 < sp.z;
    const f32x4 *s2 = two ? s1 + BT * BT / 4 : s1;
    f32x4 x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = s1[k * kThreads];
      y[k] = s2[k * kThreads];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      acc[k] += x[k];
      if (two) acc[k] += y[k];
    }
  }
  const int wave = threadIdx.x >> 6, wi = wave % T::NWI, wj = wave / T::NWI;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    finish_block<KIND, BT>(ws, mat, op, ti, tj, wi * T::TI + (q * 4 + k) / T::TJ, wj * T::TJ + (q * 4 + k) % T::TJ, acc[k]);
}

// ------------------------------------------------------------------------------------------------ small path
typedef double f64x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int pad16(int m) { return (m + 15) / 16 * 16; }

// share z of the lower triangle of A = G G^T: v_mfma_f64_16x16x4_f64.  Lane l holds row l % 16, k = l / 16 of a factor, and column l % 16,
// rows l / 16 + 0, 4, 8, 12 of the result
__global__ __launch_bounds__(kThreads) void ortho_small_gram_kernel(char *ws, const Mat *__restrict__ mats, const int *__restrict__ map) {
  __shared__ float t[kSmall][kChunk + 1];
  const Mat *__restrict__ p = mats + map[blockIdx.x];
  const int zi = blockIdx.x - p->first[kSmallGram], z = p->gram.z, mp = pad16(p->m), nb = mp / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kq = lane >> 4;
  const int blocks = nb * (nb + 1) / 2;                     // on and below the diagonal: at most 10, three a wave
  int bi[3], bj[3];
  f64x4 acc[3];
#pragma unroll
  for (int b = 0; b < 3; ++b) {
    bi[b] = triangle(min(wave + 4 * b, blocks - 1), bj[b]);
    acc[b] = f64x4{0, 0, 0, 0};
  }
  const int chunks = (p->n + kChunk - 1) / kChunk;
  for (int c = zi; c < chunks; c += z) {
    __syncthreads();
    load_tile(ws, p, c * kChunk, 0, t);
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < kChunk; k += 4) {
#pragma unroll
      for (int b = 0; b < 3; ++b)
        if (wave + 4 * b < blocks)
          acc[b] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)t[bi[b] * 16 + r][k + kq], (double)t[bj[b] * 16 + r][k + kq], acc[b], 0, 0, 0);
    }
  }
  double *o = at<double>(ws, p->norm) + zi * mp * kSmall;
#pragma unroll
  for (int b = 0; b < 3; ++b)
    if (wave + 4 * b < blocks)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = bi[b] * 16 + 4 * e + kq, j = bj[b] * 16 + r;
        if (i >= j) o[i * kSmall + j] = acc[b][e];
      }
}

constexpr int kPolyThreads = 1024, kLdd = kSmall + 2;        // doubles of an LDS row

// m[out] = alpha m[l] m[r] (+ beta m[add] + gamma I): symmetric, the blocks on and below the diagonal are computed and stored twice.  Matrices
// go by their place in LDS, not by pointers: selected pointers would be read as generic ones
template <int NB>
__device__ __forceinline__ void small_product(double (*m)[kSmall * kLdd], int l, int r, int out, int add, double alpha, double beta, double gamma) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane & 15, kq = lane >> 4;
  __syncthreads();
  if (wave < NB * (NB + 1) / 2) {                           // a wave per block (bi >= bj)
    const int bi = wave < 1 ? 0 : wave < 3 ? 1 : wave < 6 ? 2 : 3, bj = wave - bi * (bi + 1) / 2;
    const double *pl = m[l] + (bi * 16 + q) * kLdd + kq, *pr = m[r] + (bj * 16 + q) * kLdd + kq;
    double fl[NB * 4], fr[NB * 4];
#pragma unroll
    for (int k = 0; k < NB * 4; ++k) {
      fl[k] = pl[4 * k];
      fr[k] = pr[4 * k];
    }
    f64x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NB * 4; ++k) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(fl[k], fr[k], acc, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = bi * 16 + 4 * e + kq, j = bj * 16 + q;
      const double v = alpha * acc[e] + (add >= 0 ? beta * m[add < 0 ? 0 : add][i * kLdd + j] : 0.) + (i == j ? gamma : 0.);
      if (i < j) continue;                                  // a block on the diagonal: its upper half is the lower one's copy
      m[out][i * kLdd + j] = v;
      m[out][j * kLdd + i] = v;
    }
  }
  __syncthreads();
}

// A in m[0] -> Q; returns its place
template <int NB>
__device__ __forceinline__ int small_steps(double (*m)[kSmall * kLdd], int steps, float ca, float cb, float cc) {
  int q = -1;
  for (int s = 0; s < steps; ++s) {
    const int pn = q >= 0 ? 1 : 2;                          // the first polynomial is Q itself
    small_product<NB>(m, 0, 0, pn, 0, cc, cb, ca);
    if (s + 1 < steps) {                                    // A <- P A P by way of the free buffer
      const int tmp = q == 3 ? 2 : 3;
      small_product<NB>(m, pn, 0, tmp, -1, 1., 0., 0.);
      small_product<NB>(m, pn, tmp, 0, -1, 1., 0., 0.);
    }
    if (q >= 0) {
      const int nq = q == 2 ? 3 : 2;
      small_product<NB>(m, pn, q, nq, -1, 1., 0., 0.);
      q = nq;
    } else {
      q = 2;
    }
  }
  return q;
}

// all steps of one matrix: A -> Q, stored behind the parts of A
__global__ __launch_bounds__(kPolyThreads) void ortho_small_poly_kernel(char *ws, const Mat *__restrict__ mats, const int *__restrict__ map, int steps, float ca, float cb,
                                                                        float cc, float eps) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  __shared__ double trace;
  const Mat *__restrict__ p = mats + map[blockIdx.x];
  const int m = p->m, mp = pad16(m), z = p->gram.z;
  auto mats4 = reinterpret_cast<double (*)[kSmall * kLdd]>(lds);
  double *a = mats4[0];
  double s[4] = {0, 0, 0, 0};                               // 4 elements a thread, 32 loads in flight
  const double *part = at<double>(ws, p->norm);
  const int size = mp * kSmall;                             // rows of 64: no divisions
  for (int z0 = 0; z0 < z; z0 += 8) {
    double v[8][4];
#pragma unroll
    for (int y = 0; y < 8; ++y)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = threadIdx.x + k * kPolyThreads;
        v[y][k] = e < size && e / kSmall >= e % kSmall && z0 + y < z ? part[(z0 + y) * size + e] : 0.;
      }
#pragma unroll
    for (int y = 0; y < 8; ++y)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += v[y][k];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = threadIdx.x + k * kPolyThreads, i = e / kSmall, j = e % kSmall;
    if (e < size && i >= j) a[i * kLdd + j] = a[j * kLdd + i] = s[k];
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    double t = (int)threadIdx.x < m ? a[threadIdx.x * kLdd + threadIdx.x] : 0.;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
    if (threadIdx.x == 0) trace = t;
  }
  __syncthreads();
  const double inv = 1. / (sqrt(trace) + (double)eps);
  for (int k = threadIdx.x; k < size; k += kPolyThreads)
    if (k % kSmall < mp) a[k / kSmall * kLdd + k % kSmall] *= inv * inv;
  int q;
  switch (mp / 16) {
    case 1: q = small_steps<1>(mats4, steps, ca, cb, cc); break;
    case 2: q = small_steps<2>(mats4, steps, ca, cb, cc); break;
    case 3: q = small_steps<3>(mats4, steps, ca, cb, cc); break;
    default: q = small_steps<4>(mats4, steps, ca, cb, cc);
  }
  double *o = at<double>(ws, p->norm) + z * size;
  for (int k = threadIdx.x; k < size; k += kPolyThreads)
    if (k % kSmall < mp) o[k] = mats4[q][k / kSmall * kLdd + k % kSmall] * inv;
}

// acc = Q t for the 16 columns from c0 on
template <int NB> __device__ __forceinline__ void small_apply(double (*q)[kSmall + 2], float (*t)[kChunk + 1], int c0, f64x4 (&acc)[4]) {
  const int r = threadIdx.x & 15, kq = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f64x4{0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < NB * 16; k += 4) {
    const double x = (double)t[k + kq][c0 + r];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = __builtin_amdgcn_mfma_f64_16x16x4f64(q[b * 16 + r][k + kq], x, acc[b], 0, 0, 0);
  }
}

// out = Q G, 64 columns a workgroup, in double too: Q reaches a^steps in the directions of small singular values, and its rounding to fp32 would show in
// the others (1e-6).  Wave w has the columns 16 w .. 16 w + 15
__global__ __launch_bounds__(kThreads) void ortho_small_apply_kernel(char *ws, const Mat *__restrict__ mats, const int *__restrict__ map) {
  __shared__ float t[kSmall][kChunk + 1];
  __shared__ double q[kSmall][kSmall + 2];
  const Mat *__restrict__ p = mats + map[blockIdx.x];
  const int m = p->m, n = p->n, mp = pad16(m), nb = mp / 16, i0 = (blockIdx.x - p->first[kSmallApply]) * kChunk;
  const double *qs = at<double>(ws, p->norm) + p->gram.z * mp * kSmall;
#pragma unroll
  for (int k = 0; k < kSmall * kSmall / kThreads; ++k) {
    const int e = threadIdx.x + k * kThreads;
    if (e / kSmall < mp && e % kSmall < mp) q[e / kSmall][e % kSmall] = qs[e];
  }
  load_tile(ws, p, i0, 0, t);
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kq = lane >> 4;
  f64x4 acc[4];
  switch (nb) {
    case 1: small_apply<1>(q, t, wave * 16, acc); break;
    case 2: small_apply<2>(q, t, wave * 16, acc); break;
    case 3: small_apply<3>(q, t, wave * 16, acc); break;
    default: small_apply<4>(q, t, wave * 16, acc);
  }
  __syncthreads();
#pragma unroll
  for (int b = 0; b < 4; ++b)
    if (b < nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) t[b * 16 + 4 * e + kq][wave * 16 + r] = (float)acc[b][e];
  __syncthreads();
  const bool wide = p->out_i == 1;
  const long long oi = p->out_i, oj = p->out_j;
  const int f32 = !p->bf16;
  char *out = ws + p->out;
#pragma unroll 4
  for (int k = threadIdx.x; k < kSmall * kChunk; k += kThreads) {
    const int c = wide ? k % 64 : k / 64, j = wide ? k / 64 : k % 64;
    if (j >= m || i0 + c >= n) continue;
    const long long e = j * oj + (i0 + c) * oi;
    if (f32) ((float *)out)[e] = t[j][c];
    else ((__bf16 *)out)[e] = (__bf16)t[j][c];
  }
}

size_t take(size_t &at, size_t bytes) {
  const size_t here = at;
  at = mr3d_align_up(at + bytes, 256);
  return here;
}

// Splitting the k axis.  What a list (or its last round of workgroups) leaves idle is filled by computing tiles with z workgroups each: their parts travel
// through memory and back at 4 TB/s and are joined by another launch of 6 us.
//
// A list of fewer tiles than run at a time (512 of the 128-wide ones, 768 of the 64-wide ones): parts of about `len` k-steps for every matrix, so that long
// and short axes end together.  A k-step takes 0.7 us while a 128-wide tile has its CU alone, and as much longer as there are more on it; 64-wide tiles
// 0.34 us alone, 0.5 for two and 0.7 for three a CU
struct Work { long long tiles; int steps; };
Work work_of(const mr3d_matrix &g, int kind, int bt) {
  const long long m = g.rows < g.cols ? g.rows : g.cols, n = g.rows < g.cols ? g.cols : g.rows, tm = (m + bt - 1) / bt, tn = (n + bt - 1) / bt;
  if (m <= kSmall) return {0, 0};
  return {kind < 2 ? tm * (tm + 1) / 2 : tm * tn, (int)(((kind == 0 ? n : m) + 31) / 32)};
}
int part_length(const mr3d_matrix *in, int count, int kind, int bt, double &best) {
  int longest = 0;
  double total = 0;
  for (int k = 0; k < count; ++k) {
    const Work w = work_of(in[k], kind, bt);
    longest = w.steps > longest ? w.steps : longest;
    total += (double)w.tiles * w.steps;
  }
  const double part_us = bt * bt * 8. / 4e6;
  best = 1e30;
  int best_len = longest;
  for (const int div : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32}) {
    const int len = (longest + div - 1) / div;
    if (len < 4) break;
    double us = 0;
    for (int k = 0; k < count && div > 1; ++k) {
      const Work w = work_of(in[k], kind, bt);
      if (w.steps > len) us += part_us * (double)w.tiles * ((w.steps + len - 1) / len);
    }
    const double c = total / (256. * (double)len);          // workgroups a CU
    const double step = bt == 128 ? 0.7 * (c > 1 ? c : 1) : c <= 1 ? 0.34 : c <= 2 ? 0.34 + 0.16 * (c - 1) : 0.5 + 0.2 * (c - 2);
    us += (double)len * step + (div > 1 ? 6. : 0.);
    if (us < best) {
      best = us;
      best_len = len;
    }
  }
  return best_len;
}

// One matrix's share.  len > 0: parts of that many k-steps.  len 0 (a list that fills whole rounds of workgroups): the tiles left over after them, taken
// from the list's largest matrix, for the z with the least estimated time (4096 x 4096: 528 tiles on and below the diagonal, 240 -> 202 us)
Split split_for(int tiles, int steps, int len, long long list_tiles, bool carries_rest, int bt) {
  Split s{tiles, tiles, 1};
  if (len) {
    int z = (steps + len - 1) / len;
    z = z > 32 ? 32 : z;
    if (z > 1) {
      s.z = z;
      s.whole = 0;
    }
    return s;
  }
  const long long resident = bt == 128 ? 512 : 768, rest = list_tiles % resident;
  if (!rest || !carries_rest || rest > tiles) return s;
  const double tile_us = steps * (bt == 128 ? 1.4 : 0.7), part_us = bt * bt * 8. / 4e6;
  double best = tile_us;
  for (int z = 2; z <= 32 && z <= steps / 4; ++z) {
    const double us = tile_us * (double)((rest * z + resident - 1) / resident) / z + part_us * (double)rest * z + 6.;
    if (us < best) {
      best = us;
      s.z = z;
      s.whole = (int)(tiles - rest);
    }
  }
  return s;
}
int split_blocks(const Split &s) { return s.whole + (s.tiles - s.whole) * s.z; }

// Everything about the list that depends on its shapes: workspace places and workgroups.  `base` null: sizes only.
int plan_list(const mr3d_matrix *in, int count, char *base, Plan &plan, Mat *mats, bool pointers) {
  if (!in || count <= 0 || count > 65536) return MR3D_ERR_INVALID_ARG;
  plan = Plan{};
  size_t at = 0;
  plan.mats_off = take(at, (size_t)count * sizeof(Mat));
  struct { long long sym[2], apply[2], most; int carrier; } sum{};
  sum.carrier = -1;
  for (int k = 0; k < count; ++k) {
    const mr3d_matrix &g = in[k];
    if (g.rows <= 0 || g.cols <= 0 || g.rows > (1 << 20) || g.cols > (1 << 20) || (pointers && (!g.in || !g.out))) return MR3D_ERR_INVALID_ARG;
    if (g.dtype != MR3D_DTYPE_F32 && g.dtype != MR3D_DTYPE_BF16) return MR3D_ERR_UNSUPPORTED;
    const long long m = g.rows < g.cols ? g.rows : g.cols, n = g.rows < g.cols ? g.cols : g.rows;
    if (m <= kSmall) continue;
    for (int b = 0; b < 2; ++b) {
      const long long bt = b ? 128 : 64, tm = (m + bt - 1) / bt, tn = (n + bt - 1) / bt;
      sum.sym[b] += tm * (tm + 1) / 2;
      sum.apply[b] += tm * tn;
    }
    if (m * n > sum.most) {
      sum.most = m * n;
      sum.carrier = k;
    }
  }
  // tile width and part length of each product: the pair with the least estimated time; 128 once 64-wide tiles fill a round
  int bt[3], len[3];
  long long list[3];
  for (int kind = 0; kind < 3; ++kind) {
    const long long n64 = kind < 2 ? sum.sym[0] : sum.apply[0], n128 = kind < 2 ? sum.sym[1] : sum.apply[1];
    double us64 = 1e30, us128 = 1e30;
    const int l64 = n64 < 768 ? part_length(in, count, kind, 64, us64) : 0, l128 = n128 < 512 ? part_length(in, count, kind, 128, us128) : 0;
    const bool wide = n64 >= 768 || us128 < us64;
    bt[kind] = wide ? 128 : 64;
    len[kind] = wide ? l128 : l64;
    list[kind] = wide ? n128 : n64;
  }
  plan.bt_gram = bt[0];
  plan.bt_square = bt[1];
  plan.bt_apply = bt[2];
  long long blocks[kStages] = {};
  for (int k = 0; k < count; ++k) {
    const mr3d_matrix &g = in[k];
    const bool tall = g.rows > g.cols;
    Mat p{};
    p.m = (int)(tall ? g.cols : g.rows);
    p.n = (int)(tall ? g.rows : g.cols);
    p.in = (const char *)g.in - base;
    p.out = (const char *)g.out - base;
    p.in_j = tall ? g.in_col_stride : g.in_row_stride;
    p.in_i = tall ? g.in_row_stride : g.in_col_stride;
    p.out_j = tall ? 1 : g.cols;
    p.out_i = tall ? g.cols : 1;
    p.bf16 = g.dtype == MR3D_DTYPE_BF16;
    long long need[kStages] = {};
    if (p.m <= kSmall) {
      // a share of A takes at least 64 columns, at most 32 shares (one workgroup adds them up)
      const int chunks = (p.n + kChunk - 1) / kChunk, mp = (p.m + 15) / 16 * 16;
      p.gram.z = chunks < 32 ? chunks : 32;
      p.norm = take(at, ((size_t)p.gram.z + 1) * mp * kSmall * 8);
      need[kSmallGram] = p.gram.z;
      need[kSmallPoly] = 1;
      need[kSmallApply] = chunks;
    } else {
      p.ldx = (p.n + 31) / 32 * 128;
      p.lda = (p.m + 31) / 32 * 128;
      const long long tg = (p.m + plan.bt_gram - 1) / plan.bt_gram, ts = (p.m + plan.bt_square - 1) / plan.bt_square, tm = (p.m + plan.bt_apply - 1) / plan.bt_apply, tn = (p.n + plan.bt_apply - 1) / plan.bt_apply;
      const int ksm = (p.m + 31) / 32, ksn = (p.n + 31) / 32, qg = plan.bt_gram == 128 ? 4 : 1, qs = plan.bt_square == 128 ? 4 : 1, qa = plan.bt_apply == 128 ? 4 : 1;
      if (ts * (ts + 1) / 2 > 0x3fffffff || tg * (tg + 1) / 2 > 0x3fffffff || tm * tn > 0x3fffffff) return MR3D_ERR_UNSUPPORTED;
      p.gram = split_for((int)(tg * (tg + 1) / 2), ksn, len[0], list[0], k == sum.carrier, plan.bt_gram);
      p.square = split_for((int)(ts * (ts + 1) / 2), ksm, len[1], list[1], k == sum.carrier, plan.bt_square);
      p.apply = split_for((int)(tm * tn), ksm, len[2], list[2], k == sum.carrier, plan.bt_apply);
      const long long numel = (long long)p.m * p.n;
      p.norm_blocks = (int)((numel + 8191) / 8192 > 1024 ? 1024 : (numel + 8191) / 8192);
      for (int b = 0; b < kBufs; ++b) {
        const bool x = b == kX0 || b == kX1;
        p.buf[b] = take(at, (size_t)p.m * (x ? p.ldx : p.lda));
      }
      size_t part = 0;
      const struct { Split s; int bt; } uses[3] = {{p.gram, plan.bt_gram}, {p.square, plan.bt_square}, {p.apply, plan.bt_apply}};
      for (const auto &u : uses) {
        const size_t b = (size_t)(u.s.tiles - u.s.whole) * u.s.z * u.bt * u.bt * sizeof(float);
        part = b > part ? b : part;
      }
      if (part) p.part = take(at, part);
      p.norm = take(at, (size_t)p.norm_blocks * sizeof(double));
      need[kNorm] = p.norm_blocks;
      need[kPack] = (long long)((p.m + 63) / 64) * ((p.n + 63) / 64);
      need[kGram] = split_blocks(p.gram);
      need[kGramJoin] = (long long)(p.gram.tiles - p.gram.whole) * qg;
      need[kSquare] = split_blocks(p.square);
      need[kSquareJoin] = (long long)(p.square.tiles - p.square.whole) * qs;
      need[kApply] = split_blocks(p.apply);
      need[kApplyJoin] = (long long)(p.apply.tiles - p.apply.whole) * qa;
    }
    for (int s = 0; s < kStages; ++s) {
      p.first[s] = (int)blocks[s];
      blocks[s] += need[s];
      if (blocks[s] > 0x3fffffff) return MR3D_ERR_UNSUPPORTED;
    }
    if (mats) mats[k] = p;
  }
  for (int s = 0; s < kStages; ++s) {
    plan.blocks[s] = (int)blocks[s];
    plan.map_off[s] = take(at, (size_t)blocks[s] * sizeof(int));
  }
  plan.bytes = at;
  return MR3D_OK;
}

struct Launcher {
  char *ws;
  const Plan &plan;
  const Mat *mats;
  const Maps &maps;
  hipStream_t q;

  template <int KIND, int BT> void tiles(const Op &op, int stage) const {
    ortho_product_kernel<KIND, BT><<<plan.blocks[stage], kThreads, Pick<BT, KIND == 2>::T::LDS_BYTES, q>>>(ws, mats, maps.map[stage], op);
    if (plan.blocks[stage + 1]) ortho_join_kernel<KIND, BT><<<plan.blocks[stage + 1], kThreads, 0, q>>>(ws, mats, maps.map[stage + 1], op);
  }
  template <int KIND> void product(const Op &op, int stage, int bt) const { bt == 128 ? tiles<KIND, 128>(op, stage) : tiles<KIND, 64>(op, stage); }
  void step(int x, bool last, float ca, float cb, float cc) const {
    product<0>(Op{x, kSA / (kSX * kSX), 0.f, 0.f, 0}, kGram, plan.bt_gram);
    product<1>(Op{x, cc * kSP / (kSA * kSA), cb * kSP / kSA, ca * kSP, 0}, kSquare, plan.bt_square);
    product<2>(Op{x, last ? 1.f / (kSP * kSX) : 1.f / kSP, 0.f, 0.f, last}, kApply, plan.bt_apply);
  }
};

}  // namespace

extern "C" size_t mr3d_orthogonalize_workspace_bytes(const mr3d_matrix *mats_host, int count) {
  Plan plan;
  return plan_list(mats_host, count, nullptr, plan, nullptr, false) == MR3D_OK ? plan.bytes : 0;
}

extern "C" int mr3d_orthogonalize_tiles(const mr3d_matrix *mats_host, int count, mr3d_ortho_tiles *tiles_host) {
  if (!tiles_host || !mats_host || count <= 0 || count > 65536) return MR3D_ERR_INVALID_ARG;
  Mat *table = new (std::nothrow) Mat[count];
  if (!table) return MR3D_ERR_INVALID_ARG;
  Plan plan;
  const int st = plan_list(mats_host, count, nullptr, plan, table, false);
  if (st == MR3D_OK) {
    mr3d_ortho_tiles t{{plan.bt_gram, plan.bt_square, plan.bt_apply}, {}, {}, {1, 1, 1}};
    for (int k = 0; k < count; ++k) {
      if (table[k].m <= kSmall) continue;
      const Split s[3] = {table[k].gram, table[k].square, table[k].apply};
      for (int i = 0; i < 3; ++i) {
        t.whole[i] += s[i].whole;
        t.split[i] += s[i].tiles - s[i].whole;
        if (s[i].tiles > s[i].whole && s[i].z > t.parts[i]) t.parts[i] = s[i].z;
      }
    }
    *tiles_host = t;
  }
  delete[] table;
  return st;
}

extern "C" int mr3d_orthogonalize(const mr3d_matrix *mats_host, int count, int steps, float ca, float cb, float cc, float eps, void *workspace,
                                  size_t workspace_bytes, mr3d_stream_t s) {
  if (steps < 1 || steps > 100 || !(eps >= 0.f)) return MR3D_ERR_INVALID_ARG;
  if (!(ca >= -16.f && ca <= 16.f && cb >= -16.f && cb <= 16.f && cc >= -16.f && cc <= 16.f)) return MR3D_ERR_INVALID_ARG;
  if (!mats_host || count <= 0 || count > 65536) return MR3D_ERR_INVALID_ARG;
  if (!workspace || ((uintptr_t)workspace & 255)) return MR3D_ERR_WORKSPACE;
  Mat *table = new (std::nothrow) Mat[count];
  if (!table) return MR3D_ERR_INVALID_ARG;
  Plan plan;
  char *base = (char *)workspace;
  int st = plan_list(mats_host, count, base, plan, table, true);
  if (st == MR3D_OK && workspace_bytes < plan.bytes) st = MR3D_ERR_WORKSPACE;
  constexpr int kPolyLds = 4 * kSmall * kLdd * 8;
  if (st == MR3D_OK && plan.blocks[kSmallPoly] &&
      hipFuncSetAttribute(reinterpret_cast<const void *>(ortho_small_poly_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kPolyLds) != hipSuccess)
    st = MR3D_ERR_LAUNCH;
  if (st != MR3D_OK) {
    delete[] table;
    return st;
  }
  hipStream_t q = mr3d_stream(s);
  Mat *mats = (Mat *)(base + plan.mats_off);
  Maps maps;
  for (int s = 0; s < kStages; ++s) maps.map[s] = (int *)(base + plan.map_off[s]);
  for (int at = 0; at < count; at += kBatch) {
    MatBatch b;
    const int n = count - at < kBatch ? count - at : kBatch;
    for (int k = 0; k < n; ++k) b.m[k] = table[at + k];
    int most = 1;
    for (int s = 0; s < kStages; ++s) {
      maps.end[s] = at + n < count ? table[at + n].first[s] : plan.blocks[s];
      most = maps.end[s] - b.m[0].first[s] > most ? maps.end[s] - b.m[0].first[s] : most;
    }
    const int mb = (most + 255) / 256;
    ortho_table_kernel<<<dim3(mb < 256 ? mb : 256, kStages), 256, 0, q>>>(b, n, at, mats, maps);
  }
  delete[] table;
  if (plan.blocks[kSmallPoly]) {
    ortho_small_gram_kernel<<<plan.blocks[kSmallGram], kThreads, 0, q>>>(base, mats, maps.map[kSmallGram]);
    ortho_small_poly_kernel<<<plan.blocks[kSmallPoly], kPolyThreads, kPolyLds, q>>>(base, mats, maps.map[kSmallPoly], steps, ca, cb, cc, eps);
    ortho_small_apply_kernel<<<plan.blocks[kSmallApply], kThreads, 0, q>>>(base, mats, maps.map[kSmallApply]);
  }
  if (plan.blocks[kNorm]) {
    ortho_norm_kernel<<<plan.blocks[kNorm], 256, 0, q>>>(base, mats, maps.map[kNorm]);
    ortho_pack_kernel<<<plan.blocks[kPack], 256, 0, q>>>(base, mats, maps.map[kPack], eps);
    const Launcher run{base, plan, mats, maps, q};
    for (int k = 0; k < steps; ++k) run.step(k & 1 ? kX1 : kX0, k == steps - 1, ca, cb, cc);
  }
  return mr3d_launch_status();
}
