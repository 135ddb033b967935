// Orthogonalised updates: Newton-Schulz products of a LIST of matrices, all of them in one launch per stage.
//   X = G / (|G|_F + eps), wide (m <= n; a tall G is read transposed);  steps times:
//     A = X X^T          B = a I + b A + c A A          X = B X
// (a I sits inside B, so the third product needs no second read of X).  A and A A are symmetric: only the tiles on and below the diagonal are computed
// and stored twice.
// Every factor is kept as two fp16 planes (gemm16.h, split storage), scaled by powers of two into fp16's range: 22 bits, three passes of the
// 16-bit matrix pipe, fp32 accumulators.  Plain bf16 or fp16 factors would lose 2e-2 / 2e-3 of the result over five steps (the
// polynomial's slope at 0 is a = 3.4: rounding errors of the first steps are amplified a few hundred times).
// MFMA-bound on large matrices; on small ones the 4 dependent launches of a step are what counts, hence the list.
#include "gemm16.h"
#include <new>

using namespace gemm16;

namespace {

// powers of two that bring X, A and B into fp16's range: |X| < 16, |A| < 16, |B| < 64
constexpr float kSX = 4096.f, kSA = 4096.f, kSB = 1024.f;
constexpr int kT = 128;                                     // tile of every product
typedef Tile<kT, kT, 2, 2, false, false, true, 128, 2> TileGram;
typedef Tile<kT, kT, 2, 2, true, false, true, 128, 2> TileApply;
constexpr int kThreads = TileGram::THREADS;

enum Stage { kNorm, kPack, kGram, kReduce, kPoly, kApply, kStages };

struct Mat {
  const char *in;
  char *out;
  long long in_i, in_j, out_i, out_j;                       // element strides along n (i) and m (j)
  char *x[2], *a, *b;                                       // planes: [m][ldx], [m][ldx], [m][lda], [m][lda]
  float *part;                                              // [z][tiles][kT * kT]
  double *norm;
  int m, n, ldx, lda;                                       // ld in bytes
  int z, bf16, norm_blocks, pad;
  int first[kStages];                                       // first workgroup of this matrix in each stage
};

struct Plan {
  int blocks[kStages];
  size_t bytes, mats_off, map_off[kStages];
};

constexpr int kBatch = 16;
struct MatBatch { Mat m[kBatch]; };

__device__ __forceinline__ int triangle(int t, int &ti) {
  int tj = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while ((tj + 1) * (tj + 2) / 2 <= t) ++tj;
  while (tj * (tj + 1) / 2 > t) --tj;
  ti = t - tj * (tj + 1) / 2;
  return tj;
}

__global__ __launch_bounds__(64) void ortho_table_kernel(MatBatch batch, int count, int at, Mat *__restrict__ mats) {
  if ((int)threadIdx.x < count) mats[at + threadIdx.x] = batch.m[threadIdx.x];
}

// workgroup -> matrix, per stage
struct Maps { int *map[kStages]; int blocks[kStages]; };
__global__ __launch_bounds__(256) void ortho_map_kernel(const Mat *__restrict__ mats, int count, Maps maps) {
  for (int s = 0; s < kStages; ++s)
    for (int b = blockIdx.x * 256 + threadIdx.x; b < maps.blocks[s]; b += gridDim.x * 256) {
      int lo = 0, hi = count - 1;
      while (lo < hi) {                                     // the last matrix whose first workgroup is <= b
        const int mid = (lo + hi + 1) / 2;
        if (mats[mid].first[s] <= b) lo = mid; else hi = mid - 1;
      }
      maps.map[s][b] = lo;
    }
}

__device__ __forceinline__ float read_in(const Mat &p, long long off) {
  return p.bf16 ? (float)((const __bf16 *)p.in)[off] : ((const float *)p.in)[off];
}

// squares of the input in double: fp32 squares would overflow from 2^64 on
__global__ __launch_bounds__(256) void ortho_norm_kernel(const Mat *__restrict__ mats, const int *__restrict__ map) {
  const Mat p = mats[map[blockIdx.x]];
  const int chunk = blockIdx.x - p.first[kNorm];
  const bool wide = p.in_i == 1;                            // walk the contiguous axis with the threads
  const int inner = wide ? p.n : p.m, outer = wide ? p.m : p.n;
  const long long si = wide ? 1 : p.in_j, so = wide ? p.in_j : p.in_i;
  const long long total = (long long)inner * outer;
  double s = 0;
  long long e = (long long)chunk * 256 + threadIdx.x;
  const long long stride = (long long)p.norm_blocks * 256;
  if (si == 1 && so == inner && ((uintptr_t)p.in & 15) == 0) {            // packed: 16 bytes a load
    const int per = p.bf16 ? 8 : 4;
    const long long groups = total / per;
#pragma unroll 2
    for (; e < groups; e += stride) {
      float v[8];
      if (p.bf16) {
        const bf16x8 t = *reinterpret_cast<const bf16x8 *>(p.in + e * 16);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)t[k];
      } else {
        const float4 t = *reinterpret_cast<const float4 *>(p.in + e * 16);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        v[4] = v[5] = v[6] = v[7] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s += (double)v[k] * (double)v[k];
    }
    for (e = groups * per + (long long)chunk * 256 + threadIdx.x; e < total; e += stride) {
      const double v = (double)read_in(p, e);
      s += v * v;
    }
  } else {
    for (; e < total; e += stride) {
      const int o = (int)(e / inner), i = (int)(e - (long long)o * inner);
      const double v = (double)read_in(p, o * so + i * si);
      s += v * v;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  __shared__ double w[4];
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) p.norm[chunk] = w[0] + w[1] + w[2] + w[3];
}

// 64 x 64 of the input -> planes of X; the tile goes through LDS so that a tall input is read along its rows too
__global__ __launch_bounds__(256) void ortho_pack_kernel(const Mat *__restrict__ mats, const int *__restrict__ map, float eps) {
  __shared__ float t[64][65];
  __shared__ double w[4];
  const Mat p = mats[map[blockIdx.x]];
  const int tile = blockIdx.x - p.first[kPack], tn = (p.n + 63) / 64;
  const int j0 = tile / tn * 64, i0 = tile % tn * 64;
  double s = 0;
  for (int k = threadIdx.x; k < p.norm_blocks; k += 256) s += p.norm[k];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  const bool wide = p.in_i == 1;
  for (int k = threadIdx.x; k < 4096; k += 256) {
    const int q = k & 63, r = k >> 6;
    const int i = wide ? q : r, j = wide ? r : q;
    t[j][i] = (i0 + i < p.n && j0 + j < p.m) ? read_in(p, (i0 + i) * p.in_i + (j0 + j) * p.in_j) : 0.f;
  }
  __syncthreads();
  const double scale = (double)kSX / (sqrt(w[0] + w[1] + w[2] + w[3]) + (double)eps);      // may leave fp32's range where G does not
  const int np = (p.n + 31) / 32 * 32;
  for (int k = threadIdx.x; k < 64 * 16; k += 256) {
    const int j = k >> 4, i = (k & 15) * 4;
    if (j0 + j >= p.m || i0 + i >= np) continue;
    _Float16 h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split16((float)((double)t[j][i + e] * scale), h[e], l[e]);
    char *d = p.x[0] + (long long)(j0 + j) * p.ldx + (i0 + i) / 32 * 128 + (i & 31) * 2;
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

// 32 x 32 block (bi, bj) of a tile of a symmetric result: rows j of tile tj, columns i of tile ti, and mirrored off the diagonal.
// POLY: a I + b A + c acc instead of acc
template <bool POLY>
__device__ __forceinline__ void store_symmetric_block(const Mat &p, char *dst, int ti, int tj, int bi, int bj, const f32x16 &acc, float ca, float cb, float cc) {
  const int lane = threadIdx.x & 63, mp = (p.m + 31) / 32 * 32;
  const int j = tj * kT + bj * 32 + (lane & 31);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int i = ti * kT + bi * 32 + g * 8 + (lane >> 5) * 4;
    float v[4];
    if constexpr (POLY) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (j < p.m && i < mp) load_planes(p.a + (long long)j * p.lda, i, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float t = cc * (acc[g * 4 + e] * (1.f / (kSA * kSA))) + cb * (f[e] * (1.f / kSA));
        v[e] = (t + (i + e == j ? ca : 0.f)) * kSB;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[g * 4 + e] * (kSA / (kSX * kSX));
    }
    if (j < p.m && i < mp) store_planes(dst + (long long)j * p.lda, i, v);
    if (ti != tj && j < mp) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < p.m) {
          _Float16 h, l;
          split16(v[e], h, l);
          _Float16 *d = reinterpret_cast<_Float16 *>(dst + (long long)(i + e) * p.lda + (j >> 5) * 128) + (j & 31);
          d[0] = h;
          d[32] = l;
        }
    }
  }
}

template <bool POLY>
__device__ __forceinline__ void store_symmetric(const Mat &p, char *dst, int ti, int tj, const f32x16 (&acc)[2][2], float ca, float cb, float cc) {
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) store_symmetric_block<POLY>(p, dst, ti, tj, (wave & 1) * 2 + a, (wave >> 1) * 2 + b, acc[a][b], ca, cb, cc);
}

__global__ __launch_bounds__(kThreads, 2) void ortho_gram_kernel(const Mat *__restrict__ mats, const int *__restrict__ map, int cur) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const Mat p = mats[map[blockIdx.x]];
  const int local = blockIdx.x - p.first[kGram];
  int ti;
  const int t = local / p.z, zi = local % p.z, tj = triangle(t, ti);
  const int total = (p.n + 31) / 32;
  const int s0 = (int)((long long)total * zi / p.z), s1 = (int)((long long)total * (zi + 1) / p.z);
  const char *x = cur ? p.x[1] : p.x[0];
  f32x16 acc[2][2];
  run<TileGram>(lds, side_kc<TileGram>(x, p.ldx, p.m, p.ldx, ti * kT, s0), side_kc<TileGram>(x, p.ldx, p.m, p.ldx, tj * kT, s0), s1 - s0, acc);
  if (p.z == 1) {
    store_symmetric<false>(p, p.a, ti, tj, acc, 0.f, 0.f, 0.f);
  } else {
    const int tm = (p.m + kT - 1) / kT;
    float *d = p.part + ((long long)zi * (tm * (tm + 1) / 2) + t) * (kT * kT) + threadIdx.x;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) d[((a * 2 + b) * 16 + e) * kThreads] = acc[a][b][e];
  }
}

// the parts of a split Gram tile, added in a fixed order; a workgroup takes one of the four 32 x 32 blocks of every wave
__global__ __launch_bounds__(kThreads) void ortho_reduce_kernel(const Mat *__restrict__ mats, const int *__restrict__ map) {
  const Mat p = mats[map[blockIdx.x]];
  const int local = blockIdx.x - p.first[kReduce], t = local >> 2, q = local & 3;
  int ti;
  const int tj = triangle(t, ti), tm = (p.m + kT - 1) / kT;
  const long long stride = (long long)(tm * (tm + 1) / 2) * (kT * kT);
  const float *s = p.part + (long long)t * (kT * kT) + q * 16 * kThreads + threadIdx.x;
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = s[e * kThreads];
  for (int zi = 1; zi < p.z; zi += 2) {                     // 32 loads in flight
    const float *s1 = s + zi * stride, *s2 = zi + 1 < p.z ? s1 + stride : s1;
    const float keep = zi + 1 < p.z ? 1.f : 0.f;
    float u[16], v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      u[e] = s1[e * kThreads];
      v[e] = s2[e * kThreads];
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      acc[e] += u[e];
      if (keep != 0.f) acc[e] += v[e];
    }
  }
  const int wave = threadIdx.x >> 6;
  store_symmetric_block<false>(p, p.a, ti, tj, (wave & 1) * 2 + (q >> 1), (wave >> 1) * 2 + (q & 1), acc, 0.f, 0.f, 0.f);
}

__global__ __launch_bounds__(kThreads, 2) void ortho_poly_kernel(const Mat *__restrict__ mats, const int *__restrict__ map, float ca, float cb, float cc) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const Mat p = mats[map[blockIdx.x]];
  int ti;
  const int tj = triangle(blockIdx.x - p.first[kPoly], ti);
  f32x16 acc[2][2];
  run<TileGram>(lds, side_kc<TileGram>(p.a, p.lda, p.m, p.lda, ti * kT, 0), side_kc<TileGram>(p.a, p.lda, p.m, p.lda, tj * kT, 0), (p.m + 31) / 32, acc);
  store_symmetric<true>(p, p.b, ti, tj, acc, ca, cb, cc);
}

__global__ __launch_bounds__(kThreads, 2) void ortho_apply_kernel(const Mat *__restrict__ mats, const int *__restrict__ map, int cur, int last) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const Mat p = mats[map[blockIdx.x]];
  const int local = blockIdx.x - p.first[kApply], tm = (p.m + kT - 1) / kT;
  const int tj = local % tm, ti = local / tm;
  f32x16 acc[2][2];
  run<TileApply>(lds, side_ks<TileApply>(cur ? p.x[1] : p.x[0], p.ldx, p.m, p.ldx, ti * kT * 4, 0), side_kc<TileApply>(p.b, p.lda, p.m, p.lda, tj * kT, 0), (p.m + 31) / 32, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave & 1, wj = wave >> 1;
  const int np = (p.n + 31) / 32 * 32;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int j = tj * kT + (wj * 2 + b) * 32 + (lane & 31);
      if (j >= p.m) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int i = ti * kT + (wi * 2 + a) * 32 + g * 8 + (lane >> 5) * 4;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[a][b][g * 4 + e] * (last ? 1.f / (kSB * kSX) : 1.f / kSB);
        if (!last) {
          if (i < np) store_planes((cur ? p.x[0] : p.x[1]) + (long long)j * p.ldx, i, v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < p.n) {
              const long long at = j * p.out_j + (i + e) * p.out_i;
              if (p.bf16) ((__bf16 *)p.out)[at] = (__bf16)v[e];
              else ((float *)p.out)[at] = v[e];
            }
        }
      }
    }
}

size_t take(size_t &at, size_t bytes) {
  const size_t here = at;
  at = mr3d_align_up(at + bytes, 256);
  return here;
}

// Everything about the list that depends on its shapes: workspace places and workgroups.  `base` null: sizes only.
int plan_list(const mr3d_matrix *in, int count, char *base, Plan &plan, Mat *mats, bool pointers) {
  if (!in || count <= 0 || count > 65536) return MR3D_ERR_INVALID_ARG;
  plan = Plan{};
  size_t at = 0;
  plan.mats_off = take(at, (size_t)count * sizeof(Mat));
  long long gram_tiles = 0;
  for (int k = 0; k < count; ++k) {
    const mr3d_matrix &g = in[k];
    if (g.rows <= 0 || g.cols <= 0 || g.rows > (1 << 20) || g.cols > (1 << 20) || (pointers && (!g.in || !g.out))) return MR3D_ERR_INVALID_ARG;
    if (g.dtype != MR3D_DTYPE_F32 && g.dtype != MR3D_DTYPE_BF16) return MR3D_ERR_UNSUPPORTED;
    const long long m = g.rows < g.cols ? g.rows : g.cols, tm = (m + kT - 1) / kT;
    gram_tiles += tm * (tm + 1) / 2;
  }
  long long blocks[kStages] = {};
  for (int k = 0; k < count; ++k) {
    const mr3d_matrix &g = in[k];
    const bool tall = g.rows > g.cols;
    Mat p{};
    p.m = (int)(tall ? g.cols : g.rows);
    p.n = (int)(tall ? g.rows : g.cols);
    p.in = (const char *)g.in;
    p.out = (char *)g.out;
    p.in_j = tall ? g.in_col_stride : g.in_row_stride;
    p.in_i = tall ? g.in_row_stride : g.in_col_stride;
    p.out_j = tall ? 1 : g.cols;
    p.out_i = tall ? g.cols : 1;
    p.bf16 = g.dtype == MR3D_DTYPE_BF16;
    p.ldx = (p.n + 31) / 32 * 128;
    p.lda = (p.m + 31) / 32 * 128;
    const int tm = (p.m + kT - 1) / kT, tn = (p.n + kT - 1) / kT, tri = tm * (tm + 1) / 2;
    // Split the long axis of X X^T where the whole list has too few tiles to fill 256 CUs with two workgroups each; a part keeps at
    // least 8 k-steps, so that its loads and its fp32 round trip through memory pay
    const int steps = (p.n + 31) / 32;
    long long z = gram_tiles >= 512 ? 1 : 512 / gram_tiles;
    if (z > steps / 8) z = steps / 8;
    p.z = (int)(z < 1 ? 1 : z);
    const long long numel = (long long)p.m * p.n;
    p.norm_blocks = (int)((numel + 8191) / 8192 > 1024 ? 1024 : (numel + 8191) / 8192);
    const size_t ox0 = take(at, (size_t)p.m * p.ldx), ox1 = take(at, (size_t)p.m * p.ldx), oa = take(at, (size_t)p.m * p.lda), ob = take(at, (size_t)p.m * p.lda);
    const size_t op = p.z > 1 ? take(at, (size_t)p.z * tri * kT * kT * sizeof(float)) : 0, on = take(at, (size_t)p.norm_blocks * sizeof(double));
    p.x[0] = base + ox0;
    p.x[1] = base + ox1;
    p.a = base + oa;
    p.b = base + ob;
    p.part = (float *)(base + op);
    p.norm = (double *)(base + on);
    const long long need[kStages] = {p.norm_blocks, (long long)((p.m + 63) / 64) * ((p.n + 63) / 64), (long long)tri * p.z, p.z > 1 ? 4 * tri : 0, tri, (long long)tm * tn};
    for (int s = 0; s < kStages; ++s) {
      p.first[s] = (int)blocks[s];
      blocks[s] += need[s];
      if (blocks[s] > 0x7fffffff) return MR3D_ERR_UNSUPPORTED;
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

}  // namespace

extern "C" size_t mr3d_orthogonalize_workspace_bytes(const mr3d_matrix *mats_host, int count) {
  Plan plan;
  return plan_list(mats_host, count, nullptr, plan, nullptr, false) == MR3D_OK ? plan.bytes : 0;
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
  if (st != MR3D_OK) {
    delete[] table;
    return st;
  }
  hipStream_t q = mr3d_stream(s);
  Mat *mats = (Mat *)(base + plan.mats_off);
  for (int at = 0; at < count; at += kBatch) {
    MatBatch b;
    const int n = count - at < kBatch ? count - at : kBatch;
    for (int k = 0; k < n; ++k) b.m[k] = table[at + k];
    ortho_table_kernel<<<1, 64, 0, q>>>(b, n, at, mats);
  }
  delete[] table;
  Maps maps;
  int most = 0;
  for (int k = 0; k < kStages; ++k) {
    maps.map[k] = (int *)(base + plan.map_off[k]);
    maps.blocks[k] = plan.blocks[k];
    most = plan.blocks[k] > most ? plan.blocks[k] : most;
  }
  const int mb = (most + 255) / 256;
  ortho_map_kernel<<<mb < 256 ? mb : 256, 256, 0, q>>>(mats, count, maps);
  ortho_norm_kernel<<<plan.blocks[kNorm], 256, 0, q>>>(mats, maps.map[kNorm]);
  ortho_pack_kernel<<<plan.blocks[kPack], 256, 0, q>>>(mats, maps.map[kPack], eps);
  for (int k = 0; k < steps; ++k) {
    const int cur = k & 1;
    ortho_gram_kernel<<<plan.blocks[kGram], kThreads, TileGram::LDS_BYTES, q>>>(mats, maps.map[kGram], cur);
    if (plan.blocks[kReduce]) ortho_reduce_kernel<<<plan.blocks[kReduce], kThreads, 0, q>>>(mats, maps.map[kReduce]);
    ortho_poly_kernel<<<plan.blocks[kPoly], kThreads, TileGram::LDS_BYTES, q>>>(mats, maps.map[kPoly], ca, cb, cc);
    ortho_apply_kernel<<<plan.blocks[kApply], kThreads, TileApply::LDS_BYTES, q>>>(mats, maps.map[kApply], cur, k == steps - 1);
  }
  return mr3d_launch_status();
}
