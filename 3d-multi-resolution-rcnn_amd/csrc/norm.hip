// Layer norm over the last axis of [rows][cols], forward and backward (fp32 / bf16 storage, fp32 arithmetic).
//   mean = sum x / C     var = sum (x - mean)^2 / C     r = 1 / sqrt(var + eps)     h = (x - mean) r     y = h w + b
//   gh = dy w     dx = r (gh - sum gh / C - h sum(gh h) / C)     dw = sum_rows dy h     db = sum_rows dy
// HBM-bound: x is read once and y written once (backward: x, dy, dx).  A row is held in registers by `LPR` lanes (8 of a wave for 64 bf16
// channels up to a whole 1024-thread workgroup), so mean and variance are the exact two-pass form without a second read: a
// one-pass sum of squares loses the variance of rows whose mean is large.
// Backward: a workgroup walks rows in a grid-stride loop; the dw / db sums of a lane's own columns stay in registers over all its rows,
// then meet in LDS and leave as ONE partial row per workgroup; ln_param_kernel adds the partial rows in a fixed order in double
// (no atomics: run-to-run identical bits).
// Measured, forward / backward / parameter sums: 655360 x 64 bf16 37 / 55 / 5 us, 10007 x 1531 fp32 27 / 38 / 5 us -- 4.5 to 4.8 TB/s, about what a
// large copy reaches; 512 x 1024 fp32 4.6 / 5.9 / 4.0 us and 1 x 1024 2.6 us are launches.
#include "mr3d_common.h"
#include <hip/hip_bf16.h>

namespace {

typedef __bf16 bf16;

// 16 bytes of T with only T's own alignment: rows of an odd number of columns start anywhere
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Vec<bf16> {
  static constexpr int N = 8;
  typedef bf16 V __attribute__((ext_vector_type(8), aligned(2)));
};

template <typename T, int NV, int LPR>
__device__ __forceinline__ void load_row(const T *__restrict__ p, int cols, int lane, float (&f)[NV * Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * LPR + lane) * N;
    if (c + N <= cols) {
      const typename Vec<T>::V t = *reinterpret_cast<const typename Vec<T>::V *>(p + c);
#pragma unroll
      for (int e = 0; e < N; ++e) f[v * N + e] = (float)t[e];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) f[v * N + e] = c + e < cols ? (float)p[c + e] : 0.f;
    }
  }
}

template <typename T, int NV, int LPR>
__device__ __forceinline__ void store_row(T *__restrict__ p, int cols, int lane, const float (&f)[NV * Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * LPR + lane) * N;
    if (c + N <= cols) {
      typename Vec<T>::V t;
#pragma unroll
      for (int e = 0; e < N; ++e) t[e] = (T)f[v * N + e];
      *reinterpret_cast<typename Vec<T>::V *>(p + c) = t;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c + e < cols) p[c + e] = (T)f[v * N + e];
    }
  }
}

// the parameter vectors may be fp32 beside bf16 activations
template <typename T, int NV, int LPR>
__device__ __forceinline__ void load_param(const void *p, int f32, int cols, int lane, float absent, float (&f)[NV * Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int c = (v * LPR + lane) * N + e;
      float t = absent;
      if (p && c < cols) t = f32 ? ((const float *)p)[c] : (float)((const T *)p)[c];
      f[v * N + e] = t;
    }
}

// sum over the LPR lanes of a row, the same value in all of them; A sums at once.  LPR > 64: the row is the workgroup's
template <int LPR, int A>
__device__ __forceinline__ void row_sum(float (&s)[A], float *lds) {
#pragma unroll
  for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int a = 0; a < A; ++a) s[a] += __shfl_xor(s[a], o);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    __syncthreads();                                     // the previous sums have been read
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int a = 0; a < A; ++a) lds[a * W + (threadIdx.x >> 6)] = s[a];
    __syncthreads();
#pragma unroll
    for (int a = 0; a < A; ++a) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) t += lds[a * W + w];
      s[a] = t;
    }
  }
}

template <int LPR> constexpr int threads_of() { return LPR > 256 ? LPR : 256; }

template <typename T, int LPR, int NV>
__global__ __launch_bounds__(threads_of<LPR>()) void ln_fwd_kernel(const T *__restrict__ x, long long xs, const void *w, const void *b,
                                                                   int param_f32, T *__restrict__ y, float *__restrict__ mean_out,
                                                                   float *__restrict__ rstd_out, long long rows, int cols, float eps) {
  constexpr int N = NV * Vec<T>::N, TH = threads_of<LPR>(), RPB = TH / LPR;
  __shared__ float lds[LPR > 64 ? LPR / 64 : 1];
  const int lane = threadIdx.x % LPR;
  float fw[N], fb[N];
  load_param<T, NV, LPR>(w, param_f32, cols, lane, 1.f, fw);
  load_param<T, NV, LPR>(b, param_f32, cols, lane, 0.f, fb);
  const float inv = 1.f / (float)cols;
  for (long long row0 = (long long)blockIdx.x * RPB; row0 < rows; row0 += (long long)gridDim.x * RPB) {
    const long long row = row0 + threadIdx.x / LPR;
    const bool live = row < rows;                        // a dead group still takes part in the shuffles
    float f[N];
    load_row<T, NV, LPR>(x + (live ? row : row0) * xs, cols, lane, f);
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < N; ++e) s[0] += f[e];
    row_sum<LPR, 1>(s, lds);
    // the mean of what the first mean leaves takes out its error of some steps, which a small variance would show: a row of one value has variance 0.
    // (A quotient, because a product would be fused with the differences below, which would then be taken from another number than `mean`)
    float mean = s[0] / (float)cols, left[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < Vec<T>::N; ++e) left[0] += (v * LPR + lane) * Vec<T>::N + e < cols ? f[v * Vec<T>::N + e] - mean : 0.f;
    row_sum<LPR, 1>(left, lds);
    mean += left[0] * inv;
    float q[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < Vec<T>::N; ++e) {
        const float d = f[v * Vec<T>::N + e] - mean;
        q[0] += (v * LPR + lane) * Vec<T>::N + e < cols ? d * d : 0.f;
      }
    row_sum<LPR, 1>(q, lds);
    const float rstd = 1.f / sqrtf(q[0] * inv + eps);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = (f[e] - mean) * rstd * fw[e] + fb[e];
    if (live) {
      store_row<T, NV, LPR>(y + row * cols, cols, lane, f);
      if (lane == 0 && mean_out) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
      }
    }
  }
}

// partial: [gridDim.x][2][cols] (dw, db), written only when want_param
template <typename T, int LPR, int NV>
__global__ __launch_bounds__(threads_of<LPR>()) void ln_bwd_kernel(const T *__restrict__ x, long long xs, const T *__restrict__ dy, long long ds,
                                                                   const void *w, int param_f32, const float *__restrict__ mean_in,
                                                                   const float *__restrict__ rstd_in, T *__restrict__ dx, float *__restrict__ partial,
                                                                   long long rows, int cols) {
  constexpr int VN = Vec<T>::N, N = NV * VN, TH = threads_of<LPR>(), RPB = TH / LPR;
  __shared__ float lds[LPR > 64 ? 2 * (LPR / 64) : 1];
  __shared__ float acc[RPB > 1 ? TH * N : 1];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  float fw[N], aw[N], ab[N];
  load_param<T, NV, LPR>(w, param_f32, cols, lane, 1.f, fw);
#pragma unroll
  for (int e = 0; e < N; ++e) aw[e] = ab[e] = 0.f;
  const float inv = 1.f / (float)cols;
  for (long long row0 = (long long)blockIdx.x * RPB; row0 < rows; row0 += (long long)gridDim.x * RPB) {
    const long long row = row0 + group;
    const bool live = row < rows;
    const long long r = live ? row : row0;
    float f[N], g[N];
    load_row<T, NV, LPR>(x + r * xs, cols, lane, f);
    load_row<T, NV, LPR>(dy + r * ds, cols, lane, g);
    const float mean = mean_in[r], rstd = rstd_in[r];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const int i = v * VN + e;
        // columns behind the end hold x = dy = 0: h is whatever (0 - mean) r is, so it is cleared
        const float h = (v * LPR + lane) * VN + e < cols ? (f[i] - mean) * rstd : 0.f;
        if (live) {
          aw[i] += g[i] * h;
          ab[i] += g[i];
        }
        g[i] *= fw[i];
        s[0] += g[i];
        s[1] += g[i] * h;
        f[i] = h;
      }
    if (dx) {
      row_sum<LPR, 2>(s, lds);
      const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = (g[e] - c1 - f[e] * c2) * rstd;
      if (live) store_row<T, NV, LPR>(dx + row * cols, cols, lane, f);
    }
  }
  if (!partial) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float *out = partial + ((long long)blockIdx.x * 2 + which) * cols;
    if constexpr (RPB > 1) {
      // the groups of the workgroup hold the same columns: add them up in LDS, group by group in a fixed order
      __syncthreads();
#pragma unroll
      for (int e = 0; e < N; ++e) acc[(group * N + e) * LPR + lane] = which ? ab[e] : aw[e];
      __syncthreads();
      for (int i = threadIdx.x; i < LPR * N; i += TH) {
        float t = 0.f;
        for (int gr = 0; gr < RPB; ++gr) t += acc[gr * LPR * N + i];
        const int e = i / LPR, l = i % LPR, c = ((e / VN) * LPR + l) * VN + e % VN;
        if (c < cols) out[c] = t;
      }
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          const int c = (v * LPR + lane) * VN + e;
          if (c < cols) out[c] = which ? ab[v * VN + e] : aw[v * VN + e];
        }
    }
  }
}

// dw / db = sum of the partial rows: 32 columns a workgroup, 32 slices of the partial rows side by side, joined in a fixed order
__global__ __launch_bounds__(1024) void ln_param_kernel(const float *__restrict__ partial, int nparts, int cols, void *dw, void *db, int param_f32) {
  __shared__ double s[32][33];
  const int lc = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lc;
  const int which = blockIdx.y;
  double t = 0;
  if (c < cols) {
#pragma unroll 4
    for (int p = slice; p < nparts; p += 32) t += (double)partial[((long long)p * 2 + which) * cols + c];
  }
  s[slice][lc] = t;
  __syncthreads();
  if (slice == 0 && c < cols) {
    double a = 0;
    for (int i = 0; i < 32; ++i) a += s[i][lc];
    void *out = which ? db : dw;
    if (out) {
      if (param_f32) ((float *)out)[c] = (float)a;
      else ((bf16 *)out)[c] = (bf16)(float)a;
    }
  }
}

constexpr int kMaxCols = 16384;

// Workgroups of the backward pass = rows of the partial sums: four per CU keep the memory busy; a partial row costs 8 bytes a column
int bwd_blocks(long long rows, int rows_per_block) {
  const long long want = (rows + rows_per_block - 1) / rows_per_block;
  return (int)(want < 1 ? 1 : (want > 1024 ? 1024 : want));
}

// lanes per row (LPR) and 16-byte vectors per lane (NV) that hold `cols` columns: the fewest registers a lane (two vectors at most, four for the widest
// fp32 rows: the backward pass keeps x, dy, w and two sums of each column) with the fewest lanes, rows within a wave as long as they fit one
struct Shape { int lpr, nv; };
template <typename T> Shape shape_of(int cols) {
  const int vec = (cols + Vec<T>::N - 1) / Vec<T>::N;
  if (vec <= 8) return {8, 1};
  if (vec <= 16) return {16, 1};
  if (vec <= 32) return {32, 1};
  if (vec <= 64) return {64, 1};
  if (vec <= 128) return {64, 2};
  if (vec <= 256) return {256, 1};
  if (vec <= 512) return {256, 2};
  if (vec <= 1024) return {1024, 1};
  if (vec <= 2048) return {1024, 2};
  return {1024, 4};
}
int rows_per_block(Shape s) { return (s.lpr > 256 ? s.lpr : 256) / s.lpr; }

struct Args {
  const void *x, *dy, *w, *b;
  void *y, *dx;
  long long xs, ds, rows;
  float *mean, *rstd, *partial;
  int cols, param_f32, blocks;
  float eps;
  hipStream_t st;
};

template <typename T, int LPR, int NV> void launch(const Args &a, bool backward) {
  constexpr int TH = threads_of<LPR>();
  if (backward)
    ln_bwd_kernel<T, LPR, NV><<<a.blocks, TH, 0, a.st>>>((const T *)a.x, a.xs, (const T *)a.dy, a.ds, a.w, a.param_f32, a.mean, a.rstd, (T *)a.dx,
                                                         a.partial, a.rows, a.cols);
  else
    ln_fwd_kernel<T, LPR, NV><<<a.blocks, TH, 0, a.st>>>((const T *)a.x, a.xs, a.w, a.b, a.param_f32, (T *)a.y, a.mean, a.rstd, a.rows, a.cols, a.eps);
}

template <typename T> void dispatch(const Args &a, bool backward) {
  const Shape s = shape_of<T>(a.cols);
  switch (s.lpr * 8 + s.nv) {
    case 8 * 8 + 1: return launch<T, 8, 1>(a, backward);
    case 16 * 8 + 1: return launch<T, 16, 1>(a, backward);
    case 32 * 8 + 1: return launch<T, 32, 1>(a, backward);
    case 64 * 8 + 1: return launch<T, 64, 1>(a, backward);
    case 64 * 8 + 2: return launch<T, 64, 2>(a, backward);
    case 256 * 8 + 1: return launch<T, 256, 1>(a, backward);
    case 256 * 8 + 2: return launch<T, 256, 2>(a, backward);
    case 1024 * 8 + 1: return launch<T, 1024, 1>(a, backward);
    case 1024 * 8 + 2: return launch<T, 1024, 2>(a, backward);
    default:
      if constexpr (sizeof(T) == 4) return launch<T, 1024, 4>(a, backward);   // bf16: kMaxCols fits the case above
  }
}

Shape shape_for(int cols, int dtype) { return dtype == MR3D_DTYPE_BF16 ? shape_of<bf16>(cols) : shape_of<float>(cols); }

int bad(const void *x, long long stride, long long rows, int cols, int dtype, int param_dtype) {
  if (!x || rows <= 0 || cols <= 0 || stride < 0) return MR3D_ERR_INVALID_ARG;
  if ((dtype != MR3D_DTYPE_F32 && dtype != MR3D_DTYPE_BF16) || (param_dtype != MR3D_DTYPE_F32 && param_dtype != dtype)) return MR3D_ERR_UNSUPPORTED;
  if (cols > kMaxCols) return MR3D_ERR_UNSUPPORTED;
  return MR3D_OK;
}

}  // namespace

extern "C" size_t mr3d_layer_norm_workspace_bytes(long long rows, int cols, int dtype) {
  if (rows <= 0 || cols <= 0 || cols > kMaxCols) return 0;
  return (size_t)bwd_blocks(rows, rows_per_block(shape_for(cols, dtype))) * 2 * (size_t)cols * sizeof(float);
}

extern "C" int mr3d_layer_norm_forward(const void *x, long long x_stride, const void *weight, const void *bias, void *y, float *mean, float *rstd,
                                       long long rows, int cols, float eps, int dtype, int param_dtype, mr3d_stream_t s) {
  if (const int e = bad(x, x_stride, rows, cols, dtype, param_dtype)) return e;
  if (!y || !(eps >= 0.f) || (mean == nullptr) != (rstd == nullptr)) return MR3D_ERR_INVALID_ARG;
  Args a{};
  a.x = x; a.xs = x_stride; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  a.rows = rows; a.cols = cols; a.eps = eps; a.param_f32 = param_dtype == MR3D_DTYPE_F32; a.st = mr3d_stream(s);
  const int rpb = rows_per_block(shape_for(cols, dtype));
  const long long want = (rows + rpb - 1) / rpb;
  a.blocks = (int)(want > 4096 ? 4096 : want);
  if (dtype == MR3D_DTYPE_BF16) dispatch<bf16>(a, false);
  else dispatch<float>(a, false);
  return mr3d_launch_status();
}

extern "C" int mr3d_layer_norm_backward(const void *x, long long x_stride, const void *dy, long long dy_stride, const void *weight, const float *mean,
                                        const float *rstd, void *dx, void *dweight, void *dbias, long long rows, int cols, int dtype,
                                        int param_dtype, void *workspace, size_t workspace_bytes, mr3d_stream_t s) {
  if (const int e = bad(x, x_stride, rows, cols, dtype, param_dtype)) return e;
  if (!dy || dy_stride < 0 || !mean || !rstd) return MR3D_ERR_INVALID_ARG;
  const bool param = dweight || dbias;
  if (!dx && !param) return MR3D_OK;
  if (param && (!workspace || workspace_bytes < mr3d_layer_norm_workspace_bytes(rows, cols, dtype))) return MR3D_ERR_WORKSPACE;
  Args a{};
  a.x = x; a.xs = x_stride; a.dy = dy; a.ds = dy_stride; a.w = weight; a.dx = dx;
  a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd); a.partial = param ? (float *)workspace : nullptr;
  a.rows = rows; a.cols = cols; a.param_f32 = param_dtype == MR3D_DTYPE_F32; a.st = mr3d_stream(s);
  a.blocks = bwd_blocks(rows, rows_per_block(shape_for(cols, dtype)));
  if (dtype == MR3D_DTYPE_BF16) dispatch<bf16>(a, true);
  else dispatch<float>(a, true);
  if (param) ln_param_kernel<<<dim3((cols + 31) / 32, 2), 1024, 0, a.st>>>(a.partial, a.blocks, cols, dweight, dbias, a.param_f32);
  return mr3d_launch_status();
}
