// Softmax cross entropy of a linear classifier over many classes, with its gradients, without the [rows][classes] logits:
//   z = x W^T + b      loss = sum_i w_i (lse(z_i) - z_i[label_i]) / avg
//   g = (softmax(z) - onehot(label)) w / avg      dx = g W      dW = g^T x      db = sum_i g
// 6 R V K operations with gradients; the loss and the gradients leave the same call (the caller scales them by the incoming gradient).
//   rows     live rows (weight not 0, label not ignored, row < valid_rows) are numbered; the others cost nothing further, take no part
//            in any product (NaN in them stays there) and get a zero row of dx
//   pack     live rows of x (and W, where its storage is not what the products read) into gemm16.h's operand form
//   logits   z tile by tile; a wave holds 128 classes of a row: it leaves exp(z - max of the 128) and (max, sum), the label's class left out: where a
//            row is certain of its label, 1 - p of the label is a sum of small exponentials, not a difference.  The exponentials take the place
//            of the logits: fp32, or for bf16 16 bits of that (pack_exp: 2^-10 of the value, a quarter of what g's rounding to bf16 loses)
//   grad     per row: lse from the (max, sum) pairs and the label's logit, a dot product in double; loss; exponentials -> g
//   dx, dw   g W (split over the classes, parts added in a fixed order) and g^T x
// g is kept as t g', t = w (1 - p_label) / avg in fp32: a row certain of its label has gradients as exact as the others, and dx rows take t at the end.
// bf16: the label's entry of g' is -1 and loses nothing to bf16 -- a rounding there would be the same for the whole row of dx; dW takes bf16(t x) in the
// place of x, db multiplies.  fp32: dW's factor is t g' with a scale per class and 128 rows (ce_slab_kernel).
// The exponentials of at most kPiece bytes of rows exist at a time; dW accumulates over such pieces in fp32.
// Measured, 8192 x 2048 x 131072 bf16 (7782 live rows): logits 3.9 ms (1.08 PFLOP/s, exponentials and their 2 GB of stores included), grad 0.93 (4.4 TB/s),
// dx 3.5, dW 3.5 (1.2).  3001 x 515 x 20011 fp32 (2010 live): logits 162 us, losses 12, g 105, gradients
// 305, packing 34.  512 x 1024 x 1204 fp32: nine launches, 64 us in all.  One row, 1024 x 32768 bf16: logits 16 us (W at 4.2 TB/s), 13 in four small launches.
// Recomputing z for the gradient instead (no such buffer at all) costs 2 R V K more: 1.7 ps a logit at 1024 features against 0.8 ps for the
// buffer's extra trip through memory.
#include "gemm16.h"

using namespace gemm16;

namespace {

typedef __bf16 bf16;
constexpr float kLog2e = 1.44269504f;
constexpr float kSG = 16384.f;                               // fp32: g of a row relative to 1 - p_label, in [-1, 1], times this
constexpr long long kPiece = 1ll << 31;
constexpr int kStatCols = 128;                               // classes per (max, sum) pair
constexpr int kSlabRows = 128, kSlabCols = 64;               // fp32: what a workgroup turns into g; a class has a scale per kSlabRows rows
constexpr int kScaleRows = 8192;                             // fp32: rows of dW in one launch, whose classes' scales lie in LDS (8 KB)

struct Ce {
  const char *x, *w, *bias;
  const long long *labels;
  const float *row_weight, *avg_dev;
  const int *valid_rows;
  float avg_host;
  long long x_stride, w_stride, ignore;                      // strides in elements
  int rows, hidden, classes, bias_f32;
  // workspace
  int *head;                                                 // [0] live rows  [1] avg (float)  float bits of the largest: [2] |W|  [3] |x|  [4] |W| of masked classes
  int *index, *pos;                                          // live row -> row, row -> live row or -1
  int *label;                                                // of a live row; -1: outside the classes
  float *xmax, *t;                                           // of a live row.  fp32: max |x|.  bf16: w (1 - p_label) / avg
  float4 *row;                                               // of a live row, fp32: maximum, 1 / sum of the others, w (1 - p_label) / avg, scale of all x / of this
  char *xp, *xwp, *wp;                                       // packed operands (wp may be the caller's W)
  long long ldx, ldw, ldg;                                   // bytes
  char *g, *gx;                                              // exponentials, then g (fp32: for dW); fp32: g for dx
  signed char *ge;                                           // fp32: exponent of a class's scale for dW, [slab][classes]
  float2 *stats;
  float *part;
  double *row_loss;
  float *dwacc, *dbpart;
  int cap, pieces, z;                                        // rows of a piece, (max, sum) pairs of a row, parts of dx
  char *dx, *dw, *db;
  float *loss;
  int db_f32;
};

// four or eight values at any element's alignment
typedef float vf4 __attribute__((ext_vector_type(4), aligned(4)));
typedef bf16 vb4 __attribute__((ext_vector_type(4), aligned(2)));
typedef bf16 vb8 __attribute__((ext_vector_type(8), aligned(2)));

template <bool F32> __device__ __forceinline__ float elem(const char *p, long long i) {
  return F32 ? ((const float *)p)[i] : (float)((const bf16 *)p)[i];
}

// e^v for v <= 0, one instruction behind the product.  The difference comes first: logits of the type's lowest value (a mask) times log2 e would be infinite
__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * kLog2e); }

// Two exponentials in [0, 1] as 16 bits each: of an fp32 value the sign and the upper bit of the exponent are 0 there, the next 16 bits are kept
// (rounded).  2^-10 of the value over fp32's whole range down to 2^-126: fp16 would have 2^-11, but only above 2^-14 of the largest of the 128
// classes, and nothing below 2^-25, where g in bf16 still has its 8 bits
__device__ __forceinline__ unsigned pack_exp(float a, float b) {
  return (__float_as_uint(a) + 0x2000u) >> 14 | ((__float_as_uint(b) + 0x2000u) << 2 & 0xffff0000u);
}
__device__ __forceinline__ float unpack_exp(unsigned short v) { return __uint_as_float((unsigned)v << 14); }

// largest power of two that keeps |v| <= max below 2^14
__device__ __forceinline__ float scale_for(float max) {
  if (!(max > 0.f) || !(max < 3.0e38f)) return 1.f;
  int e = 14 - (ilogbf(max) + 1);
  e = e > 100 ? 100 : e;
  return ldexpf(1.f, e);
}
__device__ __forceinline__ float scale_of_x(const Ce &c) { return scale_for(__int_as_float(c.head[3])); }
// fp32: a class whose bias masks it may have any (finite) weights: they do not set the scale, and are cut off at fp16's largest value.  Where every
// class is masked, they all count
constexpr float kMasked = -1e30f;
__device__ __forceinline__ bool masked_class(const Ce &c, int v) { return c.bias && ((const float *)c.bias)[v] <= kMasked; }
__device__ __forceinline__ float scale_of_w(const Ce &c) { return scale_for(__int_as_float(c.head[2] ? c.head[2] : c.head[4])); }

// live rows in order: a prefix sum over 1024 rows at a time by one workgroup
__global__ __launch_bounds__(1024) void ce_rows_kernel(Ce c) {
  __shared__ int wsum[16], wpos[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0, positive = 0;
  const int valid = c.valid_rows ? min(max(*c.valid_rows, 0), c.rows) : c.rows;
  for (int r0 = 0; r0 < c.rows; r0 += 1024) {
    const int r = r0 + threadIdx.x;
    bool live = false, pos = false;
    if (r < valid) {
      const float w = c.row_weight ? c.row_weight[r] : 1.f;
      live = w != 0.f && c.labels[r] != c.ignore;
      pos = live && w > 0.f;
    }
    const unsigned long long bl = __ballot(live), bp = __ballot(pos);
    if (lane == 0) {
      wsum[wave] = __popcll(bl);
      wpos[wave] = __popcll(bp);
    }
    __syncthreads();
    int before = base;
    for (int k = 0; k < 16; ++k) {
      if (k < wave) before += wsum[k];
      base += wsum[k];
      positive += wpos[k];
    }
    const int at = before + __popcll(bl & ((1ull << lane) - 1));
    if (live) {
      c.index[at] = r;
      c.label[at] = c.labels[r] >= 0 && c.labels[r] < c.classes ? (int)c.labels[r] : -1;
    }
    if (r < c.rows) c.pos[r] = live ? at : -1;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    c.head[0] = base;
    ((float *)c.head)[1] = c.avg_dev ? *c.avg_dev : (c.avg_host > 0.f ? c.avg_host : (float)max(positive, 1));
    c.head[2] = c.head[3] = c.head[4] = 0;
  }
}

__device__ __forceinline__ float block_max(float v, float *lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
}

// largest |p[k]| of each of kMaxRows rows as far as this lane sees it: 16 bytes a load with the alignment of a float (odd strides), the rows side
// by side so that a short one does not leave the wave waiting.  Rows that do not exist repeat the first
constexpr int kMaxRows = 4;
__device__ __forceinline__ void rows_max(const float *const (&p)[kMaxRows], int n, float (&m)[kMaxRows]) {
#pragma unroll
  for (int r = 0; r < kMaxRows; ++r) m[r] = 0.f;
  int k = (threadIdx.x & 63) * 4;
#pragma unroll 2
  for (; k + 4 <= n; k += 256)
#pragma unroll
    for (int r = 0; r < kMaxRows; ++r) {
      const vf4 t = *reinterpret_cast<const vf4 *>(p[r] + k);
      m[r] = fmaxf(fmaxf(fmaxf(m[r], fabsf(t[0])), fabsf(t[1])), fmaxf(fabsf(t[2]), fabsf(t[3])));
    }
  for (; k < n; ++k)                                        // the last, partial group: one lane's
#pragma unroll
    for (int r = 0; r < kMaxRows; ++r) m[r] = fmaxf(m[r], fabsf(p[r][k]));
}

// fp32: the largest |x| of each live row and of all, the largest |W|; four rows a wave, the first `xblocks` workgroups take x, the rest W.
// The maximum of positive floats is the maximum of their bits: an integer atomic, whose order does not matter -- one per workgroup, because
// a thousand of them on one address take 15 us
__global__ __launch_bounds__(256) void ce_max_kernel(Ce c, int xblocks, int wblocks) {
  __shared__ float lds[4];
  float m = 0.f, mm = 0.f, v[kMaxRows];
  const float *p[kMaxRows];
  const int wave = threadIdx.x >> 6;
  const bool is_x = (int)blockIdx.x < xblocks;
  if (is_x) {
    const int live = c.head[0];
    for (int j = (blockIdx.x * 4 + wave) * kMaxRows; j < live; j += xblocks * 4 * kMaxRows) {
#pragma unroll
      for (int r = 0; r < kMaxRows; ++r) p[r] = (const float *)c.x + c.index[j + r < live ? j + r : j] * c.x_stride;
      rows_max(p, c.hidden, v);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1)
#pragma unroll
        for (int r = 0; r < kMaxRows; ++r) v[r] = fmaxf(v[r], __shfl_xor(v[r], o));
#pragma unroll
      for (int r = 0; r < kMaxRows; ++r) {
        if (j + r >= live) break;
        if ((threadIdx.x & 63) == 0) c.xmax[j + r] = v[r];
        m = fmaxf(m, v[r]);
      }
    }
  } else {
    for (int j = ((blockIdx.x - xblocks) * 4 + wave) * kMaxRows; j < c.classes; j += wblocks * 4 * kMaxRows) {
#pragma unroll
      for (int r = 0; r < kMaxRows; ++r) p[r] = (const float *)c.w + (j + r < c.classes ? j + r : j) * c.w_stride;
      rows_max(p, c.hidden, v);
#pragma unroll
      for (int r = 0; r < kMaxRows; ++r) {
        const bool masked = masked_class(c, min(j + r, c.classes - 1));
        m = fmaxf(m, masked ? 0.f : v[r]);
        mm = fmaxf(mm, masked ? v[r] : 0.f);
      }
    }
  }
  m = block_max(m, lds);
  if (threadIdx.x == 0 && m > 0.f) atomicMax(&c.head[is_x ? 3 : 2], __float_as_int(m));
  if (is_x || !c.bias) return;
  __syncthreads();
  mm = block_max(mm, lds);
  if (threadIdx.x == 0 && mm > 0.f) atomicMax(&c.head[4], __float_as_int(mm));
}

// one stored row of an operand: bf16 copied, fp32 split; zeros behind the last column
template <bool F32> __device__ __forceinline__ void pack_row(const char *src, char *dst, long long ld, int cols, float scale, float most) {
  if constexpr (F32) {
    const float *s = (const float *)src;
    for (int k = threadIdx.x * 4; k < ld / 4; k += 1024) {
      _Float16 h[4], l[4];
      float t[4];
      if (k + 4 <= cols) *reinterpret_cast<vf4 *>(t) = *reinterpret_cast<const vf4 *>(s + k);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = k + e < cols ? s[k + e] : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u = t[e] * scale;
        split16(u > most ? most : u < -most ? -most : u, h[e], l[e]);                         // NaN stays
      }
      char *d = dst + (k >> 5) * 128 + (k & 31) * 2;
      *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<uint2 *>(h);
      *reinterpret_cast<uint2 *>(d + 64) = *reinterpret_cast<uint2 *>(l);
    }
  } else {
    const bf16 *s = (const bf16 *)src;
    for (int k = threadIdx.x * 8; k < ld / 2; k += 2048) {
      bf16 t[8];
      if (k + 8 <= cols) *reinterpret_cast<vb8 *>(t) = *reinterpret_cast<const vb8 *>(s + k);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = k + e < cols ? s[k + e] : (bf16)0.f;
      *reinterpret_cast<uint4 *>(dst + 2 * k) = *reinterpret_cast<uint4 *>(t);
    }
  }
}

template <bool F32>
__global__ __launch_bounds__(256) void ce_pack_kernel(Ce c) {
  const int b = blockIdx.x;
  if (b < c.rows) {
    if (b >= c.head[0]) return;
    const int r = c.index[b];
    const char *src = c.x + r * c.x_stride * (F32 ? 4 : 2);
    pack_row<F32>(src, c.xp + b * c.ldx, c.ldx, c.hidden, F32 ? scale_for(c.xmax[b]) : 1.f, INFINITY);
  } else {
    const int v = b - c.rows;
    pack_row<F32>(c.w + v * c.w_stride * (F32 ? 4 : 2), c.wp + v * c.ldw, c.ldw, c.hidden, F32 ? scale_of_w(c) : 1.f, F32 && masked_class(c, v) ? 65504.f : INFINITY);
  }
}

// z of one tile (classes x live rows) -> exponentials and (max, sum)
template <class T, bool TRAIN>
__global__ __launch_bounds__(T::THREADS, 2) void ce_logits_kernel(Ce c, int row0) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int live = min(c.head[0] - row0, c.cap);
  if (live <= 0) return;
  const int nti = (c.classes + T::BI - 1) / T::BI, ntj = (live + T::BJ - 1) / T::BJ;
  if ((int)blockIdx.x >= nti * ntj) return;
  int ti, tj;
  tile_of(blockIdx.x, nti * ntj, nti, ntj, ti, tj);
  f32x4 acc[T::TI][T::TJ];
  run<T>(lds, side_kc<T>(c.wp, c.ldw, c.classes, c.ldx, ti * T::BI, 0), side_kc<T>(c.xp + row0 * c.ldx, c.ldx, live, c.ldx, tj * T::BJ, 0),
         (int)(c.ldx / 128), acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave % T::NWI, wj = wave / T::NWI;
  const float rsw = T::SPLIT ? 1.f / scale_of_w(c) : 1.f;
  const int vpad = (int)(c.ldg / (T::SPLIT ? 4 : 2));
  constexpr int WI = T::TI * 16;
  static_assert(kStatCols % WI == 0, "a wave's classes lie in one pair");
  const bool ragged = (ti + 1) * T::BI > c.classes;
#pragma unroll
  for (int b = 0; b < T::TJ; ++b) {
    const int jl = (wj * T::TJ + b) * 16 + (lane & 15), j = tj * T::BJ + jl;
    const float rs = T::SPLIT ? rsw / scale_for(j < live ? c.xmax[row0 + j] : 0.f) : rsw;
    const int iw = ti * T::BI + wi * WI + (lane >> 4) * 4;
    if (c.bias) {
#pragma unroll
      for (int a = 0; a < T::TI; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = min(iw + a * 16 + e, c.classes - 1);
          acc[a][b][e] = fmaf(acc[a][b][e], rs, c.bias_f32 ? ((const float *)c.bias)[i] : (float)((const bf16 *)c.bias)[i]);
        }
    } else if constexpr (T::SPLIT) {
#pragma unroll
      for (int a = 0; a < T::TI; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[a][b][e] *= rs;
    }
    if (ragged) {
#pragma unroll
      for (int a = 0; a < T::TI; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (iw + a * 16 + e >= c.classes) acc[a][b][e] = -INFINITY;
    }
    const int own = (j < live ? c.label[row0 + j] : -1) - (ti * T::BI + wi * WI);
    if (__any(own >= 0 && own < WI)) {
#pragma unroll
      for (int a = 0; a < T::TI; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (own == (lane >> 4) * 4 + a * 16 + e) acc[a][b][e] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int a = 0; a < T::TI; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, acc[a][b][e]);
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const float ms = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int a = 0; a < T::TI; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = exp_of(acc[a][b][e] - ms);
        s += p;
        acc[a][b][e] = p;
      }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < 16 && j < live) c.stats[(long long)j * c.pieces + (ti * T::BI + wi * WI) / WI] = make_float2(m, s);
    if constexpr (TRAIN && T::SPLIT) {
      if (j < live) {
        char *row = c.g + j * c.ldg;
#pragma unroll
        for (int a = 0; a < T::TI; ++a)
          if (iw + a * 16 < vpad) *reinterpret_cast<f32x4 *>(row + (iw + a * 16) * 4) = acc[a][b];
      }
    } else if constexpr (TRAIN) {
      // through LDS, so that a row leaves in whole 16-byte pieces side by side; piece u of row jl sits at u ^ jl (a lane is a row)
#pragma unroll
      for (int a = 0; a < T::TI; ++a) {
        const int u = ((wi * WI + a * 16) >> 3) + (lane >> 5);
        *reinterpret_cast<uint2 *>(lds + jl * (T::BI * 2) + ((u ^ (jl & (T::BI / 8 - 1))) << 4) + ((lane >> 4) & 1) * 8) =
            make_uint2(pack_exp(acc[a][b][0], acc[a][b][1]), pack_exp(acc[a][b][2], acc[a][b][3]));
      }
    }
  }
  if constexpr (TRAIN && !T::SPLIT) {
    constexpr int U = T::BI / 8;                             // 16-byte pieces of a row
    __syncthreads();
    const int u = threadIdx.x % U, i = ti * T::BI + u * 8;
#pragma unroll 4
    for (int jl = threadIdx.x / U; jl < T::BJ; jl += T::THREADS / U) {
      const int j = tj * T::BJ + jl;
      if (j < live && i < vpad)
        *reinterpret_cast<uint4 *>(c.g + j * c.ldg + i * 2) = *reinterpret_cast<const uint4 *>(lds + jl * (T::BI * 2) + ((u ^ (jl & (U - 1))) << 4));
    }
  }
}

__device__ __forceinline__ double block_sum(double v, double *lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

// two sums at once, the same in every thread
__device__ __forceinline__ void block_sum(double &a, double &b, double (*lds)[4]) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  if ((threadIdx.x & 63) == 0) {
    lds[0][threadIdx.x >> 6] = a;
    lds[1][threadIdx.x >> 6] = b;
  }
  __syncthreads();
  a = lds[0][0] + lds[0][1] + lds[0][2] + lds[0][3];
  b = lds[1][0] + lds[1][1] + lds[1][2] + lds[1][3];
}

// one live row: log-sum-exp, loss, and (TRAIN) the exponentials become g (fp32: what ce_slab_kernel needs for it).  `wcols`: classes of a (max, sum) pair
template <bool F32, bool TRAIN>
__global__ __launch_bounds__(256) void ce_grad_kernel(Ce c, int row0, int wcols, int want_dw) {
  __shared__ double lds[2][4];
  __shared__ float ldm[4];
  const int j = blockIdx.x;
  if (j >= min(c.head[0] - row0, c.cap)) return;
  const int r = c.index[row0 + j];
  const float2 *st = c.stats + (long long)j * c.pieces;
  // the label's logit first: its loads wait for row and label, the pairs' do not
  const int label = c.label[row0 + j];                       // -1: the loss and this row's gradient are NaN
  double dot = 0;
  if (label >= 0) {
#pragma unroll 4
    for (int k = threadIdx.x; k < c.hidden; k += 256)
      dot += (double)elem<F32>(c.x, r * c.x_stride + k) * (double)elem<F32>(c.w, label * c.w_stride + k);
    if (threadIdx.x == 0 && c.bias) dot += c.bias_f32 ? (double)((const float *)c.bias)[label] : (double)(float)((const bf16 *)c.bias)[label];
  }
  float m = -INFINITY;
  bool nan = false;
  for (int k = threadIdx.x; k < c.pieces; k += 256) {
    const float v = st[k].x;
    nan |= v != v || st[k].y != st[k].y;                     // fmaxf drops a NaN
    m = fmaxf(m, v);
  }
  m = block_max(nan ? INFINITY : m, ldm);                    // infinity less infinity: the row's sums become NaN
  const float ms = m == -INFINITY ? 0.f : m;
  double s = 0;
  for (int k = threadIdx.x; k < c.pieces; k += 256) s += (double)st[k].y * (double)exp_of(st[k].x - ms);
  block_sum(s, dot, lds);
  // the others' sum is s e^m; with the label's e^d: 1 - p_label, and lse - z_label without a difference of sums where that is small
  const double d = label >= 0 ? dot : (double)NAN, top = fmax((double)m, d);
  const double others = s * exp((double)m - top), all = others + exp(d - top), rest = others / all;
  const double ce = ((double)m < d ? log1p(s * exp((double)m - d)) : (top - d) + log(all)) + (all - all);   // NaN stays
  const float w = c.row_weight ? c.row_weight[r] : 1.f;
  if (threadIdx.x == 0) c.row_loss[row0 + j] = ce * (double)w;
  if constexpr (TRAIN) {
    // exponentials relative to their pair's maximum -> p / (1 - p_label)
    const float f = s > 0 ? (float)(1. / s) : (float)(s * 0.), t = (float)(rest * (double)w / (double)((const float *)c.head)[1]);
    if constexpr (F32) {
      if (threadIdx.x == 0) c.row[row0 + j] = make_float4(ms, f, t, scale_of_x(c) / scale_for(c.xmax[row0 + j]));
    } else {
      char *row = c.g + j * c.ldg;
      for (long long k = threadIdx.x * 8; k < c.ldg / 2; k += 2048) {
        unsigned short p[8];
        bf16 v[8];
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(row + k * 2);
        const float e = exp_of(st[k / wcols].x - ms) * f;
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = (bf16)(k + q == label ? -1.f : unpack_exp(p[q]) * e);
        *reinterpret_cast<uint4 *>(row + k * 2) = *reinterpret_cast<uint4 *>(v);
      }
      if (threadIdx.x == 0) c.t[row0 + j] = t;
      if (want_dw) {
        const char *from = c.xp + (row0 + j) * c.ldx;
        char *to = c.xwp + (row0 + j) * c.ldx;
        for (long long k = threadIdx.x * 16; k < c.ldx; k += 4096) {
          bf16x8 v = *reinterpret_cast<const bf16x8 *>(from + k);
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = (bf16)((float)v[q] * t);
          *reinterpret_cast<bf16x8 *>(to + k) = v;
        }
      }
    }
  }
}

// fp32: the exponentials of kSlabRows rows x kSlabCols classes become g, as the two products and db want it.
//   dx  g' = p / (1 - p_label), the label's -1: relative to its row, the row's factor t joins at the end
//   dW  t g' over x's own scale: a class has a scale of its own (a power of two, for these rows, undone where the product's accumulators restart).
//       Fp16 planes relative to the row would lose the classes that are unlikely in every row: 22 bits end at 2^-17, all of them at 2^-39
//   db  sums of t g' in fp32
// Two forms of g are written where both are wanted: 105 us for 2010 rows of 20011 classes (4.6 TB/s).  16 threads a row, 8 rows a thread
__global__ __launch_bounds__(256) void ce_slab_kernel(Ce c, int row0, int wcols, int want_dx, int want_dw, int want_db) {
  __shared__ float lmax[16][kSlabCols], lsum[16][kSlabCols];
  __shared__ float4 rows[kSlabRows];
  __shared__ int labels[kSlabRows];
  const int live = min(c.head[0] - row0, c.cap), j0 = blockIdx.y * kSlabRows, i0 = blockIdx.x * kSlabCols, own = i0 + threadIdx.x;
  const bool column = threadIdx.x < kSlabCols && own < c.classes;
  if (j0 >= live) {
    if (want_db && !row0 && column) c.dbpart[(long long)blockIdx.y * c.classes + own] = 0.f;
    return;
  }
  const int cg = (threadIdx.x & 15) * 4, rg = threadIdx.x >> 4, i = i0 + cg;
  const bool in = i < c.ldg / 4;
  float v[8][4], m[4], s[4], top[8];
  const int i_load = in ? i : 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {                              // all loads side by side: what lies outside repeats the last row or the first classes
    const int j = min(j0 + rg + 16 * q, live - 1);
    *reinterpret_cast<float4 *>(v[q]) = *reinterpret_cast<const float4 *>(c.g + j * c.ldg + i_load * 4);
    top[q] = c.stats[(long long)j * c.pieces + i_load / wcols].x;
  }
  if (threadIdx.x < kSlabRows && j0 + (int)threadIdx.x < live) {
    rows[threadIdx.x] = c.row[row0 + j0 + threadIdx.x];
    labels[threadIdx.x] = c.label[row0 + j0 + threadIdx.x];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e) m[e] = s[e] = 0.f;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const int r = rg + 16 * q;
    if (j0 + r >= live) break;
    const float4 f = rows[r];
    const float e2 = exp_of(top[q] - f.x) * f.y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[q][e] = i + e == labels[r] ? -1.f : v[q][e] * e2;
      s[e] += v[q][e] * f.z;
      m[e] = fmaxf(m[e], fabsf(v[q][e] * (f.z * f.w)));
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    lmax[rg][cg + e] = m[e];
    lsum[rg][cg + e] = s[e];
  }
  __syncthreads();                                           // every load of g has returned too: what follows may be stored in its place
  float scale[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t = fmaxf(t, lmax[k][cg + e]);
    int k = 0;
    if (t > 0.f && t < 3.0e38f) k = min(max(13 - ilogbf(t), -100), 120);
    scale[e] = __int_as_float((127 + k) << 23);
    if (want_dw && rg == 0 && i + e < c.classes) c.ge[(long long)blockIdx.y * c.classes + i + e] = (signed char)k;
  }
  if (want_db && column) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += lsum[k][threadIdx.x];
    float *d = c.dbpart + (long long)blockIdx.y * c.classes + own;
    *d = row0 ? *d + t : t;                                  // pieces one after the other
  }
  if (!in) return;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const int r = rg + 16 * q;
    if (j0 + r >= live) break;
    const long long at = (j0 + r) * c.ldg + (i >> 5) * 128 + (i & 31) * 2;
    _Float16 hi[4], lo[4];
    if (want_dx) {
#pragma unroll
      for (int e = 0; e < 4; ++e) split16(v[q][e] * kSG, hi[e], lo[e]);
      *reinterpret_cast<uint2 *>(c.gx + at) = *reinterpret_cast<uint2 *>(hi);
      *reinterpret_cast<uint2 *>(c.gx + at + 64) = *reinterpret_cast<uint2 *>(lo);
    }
    if (want_dw) {
      const float f = rows[r].z * rows[r].w;
#pragma unroll
      for (int e = 0; e < 4; ++e) split16(v[q][e] * f * scale[e], hi[e], lo[e]);
      *reinterpret_cast<uint2 *>(c.g + at) = *reinterpret_cast<uint2 *>(hi);
      *reinterpret_cast<uint2 *>(c.g + at + 64) = *reinterpret_cast<uint2 *>(lo);
    }
  }
}

// part z of dx: live rows x hidden, summed over the z-th share of the classes
template <class T> __device__ __forceinline__ void dx_tile(const Ce &c, int row0, int bid, char *lds) {
  const int live = min(c.head[0] - row0, c.cap);
  if (live <= 0) return;
  const int nti = (c.hidden + T::BI - 1) / T::BI, ntj = (live + T::BJ - 1) / T::BJ;
  if (bid >= nti * ntj * c.z) return;
  const int zi = bid % c.z;
  const int ti = bid / c.z % nti, tj = bid / c.z / nti;
  const int total = (c.classes + T::KK - 1) / T::KK;
  const int s0 = (int)((long long)total * zi / c.z), s1 = (int)((long long)total * (zi + 1) / c.z);
  f32x4 acc[T::TI][T::TJ];
  run<T>(lds, side_ks<T>(c.wp, c.ldw, c.classes, c.ldx, ti * T::BI * (T::SPLIT ? 4 : 2), s0), side_kc<T>(T::SPLIT ? c.gx : c.g, c.ldg, live, c.ldg, tj * T::BJ, s0),
         s1 - s0, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave % T::NWI, wj = wave / T::NWI;
  const int hp = (c.hidden + 3) / 4 * 4;
#pragma unroll
  for (int b = 0; b < T::TJ; ++b) {
    const int j = tj * T::BJ + (wj * T::TJ + b) * 16 + (lane & 15);
    if (j >= live) continue;
    float *row = c.part + ((long long)zi * c.cap + j) * hp;
#pragma unroll
    for (int a = 0; a < T::TI; ++a) {
      const int i = ti * T::BI + (wi * T::TI + a) * 16 + (lane >> 4) * 4;
      if (i < hp) *reinterpret_cast<f32x4 *>(row + i) = acc[a][b];
    }
  }
}

// dx rows of the caller: the parts of a live row added up, zeros for the others
template <bool F32> __device__ __forceinline__ void dx_row(const Ce &c, int row0, int r) {
  const int live = min(c.head[0] - row0, c.cap);
  const int hp = (c.hidden + 3) / 4 * 4;
  const int p = c.pos[r];
  if (p >= 0 && (p < row0 || p >= row0 + live)) return;                       // another piece's row
  const float t = p < 0 ? 0.f : F32 ? c.row[p].z : c.t[p], ws = F32 ? 1.f / kSG / scale_of_w(c) : 1.f;      // one by one: their product may leave fp32's range
  for (int k = threadIdx.x * 4; k < c.hidden; k += 1024) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p >= 0) {
      for (int z = 0; z < c.z; ++z) {
        const float4 a = *reinterpret_cast<const float4 *>(c.part + ((long long)z * c.cap + p - row0) * hp + k);
        v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
      }
      v.x = v.x * ws * t; v.y = v.y * ws * t; v.z = v.z * ws * t; v.w = v.w * ws * t;
    }
    const float o[4] = {v.x, v.y, v.z, v.w};
    const long long at = (long long)r * c.hidden + k;
    if (k + 4 <= c.hidden) {
      if (F32) *reinterpret_cast<vf4 *>((float *)c.dx + at) = vf4{o[0], o[1], o[2], o[3]};
      else *reinterpret_cast<vb4 *>((bf16 *)c.dx + at) = vb4{(bf16)o[0], (bf16)o[1], (bf16)o[2], (bf16)o[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k + e < c.hidden) {
          if (F32) ((float *)c.dx)[at + e] = o[e];
          else ((bf16 *)c.dx)[at + e] = (bf16)o[e];
        }
    }
  }
}

// what kSlabRows rows add to this lane's classes: their scale undone, from LDS, and that of x
template <class T> struct ClassScales {
  const signed char *at;
  float f;
  __device__ __forceinline__ float operator()(int slab, int b) const { return f * __int_as_float((127 - at[slab * T::BJ + b * 16]) << 23); }
};

// dW tile: classes x hidden, summed over the piece's live rows (fp32: kScaleRows of them, from `from` on; a loop over them here costs 25 spilled
// registers and 15 % of the time).  mode 0: store in the caller's type, 1: store to / 2: add to an fp32 accumulator
template <class T> __device__ __forceinline__ void dw_tile(const Ce &c, int row0, int mode, int from, int bid, char *lds) {
  int live = max(min(c.head[0] - row0, c.cap), 0);
  if (live <= from && row0 + from) return;
  const int nti = (c.hidden + T::BI - 1) / T::BI, ntj = (c.classes + T::BJ - 1) / T::BJ;
  int ti, tj;
  tile_of(bid, nti * ntj, nti, ntj, ti, tj);
  constexpr int E = T::SPLIT ? 4 : 2;
  const char *x = (T::SPLIT ? c.xp : c.xwp) + row0 * c.ldx;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave % T::NWI, wj = wave / T::NWI;
  f32x4 acc[T::TI][T::TJ];
  if constexpr (T::SPLIT) {
    static_assert(T::RESTART * T::KK == kSlabRows, "a part of the sums is a slab");
    live = min(live, from + kScaleRows);
    signed char *scales = reinterpret_cast<signed char *>(lds + T::LDS_BYTES);
    for (int k = threadIdx.x; k < kScaleRows / kSlabRows * T::BJ; k += T::THREADS) {
      const int j = tj * T::BJ + k % T::BJ, slab = from / kSlabRows + k / T::BJ;
      scales[k] = j < c.classes && slab * kSlabRows < live ? c.ge[(long long)slab * c.classes + j] : 0;
    }
    __syncthreads();
    const int s = from / T::KK;
    run<T>(lds, side_ks<T>(x, c.ldx, live, c.ldx, ti * T::BI * E, s), side_ks<T>(c.g, c.ldg, live, c.ldg, (long long)tj * T::BJ * E, s),
           (live - from + T::KK - 1) / T::KK, acc, ClassScales<T>{scales + wj * T::TJ * 16 + (lane & 15), 1.f / scale_of_x(c)});
  } else {
    run<T>(lds, side_ks<T>(x, c.ldx, live, c.ldx, ti * T::BI * E, 0), side_ks<T>(c.g, c.ldg, live, c.ldg, (long long)tj * T::BJ * E, 0),
           (live + T::KK - 1) / T::KK, acc);
  }
#pragma unroll
  for (int b = 0; b < T::TJ; ++b) {
    const int j = tj * T::BJ + (wj * T::TJ + b) * 16 + (lane & 15);
    if (j >= c.classes) continue;
#pragma unroll
    for (int a = 0; a < T::TI; ++a) {
      const int i = ti * T::BI + (wi * T::TI + a) * 16 + (lane >> 4) * 4;
      const f32x4 v = acc[a][b];
      const long long at = (long long)j * c.hidden + i;
      const bool whole = i + 4 <= c.hidden;
      if (T::SPLIT || mode) {
        float *d = (T::SPLIT ? (float *)c.dw : c.dwacc) + at;
        if (whole) {
          vf4 t = {v[0], v[1], v[2], v[3]};
          if (mode == 2) t += *reinterpret_cast<const vf4 *>(d);
          *reinterpret_cast<vf4 *>(d) = t;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < c.hidden) d[e] = mode == 2 ? d[e] + v[e] : v[e];
        }
      } else {
        bf16 *d = (bf16 *)c.dw + at;
        if (whole) {
          *reinterpret_cast<vb4 *>(d) = vb4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < c.hidden) d[e] = (bf16)v[e];
        }
      }
    }
  }
}

__global__ __launch_bounds__(256) void ce_dw_round_kernel(const float *__restrict__ acc, bf16 *__restrict__ dw, long long n) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) dw[i] = (bf16)acc[i];
}

// bf16's db: column sums of g.  A workgroup adds kDbRows rows of 256 columns: 8 columns (16 bytes) a thread and 8 rows side
// by side, which meet in LDS; the parts are added in order afterwards
constexpr int kDbRows = 64;
__device__ __forceinline__ void db_part(const Ce &c, int row0, int bx, int slice, char *lds) {
  float (*sum)[256] = reinterpret_cast<float (*)[256]>(lds);
  const int live = min(c.head[0] - row0, c.cap);
  const int j0 = slice * kDbRows, j1 = min(j0 + kDbRows, live);
  const int col = (threadIdx.x & 31) * 8, i = bx * 256 + col, sub = threadIdx.x >> 5;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.f;
  if (i < c.classes) {                                       // whole groups of 8 exist: rows are padded with zeros
#pragma unroll 4
    for (int j = j0 + sub; j < j1; j += 8) {
      const bf16x8 v = *reinterpret_cast<const bf16x8 *>(c.g + j * c.ldg + i * 2);
      const float t = c.t[row0 + j];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += (float)v[e] * t;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[sub][col + e] = s[e];
  __syncthreads();
  const int o = bx * 256 + threadIdx.x;
  if (o >= c.classes) return;
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) t += sum[k][threadIdx.x];
  float *d = c.dbpart + (long long)slice * c.classes + o;
  *d = row0 ? *d + t : t;                                    // pieces one after the other
}

// The gradients' launches.  Tiles of 64 and 128 (one workgroup shape) share one launch, bf16 with db's sums: each alone leaves CUs idle
template <class TX, class TW>
__global__ __launch_bounds__(256, 2) void ce_gradients_kernel(Ce c, int row0, int mode, int from, int dx_blocks, int dw_blocks, int db_blocks) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  int b = blockIdx.x;
  if (b < dx_blocks) return dx_tile<TX>(c, row0, b, lds);
  b -= dx_blocks;
  if (b < dw_blocks) return dw_tile<TW>(c, row0, mode, from, b, lds);
  b -= dw_blocks;
  if constexpr (!TX::SPLIT) db_part(c, row0, b % db_blocks, b / db_blocks, lds);
}
template <class T> __global__ __launch_bounds__(T::THREADS, 2) void ce_dx_kernel(Ce c, int row0) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  dx_tile<T>(c, row0, blockIdx.x, lds);
}
template <class T> __global__ __launch_bounds__(T::THREADS, 2) void ce_dw_kernel(Ce c, int row0, int mode) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  dw_tile<T>(c, row0, mode, 0, blockIdx.x, lds);
}
__global__ __launch_bounds__(256) void ce_db_kernel(Ce c, int row0) {
  __shared__ __attribute__((aligned(16))) char lds[8 * 256 * 4];
  db_part(c, row0, blockIdx.x, blockIdx.y, lds);
}

// live rows of dx of a piece that is not the last
template <bool F32> __global__ __launch_bounds__(256) void ce_dx_rows_kernel(Ce c, int row0) {
  if (row0 + (int)blockIdx.x < c.head[0]) dx_row<F32>(c, row0, c.index[row0 + blockIdx.x]);
}

// The last launch.  Workgroup 0: the loss, row by row in order; the next db_blocks: db, 64 columns each, the slices four side by side; the others:
// the rows of dx of the last piece (from row0 on) and those that do not count
template <bool F32> __global__ __launch_bounds__(256) void ce_finish_kernel(Ce c, int slices, int db_blocks, int row0) {
  __shared__ double sum[4][64];
  if ((int)blockIdx.x > db_blocks) return dx_row<F32>(c, row0, blockIdx.x - 1 - db_blocks);
  if (blockIdx.x == 0) {
    double s = 0;
    const int live = c.head[0];
#pragma unroll 4
    for (int j = threadIdx.x; j < live; j += 256) s += c.row_loss[j];
    s = block_sum(s, sum[0]);
    if (threadIdx.x == 0) c.loss[0] = (float)(s / (double)((const float *)c.head)[1]);
    return;
  }
  const int col = threadIdx.x & 63, sub = threadIdx.x >> 6, i = (blockIdx.x - 1) * 64 + col;
  double s = 0;
  if (i < c.classes) {
#pragma unroll 8
    for (int k = sub; k < slices; k += 4) s += (double)c.dbpart[(long long)k * c.classes + i];
  }
  sum[sub][col] = s;
  __syncthreads();
  if (sub || i >= c.classes) return;
  s = sum[0][col] + sum[1][col] + sum[2][col] + sum[3][col];
  if (c.db_f32) ((float *)c.db)[i] = (float)s;
  else ((bf16 *)c.db)[i] = (bf16)(float)s;
}

// gradients *= *factor, unless the factor is 1 (the usual root of a backward pass): then nothing is read or written.  bf16 gradients are rounded here a
// second time (2^-8 at most; exact for powers of two): kept in fp32 until now they would cost as much memory again as x and W
struct Spans { mr3d_span s[4]; };
__global__ __launch_bounds__(256) void ce_scale_kernel(Spans spans, const float *__restrict__ factor) {
  const float f = *factor;
  if (f == 1.f) return;
  const mr3d_span p = spans.s[blockIdx.y];
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < p.count; i += (long long)gridDim.x * 256) {
    if (p.dtype == MR3D_DTYPE_F32) ((float *)p.data)[i] *= f;
    else ((bf16 *)p.data)[i] = (bf16)((float)((bf16 *)p.data)[i] * f);
  }
}

// Tiles.  bf16: 256 x 256 (8 waves of 128 x 64, one workgroup a CU) has the fewest LDS bytes per product; it needs enough tiles to fill 256 CUs.
// 128 x 128 (4 waves of 64 x 64, two workgroups a CU) below that, and for fp32, whose restarted sums leave no room for the large tile's
// accumulators.  64 x 64 (three workgroups a CU) where even those would leave CUs without one: 1024^3, fp32: 25 -> 14 us.
template <bool IKS, bool JKS, bool SPLIT> struct Tiles {
  typedef Tile<64, 64, 2, 2, IKS, JKS, SPLIT, 3> Tiny;
  typedef Tile<128, 128, 2, 2, IKS, JKS, SPLIT, 2> Small;
  typedef Tile<256, 256, 2, 4, IKS, JKS, SPLIT, 2> Large;
};
template <bool IKS, bool JKS> struct Tiles<IKS, JKS, true> {
  typedef Tile<64, 64, 2, 2, IKS, JKS, true, 3> Tiny;
  typedef Tile<128, 128, 2, 2, IKS, JKS, true, 2> Small;
  typedef Small Large;
};
long long tiles_of(long long i, long long j, int bt) { return ((i + bt - 1) / bt) * ((j + bt - 1) / bt); }
// z: ways the k axis may be split
int tile_for(bool f32, long long i, long long j, long long z) {
  if (!f32 && tiles_of(i, j, 256) >= 192) return 256;
  return tiles_of(i, j, 128) * z >= 160 ? 128 : 64;
}

long long up(long long v, long long a) { return (v + a - 1) / a * a; }

struct Layout {
  size_t bytes, head, index, pos, label, xmax, row, xp, xwp, wp, g, gx, ge, stats, part, row_loss, dwacc, dbpart;
  long long ldx, ldw, ldg;
  int cap, chunks, pieces, z, wcols, db_slices;
  int bt_logits, bt_dx, bt_dw;
  bool pack_w;
};

size_t take(size_t &at, size_t bytes) {
  const size_t here = at;
  at = mr3d_align_up(at + bytes, 1024);
  return here;
}

int layout_of(const mr3d_linear_ce *a, Layout &l) {
  if (!a || a->rows <= 0 || a->hidden <= 0 || a->classes <= 0) return MR3D_ERR_INVALID_ARG;
  if (a->dtype != MR3D_DTYPE_F32 && a->dtype != MR3D_DTYPE_BF16) return MR3D_ERR_UNSUPPORTED;
  if (a->param_dtype != MR3D_DTYPE_F32 && a->param_dtype != a->dtype) return MR3D_ERR_UNSUPPORTED;
  if (a->rows > (1 << 22) || a->hidden > (1 << 16) || a->classes > (1 << 20)) return MR3D_ERR_UNSUPPORTED;
  if (a->x_stride < a->hidden || a->weight_stride < a->hidden) return MR3D_ERR_INVALID_ARG;
  const bool f32 = a->dtype == MR3D_DTYPE_F32, train = a->want_dx || a->want_dweight || a->want_dbias;
  l = Layout{};
  size_t at = 0;
  l.ldx = up(a->hidden, f32 ? 32 : 64) * (f32 ? 4 : 2);
  l.ldg = up(a->classes, f32 ? 32 : 64) * (f32 ? 4 : 2);
  // bf16 weights are read where they are when a row is whole 128-byte k-steps on 16-byte boundaries, and 256 rows lie within the 32-bit
  // offsets of a tile's loads
  l.pack_w = f32 || a->hidden % 64 || a->weight_stride % 8 || a->weight_stride > 1 << 21 || ((uintptr_t)a->weight & 15);
  l.ldw = l.pack_w ? l.ldx : a->weight_stride * 2;
  l.chunks = 1;
  // bytes a row of a piece needs: its exponentials (fp32 with dx and dW: and a second form of g), or only its (max, sum) pairs (one for 32 classes at most)
  const bool two = f32 && a->want_dx && a->want_dweight;
  const long long row_bytes = train ? l.ldg * (two ? 2 : 1) : up(a->classes, 64) / 32 * 8;
  long long cap = a->rows;
  if (cap * row_bytes > kPiece) {
    cap = kPiece / row_bytes / 256 * 256;
    if (cap < 256) cap = 256;
    l.chunks = (int)((a->rows + cap - 1) / cap);
  }
  l.cap = (int)cap;
  l.bt_logits = tile_for(f32, a->classes, cap, 1);
  l.wcols = l.bt_logits / 2;                                 // a wave's share of a tile
  l.pieces = (int)(up(a->classes, l.bt_logits) / l.wcols);
  l.head = take(at, 64);
  l.index = take(at, (size_t)a->rows * 4);
  l.pos = take(at, (size_t)a->rows * 4);
  l.row_loss = take(at, (size_t)a->rows * 8);
  l.label = take(at, (size_t)a->rows * 4);
  l.xmax = take(at, (size_t)a->rows * 4);
  l.xp = take(at, (size_t)(a->rows * l.ldx));
  if (f32 && train) l.row = take(at, (size_t)a->rows * 16);
  if (!f32 && a->want_dweight) l.xwp = take(at, (size_t)(a->rows * l.ldx));
  if (l.pack_w) l.wp = take(at, (size_t)(a->classes * l.ldx));
  l.stats = take(at, (size_t)cap * l.pieces * 8);
  if (train) l.g = l.gx = take(at, (size_t)(cap * l.ldg));
  if (two) l.gx = take(at, (size_t)(cap * l.ldg));
  if (f32 && a->want_dweight) l.ge = take(at, (size_t)((cap + kSlabRows - 1) / kSlabRows * a->classes));
  if (a->want_dx) {
    // parts over the classes until two workgroups a CU have work; a part keeps 16 k-steps
    const long long steps = l.ldg / 128, most = steps / 16 > 1 ? steps / 16 : 1;
    l.bt_dx = tile_for(f32, a->hidden, cap, most);
    long long tiles = tiles_of(a->hidden, cap, l.bt_dx), z = l.bt_dx == 256 || tiles >= 512 ? 1 : 512 / tiles;
    // the large tile with a part of the classes each, where that makes 192 to 256 workgroups (2048 x 2048 x 131072: 3.19 -> 2.97 ms in all)
    const long long large = tiles_of(a->hidden, cap, 256), zl = 256 / large;
    if (!f32 && zl > 1 && zl <= most && large * zl >= 192) {
      l.bt_dx = 256;
      z = zl;
    }
    if (z > most) z = most;
    l.z = (int)z;
    l.part = take(at, (size_t)l.z * cap * up(a->hidden, 4) * 4);
  }
  l.bt_dw = tile_for(f32, a->hidden, a->classes, 1);
  if (a->want_dweight && !f32 && l.chunks > 1) l.dwacc = take(at, (size_t)a->classes * a->hidden * 4);
  if (a->want_dbias) {
    l.db_slices = f32 ? (int)((cap + kSlabRows - 1) / kSlabRows) : (int)((cap + kDbRows - 1) / kDbRows);
    l.dbpart = take(at, (size_t)l.db_slices * a->classes * 4);
  }
  l.bytes = at;
  return MR3D_OK;
}

template <class K> int allow_lds(K kernel, int bytes) {
  return hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess ? MR3D_OK : MR3D_ERR_LAUNCH;
}

template <class T, bool TRAIN> int launch_logits(const Ce &c, int row0, hipStream_t q) {
  if (T::LDS_BYTES > 65536)
    if (const int e = allow_lds(ce_logits_kernel<T, TRAIN>, T::LDS_BYTES)) return e;
  const long long n = (long long)((c.classes + T::BI - 1) / T::BI) * ((c.cap + T::BJ - 1) / T::BJ);
  ce_logits_kernel<T, TRAIN><<<(unsigned)n, T::THREADS, T::LDS_BYTES, q>>>(c, row0);
  return MR3D_OK;
}
template <class T> int dx_blocks(const Ce &c) { return (c.hidden + T::BI - 1) / T::BI * ((c.cap + T::BJ - 1) / T::BJ) * c.z; }
template <class T> int dw_blocks(const Ce &c) { return (c.hidden + T::BI - 1) / T::BI * ((c.classes + T::BJ - 1) / T::BJ); }
template <class T> int launch_dx(const Ce &c, int row0, hipStream_t q) {
  if (T::LDS_BYTES > 65536)
    if (const int e = allow_lds(ce_dx_kernel<T>, T::LDS_BYTES)) return e;
  ce_dx_kernel<T><<<dx_blocks<T>(c), T::THREADS, T::LDS_BYTES, q>>>(c, row0);
  return MR3D_OK;
}
template <class T> int launch_dw(const Ce &c, int row0, int mode, hipStream_t q) {
  if (T::LDS_BYTES > 65536)
    if (const int e = allow_lds(ce_dw_kernel<T>, T::LDS_BYTES)) return e;
  ce_dw_kernel<T><<<dw_blocks<T>(c), T::THREADS, T::LDS_BYTES, q>>>(c, row0, mode);
  return MR3D_OK;
}
template <class TX, class TW> int launch_gradients(const mr3d_linear_ce *a, const Ce &c, int row0, int mode, hipStream_t q) {
  constexpr bool F32 = TX::SPLIT;
  constexpr int ldw = TW::LDS_BYTES + (F32 ? kScaleRows / kSlabRows * TW::BJ : 0), lds = TX::LDS_BYTES > ldw ? TX::LDS_BYTES : ldw;
  static_assert(lds <= 81920 && lds >= 8192 && TX::THREADS == 256 && TW::THREADS == 256, "two workgroups a CU");
  const int nw = a->want_dweight ? dw_blocks<TW>(c) : 0, nb = (a->classes + 255) / 256;
  if (lds > 65536)
    if (const int e = allow_lds(ce_gradients_kernel<TX, TW>, lds)) return e;
  for (int from = 0; from == 0 || (F32 && nw && from < c.cap); from += kScaleRows) {
    const int nx = a->want_dx && !from ? dx_blocks<TX>(c) : 0, n = nx + nw + (!F32 && a->want_dbias ? nb * ((c.cap + kDbRows - 1) / kDbRows) : 0);
    if (n) ce_gradients_kernel<TX, TW><<<n, 256, lds, q>>>(c, row0, from ? 2 : mode, from, nx, nw, nb);
  }
  return MR3D_OK;
}

template <class TT, class F> int pick(int bt, F f) {
  return bt == 256 ? f(typename TT::Large()) : bt == 128 ? f(typename TT::Small()) : f(typename TT::Tiny());
}

template <bool F32> int run_ce(const mr3d_linear_ce *a, const Layout &l, Ce &c, hipStream_t q) {
  const bool train = a->want_dx || a->want_dweight || a->want_dbias;
  typedef Tiles<false, false, F32> TL;
  typedef Tiles<true, false, F32> TX;
  typedef Tiles<true, true, F32> TW;
  ce_rows_kernel<<<1, 1024, 0, q>>>(c);
  if (F32) {
    const int per = 4 * kMaxRows, xb = a->rows < 128 * per ? (a->rows + per - 1) / per : 128, wb = a->classes < 512 * per ? (a->classes + per - 1) / per : 512;
    ce_max_kernel<<<xb + wb, 256, 0, q>>>(c, xb, wb);
  }
  ce_pack_kernel<F32><<<a->rows + (l.pack_w ? a->classes : 0), 256, 0, q>>>(c);
  for (int k = 0; k < l.chunks; ++k) {
    const int row0 = k * l.cap;
    int e = MR3D_OK;
    if (train) {
      e = pick<TL>(l.bt_logits, [&](auto t) { return launch_logits<decltype(t), true>(c, row0, q); });
      ce_grad_kernel<F32, true><<<l.cap, 256, 0, q>>>(c, row0, l.wcols, a->want_dweight);
    } else {
      e = pick<TL>(l.bt_logits, [&](auto t) { return launch_logits<decltype(t), false>(c, row0, q); });
      ce_grad_kernel<F32, false><<<l.cap, 256, 0, q>>>(c, row0, l.wcols, a->want_dweight);
    }
    if (e) return e;
    const int mode = k ? 2 : (l.chunks > 1 ? 1 : 0);
    if (!train) continue;
    if (F32)
      ce_slab_kernel<<<dim3((unsigned)((l.ldg / 4 + kSlabCols - 1) / kSlabCols), (l.cap + kSlabRows - 1) / kSlabRows), 256, 0, q>>>(c, row0, l.wcols, a->want_dx,
                                                                                                                     a->want_dweight, a->want_dbias);
    if (F32 || ((!a->want_dx || l.bt_dx < 256) && (!a->want_dweight || l.bt_dw < 256))) {
      if (l.bt_dx == 128 && l.bt_dw == 128) e = launch_gradients<typename TX::Small, typename TW::Small>(a, c, row0, mode, q);
      else if (l.bt_dx == 128) e = launch_gradients<typename TX::Small, typename TW::Tiny>(a, c, row0, mode, q);
      else if (l.bt_dw == 128) e = launch_gradients<typename TX::Tiny, typename TW::Small>(a, c, row0, mode, q);
      else e = launch_gradients<typename TX::Tiny, typename TW::Tiny>(a, c, row0, mode, q);
      if (e) return e;
    } else if constexpr (!F32) {
      if (a->want_dx) e = pick<TX>(l.bt_dx, [&](auto t) { return launch_dx<decltype(t)>(c, row0, q); });
      if (e) return e;
      if (a->want_dweight) e = pick<TW>(l.bt_dw, [&](auto t) { return launch_dw<decltype(t)>(c, row0, mode, q); });
      if (e) return e;
      if (a->want_dbias) ce_db_kernel<<<dim3((a->classes + 255) / 256, (l.cap + kDbRows - 1) / kDbRows), 256, 0, q>>>(c, row0);
    }
    if (a->want_dx && k + 1 < l.chunks) ce_dx_rows_kernel<F32><<<l.cap, 256, 0, q>>>(c, row0);
  }
  if (a->want_dweight && l.dwacc) ce_dw_round_kernel<<<2048, 256, 0, q>>>(c.dwacc, (bf16 *)c.dw, (long long)a->classes * a->hidden);
  const int db_blocks = a->want_dbias ? (a->classes + 63) / 64 : 0;
  ce_finish_kernel<F32><<<1 + db_blocks + (a->want_dx ? a->rows : 0), 256, 0, q>>>(c, l.db_slices, db_blocks, (l.chunks - 1) * l.cap);
  return mr3d_launch_status();
}

}  // namespace

extern "C" size_t mr3d_linear_cross_entropy_workspace_bytes(const mr3d_linear_ce *args_host) {
  Layout l;
  return layout_of(args_host, l) == MR3D_OK ? l.bytes : 0;
}

extern "C" int mr3d_linear_cross_entropy(const mr3d_linear_ce *a, void *workspace, size_t workspace_bytes, mr3d_stream_t s) {
  Layout l;
  if (const int e = layout_of(a, l)) return e;
  if (!a->x || !a->weight || !a->labels || !a->loss) return MR3D_ERR_INVALID_ARG;
  if ((a->want_dx && !a->dx) || (a->want_dweight && !a->dweight) || (a->want_dbias && (!a->dbias || !a->bias))) return MR3D_ERR_INVALID_ARG;
  if (!(a->avg_factor >= 0.f)) return MR3D_ERR_INVALID_ARG;
  if (!workspace || ((uintptr_t)workspace & 1023) || workspace_bytes < l.bytes) return MR3D_ERR_WORKSPACE;
  char *b = (char *)workspace;
  Ce c{};
  c.x = (const char *)a->x; c.w = (const char *)a->weight; c.bias = (const char *)a->bias;
  c.labels = a->labels; c.row_weight = a->row_weight; c.avg_dev = a->avg_factor_dev; c.valid_rows = a->valid_rows_dev;
  c.avg_host = a->avg_factor;
  c.x_stride = a->x_stride; c.w_stride = a->weight_stride; c.ignore = a->ignore_index;
  c.rows = a->rows; c.hidden = a->hidden; c.classes = a->classes;
  c.bias_f32 = c.db_f32 = a->param_dtype == MR3D_DTYPE_F32;
  c.head = (int *)(b + l.head); c.index = (int *)(b + l.index); c.pos = (int *)(b + l.pos);
  c.label = (int *)(b + l.label);
  c.xmax = c.t = (float *)(b + l.xmax);
  c.row = (float4 *)(b + l.row);
  c.xp = b + l.xp; c.xwp = b + l.xwp;
  c.wp = l.pack_w ? b + l.wp : (char *)const_cast<void *>(a->weight);
  c.ldx = l.ldx; c.ldw = l.ldw; c.ldg = l.ldg;
  c.g = b + l.g; c.gx = b + l.gx; c.ge = (signed char *)(b + l.ge);
  c.stats = (float2 *)(b + l.stats); c.part = (float *)(b + l.part);
  c.row_loss = (double *)(b + l.row_loss);
  c.dwacc = (float *)(b + l.dwacc); c.dbpart = (float *)(b + l.dbpart);
  c.cap = l.cap; c.pieces = l.pieces; c.z = l.z;
  c.dx = (char *)a->dx; c.dw = (char *)a->dweight; c.db = (char *)a->dbias; c.loss = a->loss;
  return a->dtype == MR3D_DTYPE_F32 ? run_ce<true>(a, l, c, mr3d_stream(s)) : run_ce<false>(a, l, c, mr3d_stream(s));
}

extern "C" int mr3d_scale_by(const mr3d_span *spans_host, int num_spans, const float *factor_dev, mr3d_stream_t s) {
  if (!spans_host || num_spans < 1 || num_spans > 4 || !factor_dev) return MR3D_ERR_INVALID_ARG;
  Spans spans{};
  long long most = 0;
  for (int i = 0; i < num_spans; ++i) {
    const mr3d_span &p = spans_host[i];
    if (p.count < 0 || (p.count && !p.data)) return MR3D_ERR_INVALID_ARG;
    if (p.dtype != MR3D_DTYPE_F32 && p.dtype != MR3D_DTYPE_BF16) return MR3D_ERR_UNSUPPORTED;
    spans.s[i] = p;
    most = p.count > most ? p.count : most;
  }
  if (!most) return MR3D_OK;
  const long long blocks = (most + 2047) / 2048;
  ce_scale_kernel<<<dim3((unsigned)(blocks > 1024 ? 1024 : blocks), num_spans), 256, 0, mr3d_stream(s)>>>(spans, factor_dev);
  return mr3d_launch_status();
}
