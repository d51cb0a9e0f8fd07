// Matrix products with what follows them, on the ordinary arithmetic units: C[m, n] = sum_k A[m, k] B[n, k]
// with any strides, 64 x 64 results per block of 256 threads, fp32 sums.
#pragma once
#include "leaf_sum.cuh"

namespace tb {

template <class T> struct Operand { // element (row, k) at p[row * sr + k * sk]
  const T *p;
  long long sr, sk;
};

__device__ __forceinline__ float act_value(float z, int act) {
  if (act == 1) return z < 0.f ? 0.f : z; // (NaN stays)
  if (act == 2) return 0.5f * z * (1.f + erff(z * 0.70710678f));
  if (act == 3) return z / (1.f + expf(-z));
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == 1) return z > 0.f ? 1.f : 0.f;
  if (act == 2) return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * expf(-0.5f * z * z);
  if (act == 3) {
    const float s = 1.f / (1.f + expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  return 1.f;
}

template <class T> struct LinearEnd {
  const T *bias, *residual;
  long long ld_residual;
  T *out, *pre;
  long long ld_out, ld_pre;
  int act;
  __device__ void tile(const float (*c)[65], long long m0, long long n0, long long M, long long N) const {
    for (int i = threadIdx.x; i < 4096; i += 256) {
      const long long m = m0 + i / 64, n = n0 + i % 64;
      if (m >= M || n >= N) continue;
      float z = c[i / 64][i % 64] + (bias ? to_float(bias[n]) : 0.f);
      if (pre) pre[m * ld_pre + n] = from_float<T>(z);
      z = act_value(z, act);
      out[m * ld_out + n] = from_float<T>(residual ? z + to_float(residual[m * ld_residual + n]) : z);
    }
  }
};

// sum over a row's scores of a tile, relative to their largest
template <class T> struct LseEnd {
  const T *bias;
  const void *labels;
  int label_bytes;
  float2 *part;  // [tiles of classes][rows]: largest, sum
  float *at;     // [rows] the label's score
  long long rows;
  __device__ void tile(const float (*c)[65], long long m0, long long n0, long long M, long long N) const {
    if (threadIdx.x >= 64 || m0 + threadIdx.x >= M) return;
    const long long m = m0 + threadIdx.x, cols = N - n0 < 64 ? N - n0 : 64;
    const long long label = label_bytes == 8 ? ((const long long *)labels)[m] : ((const int *)labels)[m];
    float top = -INFINITY, sum = 0.f;
    for (int j = 0; j < cols; ++j) top = fmaxf(top, c[threadIdx.x][j] + (bias ? to_float(bias[n0 + j]) : 0.f));
    for (int j = 0; j < cols; ++j) {
      const float z = c[threadIdx.x][j] + (bias ? to_float(bias[n0 + j]) : 0.f);
      sum += z == top ? 1.f : expf(z - top);
      if (n0 + j == label) at[m] = z;
    }
    part[(n0 / 64) * rows + m] = make_float2(top, sum);
  }
};

// gradient of the scores, rounded
template <class T> struct ScoreGradEnd {
  const T *bias;
  const void *labels;
  int label_bytes;
  const float *grad, *lse, *scale;
  T *dz;
  long long ld_dz, first, classes; // class of column 0; classes in all
  float *bias_sums;                // [tiles of rows][ld_dz] or null
  __device__ void tile(float (*c)[65], long long m0, long long n0, long long M, long long N) const {
    for (int i = threadIdx.x; i < 4096; i += 256) {
      const long long m = m0 + i / 64, n = n0 + i % 64;
      float g = 0.f;
      if (m < M && n < N) {
        const long long label = label_bytes == 8 ? ((const long long *)labels)[m] : ((const int *)labels)[m];
        if (label >= 0 && label < classes) {
          const float z = c[i / 64][i % 64] + (bias ? to_float(bias[first + n]) : 0.f);
          g = grad[m] * (expf(z - lse[m]) - (first + n == label ? 1.f : 0.f));
        }
        dz[m * ld_dz + n] = from_float<T>(g * *scale);
      }
      c[i / 64][i % 64] = g;
    }
    __syncthreads();
    if (bias_sums && threadIdx.x < 64 && n0 + threadIdx.x < N) {
      float s = 0.f;
      for (int i = 0; i < 64; ++i) s += c[i][threadIdx.x];
      bias_sums[(m0 / 64) * ld_dz + n0 + threadIdx.x] = s;
    }
  }
};

// one summand of a product that is cut along its sum
template <class T> struct SumEnd {
  float *sums; // [rows][ld]: what came before; null: the first and only part
  long long ld;
  T *out;
  long long ld_out;
  const T *skip; // added at the end, or null
  long long ld_skip;
  const float *scale; // divides the result; null: 1
  bool first, last;
  __device__ void tile(const float (*c)[65], long long m0, long long n0, long long M, long long N) const {
    for (int i = threadIdx.x; i < 4096; i += 256) {
      const long long m = m0 + i / 64, n = n0 + i % 64;
      if (m >= M || n >= N) continue;
      float v = c[i / 64][i % 64];
      if (!first) v += sums[m * ld + n];
      if (last) out[m * ld_out + n] = from_float<T>((scale ? v / *scale : v) + (skip ? to_float(skip[m * ld_skip + n]) : 0.f));
      else sums[m * ld + n] = v;
    }
  }
};

template <class T, class End>
__global__ void __launch_bounds__(256) tb_product_kernel(Operand<T> A, Operand<T> B, long long M, long long N, long long K, End end) {
  __shared__ float a[16][65], b[16][65], c[64][65];
  const long long m0 = (long long)blockIdx.y * 64, n0 = (long long)blockIdx.x * 64;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (long long k0 = 0; k0 < K; k0 += 16) {
    for (int i = threadIdx.x; i < 1024; i += 256) {
      const int r = A.sk == 1 ? i / 16 : i % 64, k = A.sk == 1 ? i % 16 : i / 64;
      a[k][r] = m0 + r < M && k0 + k < K ? to_float(A.p[(m0 + r) * A.sr + (k0 + k) * A.sk]) : 0.f;
      const int rb = B.sk == 1 ? i / 16 : i % 64, kb = B.sk == 1 ? i % 16 : i / 64;
      b[kb][rb] = n0 + rb < N && k0 + kb < K ? to_float(B.p[(n0 + rb) * B.sr + (k0 + kb) * B.sk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += a[k][ty * 4 + i] * b[k][tx * 4 + j];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[ty * 4 + i][tx * 4 + j] = acc[i][j];
  __syncthreads();
  end.tile(c, m0, n0, M, N);
}

// a row's logarithm and loss from the parts of its tiles
__global__ void tb_loss_join_kernel(const float2 *part, long long tiles, const float *at, const void *labels, int label_bytes,
                                    long long classes, float *loss, float *lse, long long rows) {
  const long long m = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (m >= rows) return;
  float top = -INFINITY, sum = 0.f;
  for (long long t = 0; t < tiles; ++t) top = fmaxf(top, part[t * rows + m].x);
  for (long long t = 0; t < tiles; ++t) {
    const float2 p = part[t * rows + m];
    if (p.x > -INFINITY || p.x != p.x || p.y != p.y) sum += p.x == top ? p.y : p.y * expf(p.x - top);
  }
  const float l = top == -INFINITY && sum == 0.f ? -INFINITY : top + logf(sum);
  const long long label = label_bytes == 8 ? ((const long long *)labels)[m] : ((const int *)labels)[m];
  lse[m] = l;
  loss[m] = label >= 0 && label < classes ? l - at[m] : 0.f;
}

// dz = grad * activation'(pre), rounded; sums of its columns over 64 rows before rounding
template <class T>
__global__ void tb_act_grad_kernel(const T *grad, long long ld_grad, const T *pre, long long ld_pre, int act, T *dz, long long ld_dz,
                                   float *bias_sums, long long rows, long long cols) {
  const long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x, r0 = (long long)blockIdx.y * 64;
  if (c >= cols) return;
  float sum = 0.f;
  for (long long r = r0; r < rows && r < r0 + 64; ++r) {
    float g = to_float(grad[r * ld_grad + c]);
    if (act) g *= act_slope(to_float(pre[r * ld_pre + c]), act);
    if (dz) dz[r * ld_dz + c] = from_float<T>(g);
    sum += g;
  }
  if (bias_sums) bias_sums[blockIdx.y * ld_dz + c] = sum;
}

template <class T>
__global__ void tb_column_sum_kernel(const float *sums, long long tiles, long long ld, T *out, long long cols) {
  const long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (long long t = 0; t < tiles; ++t) s += sums[t * ld + c];
  out[c] = from_float<T>(s);
}

// The power of two that brings the largest |v| to about 2^13 (1 where nothing finite and nonzero is there).
__global__ void __launch_bounds__(1024) tb_scale_kernel(const float *v, long long n, float *scale) {
  __shared__ float tops[32];
  float top = 0.f;
  for (long long i = threadIdx.x; i < n; i += 1024)
    if (fabsf(v[i]) < INFINITY) top = fmaxf(top, fabsf(v[i]));
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 32; ++i) top = fmaxf(top, tops[i]);
  int e = 0;
  if (top > 0.f) frexpf(top, &e);
  *scale = top > 0.f ? ldexpf(1.f, min(max(13 - e, -100), 100)) : 1.f;
}

} // namespace tb
