// Sum of the embedding rows that a forest's leaves pick, and its gradient.
//
//   out[n, :]   = sum_t table[row(t, id[n, t]), :]
//   dtable[r,:] = sum of grad[n, :] over the (n, t) with row(t, id[n, t]) = r
//
// Sums are fp32 in a fixed order (trees for the first, batch rows for the second), rounded once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace tb {

struct LeafMapView {
  const long long *tree_off; // [num_trees + 1] first node of a tree
  const int32_t *node_row;   // [nodes] table row of a leaf, -1: an inner node
  const int32_t *row_off;    // [num_trees + 1] first table row of a tree
  long long num_trees;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Table row of (tree, id); -1: the id is no leaf of the tree.
__device__ __forceinline__ int32_t leaf_row(const LeafMapView &m, long long t, int32_t id) {
  const long long first = m.tree_off[t];
  return id >= 0 && id < m.tree_off[t + 1] - first ? m.node_row[first + id] : -1;
}

// One block per batch row; a thread sums columns threadIdx.x, + blockDim.x, ... over all trees.
template <class T>
__global__ void tb_leaf_sum_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, const T *table, long long ld_table,
                                   long long width, T *out, long long ld_out, long long n_rows) {
  for (long long n = blockIdx.x; n < n_rows; n += gridDim.x)
    for (long long c = threadIdx.x; c < width; c += blockDim.x) {
      float acc = 0.f;
      for (long long t = 0; t < m.num_trees; ++t) {
        const int32_t r = leaf_row(m, t, ids[n * ld_ids + t]);
        if (r >= 0) acc += to_float(table[r * ld_table + c]);
      }
      out[n * ld_out + c] = from_float<T>(acc);
    }
}

// One block per tree and 32 columns: batch rows in order, sums in an fp32 array [table rows][width] that
// the block alone owns; then rounded to the output.
template <class T>
__global__ void tb_leaf_grad_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, const T *grad, long long ld_grad,
                                    long long width, float *sums, T *out, long long ld_out, long long n_rows) {
  const long long t = blockIdx.x, c = (long long)blockIdx.y * 32 + threadIdx.x;
  if (c >= width) return;
  const int32_t r0 = m.row_off[t], r1 = m.row_off[t + 1];
  for (long long r = r0; r < r1; ++r) sums[r * width + c] = 0.f;
  for (long long n = 0; n < n_rows; ++n) {
    const int32_t r = leaf_row(m, t, ids[n * ld_ids + t]);
    if (r >= 0) sums[r * width + c] += to_float(grad[n * ld_grad + c]);
  }
  for (long long r = r0; r < r1; ++r) out[r * ld_out + c] = from_float<T>(sums[r * width + c]);
}

} // namespace tb
