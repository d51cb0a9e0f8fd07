// Sum of the embedding rows that a forest's leaves pick, and its gradient.
//
//   out[n, :]   = sum_t table[row(t, id[n, t]), :]
//   dtable[r,:] = sum of grad[n, :] over the (n, t) with row(t, id[n, t]) = r
//
// Both move one table or gradient row per (batch row, tree) between L2 and the multiprocessors and add it up
// in registers; nothing of that size goes to memory.  Sums are fp32 in an order that the sizes alone decide,
// rounded once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace tb {

// Which table row a leaf has: leaves are numbered in node order, so a leaf's number is the count of leaves
// before it -- the leaves of earlier words of 32 nodes, kept, and those of its own word, counted from its
// bits.  A tree of 8 levels is 128 bytes of this, one line, where a number per node would be sixteen.
struct LeafMapView {
  const uint2 *words;  // per 32 nodes of a tree: which are leaves; table row of the first leaf from there on
  const int2 *trees;   // [num_trees + 1] first word, nodes
  const int32_t *rows; // [num_trees + 1] first table row
  long long num_trees;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Table row of node `id` of a tree; -1: the id is no leaf of it.
__device__ __forceinline__ int32_t leaf_row(const uint2 *words, int2 tree, int32_t id) {
  if ((uint32_t)id >= (uint32_t)tree.y) return -1;
  const uint2 w = __ldg(words + tree.x + (id >> 5));
  const uint32_t bit = 1u << (id & 31);
  return w.x & bit ? (int32_t)(w.y + __popc(w.x & (bit - 1))) : -1;
}

// A lane's share of a row: 16 bytes' worth of columns, moved V bytes at a time (V divides the rows' addresses
// and lengths, so that a piece is inside a row or outside of it as a whole).
template <class T, int V> struct Share {
  static constexpr int kElems = 16 / sizeof(T), kPieces = 16 / V, kPer = V / sizeof(T);
  // columns c .. c + kElems - 1 of the row at p; those from `width` on are zeros
  static __device__ __forceinline__ uint4 load(const T *p, long long c, long long width) {
    uint4 q = make_uint4(0, 0, 0, 0);
    unsigned char *to = reinterpret_cast<unsigned char *>(&q);
    const unsigned char *from = reinterpret_cast<const unsigned char *>(p + c);
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (c + i * kPer < width) {
        if constexpr (V == 16) q = __ldg(reinterpret_cast<const uint4 *>(from));
        else if constexpr (V == 8) *reinterpret_cast<uint2 *>(to + 8 * i) = __ldg(reinterpret_cast<const uint2 *>(from) + i);
        else if constexpr (V == 4) *reinterpret_cast<uint32_t *>(to + 4 * i) = __ldg(reinterpret_cast<const uint32_t *>(from) + i);
        else *reinterpret_cast<uint16_t *>(to + 2 * i) = __ldg(reinterpret_cast<const uint16_t *>(from) + i);
      }
    return q;
  }
  static __device__ __forceinline__ void add(float (&acc)[kElems], uint4 q) {
    const T *v = reinterpret_cast<const T *>(&q);
#pragma unroll
    for (int i = 0; i < kElems; ++i) acc[i] += to_float(v[i]);
  }
  static __device__ __forceinline__ void store(T *p, long long c, long long width, const float (&acc)[kElems]) {
    uint4 q;
    T *v = reinterpret_cast<T *>(&q);
#pragma unroll
    for (int i = 0; i < kElems; ++i) v[i] = from_float<T>(acc[i]);
    const unsigned char *from = reinterpret_cast<const unsigned char *>(&q);
    unsigned char *to = reinterpret_cast<unsigned char *>(p + c);
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (c + i * kPer < width) {
        if constexpr (V == 16) *reinterpret_cast<uint4 *>(to) = q;
        else if constexpr (V == 8) reinterpret_cast<uint2 *>(to)[i] = *reinterpret_cast<const uint2 *>(from + 8 * i);
        else if constexpr (V == 4) reinterpret_cast<uint32_t *>(to)[i] = *reinterpret_cast<const uint32_t *>(from + 4 * i);
        else reinterpret_cast<uint16_t *>(to)[i] = *reinterpret_cast<const uint16_t *>(from + 2 * i);
      }
  }
};

// ---- few batch rows: a block per row, whose lanes' groups share the trees out ---------------------
// One chain of three loads (id, words, table row) per 8 trees of a group; latency is all that counts.
template <class T, int V>
__global__ void __launch_bounds__(1024) tb_leaf_sum_row_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, const T *table, long long ld_table,
                                                               long long width, int lanes_log2, T *out, long long ld_out) {
  using S = Share<T, V>;
  constexpr int E = S::kElems;
  __shared__ float part[32 * 32 * E]; // [warp][lane of a row][element], column lanes_log2 == 5 at most
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> lanes_log2, groups = blockDim.x >> lanes_log2;
  const long long n = blockIdx.x, c = ((long long)blockIdx.y * lanes + lane) * E;
  const int32_t *id = ids + n * ld_ids;
  float acc[E] = {};
  for (long long t0 = 0; t0 < m.num_trees; t0 += (long long)groups * 8) {
    int32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long t = t0 + (long long)i * groups + group;
      r[i] = t < m.num_trees ? leaf_row(m.words, __ldg(m.trees + t), __ldg(id + t)) : -1;
    }
    uint4 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = r[i] >= 0 ? S::load(table + r[i] * ld_table, c, width) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (r[i] >= 0) S::add(acc, q[i]);
  }
  for (int d = lanes; d < 32; d <<= 1)
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] += __shfl_xor_sync(~0u, acc[i], d);
  const int warp = threadIdx.x / 32, warps = blockDim.x / 32;
  if ((threadIdx.x & 31) < lanes)
#pragma unroll
    for (int i = 0; i < E; ++i) part[(warp * 32 + lane) * E + i] = acc[i];
  __syncthreads();
  if (threadIdx.x >= lanes) return;
  for (int w = 1; w < warps; ++w)
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] += part[(w * 32 + lane) * E + i];
  S::store(out + n * ld_out, c, width, acc);
}

// ---- many batch rows: a lane group keeps the sums of eight rows -----------------------------------
// All rows of a block go through the trees side by side, so that the rows of one tree's table, of which most
// batch rows want the same few, are read from L1 once they have come; eight loads of a lane are in flight.
// blockIdx.y: columns; blockIdx.z: a range of trees, whose sums are kept in fp32 for tb_leaf_sum_join_kernel.
constexpr int kLeafRows = 8;
template <class T, int V>
__global__ void __launch_bounds__(512) tb_leaf_sum_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, const T *table, long long ld_table,
                                                          long long width, int lanes_log2, T *out, long long ld_out, float *parts, long long ld_parts,
                                                          long long n_rows, int trees_per_part) {
  using S = Share<T, V>;
  constexpr int E = S::kElems;
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), groups = blockDim.x >> lanes_log2;
  const int base = threadIdx.x & 31 & ~(lanes - 1);
  // (a warp's groups have neighbouring rows, a group's eight rows are `groups` apart)
  const long long n0 = (long long)blockIdx.x * groups * kLeafRows + (threadIdx.x >> lanes_log2), c = ((long long)blockIdx.y * lanes + lane) * E;
  const long long t_end = min(m.num_trees, (long long)(blockIdx.z + 1) * trees_per_part);
  float acc[kLeafRows][E] = {};
  for (long long t0 = (long long)blockIdx.z * trees_per_part; t0 < t_end; t0 += lanes) {
    // every lane looks up one tree of the next `lanes`
    const long long t = t0 + lane;
    const bool there = t < t_end;
    const int2 tree = there ? __ldg(m.trees + t) : make_int2(0, 0);
    int32_t id[kLeafRows], row[kLeafRows];
#pragma unroll
    for (int i = 0; i < kLeafRows; ++i) {
      const long long n = n0 + (long long)i * groups;
      id[i] = there && n < n_rows ? __ldg(ids + n * ld_ids + t) : -1;
    }
#pragma unroll
    for (int i = 0; i < kLeafRows; ++i) row[i] = leaf_row(m.words, tree, id[i]);
    const int now = (int)min((long long)lanes, t_end - t0);
    for (int j = 0; j < now; ++j) {
      uint4 q[kLeafRows];
#pragma unroll
      for (int i = 0; i < kLeafRows; ++i) {
        const int32_t r = __shfl_sync(~0u, row[i], base + j);
        q[i] = r >= 0 ? S::load(table + r * ld_table, c, width) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kLeafRows; ++i) S::add(acc[i], q[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kLeafRows; ++i) {
    const long long n = n0 + (long long)i * groups;
    if (n >= n_rows) break;
    if (!parts) {
      S::store(out + n * ld_out, c, width, acc[i]);
    } else if (c < ld_parts) {
      float4 *d = reinterpret_cast<float4 *>(parts + ((long long)blockIdx.z * n_rows + n) * ld_parts + c);
#pragma unroll
      for (int k = 0; k < E / 4; ++k) d[k] = make_float4(acc[i][4 * k], acc[i][4 * k + 1], acc[i][4 * k + 2], acc[i][4 * k + 3]);
    }
  }
}
// Adds the parts of the tree ranges up, in order.
template <class T, int V>
__global__ void __launch_bounds__(256) tb_leaf_sum_join_kernel(const float *parts, long long ld_parts, int count, T *out, long long ld_out, long long width, long long n_rows) {
  using S = Share<T, V>;
  constexpr int E = S::kElems;
  const long long per = ld_parts / E, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n_rows * per) return;
  const long long n = i / per, c = i % per * E;
  float acc[E] = {};
  for (int s = 0; s < count; ++s) {
    const float4 *d = reinterpret_cast<const float4 *>(parts + ((long long)s * n_rows + n) * ld_parts + c);
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      const float4 v = d[k];
      acc[4 * k] += v.x, acc[4 * k + 1] += v.y, acc[4 * k + 2] += v.z, acc[4 * k + 3] += v.w;
    }
  }
  S::store(out + n * ld_out, c, width, acc);
}

// ---- gradient -------------------------------------------------------------------------------------

constexpr uint32_t kNoLeaf = 0xffffffffu;

// numbers[t][n] = number of the leaf among its tree's (kNoLeaf: none): the ids the other way around, so that
// the rows of one tree lie side by side, and looked up with a tree per warp, which touches few lines.
__global__ void __launch_bounds__(256) tb_leaf_numbers_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, uint32_t *numbers, long long ld,
                                                              long long n_rows) {
  __shared__ int32_t tile[32][33];
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  const long long t0 = (long long)blockIdx.y * 32;
  for (long long n0 = (long long)blockIdx.x * 32; n0 < n_rows; n0 += (long long)gridDim.x * 32) {
    __syncthreads();
#pragma unroll
    for (int i = y; i < 32; i += 8) tile[i][x] = n0 + i < n_rows && t0 + x < m.num_trees ? ids[(n0 + i) * ld_ids + t0 + x] : -1;
    __syncthreads();
#pragma unroll
    for (int i = y; i < 32; i += 8) {
      const long long t = t0 + i;
      if (t >= m.num_trees || n0 + x >= n_rows) continue;
      const int32_t r = leaf_row(m.words, __ldg(m.trees + t), tile[x][i]);
      numbers[t * ld + n0 + x] = r < 0 ? kNoLeaf : (uint32_t)(r - __ldg(m.rows + t));
    }
  }
}

// One block per tree, range of its leaves and columns.  The batch rows are put in the order of their leaves
// (a counting sort in shared memory: every warp counts, then places, its own stretch of the rows, so that
// equal leaves keep the order of the rows); then the sorted rows are shared out evenly among the lane groups,
// which add up runs of equal leaves.  A leaf inside one group's stretch is finished there; the ends of
// stretches are joined in order afterwards.  Batches above kLeafChunk rows come in pieces, with fp32 sums in
// `sums` in between.
constexpr int kLeafRange = 1024, kLeafChunk = 32768, kLeafGradWarps = 16;
constexpr int kLeafGradFixed = kLeafRange * 4 + 16;
__host__ __device__ constexpr int leaf_grad_smem(int chunk, int range) { // counters and, after them, the ends of stretches share their place
  return kLeafGradFixed + (kLeafGradWarps * range * 4 > 16384 ? kLeafGradWarps * range * 4 : 16384) + (chunk + 7) / 8 * 16; // order: two bytes a row
}
template <class T, int V>
__global__ void __launch_bounds__(32 * kLeafGradWarps) tb_leaf_grad_kernel(LeafMapView m, const uint32_t *numbers, long long ld_numbers, const T *grad,
                                                                           long long ld_grad, long long width, int lanes_log2, float *sums, T *out,
                                                                           long long ld_out, long long n_rows, int chunk, int range) {
  using S = Share<T, V>;
  constexpr int E = S::kElems;
  extern __shared__ __align__(16) unsigned char raw[];
  uint32_t *start = reinterpret_cast<uint32_t *>(raw);              // [kLeafRange + 1] first place of a leaf
  uint32_t *count = reinterpret_cast<uint32_t *>(raw + kLeafGradFixed); // [warp][range]
  float *ends = reinterpret_cast<float *>(count);                   // [group][lanes * E] sum of a stretch's first run
  uint16_t *order = reinterpret_cast<uint16_t *>(raw + leaf_grad_smem(0, range));
  const int tid = threadIdx.x, warp = tid / 32, wl = tid % 32;
  const int lanes = 1 << lanes_log2, lane = tid & (lanes - 1), group = tid >> lanes_log2, groups = (32 * kLeafGradWarps) >> lanes_log2;
  const long long t = blockIdx.x, c = ((long long)blockIdx.y * lanes + lane) * E;
  const int32_t row0 = m.rows[t] + (int)blockIdx.z * range;
  const int leaves = min(range, m.rows[t + 1] - row0);
  if (leaves <= 0) return;
  const uint32_t first_leaf = blockIdx.z * (uint32_t)range;
  const uint32_t *mine = numbers + t * ld_numbers;

  for (long long b0 = 0; b0 < n_rows; b0 += chunk) {
    const int now = (int)min((long long)chunk, n_rows - b0);
    const bool first = b0 == 0, last = b0 + now == n_rows;
    const int per = ((now + kLeafGradWarps - 1) / kLeafGradWarps + 31) & ~31, from = warp * per, to = min(now, from + per);
    __syncthreads();
    for (int i = tid; i < kLeafGradWarps * leaves; i += 32 * kLeafGradWarps) count[i] = 0;
    __syncthreads();
    for (int i = from + wl; i < to; i += 32) {
      const uint32_t l = mine[b0 + i] - first_leaf;
      if (l < (uint32_t)leaves) atomicAdd(&count[warp * leaves + l], 1u);
    }
    __syncthreads();
    // places: leaf by leaf, within a leaf warp by warp
    for (int l = tid; l < leaves; l += 32 * kLeafGradWarps) {
      uint32_t sum = 0;
#pragma unroll
      for (int w = 0; w < kLeafGradWarps; ++w) {
        const uint32_t k = count[w * leaves + l];
        count[w * leaves + l] = sum;
        sum += k;
      }
      start[l] = sum;
    }
    __syncthreads();
    if (warp == 0) {
      uint32_t before = 0;
      for (int l0 = 0; l0 < leaves; l0 += 32) {
        uint32_t v = l0 + wl < leaves ? start[l0 + wl] : 0, s = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t o = __shfl_up_sync(~0u, s, d);
          if (wl >= d) s += o;
        }
        if (l0 + wl < leaves) start[l0 + wl] = before + s - v;
        before += __shfl_sync(~0u, s, 31);
      }
      if (wl == 0) start[leaves] = before;
    }
    __syncthreads();
    for (int i0 = from; i0 < to; i0 += 32) {
      const int i = i0 + wl;
      const uint32_t l = i < to ? mine[b0 + i] - first_leaf : kNoLeaf;
      const uint32_t same = __match_any_sync(~0u, l);
      if (l < (uint32_t)leaves) {
        const uint32_t at = count[warp * leaves + l], rank = __popc(same & ((1u << wl) - 1));
        order[start[l] + at + rank] = (uint16_t)i;
        __syncwarp(same);
        if (rank == 0) count[warp * leaves + l] = at + __popc(same);
      }
      __syncwarp();
    }
    __syncthreads();

    const int total = (int)start[leaves], piece = (total + groups - 1) / groups;
    const int a = min(total, group * piece), z = min(total, a + piece);
    // the leaf that the place `a` belongs to: the last one that starts at or before it and is not empty
    int l = 0;
    if (a < z) {
      int lo = 0, hi = leaves - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (start[mid] <= (uint32_t)a) lo = mid;
        else hi = mid - 1;
      }
      l = lo;
    }
    auto finish = [&](int leaf, float (&acc)[E]) {
      const long long r = row0 + leaf;
      float *s = sums + r * width + c;
      if (!first) {
#pragma unroll
        for (int k = 0; k < E; ++k)
          if (c + k < width) acc[k] += s[k];
      }
      if (last) S::store(out + r * ld_out, c, width, acc);
      else {
#pragma unroll
        for (int k = 0; k < E; ++k)
          if (c + k < width) s[k] = acc[k];
      }
    };
    float acc[E] = {};
    bool whole = a < z && start[l] == (uint32_t)a; // the run at hand began in this stretch
    bool open = false;                            // the stretch's last run goes on in the next one
    float *end0 = ends + (size_t)tid * E;
    if (a < z) {
      int stop = (int)start[l + 1];
      const T *g0 = grad + b0 * ld_grad;
      for (int i = a; i < z; i += 8) {
        uint4 q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = i + k < z ? S::load(g0 + (long long)order[i + k] * ld_grad, c, width) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (i + k >= z) break;
          if (i + k == stop) {
            if (whole) finish(l, acc);
            else
#pragma unroll
              for (int e = 0; e < E; ++e) end0[e] = acc[e];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = 0.f;
            whole = true;
            do ++l; while ((int)start[l + 1] <= i + k);
            stop = (int)start[l + 1];
          }
          S::add(acc, q[k]);
        }
      }
      open = stop > z;
      if (!whole)
#pragma unroll
        for (int e = 0; e < E; ++e) end0[e] = acc[e];
      else if (!open) finish(l, acc);
    }
    __syncthreads();
    if (a < z && open && whole) { // a leaf that begins here and ends in a later stretch: its parts in order
      const int stop = (int)start[l + 1];
      for (int g = group + 1; g * piece < stop; ++g) {
        const float *e0 = ends + ((size_t)g * lanes + lane) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += e0[e];
      }
      finish(l, acc);
    }
    for (int leaf = group; leaf < leaves; leaf += groups) // leaves without a row
      if (start[leaf + 1] == start[leaf] && (first || last)) {
        float none[E] = {};
        finish(leaf, none);
      }
  }
}

} // namespace tb
