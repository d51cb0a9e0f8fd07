// Sum of the embedding rows that a forest's leaves pick, and its gradient.
//
//   out[n, :]   = sum_t table[row(t, id[n, t]), :]
//   dtable[r,:] = sum of grad[n, :] over the (n, t) with row(t, id[n, t]) = r
//
// Both move one table or gradient row per (batch row, tree) between L2 and the multiprocessors and add it up
// in registers; nothing of that size goes to memory.  Sums are fp32, rounded once, in an order that sizes decide and, for
// out, whether the staged kernel takes the call (alignment, table rows one behind the other).
#pragma once
#include "element.cuh"

#include <cstdint>
#include <type_traits>

namespace tb {

// The leaf map alone is read through __ldg: it does not change while it exists.  What an earlier kernel of the stream may
// have written is not: these kernels are resident while that one still runs, and such loads may be moved ahead of the
// wait for it.
//
// Which table row a leaf has: leaves are numbered in node order, so a leaf's number is the count of leaves
// before it -- the leaves of earlier words of 32 nodes, kept, and those of its own word, counted from its
// bits.  A tree of 8 levels is 128 bytes of this, one line, where a number per node would be sixteen.
struct LeafMapView {
  const uint2 *words;  // per 32 nodes of a tree: which are leaves; table row of the first leaf from there on
  const int2 *trees;   // [num_trees + 1] first word, nodes
  const int32_t *rows; // [num_trees + 1] first table row
  long long num_trees;
};

// Table row of node `id` of a tree; -1: the id is no leaf of it.  Without branches, so that many can be under way; an
// id beyond the tree reads the tree's first word for nothing.
__device__ __forceinline__ uint2 leaf_word(const uint2 *words, int2 tree, int32_t id) {
  return __ldg(words + tree.x + ((uint32_t)id < (uint32_t)tree.y ? id >> 5 : 0));
}
__device__ __forceinline__ int32_t leaf_row(uint2 word, int2 tree, int32_t id) {
  const uint32_t bit = 1u << (id & 31);
  const int32_t r = (int32_t)(word.y + __popc(word.x & (bit - 1)));
  return (uint32_t)id < (uint32_t)tree.y && (word.x & bit) ? r : -1;
}
__device__ __forceinline__ int32_t leaf_row(const uint2 *words, int2 tree, int32_t id) { return leaf_row(leaf_word(words, tree, id), tree, id); }

// A lane's share of a row: 16 bytes' worth of columns, moved V bytes at a time (V divides the rows' addresses
// and lengths, so that a piece is inside a row or outside of it as a whole).  Sums are kept as pairs, which the
// multiprocessor adds two at a time.
template <class T, int V> struct Share {
  static constexpr int kElems = 16 / sizeof(T), kPairs = kElems / 2, kPieces = 16 / V, kPer = V / sizeof(T);
  // the columns of the row at p that begin with column c (p points there); those from `width` on are zeros
  static __device__ __forceinline__ uint4 load(const unsigned char *p, long long c, long long width) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if constexpr (V == 16) {
      if (c < width) q = load_result(reinterpret_cast<const uint4 *>(p));
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (c + i * kPer < width) {
          if constexpr (V == 8) {
            const uint2 x = load_result(reinterpret_cast<const uint2 *>(p) + i);
            w[2 * i] = x.x, w[2 * i + 1] = x.y;
          } else if constexpr (V == 4) w[i] = load_result(reinterpret_cast<const uint32_t *>(p) + i);
          else w[i / 2] |= (uint32_t)load_result(reinterpret_cast<const uint16_t *>(p) + i) << (i % 2 * 16);
        }
      q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return q;
  }
  static __device__ __forceinline__ void add(unsigned long long &acc, float2 v) {
    asm("{\n .reg .b64 t;\n mov.b64 t, {%1, %2};\n add.rn.f32x2 %0, %0, t;\n}" : "+l"(acc) : "f"(v.x), "f"(v.y));
  }
  static __device__ __forceinline__ void add(unsigned long long (&acc)[kPairs], uint4 q) {
    if constexpr (sizeof(T) == 4) {
      add(acc[0], make_float2(__uint_as_float(q.x), __uint_as_float(q.y)));
      add(acc[1], make_float2(__uint_as_float(q.z), __uint_as_float(q.w)));
    } else {
      add_halves<T>(acc[0], q.x);
      add_halves<T>(acc[1], q.y);
      add_halves<T>(acc[2], q.z);
      add_halves<T>(acc[3], q.w);
    }
  }
  static __device__ __forceinline__ float2 get(unsigned long long a) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(a));
    return v;
  }
  // p: the row's column c
  static __device__ __forceinline__ void store(T *p, long long c, long long width, const unsigned long long (&acc)[kPairs]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 v = get(acc[i]);
      if constexpr (sizeof(T) == 4) w[2 * i] = __float_as_uint(v.x), w[2 * i + 1] = __float_as_uint(v.y);
      else {
        const T h[2] = {from_float<T>(v.x), from_float<T>(v.y)};
        w[i] = *reinterpret_cast<const uint32_t *>(h);
      }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (c + i * kPer < width) {
        if constexpr (V == 16) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (V == 8) reinterpret_cast<uint2 *>(p)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
        else if constexpr (V == 4) reinterpret_cast<uint32_t *>(p)[i] = w[i];
        else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[i / 2] >> (i % 2 * 16));
      }
  }
};

// ---- few batch rows: a cluster of blocks per row, whose lane groups share the trees out ------------
// One chain of three loads (id, word, table row) per eight trees of a group: latency is all that counts, and
// as many misses as possible are under way at a time.  The blocks' sums meet in the first one's registers.
constexpr int kLeafRowThreads = 256;
template <class T, int V>
__global__ void __launch_bounds__(kLeafRowThreads) tb_leaf_sum_row_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, const T *table,
                                                                          uint32_t row_bytes, long long width, int lanes_log2, T *out,
                                                                          long long ld_out, int blocks) {
  using S = Share<T, V>;
  constexpr int P = S::kPairs, kWarps = kLeafRowThreads / 32;
  __shared__ unsigned long long part[kWarps][32][P]; // [0]: the block's sum in the end
  after_previous_kernel();
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), rank = blockIdx.x % blocks;
  const int group = rank * (kLeafRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2), groups = blocks * (kLeafRowThreads >> lanes_log2);
  const long long n = blockIdx.x / blocks, c = ((long long)blockIdx.y * lanes + lane) * S::kElems;
  const int32_t *id = ids + n * ld_ids;
  const unsigned char *from = reinterpret_cast<const unsigned char *>(table + c);
  unsigned long long acc[P] = {};
  for (long long t0 = 0; t0 < m.num_trees; t0 += (long long)groups * 8) {
    int32_t r[8];
    int2 tree[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long t = t0 + (long long)i * groups + group;
      tree[i] = t < m.num_trees ? __ldg(m.trees + t) : make_int2(0, 0);
      r[i] = t < m.num_trees ? id[t] : -1;
    }
    uint2 word[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) word[i] = leaf_word(m.words, tree[i], r[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = leaf_row(word[i], tree[i], r[i]);
    uint4 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = r[i] >= 0 ? S::load(from + (unsigned long long)r[i] * row_bytes, c, width) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (r[i] >= 0) S::add(acc, q[i]);
  }
  for (int d = lanes; d < 32; d <<= 1)
#pragma unroll
    for (int i = 0; i < P; ++i) S::add(acc[i], S::get(__shfl_xor_sync(~0u, acc[i], d)));
  const int warp = threadIdx.x / 32;
  if ((threadIdx.x & 31) < lanes)
#pragma unroll
    for (int i = 0; i < P; ++i) part[warp][lane][i] = acc[i];
  __syncthreads();
  if (threadIdx.x < lanes) {
    for (int w = 1; w < kWarps; ++w)
#pragma unroll
      for (int i = 0; i < P; ++i) S::add(acc[i], S::get(part[w][lane][i]));
#pragma unroll
    for (int i = 0; i < P; ++i) part[0][lane][i] = acc[i];
  }
  if (blocks > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && threadIdx.x < lanes) {
      const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&part[0][lane][0]);
      for (int b = 1; b < blocks; ++b) {
        uint32_t theirs;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(mine), "r"(b));
#pragma unroll
        for (int i = 0; i < P; ++i) {
          unsigned long long v;
          asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(theirs + 8 * i) : "memory");
          S::add(acc[i], S::get(v));
        }
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); // (the others' memory has been read)
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (rank == 0 && threadIdx.x < lanes) S::store(out + n * ld_out + c, c, width, acc);
}

// ---- many batch rows: a lane group keeps the sums of eight rows -----------------------------------
// All rows of a block go through the trees side by side, so that the rows of one tree's table, of which most
// batch rows want the same few, are read from L1 once they have come; eight loads of a lane are in flight.
// The work -- row tiles times batches of trees, in that order -- is dealt out evenly: a block takes a stretch
// of it, which may end one tile and begin the next.  A tile that one block has as a whole is finished there,
// the parts of the others are kept in fp32 for tb_leaf_sum_join_kernel.
constexpr int kLeafRows = 8;
struct LeafStretch {
  long long tiles, batches, blocks; // of the whole; a tile's batches of trees
  __host__ __device__ long long begin(long long block) const { return block * (tiles * batches) / blocks; }
  __host__ __device__ long long block_of(long long unit) const { // the block that has this unit
    long long b = unit * blocks / (tiles * batches);
    while (b + 1 < blocks && begin(b + 1) <= unit) ++b;
    while (b > 0 && begin(b) > unit) --b;
    return b;
  }
};
template <class T, int V>
__global__ void __launch_bounds__(512, 1) tb_leaf_sum_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, const T *table, uint32_t row_bytes,
                                                             long long width, int lanes_log2, T *out, long long ld_out, float *parts, long long ld_parts,
                                                             long long n_rows, LeafStretch work) {
  using S = Share<T, V>;
  constexpr int P = S::kPairs;
  after_previous_kernel();
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1), groups = blockDim.x >> lanes_log2;
  const int base = threadIdx.x & 31 & ~(lanes - 1);
  const long long c = ((long long)blockIdx.y * lanes + lane) * S::kElems;
  const unsigned char *from = reinterpret_cast<const unsigned char *>(table + c);
  long long u = work.begin(blockIdx.x);
  const long long u_end = work.begin(blockIdx.x + 1);
  while (u < u_end) {
    const long long tile = u / work.batches, b0 = u % work.batches, b1 = min(work.batches, b0 + (u_end - u));
    // (a warp's groups have neighbouring rows, a group's eight rows are `groups` apart)
    const long long n0 = tile * groups * kLeafRows + (threadIdx.x >> lanes_log2);
    const int32_t *id_at[kLeafRows];
#pragma unroll
    for (int i = 0; i < kLeafRows; ++i) id_at[i] = ids + min(n0 + (long long)i * groups, n_rows - 1) * ld_ids; // (what is behind the last row is not kept)
    unsigned long long acc[kLeafRows][P] = {};
    for (long long b = b0; b < b1; ++b) {
      // every lane looks up one tree of the batch
      const long long t = b * lanes + lane;
      const bool there = t < m.num_trees;
      const int2 tree = there ? __ldg(m.trees + t) : make_int2(0, 0);
      int32_t row[kLeafRows];
#pragma unroll
      for (int i = 0; i < kLeafRows; ++i) row[i] = there ? id_at[i][t] : -1;
      bool all = true;
#pragma unroll
      for (int i = 0; i < kLeafRows; ++i) {
        row[i] = leaf_row(m.words, tree, row[i]);
        all &= row[i] >= 0;
      }
      if (__all_sync(~0u, all)) {
        for (int j = 0; j < lanes; ++j) {
          uint4 q[kLeafRows];
#pragma unroll
          for (int i = 0; i < kLeafRows; ++i) q[i] = S::load(from + (unsigned long long)(uint32_t)__shfl_sync(~0u, row[i], base + j) * row_bytes, c, width);
#pragma unroll
          for (int i = 0; i < kLeafRows; ++i) S::add(acc[i], q[i]);
        }
      } else { // (some id is no leaf, or the batch ends behind the last tree)
        for (int j = 0; j < lanes; ++j)
#pragma unroll
          for (int i = 0; i < kLeafRows; ++i) {
            const int32_t r = __shfl_sync(~0u, row[i], base + j);
            if (r >= 0) S::add(acc[i], S::load(from + (unsigned long long)(uint32_t)r * row_bytes, c, width));
          }
      }
    }
    const bool whole = b0 == 0 && b1 == work.batches;
    const long long part = whole ? 0 : blockIdx.x - work.block_of(tile * work.batches);
#pragma unroll
    for (int i = 0; i < kLeafRows; ++i) {
      const long long n = n0 + (long long)i * groups;
      if (n >= n_rows) break;
      if (whole) {
        S::store(out + n * ld_out + c, c, width, acc[i]);
      } else if (c < ld_parts) {
        unsigned long long *d = reinterpret_cast<unsigned long long *>(parts + (part * n_rows + n) * ld_parts + c);
#pragma unroll
        for (int k = 0; k < P; ++k) d[k] = acc[i][k];
      }
    }
    u += b1 - b0;
  }
}
// The same where a tree's table rows fit a stage of shared memory and lie one behind the other, and where a row
// takes a quarter of a warp at least.  One warp copies the tables of the trees to come into a ring of stages, one
// bulk copy a tree; three look up, eight trees at a time, where in its stage each batch row's table row will lie;
// twelve add up, a lane group its eight rows: an address and a read of 30 cycles each, instead of the hundreds of an
// L1 miss.  A table is copied once for a block's tile of rows.  20011 rows, 1000 trees of 256 leaves, 64 bf16: 217 us
// with the join (the kernel above: 241); 60 % of shared memory's cycles and 2.1 of 4 instructions a cycle are used:
// neither is the limit, and what is was not found.  Waits are bounded: one that gives up sets
// tb_leaf_status.
__device__ int tb_leaf_status;
constexpr int kLeafAdders = 12, kLeafFinders = 3, kLeafStagedThreads = 32 * (kLeafAdders + kLeafFinders + 1);
constexpr int kLeafBatch = 8, kLeafSlots = 3, kLeafMaxStages = 16, kLeafMostRows = 384;
constexpr int kLeafStagedFixed = 512 + kLeafSlots * kLeafBatch * kLeafMostRows * 2; // barriers; places, in units of 16 bytes
constexpr int kLeafZeros = 512; // behind each stage: what an id that is no leaf adds
__device__ __forceinline__ bool leaf_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool leaf_wait(uint32_t bar, uint32_t parity) { // two seconds at most
  if (leaf_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (leaf_try(bar, parity)) return true;
    if ((i & 63) == 0 && clock64() - t0 > 4000000000ll) return false;
  }
}
__device__ __forceinline__ void leaf_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
template <class T>
__global__ void __launch_bounds__(kLeafStagedThreads, 1)
    tb_leaf_sum_staged_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, bool vec_ids, const T *table, uint32_t row_bytes, int width, int lanes_log2,
                              T *out, long long ld_out, float *parts, long long ld_parts, int n_rows, LeafStretch work, int stages, int stage_bytes) {
  using S = Share<T, 16>;
  constexpr int P = S::kPairs;
  extern __shared__ __align__(16) unsigned char raw[];
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(raw), full = base, empty = base + 128, found = base + 256, used = base + 256 + 8 * kLeafSlots;
  uint16_t *places = reinterpret_cast<uint16_t *>(raw + 512); // [slot][tree of the batch][row of the tile]
  const uint32_t stage0 = base + kLeafStagedFixed;
  const int pitch = stage_bytes + kLeafZeros, warp = threadIdx.x / 32, wl = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full + 8 * i) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty + 8 * i), "r"(kLeafAdders) : "memory");
    }
    for (int i = 0; i < kLeafSlots; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(found + 8 * i), "r"(kLeafFinders) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(used + 8 * i), "r"(kLeafAdders) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = threadIdx.x; i < stages * (kLeafZeros / 4); i += kLeafStagedThreads)
    *reinterpret_cast<uint32_t *>(raw + kLeafStagedFixed + (i / (kLeafZeros / 4)) * pitch + stage_bytes + i % (kLeafZeros / 4) * 4) = 0;
  __syncthreads();
  after_previous_kernel();
  const int lanes = 1 << lanes_log2, groups = (32 * kLeafAdders) >> lanes_log2, tile_rows = groups * kLeafRows;
  const int batches = (int)work.batches, trees = (int)m.num_trees;
  const long long u0 = work.begin(blockIdx.x);
  const int units = (int)(work.begin(blockIdx.x + 1) - u0), tile0 = (int)(u0 / batches), batch0 = (int)(u0 - (long long)tile0 * batches);
  bool ok = true;
  if (warp == kLeafAdders + kLeafFinders) {
    int stage = 0;
    uint32_t phase = 0;
    auto fetch = [&](int b) { return __ldg(m.rows + min(b * kLeafBatch + wl, trees)); }; // lanes 0 to 8: where tables begin
    int32_t next = fetch(batch0); // (a batch ahead: a load per tree would be longer than its copy)
    for (int u = 0, b = batch0; ok && u < units; ++u) {
      const int now = min(kLeafBatch, trees - b * kLeafBatch);
      const int32_t begin = next;
      if (++b == batches) b = 0;
      next = fetch(b);
      for (int j = 0; j < now; ++j) {
        const int32_t first = __shfl_sync(~0u, begin, j);
        const uint32_t bytes = (uint32_t)(__shfl_sync(~0u, begin, j + 1) - first) * row_bytes;
        if (!(ok = __all_sync(~0u, leaf_wait(empty + 8 * stage, phase ^ 1)))) break;
        if (wl == 0) {
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full + 8 * stage), "r"(bytes) : "memory");
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(stage0 + stage * pitch), "l"(reinterpret_cast<const unsigned char *>(table) + (unsigned long long)first * row_bytes), "r"(bytes),
                         "r"(full + 8 * stage) : "memory");
        }
        if (++stage == stages) stage = 0, phase ^= 1;
      }
    }
    if (!ok) // copies in flight land before the block ends
      for (int i = 0; i < stages; ++i) {
        if (stage-- == 0) stage = stages - 1, phase ^= 1;
        leaf_wait(full + 8 * stage, phase);
      }
  } else if (warp >= kLeafAdders) {
    int slot = 0;
    uint32_t phase = 0;
    const uint32_t none = (uint32_t)stage_bytes / 16, row_units = row_bytes / 16;
    constexpr int kMost = kLeafMostRows / 32 / kLeafFinders;
    const int row0 = (warp - kLeafAdders) * 32 + wl; // and every kLeafFinders * 32 rows
    int32_t id[kMost][kLeafBatch], next[kMost][kLeafBatch];
    int2 tree, next_tree; // of a batch's tree: lanes 0 to 7 have one each
    int32_t first, next_first;
    auto fetch = [&](int tile, int b) { // a batch's ids, one batch ahead of their use
      const int t0 = b * kLeafBatch, now = min(kLeafBatch, trees - t0);
#pragma unroll
      for (int k = 0; k < kMost; ++k) {
        const int row = row0 + kLeafFinders * 32 * k;
        // (what is behind the tile's or the batch's last row is not kept)
        const int32_t *at = ids + (long long)min(tile * tile_rows + min(row, tile_rows - 1), n_rows - 1) * ld_ids + t0;
        if (vec_ids && now == kLeafBatch) {
          const int4 a = reinterpret_cast<const int4 *>(at)[0], b = reinterpret_cast<const int4 *>(at)[1];
          next[k][0] = a.x, next[k][1] = a.y, next[k][2] = a.z, next[k][3] = a.w, next[k][4] = b.x, next[k][5] = b.y, next[k][6] = b.z, next[k][7] = b.w;
        } else {
#pragma unroll
          for (int j = 0; j < kLeafBatch; ++j) next[k][j] = j < now ? at[j] : -1;
        }
      }
      const bool there = wl < now; // (of the trees behind the last one nothing is found)
      next_tree = there ? __ldg(m.trees + t0 + wl) : make_int2(0, 0);
      next_first = there ? __ldg(m.rows + t0 + wl) : 0;
    };
    if (units) fetch(tile0, batch0);
    for (int u = 0, tile = tile0, b = batch0; ok && u < units; ++u) {
#pragma unroll
      for (int k = 0; k < kMost; ++k)
#pragma unroll
        for (int j = 0; j < kLeafBatch; ++j) id[k][j] = next[k][j];
      tree = next_tree, first = next_first;
      if (++b == batches) b = 0, ++tile;
      if (u + 1 < units) fetch(tile, b);
      if (!(ok = __all_sync(~0u, leaf_wait(used + 8 * slot, phase ^ 1)))) break;
      uint16_t *to = places + slot * kLeafBatch * kLeafMostRows + row0;
#pragma unroll
      for (int j0 = 0; j0 < kLeafBatch; j0 += 4) {
        uint2 word[4][kMost]; // (sixteen reads under way)
        int2 of[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          of[j] = make_int2(__shfl_sync(~0u, tree.x, j0 + j), __shfl_sync(~0u, tree.y, j0 + j));
#pragma unroll
          for (int k = 0; k < kMost; ++k) word[j][k] = leaf_word(m.words, of[j], id[k][j0 + j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int32_t from = __shfl_sync(~0u, first, j0 + j);
#pragma unroll
          for (int k = 0; k < kMost; ++k) {
            const int32_t r = leaf_row(word[j][k], of[j], id[k][j0 + j]);
            if (row0 + kLeafFinders * 32 * k < tile_rows) to[(j0 + j) * kLeafMostRows + kLeafFinders * 32 * k] = (uint16_t)(r < 0 ? none : (uint32_t)(r - from) * row_units);
          }
        }
      }
      __syncwarp();
      if (wl == 0) leaf_arrive(found + 8 * slot);
      if (++slot == kLeafSlots) slot = 0, phase ^= 1;
    }
  } else {
    const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> lanes_log2;
    const int c = lane * S::kElems;
    int stage = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0;
    int tile = tile0, b0 = batch0;
    for (int u = 0; ok && u < units; ++tile, b0 = 0) {
      const int b1 = min(batches, b0 + (units - u));
      unsigned long long acc[kLeafRows][P] = {};
      for (int b = b0; b < b1; ++b) { // (all lanes leave it together: the warp votes)
        const int now = min(kLeafBatch, trees - b * kLeafBatch);
        if (!(ok = __all_sync(~0u, ok && leaf_wait(found + 8 * slot, slot_phase)))) break;
        const uint16_t *place = places + slot * kLeafBatch * kLeafMostRows + group * kLeafRows;
        // two trees at a time; a wait that gave up is looked at after the batch (what is read is shared memory still)
        for (int j = 0; j < now; j += 2) {
          const bool two = j + 1 < now;
          const int other = stage + 1 == stages ? 0 : stage + 1;
          const uint32_t other_phase = phase ^ (other == 0);
          uint4 o[2];
          o[0] = *reinterpret_cast<const uint4 *>(place + j * kLeafMostRows);
          if (two) o[1] = *reinterpret_cast<const uint4 *>(place + (j + 1) * kLeafMostRows);
          if (ok) ok = leaf_wait(full + 8 * stage, phase);
          if (two && ok) ok = leaf_wait(full + 8 * other, other_phase);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && !two) break;
            const uint32_t at = stage0 + (h ? other : stage) * pitch + lane * 16, w[4] = {o[h].x, o[h].y, o[h].z, o[h].w};
            uint4 q[kLeafRows];
#pragma unroll
            for (int i = 0; i < kLeafRows; ++i) {
              const uint32_t from = at + (i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu) * 16;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q[i].x), "=r"(q[i].y), "=r"(q[i].z), "=r"(q[i].w) : "r"(from));
            }
#pragma unroll
            for (int i = 0; i < kLeafRows; ++i) S::add(acc[i], q[i]);
          }
          __syncwarp();
          if (wl == 0) {
            leaf_arrive(empty + 8 * stage);
            if (two) leaf_arrive(empty + 8 * other);
          }
          for (int k = 0; k < 1 + two; ++k)
            if (++stage == stages) stage = 0, phase ^= 1;
        }
        if (wl == 0) leaf_arrive(used + 8 * slot);
        if (++slot == kLeafSlots) slot = 0, slot_phase ^= 1;
      }
      ok = __all_sync(~0u, ok);
      const bool whole = b0 == 0 && b1 == batches;
      const long long part = whole ? 0 : blockIdx.x - work.block_of((long long)tile * batches);
#pragma unroll
      for (int i = 0; i < kLeafRows; ++i) {
        const long long n = (long long)tile * tile_rows + group * kLeafRows + i;
        if (n >= n_rows) break;
        if (whole) {
          S::store(out + n * ld_out + c, c, width, acc[i]);
        } else if (c < ld_parts) {
          unsigned long long *d = reinterpret_cast<unsigned long long *>(parts + (part * n_rows + n) * ld_parts + c);
#pragma unroll
          for (int k = 0; k < P; ++k) d[k] = acc[i][k];
        }
      }
      u += b1 - b0;
    }
  }
  if (!ok) atomicExch(&tb_leaf_status, 4);
}
// Adds the parts of the tiles that several blocks had, in order.
template <class T, int V>
__global__ void __launch_bounds__(256) tb_leaf_sum_join_kernel(const float *parts, long long ld_parts, int tile_rows, T *out, long long ld_out,
                                                               long long width, long long n_rows, LeafStretch work) {
  using S = Share<T, V>;
  constexpr int P = S::kPairs;
  after_previous_kernel();
  const long long per = ld_parts / S::kElems, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n_rows * per) return;
  const long long n = i / per, c = i % per * S::kElems, tile = n / tile_rows;
  const long long count = work.block_of((tile + 1) * work.batches - 1) - work.block_of(tile * work.batches) + 1;
  if (count == 1) return;
  unsigned long long acc[P] = {};
  for (long long s = 0; s < count; ++s) {
    const unsigned long long *d = reinterpret_cast<const unsigned long long *>(parts + (s * n_rows + n) * ld_parts + c);
#pragma unroll
    for (int k = 0; k < P; ++k) S::add(acc[k], S::get(d[k]));
  }
  S::store(out + n * ld_out + c, c, width, acc);
}

// ---- gradient -------------------------------------------------------------------------------------

// numbers[t][n] = number of the leaf among its tree's (all ones: none): the ids the other way around, so that
// the rows of one tree lie side by side, and looked up with a tree per warp, which touches few lines.
constexpr int kNumberRows = 128;
template <class N>
__global__ void __launch_bounds__(256) tb_leaf_numbers_kernel(LeafMapView m, const int32_t *ids, long long ld_ids, N *numbers, long long ld,
                                                              long long n_rows) {
  __shared__ int2 tile[32][kNumberRows / 2 + 1]; // [tree][pair of rows]
  after_previous_kernel();
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  const int t0 = blockIdx.y * 32, trees = (int)min(32ll, m.num_trees - t0);
  for (long long n0 = (long long)blockIdx.x * kNumberRows; n0 < n_rows; n0 += (long long)gridDim.x * kNumberRows) {
    const int rows = (int)min((long long)kNumberRows, n_rows - n0);
    __syncthreads();
    const int32_t *from = ids + n0 * ld_ids + t0 + x;
    int32_t v[kNumberRows / 8]; // of rows 16 i + 2 y and the next
#pragma unroll
    for (int i = 0; i < kNumberRows / 8; ++i) {
      const int row = i / 2 * 16 + 2 * y + i % 2;
      v[i] = row < rows && x < trees ? from[row * ld_ids] : -1;
    }
#pragma unroll
    for (int i = 0; i < kNumberRows / 16; ++i) tile[x][i * 8 + y] = make_int2(v[2 * i], v[2 * i + 1]);
    __syncthreads();
    for (int i = y; i < trees; i += 8) {
      const int2 tree = __ldg(m.trees + t0 + i);
      const int32_t first = __ldg(m.rows + t0 + i);
      N *to = numbers + (t0 + i) * ld + n0;
#pragma unroll
      for (int k = 0; k < kNumberRows / 64; ++k) {
        const int2 id = tile[i][x + 32 * k];
        const int32_t a = leaf_row(m.words, tree, id.x), b = leaf_row(m.words, tree, id.y);
        const N pair[2] = {a < 0 ? (N)~(N)0 : (N)(a - first), b < 0 ? (N)~(N)0 : (N)(b - first)};
        const int row = 2 * (x + 32 * k); // (ld is a multiple of 8: the second of a pair is there, used or not)
        if (row < rows) {
          if constexpr (sizeof(N) == 2) *reinterpret_cast<uint32_t *>(to + row) = *reinterpret_cast<const uint32_t *>(pair);
          else *reinterpret_cast<uint2 *>(to + row) = *reinterpret_cast<const uint2 *>(pair);
        }
      }
    }
  }
}

// One block per tree, range of its leaves and columns.  The batch rows are put in the order of their leaves
// (a counting sort in shared memory: every warp counts, then places, its own stretch of the rows, so that
// equal leaves keep the order of the rows); then the sorted rows are shared out evenly among the lane groups,
// which add up runs of equal leaves.  A leaf inside one group's stretch is finished there; the ends of
// stretches are joined in order afterwards.  Batches above kLeafChunk rows come in pieces, with fp32 sums in
// `sums` in between.  20011 rows, 1000 trees of 256 leaves, 64 bf16: 304 us and 41 for the numbers; 2.75 of 4
// instructions a cycle, 8.8 TB/s from L2: instructions bound it.
constexpr int kLeafRange = 1024, kLeafChunk = 32768, kLeafGradWarps = 16;
constexpr int kLeafGradFixed = kLeafRange * 4 + 16;
__host__ __device__ constexpr int leaf_grad_smem(int chunk, int range) { // counters and, after them, the ends of stretches share their place
  return kLeafGradFixed + (kLeafGradWarps * range * 4 > kLeafGradWarps * 1024 ? kLeafGradWarps * range * 4 : kLeafGradWarps * 1024) +
         (chunk + 15) / 8 * 16; // order: two bytes a row
}
template <class T, int V, class N>
__global__ void __launch_bounds__(32 * kLeafGradWarps, 2) tb_leaf_grad_kernel(LeafMapView m, const N *numbers, long long ld_numbers, const T *grad,
                                                                              uint32_t row_bytes, long long width, int lanes_log2, float *sums, T *out,
                                                                              long long ld_out, long long n_rows, int chunk, int range) {
  using S = Share<T, V>;
  constexpr int P = S::kPairs;
  // N: two- or four-byte leaf numbers of tb_leaf_numbers_kernel, or (int32_t) the ids themselves, looked up here
  // twice: of few rows and trees that is less than another launch
  constexpr bool kIds = std::is_same<N, int32_t>::value;
  constexpr uint32_t kNone = kIds ? 0xffffffffu : (uint32_t)(N)~(N)0;
  extern __shared__ __align__(16) unsigned char raw[];
  after_previous_kernel();
  uint32_t *start = reinterpret_cast<uint32_t *>(raw);                  // [leaves + 1] first place of a leaf
  uint32_t *count = reinterpret_cast<uint32_t *>(raw + kLeafGradFixed); // [warp][leaves]
  unsigned long long *ends = reinterpret_cast<unsigned long long *>(count); // [thread][P] sum of a stretch's first run
  uint16_t *order = reinterpret_cast<uint16_t *>(raw + leaf_grad_smem(0, range) - 16);
  const int tid = threadIdx.x, warp = tid / 32, wl = tid % 32;
  const int lanes = 1 << lanes_log2, lane = tid & (lanes - 1), group = tid >> lanes_log2, groups = (32 * kLeafGradWarps) >> lanes_log2;
  const long long t = blockIdx.x, c = ((long long)blockIdx.y * lanes + lane) * S::kElems;
  const int32_t row0 = m.rows[t] + (int)blockIdx.z * range;
  const int leaves = min(range, m.rows[t + 1] - row0);
  if (leaves <= 0) return;
  const uint32_t first_leaf = blockIdx.z * (uint32_t)range;
  const N *mine = kIds ? numbers + t : numbers + t * ld_numbers;
  const int2 tree = kIds ? __ldg(m.trees + t) : make_int2(0, 0);
  const int32_t tree_row = kIds ? __ldg(m.rows + t) : 0;
  auto number = [&](long long i) -> uint32_t {
    if constexpr (kIds) {
      const int32_t r = leaf_row(m.words, tree, mine[i * ld_numbers]);
      return r < 0 ? kNone : (uint32_t)(r - tree_row);
    } else {
      return mine[i];
    }
  };

  for (long long b0 = 0; b0 < n_rows; b0 += chunk) {
    const int now = (int)min((long long)chunk, n_rows - b0);
    const bool first = b0 == 0, last = b0 + now == n_rows;
    const int per = ((now + kLeafGradWarps - 1) / kLeafGradWarps + 31) & ~31, from = warp * per, to = min(now, from + per);
    __syncthreads();
    for (int i = tid; i < kLeafGradWarps * leaves; i += 32 * kLeafGradWarps) count[i] = 0;
    __syncthreads();
    uint32_t *own = count + warp * leaves;
    constexpr int kAhead = 8; // numbers of a lane that are loaded at a time
    for (int i0 = from + wl; i0 < to; i0 += 32 * kAhead) {
      uint32_t l[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) l[k] = i0 + 32 * k < to ? number(b0 + i0 + 32 * k) : kNone;
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (l[k] != kNone && l[k] - first_leaf < (uint32_t)leaves) atomicAdd(own + (l[k] - first_leaf), 1u);
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
      if (wl < 8) order[before + wl] = 0; // (read, never added)
    }
    __syncthreads();
    for (int l = tid; l < leaves; l += 32 * kLeafGradWarps)
#pragma unroll
      for (int w = 0; w < kLeafGradWarps; ++w) count[w * leaves + l] += start[l];
    __syncthreads();
    for (int i0 = from; i0 < to; i0 += 32 * kAhead) {
      uint32_t ls[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) ls[k] = i0 + 32 * k + wl < to ? number(b0 + i0 + 32 * k + wl) : kNone;
      // (the equal ones of 32 rows get their places from one of them, whose counter tells how many came before;
      // a warp's additions to a counter happen in the order of the program, so all eight can be under way)
      uint32_t same[kAhead], at[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        ls[k] = ls[k] == kNone || ls[k] - first_leaf >= (uint32_t)leaves ? kNone : ls[k] - first_leaf;
        const uint32_t there = __ballot_sync(~0u, ls[k] != kNone);
        same[k] = ls[k] != kNone ? there : ~there;
      }
      for (int b = 0; (1 << b) < leaves; ++b) // (a vote a bit: several times faster than a match instruction)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const bool set = ls[k] >> b & 1;
          const uint32_t with = __ballot_sync(~0u, set);
          same[k] &= set ? with : ~with;
        }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const bool leads = (same[k] & ((1u << wl) - 1)) == 0 && ls[k] != kNone;
        at[k] = leads ? atomicAdd(own + ls[k], (uint32_t)__popc(same[k])) : 0;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint32_t place = __shfl_sync(~0u, at[k], __ffs(same[k]) - 1) + __popc(same[k] & ((1u << wl) - 1));
        if (ls[k] != kNone) order[place] = (uint16_t)(i0 + 32 * k + wl);
      }
    }
    __syncthreads();

    const int total = (int)start[leaves], piece = ((total + groups - 1) / groups + 7) & ~7;
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
    auto finish = [&](int leaf, unsigned long long (&acc)[P]) {
      const long long r = row0 + leaf;
      float *s = sums + r * width + c;
      if (!first) {
#pragma unroll
        for (int k = 0; k < P; ++k) S::add(acc[k], make_float2(c + 2 * k < width ? s[2 * k] : 0.f, c + 2 * k + 1 < width ? s[2 * k + 1] : 0.f));
      }
      if (last) S::store(out + r * ld_out + c, c, width, acc);
      else {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const float2 v = S::get(acc[k]);
          if (c + 2 * k < width) s[2 * k] = v.x;
          if (c + 2 * k + 1 < width) s[2 * k + 1] = v.y;
        }
      }
    };
    unsigned long long acc[P] = {};
    bool whole = a < z && start[l] == (uint32_t)a; // the run at hand began in this stretch
    bool open = false;                            // the stretch's last run goes on in the next one
    unsigned long long *end0 = ends + tid * P;
    if (a < z) {
      int stop = (int)start[l + 1];
      const unsigned char *g0 = reinterpret_cast<const unsigned char *>(grad + c) + (unsigned long long)b0 * row_bytes;
      for (int i = a; i < z; i += 8) {
        const uint4 o = *reinterpret_cast<const uint4 *>(order + i);
        const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
        uint4 q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = S::load(g0 + (unsigned long long)(k % 2 ? ow[k / 2] >> 16 : ow[k / 2] & 0xffffu) * row_bytes, c, width);
        if (stop >= i + 8 && z >= i + 8) { // (one run)
#pragma unroll
          for (int k = 0; k < 8; ++k) S::add(acc, q[k]);
          continue;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (i + k >= z) break;
          if (i + k == stop) {
            if (whole) finish(l, acc);
            else
#pragma unroll
              for (int e = 0; e < P; ++e) end0[e] = acc[e];
#pragma unroll
            for (int e = 0; e < P; ++e) acc[e] = 0;
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
        for (int e = 0; e < P; ++e) end0[e] = acc[e];
      else if (!open) finish(l, acc);
    }
    __syncthreads();
    if (a < z && open && whole) { // a leaf that begins here and ends in a later stretch: its parts in order
      const int stop = (int)start[l + 1];
      for (int g = group + 1; g * piece < stop; ++g) {
        const unsigned long long *e0 = ends + ((g << lanes_log2) + lane) * P;
#pragma unroll
        for (int e = 0; e < P; ++e) S::add(acc[e], S::get(e0[e]));
      }
      finish(l, acc);
    }
    for (int leaf = group; leaf < leaves; leaf += groups) // leaves without a row
      if (start[leaf + 1] == start[leaf] && (first || last)) {
        unsigned long long none[P] = {};
        finish(leaf, none);
      }
  }
}

} // namespace tb
