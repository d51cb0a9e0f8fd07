// C ABI of the leaf sums (include/tbk_leaf.h): the leaf map, plans, launches.
#include "leaf_api.h"
#include "leaf_sum.cuh"

#include <cstring>
#include <memory>
#include <new>
#include <type_traits>
#include <vector>

struct tbk_leaf_map {
  int device = 0;
  int64_t rows = 0, max_rows = 0; // table rows in all, of the largest tree
  tb::LeafMapView view{};
  void *mem = nullptr;
};

namespace {

// f(element type, bytes that are moved at a time)
template <class F> int with_piece(int32_t type, int bytes, F f) {
  auto sized = [&](auto t) {
    switch (bytes) {
    case 16: return f(t, std::integral_constant<int, 16>());
    case 8: return f(t, std::integral_constant<int, 8>());
    case 4: return f(t, std::integral_constant<int, 4>());
    default:
      if constexpr (sizeof(t) == 2) return f(t, std::integral_constant<int, 2>());
      else return f(t, std::integral_constant<int, 4>());
    }
  };
  return type == TBK_TYPE_F32 ? sized(float()) : type == TBK_TYPE_F16 ? sized(__half()) : sized(__nv_bfloat16());
}
// The largest power of two, 16 at most, that divides the addresses and lengths of all rows of two matrices.
int piece_bytes(int32_t type, int64_t width, const void *p, int64_t ld_p, int64_t rows_p, const void *q, int64_t ld_q, int64_t rows_q) {
  const uint64_t size = type == TBK_TYPE_F32 ? 4 : 2;
  const uint64_t all = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | width * size | (rows_p > 1 ? ld_p * size : 0) |
                       (rows_q > 1 ? ld_q * size : 0) | 16;
  return (int)(all & (~all + 1));
}
// Lanes (as a power of two) that share a row, 16 bytes each.
int lanes_of(int64_t width, int32_t type) {
  const int64_t wanted = tiles_of(width, type == TBK_TYPE_F32 ? 4 : 8);
  int log2 = 0;
  while (log2 < 5 && (1 << log2) < wanted) ++log2;
  return log2;
}

constexpr int kLeafStagedSmem = 227 * 1024 - tb::kLeafStagedFixed;

// How a leaf sum is cut.  Up to six rows per multiprocessor: a cluster of blocks per row (1000 trees, width 64: 4.5 us
// for 64 rows, 13 for 296, 20 for 512, 37 for 1024; tiles take 35 to 38 us for all of them).  Above that: tiles of
// eight rows per lane group, of as few warps as it takes to have enough tiles, whose trees the blocks share
// out (a block to a multiprocessor, 16 warps, where tiles are many; at most about 16 parts of a tile).  With
// very many tiles each has a block of its own and there are no parts.
struct LeafSumPlan {
  bool by_row;
  int64_t staged_rows = 0; // of a tile
  int lanes_log2, threads, cluster = 1, tile_rows = 0;
  unsigned columns;
  int64_t ld_parts, max_parts = 0;
  tb::LeafStretch work{}, staged_work{}; // in batches of a tree per lane; of kLeafBatch trees
  LeafSumPlan(int64_t n, int64_t width, int32_t type, int64_t trees, int sms) {
    const int elems = type == TBK_TYPE_F32 ? 4 : 8;
    lanes_log2 = lanes_of(width, type);
    const int lanes = 1 << lanes_log2;
    columns = (unsigned)tiles_of(width, (int64_t)elems << lanes_log2);
    ld_parts = tiles_of(width, elems) * elems;
    by_row = n <= 6 * sms;
    if (by_row) {
      threads = tb::kLeafRowThreads;
      while (cluster < 8 && (int64_t)cluster * 8 * (threads / lanes) < trees) cluster *= 2;
      return;
    }
    const int64_t rows_per_warp = (32 / lanes) * tb::kLeafRows;
    int warps = 16;
    while (warps > 2 && tiles_of(n, warps * rows_per_warp) * 8 < sms) warps /= 2;
    threads = 32 * warps;
    tile_rows = (int)(warps * rows_per_warp);
    work.tiles = tiles_of(n, tile_rows);
    work.batches = tiles_of(trees, lanes);
    staged_rows = tb::kLeafAdders * rows_per_warp;
    staged_work.tiles = tiles_of(n, staged_rows), staged_work.batches = tiles_of(trees, tb::kLeafBatch);
    for (tb::LeafStretch *w : {&work, &staged_work}) {
      w->blocks = w->tiles;
      if (w->tiles >= 8 * sms) continue;
      w->blocks = std::min(std::max<int64_t>(1, sms / columns) * (16 / warps), std::min<int64_t>(16 * w->tiles, w->tiles * w->batches));
      max_parts = std::max(max_parts, std::min<int64_t>(w->blocks, w->batches / (w->tiles * w->batches / w->blocks) + 2));
    }
  }
  // Tables of trees are staged where three stages hold the largest and a tile has as many rows as the
  // largest tree leaves (with fewer, more bytes are copied than read).  A tile's places have room for kLeafMostRows,
  // which shuts out rows of less than eight lanes: an array's size, no measured border.
  bool staged(int64_t max_rows, int64_t row_bytes) const {
    return !by_row && columns == 1 && threads == 512 && staged_rows <= tb::kLeafMostRows && max_rows <= staged_rows && max_rows * row_bytes + tb::kLeafZeros <= kLeafStagedSmem / 3;
  }
};

// Up to so many ids the gradient looks them up itself, above that a kernel of their own does (100 trees of 8 levels,
// width 64: 15.1 and 17.6 us for 1024 rows, 35.9 and 34.4 for 5243, 90 and 99 for 20000).
constexpr int64_t kFewIds = 1 << 21;

struct LeafGradParts {
  int64_t ld;
  unsigned char *numbers; // two bytes each, or four where a tree has very many leaves
  float *sums;
  LeafGradParts(Parts &w, int64_t n, int64_t width, int64_t trees, int64_t rows, bool narrow)
      : ld(up8(n)), numbers(w.take<unsigned char>(n * trees <= kFewIds ? 0 : (uint64_t)trees * ld * (narrow ? 2 : 4))), sums(w.take<float>(n > tb::kLeafChunk ? rows * width : 0)) {}
};

} // namespace

extern "C" {

int tbk_leaf_map_create(const tbk_forest_arrays *fa, int32_t device, tbk_leaf_map **out) {
  if (!out) return fail(TBK_ERR_INVALID, "null argument");
  *out = nullptr;
  if (!fa || !fa->tree_off || !fa->left) return fail(TBK_ERR_INVALID, "null forest array");
  if (fa->num_trees < 1) return fail(TBK_ERR_INVALID, "a leaf map needs a tree at least");
  if (fa->num_trees > 65535 * 32) return fail(TBK_ERR_UNSUPPORTED, "more than %d trees", 65535 * 32); // (32 to a row of a grid)
  if (fa->tree_off[0] != 0) return fail(TBK_ERR_INVALID, "tree_off does not begin with 0");
  for (int64_t t = 0; t < fa->num_trees; ++t)
    if (fa->tree_off[t + 1] <= fa->tree_off[t] || fa->tree_off[t + 1] - fa->tree_off[t] > kMost) return fail(TBK_ERR_INVALID, "tree %lld has no nodes, or too many", (long long)t);
  try {
    std::unique_ptr<tbk_leaf_map> map(new tbk_leaf_map);
    const int64_t trees = fa->num_trees;
    std::vector<uint2> words;
    std::vector<int2> tree((size_t)trees + 1);
    std::vector<int32_t> row_off((size_t)trees + 1);
    int64_t rows = 0;
    for (int64_t t = 0; t < trees; ++t) {
      const int64_t nodes = fa->tree_off[t + 1] - fa->tree_off[t];
      const int32_t *left = fa->left + fa->tree_off[t];
      tree[t] = make_int2((int)words.size(), (int)nodes);
      row_off[t] = (int32_t)rows;
      for (int64_t i = 0; i < nodes; i += 32) {
        uint2 w = make_uint2(0, (uint32_t)rows);
        for (int64_t k = i; k < std::min(nodes, i + 32); ++k)
          if (left[k] < 0) w.x |= 1u << (k - i), ++rows;
        words.push_back(w);
      }
      if (rows > kMost || words.size() > (size_t)kMost) return fail(TBK_ERR_UNSUPPORTED, "more than %lld leaves", (long long)kMost);
      if (rows == row_off[t]) return fail(TBK_ERR_INVALID, "tree %lld has no leaf", (long long)t);
      map->max_rows = std::max<int64_t>(map->max_rows, rows - row_off[t]);
    }
    tree[trees] = make_int2((int)words.size(), 0);
    row_off[trees] = (int32_t)rows;
    map->device = device;
    map->rows = rows;
    const size_t a = words.size() * 8, b = tree.size() * 8, c = row_off.size() * 4;
    std::vector<unsigned char> image(a + b + c);
    std::memcpy(image.data(), words.data(), a);
    std::memcpy(image.data() + a, tree.data(), b);
    std::memcpy(image.data() + a + b, row_off.data(), c);
    OnDevice on(device);
    CUDA_TRY(on.error);
    CUDA_TRY(cudaMalloc(&map->mem, image.size()));
    unsigned char *p = static_cast<unsigned char *>(map->mem);
    map->view = {reinterpret_cast<uint2 *>(p), reinterpret_cast<int2 *>(p + a), reinterpret_cast<int32_t *>(p + a + b), trees};
    const cudaError_t e = cudaMemcpy(p, image.data(), image.size(), cudaMemcpyHostToDevice);
    if (e != cudaSuccess) {
      cudaFree(map->mem);
      return fail(TBK_ERR_CUDA, "upload of the leaf map failed: %s", cudaGetErrorString(e));
    }
    *out = map.release();
    return TBK_OK;
  } catch (const std::bad_alloc &) {
    return fail(TBK_ERR_INVALID, "out of host memory");
  }
}

int tbk_leaf_map_free(tbk_leaf_map *map) {
  if (!map) return TBK_OK;
  OnDevice on(map->device);
  if (on.error == cudaSuccess) cudaFree(map->mem);
  delete map;
  return TBK_OK;
}

int64_t tbk_leaf_map_rows(const tbk_leaf_map *map) { return map ? map->rows : -1; }

static int check_leaf_call(const tbk_leaf_map *map, const int32_t *ids, int64_t n, int64_t ld_ids, int64_t width, int32_t type) {
  if (!map) return fail(TBK_ERR_INVALID, "null leaf map");
  TRY(check_sizes("leaf sum", n, width, 1));
  if (type != TBK_TYPE_F32 && type != TBK_TYPE_F16 && type != TBK_TYPE_BF16) return fail(TBK_ERR_INVALID, "unknown element type %d", type);
  if (width > 1 << 20) return fail(TBK_ERR_UNSUPPORTED, "leaf sum: %lld columns", (long long)width);
  return check_matrix("leaf_ids", ids, ld_ids, n, map->view.num_trees, 4);
}

static int element_bytes(int32_t type) { return type == TBK_TYPE_F32 ? 4 : 2; }
// (the kernels multiply row numbers with 32-bit strides)
static int check_stride(const char *what, int64_t ld, int32_t type) {
  if (ld * element_bytes(type) > 0xffffffffll) return fail(TBK_ERR_UNSUPPORTED, "%s: %lld elements from row to row", what, (long long)ld);
  return TBK_OK;
}

int tbk_leaf_sum_workspace(const tbk_leaf_map *map, int64_t n, int64_t width, int32_t type, uint64_t *bytes) {
  if (!map || !bytes) return fail(TBK_ERR_INVALID, "null argument");
  TRY(check_sizes("leaf sum", n, width, 1));
  const LeafSumPlan plan(n, width, type, map->view.num_trees, multiprocessors(map->device));
  *bytes = (uint64_t)plan.max_parts * n * plan.ld_parts * 4;
  return TBK_OK;
}

int tbk_leaf_sum(const tbk_leaf_map *map, const int32_t *ids, int64_t n, int64_t ld_ids, const void *table, int64_t ld_table,
                 int64_t width, int32_t type, void *out, int64_t ld_out, void *ws, uint64_t ws_bytes, void *stream_) {
  TRY(check_leaf_call(map, ids, n, ld_ids, width, type));
  TRY(check_matrix("table", table, ld_table, map->rows, width, element_bytes(type)));
  TRY(check_matrix("out", out, ld_out, n, width, element_bytes(type)));
  TRY(check_stride("table", ld_table, type));
  if (n == 0) return TBK_OK;
  uint64_t need = 0;
  TRY(tbk_leaf_sum_workspace(map, n, width, type, &need));
  TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(map->device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  const LeafSumPlan plan(n, width, type, map->view.num_trees, multiprocessors(map->device));
  return with_piece(type, piece_bytes(type, width, table, ld_table, map->rows, out, ld_out, n), [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const uint32_t row_bytes = (uint32_t)(ld_table * sizeof(T));
    if (plan.by_row) {
      return launch(tb::tb_leaf_sum_row_kernel<T, V>, dim3((unsigned)(n * plan.cluster), plan.columns), plan.threads, 0, stream, plan.cluster, map->view, ids, ld_ids,
                    (const T *)table, row_bytes, width, plan.lanes_log2, (T *)out, ld_out, plan.cluster);
    }
    float *parts = (float *)ws;
    tb::LeafStretch work = plan.work;
    int tile_rows = plan.tile_rows;
    if (V == 16 && plan.staged(map->max_rows, row_bytes) && ld_table == width && n < kMost) {
      const int stage_bytes = (int)(map->max_rows * row_bytes), stages = std::min(tb::kLeafMaxStages, kLeafStagedSmem / (stage_bytes + tb::kLeafZeros));
      const int smem = tb::kLeafStagedFixed + stages * (stage_bytes + tb::kLeafZeros);
      const bool vec_ids = reinterpret_cast<uintptr_t>(ids) % 16 == 0 && ld_ids % 4 == 0;
      work = plan.staged_work, tile_rows = (int)plan.staged_rows;
      CUDA_TRY(cudaFuncSetAttribute(tb::tb_leaf_sum_staged_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, tb::kLeafStagedFixed + kLeafStagedSmem));
      TRY(launch(tb::tb_leaf_sum_staged_kernel<T>, dim3((unsigned)work.blocks), tb::kLeafStagedThreads, smem, stream, 1, map->view, ids, ld_ids, vec_ids, (const T *)table,
                 row_bytes, (int)width, plan.lanes_log2, (T *)out, ld_out, parts, plan.ld_parts, (int)n, work, stages, stage_bytes));
    } else {
      TRY(launch(tb::tb_leaf_sum_kernel<T, V>, dim3((unsigned)work.blocks, plan.columns), plan.threads, 0, stream, 1, map->view, ids, ld_ids, (const T *)table, row_bytes, width,
                 plan.lanes_log2, (T *)out, ld_out, parts, plan.ld_parts, n, work));
    }
    if (plan.max_parts)
      TRY(launch(tb::tb_leaf_sum_join_kernel<T, V>, (unsigned)tiles_of(n * plan.ld_parts / tb::Share<T, V>::kElems, 256), 256, 0, stream, 1, parts, plan.ld_parts, tile_rows,
                 (T *)out, ld_out, width, n, work));
    return (int)TBK_OK;
  });
}

// The status word of the staged leaf sum (see tbk_leaf_check_status).
int leaf_sum_status(int *word) {
  int zero = 0;
  CUDA_TRY(cudaMemcpyFromSymbol(word, tb::tb_leaf_status, sizeof *word));
  if (*word) CUDA_TRY(cudaMemcpyToSymbol(tb::tb_leaf_status, &zero, sizeof zero));
  return TBK_OK;
}

int tbk_leaf_sum_backward_workspace(const tbk_leaf_map *map, int64_t n, int64_t width, int32_t type, uint64_t *bytes) {
  if (!map || !bytes) return fail(TBK_ERR_INVALID, "null argument");
  (void)type;
  TRY(check_sizes("leaf sum", n, width, 1));
  Parts w{nullptr};
  LeafGradParts parts(w, n, width, map->view.num_trees, map->rows, map->max_rows < 0xffff);
  *bytes = w.used;
  return TBK_OK;
}

int tbk_leaf_sum_backward(const tbk_leaf_map *map, const int32_t *ids, int64_t n, int64_t ld_ids, const void *grad, int64_t ld_grad,
                          int64_t width, int32_t type, void *out, int64_t ld_out, void *ws, uint64_t ws_bytes, void *stream_) {
  TRY(check_leaf_call(map, ids, n, ld_ids, width, type));
  TRY(check_matrix("grad", grad, ld_grad, n, width, element_bytes(type)));
  TRY(check_matrix("out", out, ld_out, map->rows, width, element_bytes(type)));
  TRY(check_stride("grad", ld_grad, type));
  uint64_t need = 0;
  TRY(tbk_leaf_sum_backward_workspace(map, n, width, type, &need));
  OnDevice on(map->device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  const size_t size = element_bytes(type);
  if (n == 0) {
    CUDA_TRY(cudaMemset2DAsync(out, (size_t)ld_out * size, 0, (size_t)width * size, (size_t)map->rows, stream));
    return TBK_OK;
  }
  TRY(check_workspace(ws, ws_bytes, need));
  Parts w{(unsigned char *)ws};
  const int64_t trees = map->view.num_trees;
  const bool narrow = map->max_rows < 0xffff;
  LeafGradParts parts(w, n, width, trees, map->rows, narrow);
  const dim3 blocks((unsigned)std::min<int64_t>(tiles_of(n, tb::kNumberRows), 4096), (unsigned)tiles_of(trees, 32));
  const bool few = n * trees <= kFewIds;
  if (few) ;
  else if (narrow) TRY(launch(tb::tb_leaf_numbers_kernel<uint16_t>, blocks, 256, 0, stream, 1, map->view, ids, ld_ids, (uint16_t *)parts.numbers, parts.ld, n));
  else TRY(launch(tb::tb_leaf_numbers_kernel<uint32_t>, blocks, 256, 0, stream, 1, map->view, ids, ld_ids, (uint32_t *)parts.numbers, parts.ld, n));
  return with_piece(type, piece_bytes(type, width, grad, ld_grad, n, out, ld_out, map->rows), [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const int lanes_log2 = lanes_of(width, type), range = (int)std::min<int64_t>(map->max_rows, tb::kLeafRange);
    const int chunk = (int)std::min<int64_t>(n, tb::kLeafChunk), smem = tb::leaf_grad_smem(chunk, range);
    const dim3 grid((unsigned)trees, (unsigned)tiles_of(width, (int64_t)(16 / size) << lanes_log2), (unsigned)tiles_of(map->max_rows, range));
    if (grid.y > 65535 || grid.z > 65535) return fail(TBK_ERR_UNSUPPORTED, "leaf_sum_backward: too many columns, or leaves of a tree");
    auto sorted = [&](auto number) {
      using N = decltype(number);
      const auto kernel = tb::tb_leaf_grad_kernel<T, V, N>;
      CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tb::leaf_grad_smem(tb::kLeafChunk, tb::kLeafRange)));
      return launch(kernel, grid, 32 * tb::kLeafGradWarps, smem, stream, 1, map->view, few ? (const N *)ids : (const N *)parts.numbers, few ? ld_ids : parts.ld, (const T *)grad, (uint32_t)(ld_grad * sizeof(T)), width,
                    lanes_log2, parts.sums, (T *)out, ld_out, n, chunk, range);
    };
    return few ? sorted(int32_t()) : narrow ? sorted(uint16_t()) : sorted(uint32_t());
  });
}

} // extern "C"
