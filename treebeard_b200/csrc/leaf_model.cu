// C ABI of the operators behind a forest's leaves (include/tbk_leaf.h): checks, plans, launches.
#include "../../include/tbk_leaf.h"
#include "dense.cuh"
#include "last_error.h"

#include <cudaTypedefs.h>
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <type_traits>
#include <vector>

#define CUDA_TRY(expr)                                                                                            \
  do {                                                                                                            \
    cudaError_t e__ = (expr);                                                                                     \
    if (e__ != cudaSuccess)                                                                                       \
      return fail(TBK_ERR_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e__), __FILE__, __LINE__);     \
  } while (0)

using tb::fail;

struct tbk_leaf_map {
  int device = 0;
  int64_t rows = 0, max_rows = 0; // table rows in all, of the largest tree
  tb::LeafMapView view{};
  void *mem = nullptr;
};

namespace {

// Makes a device current for a call's launches and puts the old one back.
struct OnDevice {
  int before = -1;
  cudaError_t error;
  explicit OnDevice(int device) {
    error = cudaGetDevice(&before);
    if (error == cudaSuccess && before != device) error = cudaSetDevice(device);
    else if (error == cudaSuccess) before = -1;
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

constexpr int64_t kMost = 0x7ffff000; // of every size: coordinates of tiles behind the last one fit 32 bits

// A workspace cut into 256-byte aligned parts; with a null base only their sizes are added up.
struct Parts {
  unsigned char *base;
  uint64_t used = 0;
  template <class P> P *take(uint64_t count) {
    P *p = base ? reinterpret_cast<P *>(base + used) : nullptr;
    used += (count * sizeof(P) + 255) / 256 * 256;
    return p;
  }
};

int64_t tiles_of(int64_t n, int64_t tile) { return (n + tile - 1) / tile; }

int half_type(int32_t type, const char *what) {
  if (type == TBK_TYPE_F16 || type == TBK_TYPE_BF16) return TBK_OK;
  if (type == TBK_TYPE_F32) return fail(TBK_ERR_UNSUPPORTED, "%s takes 16-bit floating point types (fp16, bf16)", what);
  return fail(TBK_ERR_INVALID, "unknown element type %d", type);
}

int check_sizes(const char *what, int64_t n, int64_t a, int64_t b) {
  if (n < 0 || a < 1 || b < 1) return fail(TBK_ERR_INVALID, "%s: sizes %lld, %lld, %lld are not >= 0, >= 1, >= 1", what, (long long)n, (long long)a, (long long)b);
  if (n > kMost || a > kMost || b > kMost) return fail(TBK_ERR_UNSUPPORTED, "%s: a size is above %lld", what, (long long)kMost);
  return TBK_OK;
}

int check_matrix(const char *what, const void *p, int64_t ld, int64_t rows, int64_t cols) {
  if (!p && rows > 0) return fail(TBK_ERR_INVALID, "%s is null", what);
  if (ld < cols && rows > 1) return fail(TBK_ERR_INVALID, "%s: %lld elements from row to row are less than its %lld columns", what, (long long)ld, (long long)cols);
  if (ld > ((int64_t)1 << 38)) return fail(TBK_ERR_UNSUPPORTED, "%s: %lld elements from row to row", what, (long long)ld);
  return TBK_OK;
}

int check_workspace(const void *p, uint64_t have, uint64_t need) {
  if (need == 0) return TBK_OK;
  if (!p || have < need) return fail(TBK_ERR_INVALID, "the workspace has %llu of %llu bytes", (unsigned long long)(p ? have : 0), (unsigned long long)need);
  if (reinterpret_cast<uintptr_t>(p) % 256) return fail(TBK_ERR_INVALID, "the workspace is not 256-byte aligned");
  return TBK_OK;
}

#define TRY(expr)               \
  do {                          \
    const int rc__ = (expr);    \
    if (rc__) return rc__;      \
  } while (0)

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
template <class F> int with_half(int32_t type, F f) { return type == TBK_TYPE_F16 ? f(__half()) : f(__nv_bfloat16()); }

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// Multiprocessors of a device; the figure of the architecture where there is none (workspace sizes on a host).
int multiprocessors(int device) {
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 2) {
    cudaGetLastError();
    return 148;
  }
  return n;
}

// How a product is cut: 256 x 256 tiles of two blocks or 128 x 128 tiles of one, and, where that leaves
// multiprocessors without work, the sum into parts that a second kernel joins.  Cycles per 64 k of a tile, around
// a tile and for the second kernel were measured (see tb_dense_kernel); the cheapest cut is taken.
struct ProductPlan {
  bool pair = false;
  int splits = 1;
};
ProductPlan plan_product(int64_t m, int64_t n, int64_t k, int sms, bool may_split) {
  ProductPlan best;
  double least = 1e300;
  const int64_t kb = tiles_of(k, 64);
  for (int pair = 0; pair < 2; ++pair) {
    const double tiles = (double)tiles_of(m, pair ? 256 : 128) * tiles_of(n, pair ? 256 : 128), slots = pair ? sms / 2 : sms;
    for (int64_t splits = 1; splits <= (may_split ? std::min<int64_t>(kb, 32) : 1); ++splits) {
      double cost = std::ceil(tiles * splits / slots) * (tiles_of(kb, splits) * (pair ? 530.0 : 300.0) + (pair ? 1400 : 900)) + 2500;
      if (splits > 1) cost += 5000 + (double)m * n * 8 * splits / 2500;
      if (cost < least) least = cost, best.pair = pair, best.splits = (int)splits;
    }
  }
  return best;
}
uint64_t part_floats(int64_t m, int64_t n, int64_t k, int sms) {
  const ProductPlan plan = plan_product(m, n, k, sms, true);
  return plan.splits > 1 ? (uint64_t)plan.splits * m * up8(n) : 0;
}

// An operand of a product: rows x sum matrix at p, row-major, or (rows_inner) sum x rows.
struct Side {
  const void *p;
  int64_t ld;
  bool rows_inner;
};

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled f = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}
template <class T> int tensor_map(CUtensorMap *map, const Side &s, int64_t rows, int64_t k) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return fail(TBK_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const int64_t inner = s.rows_inner ? rows : k, outer = s.rows_inner ? k : rows;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer}, strides[1] = {(cuuint64_t)(outer > 1 ? s.ld : up8(inner)) * 2};
  const cuuint32_t box[2] = {64, s.rows_inner ? 64u : 128u}, one[2] = {1, 1};
  const CUresult rc = encode(map, sizeof(T) == 2 && std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                             const_cast<void *>(s.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? TBK_OK : fail(TBK_ERR_CUDA, "cuTensorMapEncodeTiled: %d (%lld x %lld, %lld)", (int)rc, (long long)outer, (long long)inner, (long long)s.ld);
}

template <class T, bool PAIR, class End>
int launch_dense(const Side &a, const Side &b, int64_t m, int64_t n, int64_t k, int splits, int run, int sms, const End &end, cudaStream_t stream) {
  constexpr int tile = PAIR ? 256 : 128;
  tb::DenseProblem p;
  TRY(tensor_map<T>(&p.a, a, m, k));
  TRY(tensor_map<T>(&p.b, b, n, k));
  p.M = m, p.N = n;
  p.a_rows_inner = a.rows_inner, p.b_rows_inner = b.rows_inner;
  p.m_tiles = (int)tiles_of(m, tile), p.n_tiles = (int)tiles_of(n, tile), p.k_blocks = (int)tiles_of(k, 64);
  const int64_t slots = PAIR ? sms / 2 : sms;
  p.chunk = run;
  p.chunks = (int)tiles_of(p.n_tiles, p.chunk);
  p.splits = splits;
  p.group = PAIR ? 8 : 16;
  p.units = (long long)p.m_tiles * p.chunks * splits;
  static std::atomic<uint64_t> ready{0}; // devices on which the kernel may use its shared memory
  int device = 0;
  CUDA_TRY(cudaGetDevice(&device));
  if (device > 63 || !(ready.load() >> device & 1)) {
    CUDA_TRY(cudaFuncSetAttribute(tb::tb_dense_kernel<T, PAIR, End>, cudaFuncAttributeMaxDynamicSharedMemorySize, tb::kDenseSmem));
    if (device <= 63) ready.fetch_or(1ull << device);
  }
  const unsigned grid = (unsigned)std::min<int64_t>(p.units, slots) * (PAIR ? 2 : 1);
  tb::tb_dense_kernel<T, PAIR, End><<<grid, tb::kDenseThreads, tb::kDenseSmem, stream>>>(p, end);
  CUDA_TRY(cudaGetLastError());
  return TBK_OK;
}

// C[m, n] = sum_k A[m, k] B[n, k], finished by F.  parts: room for what part_floats says.
template <class T, class F>
int product(const Side &a, const Side &b, int64_t m, int64_t n, int64_t k, const F &f, float *parts, int sms, cudaStream_t stream) {
  const ProductPlan plan = plan_product(m, n, k, sms, true);
  if (plan.splits == 1) {
    const tb::WholeEnd<F> end{f};
    return plan.pair ? launch_dense<T, true>(a, b, m, n, k, 1, 1, sms, end, stream)
                     : launch_dense<T, false>(a, b, m, n, k, 1, 1, sms, end, stream);
  }
  const int64_t ld = up8(n);
  const tb::PartEnd end{parts, ld};
  if (plan.pair) TRY((launch_dense<T, true>(a, b, m, n, k, plan.splits, 1, sms, end, stream)));
  else TRY((launch_dense<T, false>(a, b, m, n, k, plan.splits, 1, sms, end, stream)));
  tb::tb_dense_join_kernel<F><<<(unsigned)tiles_of(m * (ld / 8), 256), 256, 0, stream>>>(parts, plan.splits, ld, m, n, f);
  CUDA_TRY(cudaGetLastError());
  return TBK_OK;
}

// Whether tensor copies can read a matrix: rows begin at multiples of 16 bytes.
bool tma_rows(const void *p, int64_t ld, int64_t rows) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld % 8 == 0 || rows <= 1);
}
// The matrix itself, or a copy that tensor copies can read (in `room`, rows x up8(cols)).
template <class T> int readable(const void **p, int64_t *ld, int64_t rows, int64_t cols, T *room, cudaStream_t stream) {
  if (tma_rows(*p, *ld, rows)) return TBK_OK;
  tb::tb_align_rows_kernel<T><<<(unsigned)std::min<int64_t>(rows, 148 * 16), 256, 0, stream>>>((const T *)*p, *ld, room, up8(cols), rows, cols);
  CUDA_TRY(cudaGetLastError());
  *p = room;
  *ld = up8(cols);
  return TBK_OK;
}
// Whether 16 bytes at a time can be read or written at every eighth column.
bool vec_rows(const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

typedef unsigned short Half; // an element of either 16-bit type

struct LinearParts {
  Half *x, *weight;
  float *parts;
  LinearParts(Parts &w, int64_t n, int64_t inputs, int64_t outputs, bool aligned, int sms)
      : x(w.take<Half>(aligned ? 0 : n * up8(inputs))), weight(w.take<Half>(aligned ? 0 : outputs * up8(inputs))),
        parts(w.take<float>(part_floats(n, outputs, inputs, sms))) {}
};
struct LinearGradParts {
  int64_t ld;
  Half *x, *weight, *dz;
  float *bias_sums, *parts;
  LinearGradParts(Parts &w, int64_t n, int64_t inputs, int64_t outputs, bool aligned, int sms)
      : ld(up8(outputs)), x(w.take<Half>(aligned ? 0 : n * up8(inputs))), weight(w.take<Half>(aligned ? 0 : outputs * up8(inputs))),
        dz(w.take<Half>(n * ld)), bias_sums(w.take<float>(tiles_of(n, 32) * ld)),
        parts(w.take<float>(std::max(part_floats(n, inputs, outputs, sms), part_floats(outputs, inputs, n, sms)))) {}
};

// How the scores of a loss are cut: a unit goes through a run of column tiles, as long as every slot still gets
// eight units, so that the last ones end together.
struct LossCut {
  bool pair;
  int run, parts; // column tiles of a unit; partial sums of a row
  LossCut(int64_t n, int64_t width, int64_t classes, int sms) {
    pair = plan_product(n, classes, width, sms, false).pair;
    const int64_t tile = pair ? 256 : 128, slots = pair ? sms / 2 : sms, cols = tiles_of(classes, tile);
    run = (int)std::clamp<int64_t>(tiles_of(n, tile) * cols / (8 * slots), 1, 8);
    parts = 2 * (int)tiles_of(cols, run);
  }
};

struct LossParts {
  LossCut cut;
  Half *x, *weight;
  float2 *part;
  float *at;
  LossParts(Parts &w, int64_t n, int64_t width, int64_t classes, bool aligned, int sms)
      : cut(n, width, classes, sms), x(w.take<Half>(aligned ? 0 : n * up8(width))), weight(w.take<Half>(aligned ? 0 : classes * up8(width))),
        part(w.take<float2>((uint64_t)n * cut.parts)), at(w.take<float>(n)) {}
};

// Classes of a piece of dz: about 64 MB, so that a piece that has just been written is read from L2.
int64_t piece_classes(int64_t n, int64_t classes) {
  const int64_t fits = ((int64_t)32 << 20) / std::max<int64_t>(1, n) / 256 * 256;
  return std::min(up8(classes), std::max<int64_t>(256, fits));
}
struct LossGradParts {
  int64_t piece, ld_sums;
  float *scale;
  Half *x, *weight, *dz;
  float *bias_sums, *sums, *parts;
  LossGradParts(Parts &w, int64_t n, int64_t width, int64_t classes, bool aligned, int sms)
      : piece(piece_classes(n, classes)), ld_sums(up8(width)), scale(w.take<float>(1)), x(w.take<Half>(aligned ? 0 : n * up8(width))),
        weight(w.take<Half>(aligned ? 0 : classes * up8(width))), dz(w.take<Half>((uint64_t)n * piece)),
        bias_sums(w.take<float>(tiles_of(n, 32) * piece)), sums(w.take<float>(piece < classes ? n * ld_sums : 0)) {
    uint64_t most = 0; // of a full piece's products and the last one's
    for (const int64_t now : {std::min(piece, classes), (classes - 1) % piece + 1})
      if (n > 0) most = std::max({most, part_floats(n, width, now, sms), part_floats(now, width, n, sms)});
    parts = w.take<float>(most);
  }
};

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

// How a leaf sum is cut.  Up to two rows per multiprocessor: a block per row, trees over its lane groups.
// Above that: blocks of 64 rows per lane group and warp, and ranges of trees (joined afterwards) so that the
// multiprocessors are evenly filled; a range costs a round trip of its fp32 sums.
struct LeafSumPlan {
  bool by_row;
  int lanes_log2, threads, trees_per_part;
  unsigned columns, blocks, parts = 1;
  int64_t ld_parts;
  LeafSumPlan(int64_t n, int64_t width, int32_t type, int64_t trees, int sms) {
    const int elems = type == TBK_TYPE_F32 ? 4 : 8;
    lanes_log2 = lanes_of(width, type);
    const int lanes = 1 << lanes_log2;
    columns = (unsigned)tiles_of(width, (int64_t)elems << lanes_log2);
    ld_parts = tiles_of(width, elems) * elems;
    by_row = n <= 2 * sms;
    trees_per_part = (int)trees;
    if (by_row) {
      threads = (int)std::clamp<int64_t>(tiles_of(tiles_of(trees, 8) * lanes, 32) * 32, 32, 1024);
      blocks = (unsigned)n;
      return;
    }
    const int64_t rows_per_warp = (32 / lanes) * tb::kLeafRows;
    threads = (int)std::min<int64_t>(512, tiles_of(n, rows_per_warp) * 32);
    blocks = (unsigned)tiles_of(n, threads / 32 * rows_per_warp);
    const double gather = (double)n * trees * width * (32 / elems) / 8 / 15e6, trip = (double)n * ld_parts * 8 / 4e6; // us
    double least = 1e300;
    for (int64_t p = 1; p <= std::min<int64_t>(64, tiles_of(trees, 2 * lanes)); ++p) {
      const double units = (double)blocks * columns * p, cost = gather * std::ceil(units / sms) * sms / units + (p > 1 ? trip * p + 4 : 0);
      if (cost < least) least = cost, parts = (unsigned)p;
    }
    trees_per_part = (int)tiles_of(tiles_of(trees, parts), lanes) * lanes;
    parts = (unsigned)tiles_of(trees, trees_per_part);
  }
};

struct LeafGradParts {
  int64_t ld;
  uint32_t *numbers;
  float *sums;
  LeafGradParts(Parts &w, int64_t n, int64_t width, int64_t trees, int64_t rows)
      : ld(up8(n)), numbers(w.take<uint32_t>(trees * ld)), sums(w.take<float>(n > tb::kLeafChunk ? rows * width : 0)) {}
};

} // namespace

extern "C" {

int tbk_leaf_map_create(const tbk_forest_arrays *fa, int32_t device, tbk_leaf_map **out) {
  if (!out) return fail(TBK_ERR_INVALID, "null argument");
  *out = nullptr;
  if (!fa || !fa->tree_off || !fa->left) return fail(TBK_ERR_INVALID, "null forest array");
  if (fa->num_trees < 1) return fail(TBK_ERR_INVALID, "a leaf map needs a tree at least");
  if (fa->num_trees > 1 << 21) return fail(TBK_ERR_UNSUPPORTED, "more than %d trees", 1 << 21);
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
  return check_matrix("leaf_ids", ids, ld_ids, n, map->view.num_trees);
}

int tbk_leaf_sum_workspace(const tbk_leaf_map *map, int64_t n, int64_t width, int32_t type, uint64_t *bytes) {
  if (!map || !bytes) return fail(TBK_ERR_INVALID, "null argument");
  TRY(check_sizes("leaf sum", n, width, 1));
  const LeafSumPlan plan(n, width, type, map->view.num_trees, multiprocessors(map->device));
  *bytes = plan.parts > 1 ? (uint64_t)plan.parts * n * plan.ld_parts * 4 : 0;
  return TBK_OK;
}

int tbk_leaf_sum(const tbk_leaf_map *map, const int32_t *ids, int64_t n, int64_t ld_ids, const void *table, int64_t ld_table,
                 int64_t width, int32_t type, void *out, int64_t ld_out, void *ws, uint64_t ws_bytes, void *stream_) {
  TRY(check_leaf_call(map, ids, n, ld_ids, width, type));
  TRY(check_matrix("table", table, ld_table, map->rows, width));
  TRY(check_matrix("out", out, ld_out, n, width));
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
    if (plan.by_row) {
      tb::tb_leaf_sum_row_kernel<T, V><<<dim3((unsigned)n, plan.columns), plan.threads, 0, stream>>>(map->view, ids, ld_ids, (const T *)table, ld_table,
                                                                                                     width, plan.lanes_log2, (T *)out, ld_out);
      CUDA_TRY(cudaGetLastError());
      return (int)TBK_OK;
    }
    float *parts = plan.parts > 1 ? (float *)ws : nullptr;
    tb::tb_leaf_sum_kernel<T, V><<<dim3(plan.blocks, plan.columns, plan.parts), plan.threads, 0, stream>>>(
        map->view, ids, ld_ids, (const T *)table, ld_table, width, plan.lanes_log2, (T *)out, ld_out, parts, plan.ld_parts, n, plan.trees_per_part);
    CUDA_TRY(cudaGetLastError());
    if (parts) {
      const int64_t threads = n * plan.ld_parts / tb::Share<T, V>::kElems;
      tb::tb_leaf_sum_join_kernel<T, V><<<(unsigned)tiles_of(threads, 256), 256, 0, stream>>>(parts, plan.ld_parts, plan.parts, (T *)out, ld_out, width, n);
      CUDA_TRY(cudaGetLastError());
    }
    return (int)TBK_OK;
  });
}

int tbk_leaf_sum_backward_workspace(const tbk_leaf_map *map, int64_t n, int64_t width, int32_t type, uint64_t *bytes) {
  if (!map || !bytes) return fail(TBK_ERR_INVALID, "null argument");
  (void)type;
  TRY(check_sizes("leaf sum", n, width, 1));
  Parts w{nullptr};
  LeafGradParts parts(w, n, width, map->view.num_trees, map->rows);
  *bytes = w.used;
  return TBK_OK;
}

int tbk_leaf_sum_backward(const tbk_leaf_map *map, const int32_t *ids, int64_t n, int64_t ld_ids, const void *grad, int64_t ld_grad,
                          int64_t width, int32_t type, void *out, int64_t ld_out, void *ws, uint64_t ws_bytes, void *stream_) {
  TRY(check_leaf_call(map, ids, n, ld_ids, width, type));
  TRY(check_matrix("grad", grad, ld_grad, n, width));
  TRY(check_matrix("out", out, ld_out, map->rows, width));
  uint64_t need = 0;
  TRY(tbk_leaf_sum_backward_workspace(map, n, width, type, &need));
  OnDevice on(map->device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  const size_t size = type == TBK_TYPE_F32 ? 4 : 2;
  if (n == 0) {
    CUDA_TRY(cudaMemset2DAsync(out, (size_t)ld_out * size, 0, (size_t)width * size, (size_t)map->rows, stream));
    return TBK_OK;
  }
  TRY(check_workspace(ws, ws_bytes, need));
  Parts w{(unsigned char *)ws};
  const int64_t trees = map->view.num_trees;
  LeafGradParts parts(w, n, width, trees, map->rows);
  tb::tb_leaf_numbers_kernel<<<dim3((unsigned)std::min<int64_t>(tiles_of(n, 32), 4096), (unsigned)tiles_of(trees, 32)), 256, 0, stream>>>(map->view, ids, ld_ids, parts.numbers, parts.ld, n);
  CUDA_TRY(cudaGetLastError());
  return with_piece(type, piece_bytes(type, width, grad, ld_grad, n, out, ld_out, map->rows), [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const auto kernel = tb::tb_leaf_grad_kernel<T, V>;
    const int lanes_log2 = lanes_of(width, type), range = (int)std::min<int64_t>(map->max_rows, tb::kLeafRange);
    const int chunk = (int)std::min<int64_t>(n, tb::kLeafChunk), smem = tb::leaf_grad_smem(chunk, range);
    CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tb::leaf_grad_smem(tb::kLeafChunk, tb::kLeafRange)));
    const dim3 grid((unsigned)trees, (unsigned)tiles_of(width, (16 / size) << lanes_log2), (unsigned)tiles_of(map->max_rows, range));
    if (grid.y > 65535 || grid.z > 65535) return fail(TBK_ERR_UNSUPPORTED, "leaf_sum_backward: too many columns or leaves of a tree");
    kernel<<<grid, 32 * tb::kLeafGradWarps, smem, stream>>>(map->view, parts.numbers, parts.ld, (const T *)grad, ld_grad, width, lanes_log2, parts.sums,
                                                            (T *)out, ld_out, n, chunk, range);
    CUDA_TRY(cudaGetLastError());
    return (int)TBK_OK;
  });
}

int tbk_linear_workspace(int64_t n, int64_t inputs, int64_t outputs, int32_t type, int32_t aligned, int32_t device, uint64_t *bytes) {
  if (!bytes) return fail(TBK_ERR_INVALID, "null argument");
  TRY(half_type(type, "linear"));
  TRY(check_sizes("linear", n, inputs, outputs));
  Parts w{nullptr};
  LinearParts parts(w, n, inputs, outputs, aligned != 0, multiprocessors(device));
  *bytes = w.used;
  return TBK_OK;
}

int tbk_linear(const void *x, int64_t ld_x, const void *weight, int64_t ld_w, const void *bias, int32_t act, const void *residual,
               int64_t ld_res, void *out, int64_t ld_out, void *pre, int64_t ld_pre, int64_t n, int64_t inputs, int64_t outputs,
               int32_t type, void *ws, uint64_t ws_bytes, int32_t device, void *stream_) {
  uint64_t need = 0;
  const bool aligned = tma_rows(x, ld_x, n) && tma_rows(weight, ld_w, outputs);
  TRY(tbk_linear_workspace(n, inputs, outputs, type, aligned, device, &need));
  if (act < TBK_ACT_IDENTITY || act > TBK_ACT_SILU) return fail(TBK_ERR_INVALID, "unknown activation %d", act);
  TRY(check_matrix("x", x, ld_x, n, inputs));
  TRY(check_matrix("weight", weight, ld_w, outputs, inputs));
  if (residual) TRY(check_matrix("residual", residual, ld_res, n, outputs));
  TRY(check_matrix("out", out, ld_out, n, outputs));
  if (pre) TRY(check_matrix("pre", pre, ld_pre, n, outputs));
  if (n == 0) return TBK_OK;
  TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    const int sms = multiprocessors(device);
    Parts w{(unsigned char *)ws};
    LinearParts parts(w, n, inputs, outputs, aligned, sms);
    TRY(readable(&x, &ld_x, n, inputs, (T *)parts.x, stream));
    TRY(readable(&weight, &ld_w, outputs, inputs, (T *)parts.weight, stream));
    const tb::LinearEnd<T> end{(const T *)bias, (const T *)residual, (T *)out, (T *)pre, ld_res, ld_out, ld_pre, act,
                               vec_rows(residual, ld_res), vec_rows(out, ld_out), vec_rows(pre, ld_pre), vec_rows(bias, 0)};
    return product<T>({x, ld_x, false}, {weight, ld_w, false}, n, outputs, inputs, end, parts.parts, sms, stream);
  });
}

int tbk_linear_backward_workspace(int64_t n, int64_t inputs, int64_t outputs, int32_t type, int32_t aligned, int32_t device, uint64_t *bytes) {
  if (!bytes) return fail(TBK_ERR_INVALID, "null argument");
  TRY(half_type(type, "linear_backward"));
  TRY(check_sizes("linear_backward", n, inputs, outputs));
  Parts w{nullptr};
  LinearGradParts parts(w, n, inputs, outputs, aligned != 0, multiprocessors(device));
  *bytes = w.used;
  return TBK_OK;
}

// Gradients of a call without rows.
static int clear_rows(void *p, int64_t ld, int64_t rows, int64_t cols, cudaStream_t stream) {
  if (p) CUDA_TRY(cudaMemset2DAsync(p, (size_t)ld * 2, 0, (size_t)cols * 2, (size_t)rows, stream));
  return TBK_OK;
}

int tbk_linear_backward(const void *grad, int64_t ld_grad, const void *x, int64_t ld_x, const void *weight, int64_t ld_w, const void *pre,
                        int64_t ld_pre, int32_t act, const void *skip, int64_t ld_skip, void *grad_x, int64_t ld_gx, void *grad_w,
                        int64_t ld_gw, void *grad_b, int64_t n, int64_t inputs, int64_t outputs, int32_t type, void *ws, uint64_t ws_bytes,
                        int32_t device, void *stream_) {
  uint64_t need = 0;
  const bool aligned = tma_rows(x, ld_x, n) && tma_rows(weight, ld_w, outputs);
  TRY(tbk_linear_backward_workspace(n, inputs, outputs, type, aligned, device, &need));
  if (act < TBK_ACT_IDENTITY || act > TBK_ACT_SILU) return fail(TBK_ERR_INVALID, "unknown activation %d", act);
  TRY(check_matrix("grad", grad, ld_grad, n, outputs));
  TRY(check_matrix("x", x, ld_x, n, inputs));
  TRY(check_matrix("weight", weight, ld_w, outputs, inputs));
  if (act != TBK_ACT_IDENTITY) TRY(check_matrix("pre", pre, ld_pre, n, outputs));
  if (skip) TRY(check_matrix("skip", skip, ld_skip, n, inputs));
  if (grad_x) TRY(check_matrix("grad_x", grad_x, ld_gx, n, inputs));
  if (grad_w) TRY(check_matrix("grad_weight", grad_w, ld_gw, outputs, inputs));
  if (n > 0) TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (n == 0) {
    TRY(clear_rows(grad_w, ld_gw, outputs, inputs, stream));
    return clear_rows(grad_b, outputs, 1, outputs, stream);
  }
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    const int sms = multiprocessors(device);
    Parts w{(unsigned char *)ws};
    LinearGradParts parts(w, n, inputs, outputs, aligned, sms);
    T *dz = (T *)parts.dz;
    if (grad_w) TRY(readable(&x, &ld_x, n, inputs, (T *)parts.x, stream));
    if (grad_x) TRY(readable(&weight, &ld_w, outputs, inputs, (T *)parts.weight, stream));
    tb::tb_act_grad_kernel<T><<<dim3((unsigned)tiles_of(outputs, 256), (unsigned)std::min<int64_t>(tiles_of(n, 256), 65535)), 256, 0, stream>>>(
        (const T *)grad, ld_grad, vec_rows(grad, ld_grad), (const T *)pre, ld_pre, vec_rows(pre, ld_pre), act, dz, parts.ld,
        grad_b ? parts.bias_sums : nullptr, n, outputs);
    CUDA_TRY(cudaGetLastError());
    if (grad_b) {
      tb::tb_column_sum_kernel<T><<<(unsigned)tiles_of(outputs, 32), 256, 0, stream>>>(parts.bias_sums, tiles_of(n, 32), parts.ld, (T *)grad_b, outputs, nullptr);
      CUDA_TRY(cudaGetLastError());
    }
    if (grad_x) {
      const tb::SumEnd<T> end{nullptr, 0, (T *)grad_x, (const T *)skip, ld_gx, ld_skip, nullptr, true, true, vec_rows(grad_x, ld_gx), vec_rows(skip, ld_skip)};
      TRY((product<T>({dz, parts.ld, false}, {weight, ld_w, true}, n, inputs, outputs, end, parts.parts, sms, stream)));
    }
    if (grad_w) {
      const tb::SumEnd<T> end{nullptr, 0, (T *)grad_w, nullptr, ld_gw, 0, nullptr, true, true, vec_rows(grad_w, ld_gw), false};
      TRY((product<T>({dz, parts.ld, true}, {x, ld_x, true}, outputs, inputs, n, end, parts.parts, sms, stream)));
    }
    return (int)TBK_OK;
  });
}

int tbk_class_loss_workspace(int64_t n, int64_t width, int64_t classes, int32_t type, int32_t aligned, int32_t device, uint64_t *bytes) {
  if (!bytes) return fail(TBK_ERR_INVALID, "null argument");
  TRY(half_type(type, "class_loss"));
  TRY(check_sizes("class_loss", n, width, classes));
  Parts w{nullptr};
  LossParts parts(w, n, width, classes, aligned != 0, multiprocessors(device));
  *bytes = w.used;
  return TBK_OK;
}

static int check_labels(const void *labels, int32_t label_bytes, int64_t n) {
  if (!labels && n > 0) return fail(TBK_ERR_INVALID, "labels is null");
  if (label_bytes != 4 && label_bytes != 8) return fail(TBK_ERR_INVALID, "labels of %d bytes", label_bytes);
  return TBK_OK;
}

int tbk_class_loss(const void *x, int64_t ld_x, const void *weight, int64_t ld_w, const void *bias, const void *labels, int32_t label_bytes,
                   float *loss, float *lse, int64_t n, int64_t width, int64_t classes, int32_t type, void *ws, uint64_t ws_bytes,
                   int32_t device, void *stream_) {
  uint64_t need = 0;
  const bool aligned = tma_rows(x, ld_x, n) && tma_rows(weight, ld_w, classes);
  TRY(tbk_class_loss_workspace(n, width, classes, type, aligned, device, &need));
  TRY(check_matrix("x", x, ld_x, n, width));
  TRY(check_matrix("weight", weight, ld_w, classes, width));
  TRY(check_labels(labels, label_bytes, n));
  if (n > 0 && (!loss || !lse)) return fail(TBK_ERR_INVALID, "null output pointer");
  if (n == 0) return TBK_OK;
  TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    const int sms = multiprocessors(device);
    Parts w{(unsigned char *)ws};
    LossParts parts(w, n, width, classes, aligned, sms);
    TRY(readable(&x, &ld_x, n, width, (T *)parts.x, stream));
    TRY(readable(&weight, &ld_w, classes, width, (T *)parts.weight, stream));
    const Side a{x, ld_x, false}, b{weight, ld_w, false};
    if (parts.cut.pair) {
      const tb::LseEnd<T, 128> end{(const T *)bias, labels, label_bytes, parts.part, parts.at};
      TRY((launch_dense<T, true>(a, b, n, classes, width, 1, parts.cut.run, sms, end, stream)));
    } else {
      const tb::LseEnd<T, 64> end{(const T *)bias, labels, label_bytes, parts.part, parts.at};
      TRY((launch_dense<T, false>(a, b, n, classes, width, 1, parts.cut.run, sms, end, stream)));
    }
    tb::tb_loss_join_kernel<<<(unsigned)tiles_of(n, 128), 128, 0, stream>>>(parts.part, parts.cut.parts, parts.at, labels, label_bytes, classes, loss, lse, n);
    CUDA_TRY(cudaGetLastError());
    return (int)TBK_OK;
  });
}

int tbk_class_loss_backward_workspace(int64_t n, int64_t width, int64_t classes, int32_t type, int32_t aligned, int32_t device, uint64_t *bytes) {
  if (!bytes) return fail(TBK_ERR_INVALID, "null argument");
  TRY(half_type(type, "class_loss_backward"));
  TRY(check_sizes("class_loss_backward", n, width, classes));
  Parts w{nullptr};
  LossGradParts parts(w, n, width, classes, aligned != 0, multiprocessors(device));
  *bytes = w.used;
  return TBK_OK;
}

int tbk_class_loss_backward(const float *grad, const void *x, int64_t ld_x, const void *weight, int64_t ld_w, const void *bias,
                            const void *labels, int32_t label_bytes, const float *lse, void *grad_x, int64_t ld_gx, void *grad_w,
                            int64_t ld_gw, void *grad_b, int64_t n, int64_t width, int64_t classes, int32_t type, void *ws,
                            uint64_t ws_bytes, int32_t device, void *stream_) {
  uint64_t need = 0;
  const bool aligned = tma_rows(x, ld_x, n) && tma_rows(weight, ld_w, classes);
  TRY(tbk_class_loss_backward_workspace(n, width, classes, type, aligned, device, &need));
  TRY(check_matrix("x", x, ld_x, n, width));
  TRY(check_matrix("weight", weight, ld_w, classes, width));
  TRY(check_labels(labels, label_bytes, n));
  if (n > 0 && (!grad || !lse)) return fail(TBK_ERR_INVALID, "null input pointer");
  if (grad_x) TRY(check_matrix("grad_x", grad_x, ld_gx, n, width));
  if (grad_w) TRY(check_matrix("grad_weight", grad_w, ld_gw, classes, width));
  if (n > 0) TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  if (n == 0) {
    TRY(clear_rows(grad_w, ld_gw, classes, width, stream));
    return clear_rows(grad_b, classes, 1, classes, stream);
  }
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    const int sms = multiprocessors(device);
    Parts w{(unsigned char *)ws};
    LossGradParts parts(w, n, width, classes, aligned, sms);
    TRY(readable(&x, &ld_x, n, width, (T *)parts.x, stream));
    TRY(readable(&weight, &ld_w, classes, width, (T *)parts.weight, stream));
    const T *W = (const T *)weight;
    T *dz = (T *)parts.dz;
    const int64_t ld = parts.piece;
    tb::tb_scale_kernel<<<1, 1024, 0, stream>>>(grad, n, parts.scale);
    CUDA_TRY(cudaGetLastError());
    for (int64_t v = 0; v < classes; v += ld) {
      const int64_t now = std::min(ld, classes - v);
      const Side xs{x, ld_x, false}, ws_{W + v * ld_w, ld_w, false};
      const T *b = bias ? (const T *)bias + v : nullptr;
      float *sums = grad_b ? parts.bias_sums : nullptr;
      if (plan_product(n, now, width, sms, false).pair) {
        const tb::ScoreGradEnd<T, 128> end{b, labels, label_bytes, grad, lse, parts.scale, dz, ld, v, classes, sums};
        TRY((launch_dense<T, true>(xs, ws_, n, now, width, 1, 1, sms, end, stream)));
      } else {
        const tb::ScoreGradEnd<T, 64> end{b, labels, label_bytes, grad, lse, parts.scale, dz, ld, v, classes, sums};
        TRY((launch_dense<T, false>(xs, ws_, n, now, width, 1, 1, sms, end, stream)));
      }
      if (grad_b) {
        tb::tb_column_sum_kernel<T><<<(unsigned)tiles_of(now, 32), 256, 0, stream>>>(parts.bias_sums, tiles_of(n, 32), ld, (T *)grad_b + v, now, parts.scale);
        CUDA_TRY(cudaGetLastError());
      }
      if (grad_x) {
        const tb::SumEnd<T> end{parts.sums, parts.ld_sums, (T *)grad_x, nullptr, ld_gx, 0, parts.scale, v == 0, v + now == classes, vec_rows(grad_x, ld_gx), false};
        TRY((product<T>({dz, ld, false}, {W + v * ld_w, ld_w, true}, n, width, now, end, parts.parts, sms, stream)));
      }
      if (grad_w) {
        T *to = (T *)grad_w + v * ld_gw;
        const tb::SumEnd<T> end{nullptr, 0, to, nullptr, ld_gw, 0, parts.scale, true, true, vec_rows(to, ld_gw), false};
        TRY((product<T>({dz, ld, true}, {x, ld_x, true}, now, width, n, end, parts.parts, sms, stream)));
      }
    }
    return (int)TBK_OK;
  });
}

int tbk_leaf_check_status(int32_t device) {
  OnDevice on(device);
  CUDA_TRY(on.error);
  int word = 0, zero = 0;
  CUDA_TRY(cudaMemcpyFromSymbol(&word, tb::tb_dense_status, sizeof word));
  if (!word) return TBK_OK;
  CUDA_TRY(cudaMemcpyToSymbol(tb::tb_dense_status, &zero, sizeof zero));
  return fail(TBK_ERR_DEVICE_WAIT, "a wait inside a matrix product gave up");
}

} // extern "C"
