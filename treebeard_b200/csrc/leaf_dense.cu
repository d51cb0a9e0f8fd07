// C ABI of the linear layers and the class loss (include/tbk_leaf.h): plans, launches.
#include "../../include/tbk_leaf.h"
#include "dense.cuh"
#include "leaf_api.h"

#include <cudaTypedefs.h>
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace {

int half_type(int32_t type, const char *what) {
  if (type == TBK_TYPE_F16 || type == TBK_TYPE_BF16) return TBK_OK;
  if (type == TBK_TYPE_F32) return fail(TBK_ERR_UNSUPPORTED, "%s takes 16-bit floating point types (fp16, bf16)", what);
  return fail(TBK_ERR_INVALID, "unknown element type %d", type);
}

template <class F> int with_half(int32_t type, F f) { return type == TBK_TYPE_F16 ? f(__half()) : f(__nv_bfloat16()); }

// How products are cut: into tiles of one of the three shapes of tb_dense_kernel and, where that leaves
// multiprocessors without work, the sums into parts that a second kernel joins.  Cycles per 64 k of a tile, around a
// tile (`heavy`: with an activation of many instructions a result) and for the join follow measurements; the cheapest
// cut of a launch's one or two products is taken.
struct Size {
  int64_t m, n, k;
};
struct Cut {
  int shape = tb::kDenseOne;
  int splits[2] = {1, 1};
};
Cut find_cut(const Size *sizes, int count, int sms, bool may_split, bool heavy) {
  static const int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32};
  constexpr double kPer64[] = {700, 750, 1385};
  const double kAround[] = {900, heavy ? 3300. : 900., heavy ? 10000. : 2900.};
  Cut best;
  double least = 1e300;
  for (int shape = 0; shape < 3; ++shape) {
    const int64_t slots = shape == tb::kDenseOne ? sms : sms / 2;
    double tiles[2] = {}, kb[2] = {};
    for (int i = 0; i < count; ++i) {
      tiles[i] = (double)tiles_of(sizes[i].m, tb::dense_rows(shape)) * tiles_of(sizes[i].n, tb::dense_cols(shape));
      kb[i] = (double)tiles_of(sizes[i].k, 64);
    }
    for (const int s0 : kSplits) {
      if (s0 > 1 && (!may_split || s0 > kb[0])) break;
      for (const int s1 : kSplits) {
        if (s1 > 1 && (!may_split || count < 2 || s1 > kb[1])) break;
        const int s[2] = {s0, s1};
        double per[2] = {}, join = 0;
        int64_t units[2] = {};
        for (int i = 0; i < count; ++i) {
          per[i] = std::ceil(kb[i] / s[i]) * kPer64[shape] + kAround[shape];
          units[i] = (int64_t)tiles[i] * s[i];
          if (s[i] > 1) join += 5000 + (double)sizes[i].m * sizes[i].n * 8 * s[i] / 2500;
        }
        // slot i has units i, i + slots, ... of both products' one after the other: some slots have one more of the
        // first's, some one more in all
        const int64_t all = units[0] + units[1], a = units[0] / slots, ra = units[0] % slots, b = all / slots, rb = all % slots;
        auto load = [&](int64_t of_first, int64_t of_all) { return of_first * per[0] + (of_all - of_first) * per[1]; };
        double cost = 0;
        if (ra > 0 && rb > 0) cost = std::max(cost, load(a + 1, b + 1));
        if (rb > ra) cost = std::max(cost, load(a, b + 1));
        if (ra > rb) cost = std::max(cost, load(a + 1, b));
        if (std::max(ra, rb) < slots) cost = std::max(cost, load(a, b));
        cost += join;
        if (cost < least) least = cost, best.shape = shape, best.splits[0] = s0, best.splits[1] = s1;
      }
    }
  }
  return best;
}
// The same, remembered: a program's sizes are mostly alike, and a search takes microseconds.
Cut plan_products(const Size *sizes, int count, int sms, bool may_split, bool heavy = false) {
  struct Entry {
    int64_t key[8] = {-1};
    Cut cut;
  };
  static thread_local Entry entries[64];
  int64_t key[8] = {count * 4 + may_split * 2 + heavy, sms, sizes[0].m, sizes[0].n, sizes[0].k, 0, 0, 0};
  if (count > 1) key[5] = sizes[1].m, key[6] = sizes[1].n, key[7] = sizes[1].k;
  uint64_t h = 0;
  for (const int64_t k : key) h = (h ^ (uint64_t)k) * 0x9e3779b97f4a7c15ull;
  Entry &e = entries[h >> 58];
  if (std::memcmp(e.key, key, sizeof key) != 0) {
    e.cut = find_cut(sizes, count, sms, may_split, heavy);
    std::memcpy(e.key, key, sizeof key);
  }
  return e.cut;
}
// fp32 room for the parts of a launch's products
uint64_t part_floats(const Size *sizes, int count, int sms, bool heavy = false) {
  const Cut cut = plan_products(sizes, count, sms, true, heavy);
  uint64_t sum = 0;
  for (int i = 0; i < count; ++i)
    if (cut.splits[i] > 1) sum += (uint64_t)cut.splits[i] * sizes[i].m * up8(sizes[i].n);
  return sum;
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
template <class T> int encode_map(CUtensorMap *map, const void *p, int64_t inner, int64_t outer, int64_t ld, uint32_t box_inner, uint32_t box_outer) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return fail(TBK_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer}, strides[1] = {(cuuint64_t)(outer > 1 ? ld : up8(inner)) * 2};
  const cuuint32_t box[2] = {box_inner, box_outer}, one[2] = {1, 1};
  const CUresult rc = encode(map, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(p),
                             dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, box_inner == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? TBK_OK : fail(TBK_ERR_CUDA, "cuTensorMapEncodeTiled: %d (%lld x %lld, %lld)", (int)rc, (long long)outer, (long long)inner, (long long)ld);
}
template <class T> int side_map(CUtensorMap *map, const Side &s, int64_t rows, int64_t k) {
  return encode_map<T>(map, s.p, s.rows_inner ? rows : k, s.rows_inner ? k : rows, s.ld, 64, s.rows_inner ? 64 : 128);
}
// Where a warp's 32 rows and columns of a result go.
template <class T> int out_map(CUtensorMap *map, const void *p, int64_t rows, int64_t cols, int64_t ld) { return encode_map<T>(map, p, cols, rows, ld, 32, 32); }

// Parts of sums, fp32: [splits][rows][ld], 32 x 32 at a time.
int parts_map(CUtensorMap *map, const void *p, int splits, int64_t rows, int64_t cols, int64_t ld) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return fail(TBK_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)splits}, strides[2] = {(cuuint64_t)ld * 4, (cuuint64_t)(ld * rows) * 4};
  const cuuint32_t box[3] = {32, 32, 1}, one[3] = {1, 1, 1};
  const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? TBK_OK : fail(TBK_ERR_CUDA, "cuTensorMapEncodeTiled: %d (%d x %lld x %lld)", (int)rc, splits, (long long)rows, (long long)cols);
}

template <class T> int set_problem(tb::DenseProblem *p, int shape, const Side &a, const Side &b, const Size &size, int splits, int run) {
  TRY(side_map<T>(&p->a, a, size.m, size.k));
  TRY(side_map<T>(&p->b, b, size.n, size.k));
  p->M = (int)size.m, p->N = (int)size.n;
  p->a_rows_inner = a.rows_inner, p->b_rows_inner = b.rows_inner;
  p->m_tiles = (int)tiles_of(size.m, tb::dense_rows(shape)), p->n_tiles = (int)tiles_of(size.n, tb::dense_cols(shape));
  p->k_blocks = (int)tiles_of(size.k, 64);
  p->chunk = run;
  p->chunks = (int)tiles_of(p->n_tiles, run);
  p->splits = splits;
  p->group = shape == tb::kDenseOne ? 16 : shape == tb::kDensePair ? 8 : 4;
  const int64_t units = (int64_t)p->m_tiles * p->chunks * splits;
  if (units > 1 << 30) return fail(TBK_ERR_UNSUPPORTED, "a product of %lld x %lld", (long long)size.m, (long long)size.n);
  p->units = (int)units;
  return TBK_OK;
}
// Launches what stands in jobs.p, jobs.end.
template <class T, int SHAPE, class End, int JOBS> int launch_shape(const tb::DenseJobs<End, JOBS> &jobs, int slots, cudaStream_t stream) {
  static std::atomic<uint64_t> ready{0}; // devices on which the kernel may use its shared memory
  constexpr int smem = tb::dense_smem_bytes(SHAPE);
  const auto kernel = tb::tb_dense_kernel<T, SHAPE, End, JOBS>;
  int device = 0;
  CUDA_TRY(cudaGetDevice(&device));
  if (device > 63 || !(ready.load() >> device & 1)) {
    CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (device <= 63) ready.fetch_or(1ull << device);
  }
  const unsigned grid = (unsigned)std::min(jobs.units, slots) * (SHAPE == tb::kDenseOne ? 1 : 2);
  return launch(kernel, grid, tb::kDenseThreads, smem, stream, 1, jobs); // (its cluster is part of the kernel)
}
template <class T, class End, int JOBS> int launch_jobs(int shape, tb::DenseJobs<End, JOBS> &jobs, int sms, cudaStream_t stream) {
  jobs.units = jobs.p[0].units + (JOBS > 1 ? jobs.p[JOBS - 1].units : 0);
  return shape == tb::kDenseOne    ? launch_shape<T, tb::kDenseOne, End, JOBS>(jobs, sms, stream)
         : shape == tb::kDensePair ? launch_shape<T, tb::kDensePair, End, JOBS>(jobs, sms / 2, stream)
                                   : launch_shape<T, tb::kDenseTall, End, JOBS>(jobs, sms / 2, stream);
}
// The first `count` products of two.
template <class T, class End> int launch_some(int shape, tb::DenseJobs<End, 2> &jobs, int count, int sms, cudaStream_t stream) {
  if (count == 2) return launch_jobs<T, End, 2>(shape, jobs, sms, stream);
  tb::DenseJobs<End, 1> one;
  one.p[0] = jobs.p[0], one.end[0] = jobs.end[0];
  return launch_jobs<T, End, 1>(shape, one, sms, stream);
}

// A launch's product: C[m, n] = sum_k A[m, k] B[n, k], finished by `end`.
template <class T> struct Product {
  Side a, b;
  Size size;
  tb::Result<T> end;
};
// Column sums that are added up with a call's joins.
template <class T> struct ColumnSums {
  const float *rows = nullptr; // [count][ld]
  int64_t count = 0, ld = 0, columns = 0;
  T *out = nullptr;
  const float *scale = nullptr;
};
// One or two products, which do not depend on one another.  parts: room for what part_floats says.
template <class T>
int products(const Product<T> *list, int count, const ColumnSums<T> &sums, float *parts, int sms, cudaStream_t stream) {
  tb::FinishJobs<T> finish;
  std::memset(static_cast<void *>(&finish), 0, sizeof finish);
  if (count) {
    Size sizes[2];
    for (int i = 0; i < count; ++i) sizes[i] = list[i].size;
    const bool heavy = list[0].end.act >= tb::kActGelu; // (a layer's product is alone)
    const Cut cut = plan_products(sizes, count, sms, true, heavy);
    tb::DenseJobs<tb::ResultEnd<T>, 2> jobs;
    for (int i = 0; i < count; ++i) {
      const Product<T> &x = list[i];
      TRY(set_problem<T>(&jobs.p[i], cut.shape, x.a, x.b, x.size, cut.splits[i], 1));
      jobs.end[i].f = x.end;
      if (cut.splits[i] == 1) continue;
      jobs.end[i].f.parts = parts, jobs.end[i].f.ld_parts = up8(x.size.n);
      TRY(parts_map(&jobs.end[i].f.parts_map, parts, cut.splits[i], x.size.m, up8(x.size.n), up8(x.size.n)));
      finish.end[i] = jobs.end[i].f;
      finish.splits[i] = cut.splits[i], finish.M[i] = x.size.m, finish.N[i] = x.size.n;
      finish.blocks[i] = (unsigned)tiles_of(x.size.m * (up8(x.size.n) / 8), 256);
      parts += (uint64_t)cut.splits[i] * x.size.m * up8(x.size.n);
    }
    TRY((launch_some<T, tb::ResultEnd<T>>(cut.shape, jobs, count, sms, stream)));
  }
  if (sums.out) {
    finish.rows = sums.rows, finish.count = sums.count, finish.ld_rows = sums.ld, finish.columns = sums.columns;
    finish.column_sums = sums.out, finish.scale = sums.scale;
    finish.blocks[2] = (unsigned)tiles_of(sums.columns, 32);
  }
  const unsigned blocks = finish.blocks[0] + finish.blocks[1] + finish.blocks[2];
  return blocks ? launch(tb::tb_dense_finish_kernel<T>, blocks, 256, 0, stream, 1, finish) : (int)TBK_OK;
}

// Whether tensor copies can read a matrix: rows begin at multiples of 16 bytes.
bool tma_rows(const void *p, int64_t ld, int64_t rows) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld % 8 == 0 || rows <= 1);
}
// Has a matrix copied to `room` (rows x up8(cols)) where tensor copies cannot read it as it is.
template <class T> void make_readable(tb::PrepareJobs<T> *jobs, int which, const void **p, int64_t *ld, int64_t rows, int64_t cols, void *room) {
  if (tma_rows(*p, *ld, rows)) return;
  jobs->copy[which] = {(const T *)*p, (T *)room, *ld, up8(cols), rows, cols};
  jobs->blocks[2 + which] = (unsigned)tiles_of(rows * (up8(cols) / 8), 256);
  *p = room;
  *ld = up8(cols);
}
template <class T> tb::PrepareJobs<T> no_jobs() {
  tb::PrepareJobs<T> jobs;
  std::memset(static_cast<void *>(&jobs), 0, sizeof jobs);
  return jobs;
}
template <class T> int prepare(const tb::PrepareJobs<T> &jobs, int act, cudaStream_t stream) {
  const unsigned blocks = jobs.blocks[0] + jobs.blocks[1] + jobs.blocks[2] + jobs.blocks[3];
  if (!blocks) return TBK_OK;
  switch (act) {
  case TBK_ACT_RELU: return launch(tb::tb_dense_prepare_kernel<T, tb::kActRelu>, blocks, 256, 0, stream, 1, jobs);
  case TBK_ACT_GELU: return launch(tb::tb_dense_prepare_kernel<T, tb::kActGelu>, blocks, 256, 0, stream, 1, jobs);
  case TBK_ACT_SILU: return launch(tb::tb_dense_prepare_kernel<T, tb::kActSilu>, blocks, 256, 0, stream, 1, jobs);
  default: return launch(tb::tb_dense_prepare_kernel<T, tb::kActNone>, blocks, 256, 0, stream, 1, jobs);
  }
}
// Whether 16 bytes at a time can be read or written at every eighth column.
bool vec_rows(const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

// Where a product's whole sums go: out = sum / *scale + addend, before an activation and a bias are set.
template <class T>
int set_result(tb::Result<T> *end, void *out, int64_t ld, int64_t rows, int64_t cols, const void *addend, int64_t ld_addend, void *pre, int64_t ld_pre) {
  std::memset(static_cast<void *>(end), 0, sizeof *end);
  end->out = (T *)out, end->ld_out = ld, end->vec_out = vec_rows(out, ld);
  end->addend = (const T *)addend, end->ld_addend = ld_addend, end->vec_addend = vec_rows(addend, ld_addend);
  end->pre = (T *)pre, end->ld_pre = ld_pre, end->vec_pre = vec_rows(pre, ld_pre);
  end->first = end->last = true;
  end->tma_out = tma_rows(out, ld, rows), end->tma_addend = addend && tma_rows(addend, ld_addend, rows), end->tma_pre = pre && tma_rows(pre, ld_pre, rows);
  if (end->tma_out) TRY(out_map<T>(&end->out_map, out, rows, cols, ld));
  if (end->tma_addend) TRY(out_map<T>(&end->addend_map, addend, rows, cols, ld_addend));
  if (end->tma_pre) TRY(out_map<T>(&end->pre_map, pre, rows, cols, ld_pre));
  return TBK_OK;
}

// A layer of at most kFewRows rows.
template <class T>
int few_rows(const T *x, int64_t ld_x, const T *weight, int64_t ld_w, const T *bias, int act, const T *residual, int64_t ld_res, T *out, int64_t ld_out, T *pre, int64_t ld_pre,
             int n, int inputs, int outputs, int sms, cudaStream_t stream) {
  tb::Result<T> end;
  std::memset(static_cast<void *>(&end), 0, sizeof end);
  end.bias = bias, end.act = act, end.addend = residual, end.ld_addend = ld_res, end.out = out, end.ld_out = ld_out, end.pre = pre, end.ld_pre = ld_pre;
  const bool vec = tma_rows(x, ld_x, n) && tma_rows(weight, ld_w, outputs);
  const unsigned blocks = (unsigned)std::min<int64_t>(tiles_of(outputs, 8), 8 * sms);
  auto run = [&](auto rows) {
    constexpr int R = decltype(rows)::value;
    return vec ? launch(tb::tb_linear_rows_kernel<T, true, R>, blocks, 256, 0, stream, 1, x, ld_x, weight, ld_w, end, n, inputs, outputs)
               : launch(tb::tb_linear_rows_kernel<T, false, R>, blocks, 256, 0, stream, 1, x, ld_x, weight, ld_w, end, n, inputs, outputs);
  };
  return n == 1 ? run(std::integral_constant<int, 1>()) : n <= 4 ? run(std::integral_constant<int, 4>()) : run(std::integral_constant<int, 8>());
}

// Whether a layer goes to tb_linear_rows_kernel.  Its time grows with the rows, the other kernel's hardly: 1, 4, 8 rows
// of 1024 x 1024 take 2.5, 4.8, 8.5 us (8.6, 8.7, 9.1 there), of 4096 x 4096 8, 17, 31 (13 to 15).
bool is_few_rows(int64_t n, int64_t inputs, int64_t outputs) {
  return n == 1 || (n <= tb::kFewRows && (double)(n * n) * inputs * outputs <= 1 << 26);
}

typedef unsigned short Half; // an element of either 16-bit type

struct LinearParts {
  Half *x, *weight;
  float *parts;
  LinearParts(Parts &w, int64_t n, int64_t inputs, int64_t outputs, bool aligned, int sms) : x(nullptr), weight(nullptr), parts(nullptr) {
    if (is_few_rows(n, inputs, outputs)) return; // (read and written as they are)
    const Size size{n, outputs, inputs};
    x = w.take<Half>(aligned ? 0 : n * up8(inputs)), weight = w.take<Half>(aligned ? 0 : outputs * up8(inputs));
    parts = w.take<float>(std::max(part_floats(&size, 1, sms), part_floats(&size, 1, sms, true)));
  }
};
struct LinearGradParts {
  int64_t ld;
  Half *x, *weight, *dz;
  float *bias_sums, *parts;
  LinearGradParts(Parts &w, int64_t n, int64_t inputs, int64_t outputs, bool aligned, int sms)
      : ld(up8(outputs)), x(w.take<Half>(aligned ? 0 : n * up8(inputs))), weight(w.take<Half>(aligned ? 0 : outputs * up8(inputs))),
        dz(w.take<Half>(n * ld)), bias_sums(w.take<float>(tiles_of(n, 32) * ld)),
        parts(nullptr) {
    const Size both[2] = {{n, inputs, outputs}, {outputs, inputs, n}};
    if (n > 0) parts = w.take<float>(std::max({part_floats(both, 2, sms), part_floats(both, 1, sms), part_floats(both + 1, 1, sms)}));
  }
};

// How the scores of a loss are cut: a unit goes through a run of column tiles, as long as every slot still gets
// eight units, so that the last ones end together.
struct LossCut {
  int shape, run, parts; // column tiles of a unit; partial sums of a row
  LossCut(int64_t n, int64_t width, int64_t classes, int sms) {
    const Size size{n, classes, width};
    shape = plan_products(&size, 1, sms, false).shape;
    const int64_t slots = shape == tb::kDenseOne ? sms : sms / 2, cols = tiles_of(classes, tb::dense_cols(shape));
    run = (int)std::clamp<int64_t>(tiles_of(n, tb::dense_rows(shape)) * cols / (8 * slots), 1, 8);
    parts = 4 * (int)tiles_of(cols, run);
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

// Classes of a piece of dz, which is about 256 MB: enough tiles to fill the multiprocessors evenly.
int64_t piece_classes(int64_t n, int64_t classes) {
  const int64_t fits = ((int64_t)128 << 20) / std::max<int64_t>(1, n) / 256 * 256;
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
      if (n > 0) {
        const Size both[2] = {{n, width, now}, {now, width, n}};
        most = std::max({most, part_floats(both, 2, sms), part_floats(both, 1, sms), part_floats(both + 1, 1, sms)});
      }
    parts = w.take<float>(most);
  }
};

} // namespace

extern "C" {

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
  TRY(check_matrix("x", x, ld_x, n, inputs, 2));
  TRY(check_matrix("weight", weight, ld_w, outputs, inputs, 2));
  if (residual) TRY(check_matrix("residual", residual, ld_res, n, outputs, 2));
  TRY(check_matrix("out", out, ld_out, n, outputs, 2));
  if (pre) TRY(check_matrix("pre", pre, ld_pre, n, outputs, 2));
  TRY(check_address("bias", bias, 2));
  if (n == 0) return TBK_OK;
  TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    const int sms = multiprocessors(device);
    if (is_few_rows(n, inputs, outputs)) return few_rows<T>((const T *)x, ld_x, (const T *)weight, ld_w, (const T *)bias, act, (const T *)residual, ld_res, (T *)out, ld_out, (T *)pre,
                                              ld_pre, (int)n, (int)inputs, (int)outputs, sms, stream);
    Parts w{(unsigned char *)ws};
    LinearParts parts(w, n, inputs, outputs, aligned, sms);
    tb::PrepareJobs<T> before = no_jobs<T>();
    make_readable(&before, 0, &x, &ld_x, n, inputs, parts.x);
    make_readable(&before, 1, &weight, &ld_w, outputs, inputs, parts.weight);
    TRY(prepare(before, TBK_ACT_IDENTITY, stream));
    Product<T> product{{x, ld_x, false}, {weight, ld_w, false}, {n, outputs, inputs}, {}};
    TRY(set_result<T>(&product.end, out, ld_out, n, outputs, residual, ld_res, pre, ld_pre));
    product.end.bias = (const T *)bias, product.end.vec_bias = vec_rows(bias, 0);
    product.end.act = act;
    return products<T>(&product, 1, {}, parts.parts, sms, stream);
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
  TRY(check_matrix("grad", grad, ld_grad, n, outputs, 2));
  TRY(check_matrix("x", x, ld_x, n, inputs, 2));
  TRY(check_matrix("weight", weight, ld_w, outputs, inputs, 2));
  if (act != TBK_ACT_IDENTITY) TRY(check_matrix("pre", pre, ld_pre, n, outputs, 2));
  if (skip) TRY(check_matrix("skip", skip, ld_skip, n, inputs, 2));
  if (grad_x) TRY(check_matrix("grad_x", grad_x, ld_gx, n, inputs, 2));
  if (grad_w) TRY(check_matrix("grad_weight", grad_w, ld_gw, outputs, inputs, 2));
  TRY(check_address("grad_bias", grad_b, 2));
  if (outputs > 1 << 24) return fail(TBK_ERR_UNSUPPORTED, "linear_backward: %lld outputs", (long long)outputs);
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
    tb::PrepareJobs<T> before = no_jobs<T>();
    if (grad_w) make_readable(&before, 0, &x, &ld_x, n, inputs, parts.x);
    if (grad_x) make_readable(&before, 1, &weight, &ld_w, outputs, inputs, parts.weight);
    before.grad = (const T *)grad, before.ld_grad = ld_grad, before.vec_grad = vec_rows(grad, ld_grad);
    before.pre = (const T *)pre, before.ld_pre = ld_pre, before.vec_pre = vec_rows(pre, ld_pre);
    before.dz = dz, before.ld_dz = parts.ld, before.bias_sums = grad_b ? parts.bias_sums : nullptr;
    before.rows = (int)n, before.cols = (int)outputs;
    before.row_blocks = (unsigned)tiles_of(n, 32);
    before.blocks[1] = before.row_blocks * (unsigned)tiles_of(outputs, 256);
    TRY(prepare(before, act, stream));
    ColumnSums<T> sums;
    if (grad_b) sums = {parts.bias_sums, tiles_of(n, 32), parts.ld, outputs, (T *)grad_b, nullptr};
    Product<T> list[2];
    int count = 0;
    if (grad_x) {
      Product<T> &q = list[count++];
      q.a = {dz, parts.ld, false}, q.b = {weight, ld_w, true}, q.size = {n, inputs, outputs};
      TRY(set_result<T>(&q.end, grad_x, ld_gx, n, inputs, skip, ld_skip, nullptr, 0));
    }
    if (grad_w) {
      Product<T> &q = list[count++];
      q.a = {dz, parts.ld, true}, q.b = {x, ld_x, true}, q.size = {outputs, inputs, n};
      TRY(set_result<T>(&q.end, grad_w, ld_gw, outputs, inputs, nullptr, 0, nullptr, 0));
    }
    return products<T>(list, count, sums, parts.parts, sms, stream);
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
  TRY(check_address("labels", labels, label_bytes));
  return TBK_OK;
}

int tbk_class_loss(const void *x, int64_t ld_x, const void *weight, int64_t ld_w, const void *bias, const void *labels, int32_t label_bytes,
                   float *loss, float *lse, int64_t n, int64_t width, int64_t classes, int32_t type, void *ws, uint64_t ws_bytes,
                   int32_t device, void *stream_) {
  uint64_t need = 0;
  const bool aligned = tma_rows(x, ld_x, n) && tma_rows(weight, ld_w, classes);
  TRY(tbk_class_loss_workspace(n, width, classes, type, aligned, device, &need));
  TRY(check_matrix("x", x, ld_x, n, width, 2));
  TRY(check_matrix("weight", weight, ld_w, classes, width, 2));
  TRY(check_labels(labels, label_bytes, n));
  if (n > 0 && (!loss || !lse)) return fail(TBK_ERR_INVALID, "null output pointer");
  TRY(check_address("bias", bias, 2));
  TRY(check_address("loss", loss, 4));
  TRY(check_address("lse", lse, 4));
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
    tb::PrepareJobs<T> before = no_jobs<T>();
    make_readable(&before, 0, &x, &ld_x, n, width, parts.x);
    make_readable(&before, 1, &weight, &ld_w, classes, width, parts.weight);
    TRY(prepare(before, TBK_ACT_IDENTITY, stream));
    const Side a{x, ld_x, false}, b{weight, ld_w, false};
    auto scores = [&](auto cols) {
      using End = tb::LseEnd<T, decltype(cols)::value>;
      tb::DenseJobs<End, 1> jobs;
      TRY(set_problem<T>(&jobs.p[0], parts.cut.shape, a, b, {n, classes, width}, 1, parts.cut.run));
      jobs.end[0] = {(const T *)bias, labels, label_bytes, parts.part, parts.at};
      return launch_jobs<T, End, 1>(parts.cut.shape, jobs, sms, stream);
    };
    if (parts.cut.shape == tb::kDenseOne) TRY(scores(std::integral_constant<int, 32>()));
    else TRY(scores(std::integral_constant<int, 64>()));
    return launch(tb::tb_loss_join_kernel, (unsigned)tiles_of(n, 32), 32 * (unsigned)std::clamp(parts.cut.parts / 4, 1, tb::kJoinWarps), 0, stream, 1, parts.part, parts.cut.parts, parts.at, labels, label_bytes, classes, loss,
                  lse, n);
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
  TRY(check_matrix("x", x, ld_x, n, width, 2));
  TRY(check_matrix("weight", weight, ld_w, classes, width, 2));
  TRY(check_labels(labels, label_bytes, n));
  if (n > 0 && (!grad || !lse)) return fail(TBK_ERR_INVALID, "null input pointer");
  TRY(check_address("bias", bias, 2));
  TRY(check_address("grad_bias", grad_b, 2));
  TRY(check_address("grad_loss", grad, 4));
  TRY(check_address("lse", lse, 4));
  if (grad_x) TRY(check_matrix("grad_x", grad_x, ld_gx, n, width, 2));
  if (grad_w) TRY(check_matrix("grad_weight", grad_w, ld_gw, classes, width, 2));
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
    tb::PrepareJobs<T> before = no_jobs<T>();
    make_readable(&before, 0, &x, &ld_x, n, width, parts.x);
    make_readable(&before, 1, &weight, &ld_w, classes, width, parts.weight);
    before.weights = grad, before.num_weights = n, before.scale = parts.scale;
    before.labels = labels, before.label_bytes = label_bytes, before.classes = classes;
    before.blocks[0] = 1;
    TRY(prepare(before, TBK_ACT_IDENTITY, stream));
    const T *W = (const T *)weight;
    T *dz = (T *)parts.dz;
    const int64_t ld = parts.piece;
    for (int64_t v = 0; v < classes; v += ld) {
      const int64_t now = std::min(ld, classes - v);
      const Side xs{x, ld_x, false}, ws_{W + v * ld_w, ld_w, false};
      const T *b = bias ? (const T *)bias + v : nullptr;
      float *sums = grad_b ? parts.bias_sums : nullptr;
      CUtensorMap dz_map;
      TRY(out_map<T>(&dz_map, dz, n, now, ld));
      const Size size{n, now, width};
      const int shape = plan_products(&size, 1, sms, false).shape;
      auto gradients = [&](auto cols) {
        using End = tb::ScoreGradEnd<T, decltype(cols)::value>;
        tb::DenseJobs<End, 1> jobs;
        TRY(set_problem<T>(&jobs.p[0], shape, xs, ws_, size, 1, 1));
        jobs.end[0] = {dz_map, b, labels, label_bytes, grad, lse, parts.scale, ld, v, classes, sums};
        return launch_jobs<T, End, 1>(shape, jobs, sms, stream);
      };
      if (shape == tb::kDenseOne) TRY(gradients(std::integral_constant<int, 32>()));
      else TRY(gradients(std::integral_constant<int, 64>()));
      ColumnSums<T> column_sums;
      if (grad_b) column_sums = {parts.bias_sums, tiles_of(n, 32), ld, now, (T *)grad_b + v, parts.scale};
      Product<T> list[2];
      int count = 0;
      if (grad_x) {
        Product<T> &q = list[count++];
        q.a = {dz, ld, false}, q.b = {W + v * ld_w, ld_w, true}, q.size = {n, width, now};
        TRY(set_result<T>(&q.end, grad_x, ld_gx, n, width, nullptr, 0, nullptr, 0));
        q.end.scale = parts.scale;
        if (ld < classes) { // (several pieces)
          q.end.sums = parts.sums, q.end.ld_sums = parts.ld_sums;
          q.end.first = v == 0, q.end.last = v + now == classes;
        }
      }
      if (grad_w) {
        Product<T> &q = list[count++];
        T *to = (T *)grad_w + v * ld_gw;
        q.a = {dz, ld, true}, q.b = {x, ld_x, true}, q.size = {now, width, n};
        TRY(set_result<T>(&q.end, to, ld_gw, now, width, nullptr, 0, nullptr, 0));
        q.end.scale = parts.scale;
      }
      TRY(products<T>(list, count, column_sums, parts.parts, sms, stream));
    }
    return (int)TBK_OK;
  });
}

int leaf_sum_status(int *word); // (leaf_sum.cu)

int tbk_leaf_check_status(int32_t device) {
  OnDevice on(device);
  CUDA_TRY(on.error);
  int dense = 0, leaf = 0, zero = 0;
  CUDA_TRY(cudaDeviceSynchronize()); // (copies of symbols wait for no stream that was made non-blocking)
  CUDA_TRY(cudaMemcpyFromSymbol(&dense, tb::tb_dense_status, sizeof dense));
  if (dense) CUDA_TRY(cudaMemcpyToSymbol(tb::tb_dense_status, &zero, sizeof zero));
  TRY(leaf_sum_status(&leaf));
  if (!dense && !leaf) return TBK_OK;
  return fail(TBK_ERR_DEVICE_WAIT, "a wait inside a %s gave up", dense ? "matrix product" : "leaf sum");
}

} // extern "C"
