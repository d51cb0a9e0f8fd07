// C ABI of the operators behind a forest's leaves (include/tbk_leaf.h): checks, plans, launches.
#include "../../include/tbk_leaf.h"
#include "dense_simple.cuh"
#include "last_error.h"

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>
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

constexpr int64_t kMost = 0x7fffffff; // of every size

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

template <class F> int with_type(int32_t type, F f) {
  switch (type) {
  case TBK_TYPE_F32: return f(float());
  case TBK_TYPE_F16: return f(__half());
  default: return f(__nv_bfloat16());
  }
}
template <class F> int with_half(int32_t type, F f) { return type == TBK_TYPE_F16 ? f(__half()) : f(__nv_bfloat16()); }

// C[m, n] = sum_k A[m, k] B[n, k], then `end`
template <class T, class End>
int product(tb::Operand<T> a, tb::Operand<T> b, int64_t m, int64_t n, int64_t k, const End &end, cudaStream_t stream) {
  const dim3 grid((unsigned)tiles_of(n, 64), (unsigned)tiles_of(m, 64));
  if (grid.y > 65535) return fail(TBK_ERR_UNSUPPORTED, "too many rows");
  tb::tb_product_kernel<T, End><<<grid, 256, 0, stream>>>(a, b, m, n, k, end);
  CUDA_TRY(cudaGetLastError());
  return TBK_OK;
}

struct LossParts {
  float2 *part;
  float *at;
  LossParts(Parts &w, int64_t n, int64_t classes) : part(w.take<float2>((uint64_t)n * tiles_of(classes, 64))), at(w.take<float>(n)) {}
};

// Classes of a piece of dz: about 64 MB, so that a piece that has just been written is read from L2.
int64_t piece_classes(int64_t n, int64_t classes) {
  const int64_t fits = ((int64_t)32 << 20) / std::max<int64_t>(1, n) / 256 * 256;
  return std::min((classes + 7) / 8 * 8, std::max<int64_t>(256, fits));
}
struct LossGradParts {
  int64_t piece;
  float *scale;
  unsigned char *dz;
  float *bias_sums, *sums;
  LossGradParts(Parts &w, int64_t n, int64_t width, int64_t classes)
      : piece(piece_classes(n, classes)), scale(w.take<float>(1)), dz(w.take<unsigned char>((uint64_t)n * piece * 2)),
        bias_sums(w.take<float>(tiles_of(n, 64) * piece)), sums(w.take<float>(piece < classes ? n * width : 0)) {}
};
struct LinearGradParts {
  int64_t ld;
  unsigned char *dz;
  float *bias_sums;
  LinearGradParts(Parts &w, int64_t n, int64_t outputs)
      : ld((outputs + 7) / 8 * 8), dz(w.take<unsigned char>((uint64_t)n * ld * 2)), bias_sums(w.take<float>(tiles_of(n, 64) * ld)) {}
};

} // namespace

extern "C" {

int tbk_leaf_map_create(const tbk_forest_arrays *fa, int32_t device, tbk_leaf_map **out) {
  if (!out) return fail(TBK_ERR_INVALID, "null argument");
  *out = nullptr;
  if (!fa || !fa->tree_off || !fa->left) return fail(TBK_ERR_INVALID, "null forest array");
  if (fa->num_trees < 1 || fa->num_trees > kMost) return fail(TBK_ERR_INVALID, "a leaf map needs a tree at least");
  if (fa->tree_off[0] != 0) return fail(TBK_ERR_INVALID, "tree_off does not begin with 0");
  for (int64_t t = 0; t < fa->num_trees; ++t)
    if (fa->tree_off[t + 1] <= fa->tree_off[t] || fa->tree_off[t + 1] - fa->tree_off[t] > kMost) return fail(TBK_ERR_INVALID, "tree %lld has no nodes, or too many", (long long)t);
  try {
    std::unique_ptr<tbk_leaf_map> map(new tbk_leaf_map);
    const int64_t trees = fa->num_trees, nodes = fa->tree_off[trees];
    std::vector<long long> tree_off(fa->tree_off, fa->tree_off + trees + 1);
    std::vector<int32_t> node_row((size_t)nodes), row_off((size_t)trees + 1);
    int64_t rows = 0;
    for (int64_t t = 0; t < trees; ++t) {
      row_off[t] = (int32_t)rows;
      for (int64_t i = tree_off[t]; i < tree_off[t + 1]; ++i) node_row[i] = fa->left[i] < 0 ? (int32_t)rows++ : -1;
      if (rows > kMost) return fail(TBK_ERR_UNSUPPORTED, "more than %lld leaves", (long long)kMost);
      map->max_rows = std::max<int64_t>(map->max_rows, rows - row_off[t]);
    }
    row_off[trees] = (int32_t)rows;
    map->device = device;
    map->rows = rows;
    const size_t a = tree_off.size() * 8, b = (node_row.size() * 4 + 15) / 16 * 16, c = row_off.size() * 4;
    OnDevice on(device);
    CUDA_TRY(on.error);
    CUDA_TRY(cudaMalloc(&map->mem, a + 16 + b + c));
    unsigned char *p = static_cast<unsigned char *>(map->mem), *pb = p + (a + 15) / 16 * 16, *pc = pb + b;
    map->view = {reinterpret_cast<long long *>(p), reinterpret_cast<int32_t *>(pb), reinterpret_cast<int32_t *>(pc), trees};
    cudaError_t e = cudaMemcpy(p, tree_off.data(), a, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemcpy(pb, node_row.data(), node_row.size() * 4, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemcpy(pc, row_off.data(), c, cudaMemcpyHostToDevice);
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

int tbk_leaf_sum(const tbk_leaf_map *map, const int32_t *ids, int64_t n, int64_t ld_ids, const void *table, int64_t ld_table,
                 int64_t width, int32_t type, void *out, int64_t ld_out, void *stream) {
  TRY(check_leaf_call(map, ids, n, ld_ids, width, type));
  TRY(check_matrix("table", table, ld_table, map->rows, width));
  TRY(check_matrix("out", out, ld_out, n, width));
  if (n == 0) return TBK_OK;
  OnDevice on(map->device);
  CUDA_TRY(on.error);
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    tb::tb_leaf_sum_kernel<T><<<(unsigned)n, (unsigned)std::min<int64_t>(256, (width + 31) / 32 * 32), 0, (cudaStream_t)stream>>>(
        map->view, ids, ld_ids, (const T *)table, ld_table, width, (T *)out, ld_out, n);
    CUDA_TRY(cudaGetLastError());
    return (int)TBK_OK;
  });
}

int tbk_leaf_sum_backward_workspace(const tbk_leaf_map *map, int64_t n, int64_t width, int32_t type, uint64_t *bytes) {
  if (!map || !bytes) return fail(TBK_ERR_INVALID, "null argument");
  (void)type;
  TRY(check_sizes("leaf sum", n, width, 1));
  *bytes = (uint64_t)map->rows * width * 4;
  return TBK_OK;
}

int tbk_leaf_sum_backward(const tbk_leaf_map *map, const int32_t *ids, int64_t n, int64_t ld_ids, const void *grad, int64_t ld_grad,
                          int64_t width, int32_t type, void *out, int64_t ld_out, void *ws, uint64_t ws_bytes, void *stream) {
  TRY(check_leaf_call(map, ids, n, ld_ids, width, type));
  TRY(check_matrix("grad", grad, ld_grad, n, width));
  TRY(check_matrix("out", out, ld_out, map->rows, width));
  uint64_t need = 0;
  TRY(tbk_leaf_sum_backward_workspace(map, n, width, type, &need));
  TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(map->device);
  CUDA_TRY(on.error);
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    tb::tb_leaf_grad_kernel<T><<<dim3((unsigned)map->view.num_trees, (unsigned)tiles_of(width, 32)), 32, 0, (cudaStream_t)stream>>>(
        map->view, ids, ld_ids, (const T *)grad, ld_grad, width, (float *)ws, (T *)out, ld_out, n);
    CUDA_TRY(cudaGetLastError());
    return (int)TBK_OK;
  });
}

int tbk_linear_workspace(int64_t n, int64_t inputs, int64_t outputs, int32_t type, int32_t device, uint64_t *bytes) {
  if (!bytes) return fail(TBK_ERR_INVALID, "null argument");
  (void)device;
  TRY(half_type(type, "linear"));
  TRY(check_sizes("linear", n, inputs, outputs));
  *bytes = 0;
  return TBK_OK;
}

int tbk_linear(const void *x, int64_t ld_x, const void *weight, int64_t ld_w, const void *bias, int32_t act, const void *residual,
               int64_t ld_res, void *out, int64_t ld_out, void *pre, int64_t ld_pre, int64_t n, int64_t inputs, int64_t outputs,
               int32_t type, void *ws, uint64_t ws_bytes, int32_t device, void *stream) {
  uint64_t need = 0;
  TRY(tbk_linear_workspace(n, inputs, outputs, type, device, &need));
  if (act < TBK_ACT_IDENTITY || act > TBK_ACT_SILU) return fail(TBK_ERR_INVALID, "unknown activation %d", act);
  TRY(check_matrix("x", x, ld_x, n, inputs));
  TRY(check_matrix("weight", weight, ld_w, outputs, inputs));
  if (residual) TRY(check_matrix("residual", residual, ld_res, n, outputs));
  TRY(check_matrix("out", out, ld_out, n, outputs));
  if (pre) TRY(check_matrix("pre", pre, ld_pre, n, outputs));
  TRY(check_workspace(ws, ws_bytes, need));
  if (n == 0) return TBK_OK;
  OnDevice on(device);
  CUDA_TRY(on.error);
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    const tb::LinearEnd<T> end{(const T *)bias, (const T *)residual, ld_res, (T *)out, (T *)pre, ld_out, ld_pre, act};
    return product<T>({(const T *)x, ld_x, 1}, {(const T *)weight, ld_w, 1}, n, outputs, inputs, end, (cudaStream_t)stream);
  });
}

int tbk_linear_backward_workspace(int64_t n, int64_t inputs, int64_t outputs, int32_t type, int32_t device, uint64_t *bytes) {
  if (!bytes) return fail(TBK_ERR_INVALID, "null argument");
  (void)device;
  TRY(half_type(type, "linear_backward"));
  TRY(check_sizes("linear_backward", n, inputs, outputs));
  Parts w{nullptr};
  LinearGradParts parts(w, n, outputs);
  *bytes = w.used;
  return TBK_OK;
}

int tbk_linear_backward(const void *grad, int64_t ld_grad, const void *x, int64_t ld_x, const void *weight, int64_t ld_w, const void *pre,
                        int64_t ld_pre, int32_t act, const void *skip, int64_t ld_skip, void *grad_x, int64_t ld_gx, void *grad_w,
                        int64_t ld_gw, void *grad_b, int64_t n, int64_t inputs, int64_t outputs, int32_t type, void *ws, uint64_t ws_bytes, int32_t device, void *stream_) {
  uint64_t need = 0;
  TRY(tbk_linear_backward_workspace(n, inputs, outputs, type, device, &need));
  if (act < TBK_ACT_IDENTITY || act > TBK_ACT_SILU) return fail(TBK_ERR_INVALID, "unknown activation %d", act);
  TRY(check_matrix("grad", grad, ld_grad, n, outputs));
  TRY(check_matrix("x", x, ld_x, n, inputs));
  TRY(check_matrix("weight", weight, ld_w, outputs, inputs));
  if (act != TBK_ACT_IDENTITY) TRY(check_matrix("pre", pre, ld_pre, n, outputs));
  if (skip) TRY(check_matrix("skip", skip, ld_skip, n, inputs));
  if (grad_x) TRY(check_matrix("grad_x", grad_x, ld_gx, n, inputs));
  if (grad_w) TRY(check_matrix("grad_weight", grad_w, ld_gw, outputs, inputs));
  TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    Parts w{(unsigned char *)ws};
    LinearGradParts parts(w, n, outputs);
    T *dz = (T *)parts.dz;
    if (n > 0) {
      tb::tb_act_grad_kernel<T><<<dim3((unsigned)tiles_of(outputs, 128), (unsigned)tiles_of(n, 64)), 128, 0, stream>>>(
          (const T *)grad, ld_grad, (const T *)pre, ld_pre, act, dz, parts.ld, grad_b ? parts.bias_sums : nullptr, n, outputs);
      CUDA_TRY(cudaGetLastError());
    }
    if (grad_b) {
      tb::tb_column_sum_kernel<T><<<(unsigned)tiles_of(outputs, 128), 128, 0, stream>>>(parts.bias_sums, tiles_of(n, 64), parts.ld, (T *)grad_b, outputs);
      CUDA_TRY(cudaGetLastError());
    }
    if (grad_x && n > 0)
      TRY((product<T, tb::SumEnd<T>>({dz, parts.ld, 1}, {(const T *)weight, 1, ld_w}, n, inputs, outputs,
                                     {nullptr, 0, (T *)grad_x, ld_gx, (const T *)skip, ld_skip, nullptr, true, true}, stream)));
    if (grad_w)
      TRY((product<T, tb::SumEnd<T>>({dz, 1, parts.ld}, {(const T *)x, 1, ld_x}, outputs, inputs, n,
                                     {nullptr, 0, (T *)grad_w, ld_gw, nullptr, 0, nullptr, true, true}, stream)));
    return (int)TBK_OK;
  });
}

int tbk_class_loss_workspace(int64_t n, int64_t width, int64_t classes, int32_t type, int32_t device, uint64_t *bytes) {
  if (!bytes) return fail(TBK_ERR_INVALID, "null argument");
  (void)device;
  TRY(half_type(type, "class_loss"));
  TRY(check_sizes("class_loss", n, width, classes));
  Parts w{nullptr};
  LossParts parts(w, n, classes);
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
  TRY(tbk_class_loss_workspace(n, width, classes, type, device, &need));
  TRY(check_matrix("x", x, ld_x, n, width));
  TRY(check_matrix("weight", weight, ld_w, classes, width));
  TRY(check_labels(labels, label_bytes, n));
  if (n > 0 && (!loss || !lse)) return fail(TBK_ERR_INVALID, "null output pointer");
  TRY(check_workspace(ws, ws_bytes, need));
  if (n == 0) return TBK_OK;
  OnDevice on(device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    Parts w{(unsigned char *)ws};
    LossParts parts(w, n, classes);
    const tb::LseEnd<T> end{(const T *)bias, labels, label_bytes, parts.part, parts.at, n};
    TRY(product<T>({(const T *)x, ld_x, 1}, {(const T *)weight, ld_w, 1}, n, classes, width, end, stream));
    tb::tb_loss_join_kernel<<<(unsigned)tiles_of(n, 128), 128, 0, stream>>>(parts.part, tiles_of(classes, 64), parts.at, labels, label_bytes, classes, loss, lse, n);
    CUDA_TRY(cudaGetLastError());
    return (int)TBK_OK;
  });
}

int tbk_class_loss_backward_workspace(int64_t n, int64_t width, int64_t classes, int32_t type, int32_t device, uint64_t *bytes) {
  if (!bytes) return fail(TBK_ERR_INVALID, "null argument");
  (void)device;
  TRY(half_type(type, "class_loss_backward"));
  TRY(check_sizes("class_loss_backward", n, width, classes));
  Parts w{nullptr};
  LossGradParts parts(w, n, width, classes);
  *bytes = w.used;
  return TBK_OK;
}

int tbk_class_loss_backward(const float *grad, const void *x, int64_t ld_x, const void *weight, int64_t ld_w, const void *bias,
                            const void *labels, int32_t label_bytes, const float *lse, void *grad_x, int64_t ld_gx, void *grad_w,
                            int64_t ld_gw, void *grad_b, int64_t n, int64_t width, int64_t classes, int32_t type, void *ws,
                            uint64_t ws_bytes, int32_t device, void *stream_) {
  uint64_t need = 0;
  TRY(tbk_class_loss_backward_workspace(n, width, classes, type, device, &need));
  TRY(check_matrix("x", x, ld_x, n, width));
  TRY(check_matrix("weight", weight, ld_w, classes, width));
  TRY(check_labels(labels, label_bytes, n));
  if (n > 0 && (!grad || !lse)) return fail(TBK_ERR_INVALID, "null input pointer");
  if (grad_x) TRY(check_matrix("grad_x", grad_x, ld_gx, n, width));
  if (grad_w) TRY(check_matrix("grad_weight", grad_w, ld_gw, classes, width));
  TRY(check_workspace(ws, ws_bytes, need));
  OnDevice on(device);
  CUDA_TRY(on.error);
  cudaStream_t stream = (cudaStream_t)stream_;
  return with_half(type, [&](auto t) {
    using T = decltype(t);
    Parts w{(unsigned char *)ws};
    LossGradParts parts(w, n, width, classes);
    const T *W = (const T *)weight;
    T *dz = (T *)parts.dz;
    const int64_t ld = parts.piece;
    if (n > 0) {
      tb::tb_scale_kernel<<<1, 1024, 0, stream>>>(grad, n, parts.scale);
      CUDA_TRY(cudaGetLastError());
    }
    for (int64_t v = 0; v < classes; v += ld) {
      const int64_t now = std::min(ld, classes - v);
      if (n > 0)
        TRY((product<T, tb::ScoreGradEnd<T>>({(const T *)x, ld_x, 1}, {W + v * ld_w, ld_w, 1}, n, now, width,
                                             {(const T *)bias, labels, label_bytes, grad, lse, parts.scale, dz, ld, v, classes,
                                              grad_b ? parts.bias_sums : nullptr}, stream)));
      if (grad_b) {
        tb::tb_column_sum_kernel<T><<<(unsigned)tiles_of(now, 128), 128, 0, stream>>>(parts.bias_sums, tiles_of(n, 64), ld, (T *)grad_b + v, now);
        CUDA_TRY(cudaGetLastError());
      }
      if (grad_x && n > 0)
        TRY((product<T, tb::SumEnd<T>>({dz, ld, 1}, {W + v * ld_w, 1, ld_w}, n, width, now,
                                       {parts.sums, width, (T *)grad_x, ld_gx, nullptr, 0, parts.scale, v == 0, v + now == classes}, stream)));
      if (grad_w)
        TRY((product<T, tb::SumEnd<T>>({dz, 1, ld}, {(const T *)x, 1, ld_x}, now, width, n,
                                       {nullptr, 0, (T *)grad_w + v * ld_gw, ld_gw, nullptr, 0, n > 0 ? parts.scale : nullptr, true, true}, stream)));
    }
    return (int)TBK_OK;
  });
}

} // extern "C"
