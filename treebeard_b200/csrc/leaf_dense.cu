// C ABI of the linear layers and the class loss (include/tbk_leaf.h): plans, launches.
#include "../../include/tbk_leaf.h"
#include "dense.cuh"
#include "leaf_api.h"

#include <cudaTypedefs.h>
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace {

int half_type(int32_t type, const char *what) {
  if (type == TBK_TYPE_F16 || type == TBK_TYPE_BF16) return TBK_OK;
  if (type == TBK_TYPE_F32) return fail(TBK_ERR_UNSUPPORTED, "%s takes 16-bit floating point types (fp16, bf16)", what);
  return fail(TBK_ERR_INVALID, "unknown element type %d", type);
}

template <class F> int with_half(int32_t type, F f) { return type == TBK_TYPE_F16 ? f(__half()) : f(__nv_bfloat16()); }

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
  tb::tb_align_rows_kernel<T><<<(unsigned)std::min<int64_t>(tiles_of(rows * (up8(cols) / 8), 256), 1 << 16), 256, 0, stream>>>((const T *)*p, *ld, room, up8(cols), rows, cols);
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
    if (grad_w) TRY(readable(&x, &ld_x, n, inputs, (T *)parts.x, stream));
    if (grad_x) TRY(readable(&weight, &ld_w, outputs, inputs, (T *)parts.weight, stream));
    tb::tb_act_grad_kernel<T><<<dim3((unsigned)tiles_of(n, 32), (unsigned)tiles_of(outputs, 256)), 256, 0, stream>>>(
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
    tb::tb_loss_join_kernel<<<(unsigned)tiles_of(n, 32), 32 * tb::kJoinWarps, 0, stream>>>(parts.part, parts.cut.parts, parts.at, labels, label_bytes, classes, loss, lse, n);
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
