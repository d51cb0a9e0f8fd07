/*
 * tbk_leaf.h -- C ABI of the operators of a second model that stands behind a forest: the leaf of every
 * (row, tree) that tbk_predict_leaf_ids selects picks a row of an embedding table, a row's embeddings are
 * summed, linear layers follow, and a softmax over many classes ends it.  Forward and backward.  The
 * reference stops at the forest's own prediction (src/mlir/LowerToMidLevelIR.cpp:596-648) and has no
 * counterpart.
 *
 * Conventions as in tbk.h: plain pointers and sizes, an int status (TBK_OK = 0), nothing aborts,
 * tbk_last_error() has the message.  Matrices are row-major, `ld_*` elements from row to row (columns lie
 * one behind the other).  All device pointers belong to `device`, which need not be the current one; the
 * current device is left as it was.  Calls are ordered by `stream` and may be captured; nothing is
 * allocated, and nothing is kept between calls but how sizes are cut, which the sizes decide.  A call that asks for a workspace takes device memory of
 * the size that its *_workspace function states, 256-byte aligned, for its own use until its work on the
 * stream is done: calls that may run at the same time need workspaces of their own.
 * `aligned` of these functions: 1 if x and weight begin at 16-byte boundaries and have row strides that are
 * multiples of 8 elements; otherwise every call copies them first, as a whole, and its workspace has room for
 * that (4096 rows of 513 columns, 100003 classes: 442 us, with 512 columns 332).
 * Inputs and outputs of one call must not overlap, except that `out` may be `residual`.
 *
 * Sums are held in fp32 and every output is rounded once from there.  The order of all sums is fixed: equal calls
 * give equal bits.  It depends on sizes and, in tbk_leaf_sum, on strides and alignment too (a table whose rows do not
 * lie one behind the other takes another kernel, which joins other parts).
 */
#ifndef TBK_LEAF_H
#define TBK_LEAF_H

#include "tbk.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of matrices and vectors */
enum { TBK_TYPE_F32 = 0, TBK_TYPE_F16 = 1, TBK_TYPE_BF16 = 2 };

/* activations of a linear layer: z, max(z, 0), z * Phi(z) (Phi: the normal distribution), z / (1 + exp(-z)) */
enum { TBK_ACT_IDENTITY = 0, TBK_ACT_RELU = 1, TBK_ACT_GELU = 2, TBK_ACT_SILU = 3 };

/* Which table row a leaf stands for: the leaves of all trees, numbered tree by tree in the order of their
 * nodes (node numbering of tbk_forest_arrays, the one tbk_predict_leaf_ids answers in).  Only num_trees,
 * tree_off and left of the forest are read. */
typedef struct tbk_leaf_map tbk_leaf_map;
TBK_EXPORT int tbk_leaf_map_create(const tbk_forest_arrays *forest, int32_t device, tbk_leaf_map **out);
TBK_EXPORT int tbk_leaf_map_free(tbk_leaf_map *map);
TBK_EXPORT int64_t tbk_leaf_map_rows(const tbk_leaf_map *map); /* leaves of all trees = rows of a table */

/* out[n, :] = sum over trees t of table[row(t, leaf_ids[n, t]), :].  An id that is no leaf of its tree
 * (negative, an inner node, beyond the tree) adds nothing; a row without any leaf gets zeros.
 * type: any TBK_TYPE_*, of table and out. */
TBK_EXPORT int tbk_leaf_sum_workspace(const tbk_leaf_map *map, int64_t n_rows, int64_t width, int32_t type, uint64_t *bytes);
TBK_EXPORT int tbk_leaf_sum(const tbk_leaf_map *map, const int32_t *leaf_ids, int64_t n_rows, int64_t ld_ids,
                            const void *table, int64_t ld_table, int64_t width, int32_t type, void *out,
                            int64_t ld_out, void *workspace, uint64_t workspace_bytes, void *stream);

/* The gradient of tbk_leaf_sum with respect to the table: out[r, :] = sum of grad[n, :] over the (n, t)
 * with row(t, leaf_ids[n, t]) = r, zeros for leaves that no row reached. */
TBK_EXPORT int tbk_leaf_sum_backward_workspace(const tbk_leaf_map *map, int64_t n_rows, int64_t width, int32_t type,
                                               uint64_t *bytes);
TBK_EXPORT int tbk_leaf_sum_backward(const tbk_leaf_map *map, const int32_t *leaf_ids, int64_t n_rows, int64_t ld_ids,
                                     const void *grad, int64_t ld_grad, int64_t width, int32_t type, void *out,
                                     int64_t ld_out, void *workspace, uint64_t workspace_bytes, void *stream);

/* out = activation(z) + residual, z = x weight^T + bias, and, where pre is given, pre = z.
 * x [n_rows, inputs], weight [outputs, inputs], bias [outputs] or NULL, residual [n_rows, outputs] or NULL.
 * type: TBK_TYPE_F16 or TBK_TYPE_BF16, of all of them. */
TBK_EXPORT int tbk_linear_workspace(int64_t n_rows, int64_t inputs, int64_t outputs, int32_t type, int32_t aligned,
                                    int32_t device, uint64_t *bytes);
TBK_EXPORT int tbk_linear(const void *x, int64_t ld_x, const void *weight, int64_t ld_weight, const void *bias,
                          int32_t activation, const void *residual, int64_t ld_residual, void *out, int64_t ld_out,
                          void *pre, int64_t ld_pre, int64_t n_rows, int64_t inputs, int64_t outputs, int32_t type,
                          void *workspace, uint64_t workspace_bytes, int32_t device, void *stream);

/* Gradients of tbk_linear from grad [n_rows, outputs], the gradient of out (which is also residual's):
 * with dz = grad * activation'(pre), grad_x = dz weight + skip, grad_weight = dz^T x, grad_bias = sum of dz's
 * rows.  skip [n_rows, inputs] or NULL: what else reaches x's gradient, as where x is the residual too (then
 * skip is grad).
 * pre may be NULL with TBK_ACT_IDENTITY; grad_x, grad_weight, grad_bias may each be NULL (not wanted).
 * dz is rounded to `type` before the two products (grad_bias is summed before that), without a scale: in fp16
 * a |dz| above 65504 becomes infinite and one below 6e-5 loses digits, so grad has to come scaled. */
TBK_EXPORT int tbk_linear_backward_workspace(int64_t n_rows, int64_t inputs, int64_t outputs, int32_t type,
                                               int32_t aligned, int32_t device, uint64_t *bytes);
TBK_EXPORT int tbk_linear_backward(const void *grad, int64_t ld_grad, const void *x, int64_t ld_x, const void *weight,
                                   int64_t ld_weight, const void *pre, int64_t ld_pre, int32_t activation,
                                   const void *skip, int64_t ld_skip, void *grad_x, int64_t ld_grad_x, void *grad_weight, int64_t ld_grad_weight,
                                   void *grad_bias, int64_t n_rows, int64_t inputs, int64_t outputs, int32_t type,
                                   void *workspace, uint64_t workspace_bytes, int32_t device, void *stream);

/* Softmax cross entropy over `classes` classes without keeping the scores z = x weight^T + bias:
 * lse[n] = log sum_v exp(z[n, v]), loss[n] = lse[n] - z[n, labels[n]], both fp32.  A label outside
 * 0 .. classes-1 leaves its row out: loss 0.  labels: int64 (label_bytes 8) or int32 (4).  A class whose
 * bias is -inf has probability 0; a row of such classes only has lse = -inf and, with a label, a loss and
 * gradients that are not numbers. */
TBK_EXPORT int tbk_class_loss_workspace(int64_t n_rows, int64_t width, int64_t classes, int32_t type,
                                               int32_t aligned, int32_t device, uint64_t *bytes);
TBK_EXPORT int tbk_class_loss(const void *x, int64_t ld_x, const void *weight, int64_t ld_weight, const void *bias,
                              const void *labels, int32_t label_bytes, float *loss, float *lse, int64_t n_rows,
                              int64_t width, int64_t classes, int32_t type, void *workspace, uint64_t workspace_bytes,
                              int32_t device, void *stream);

/* Gradients of sum_n grad_loss[n] * loss[n] (grad_loss fp32): with dz[n, v] = grad_loss[n] * (exp(z[n, v] -
 * lse[n]) - [v = labels[n]]), grad_x = dz weight, grad_weight = dz^T x, grad_bias = sum of dz's rows; each may
 * be NULL (not wanted).  A row without a label has zeros for dz, which its x is multiplied with: x has to be finite
 * there too.  The scores are computed again, a piece of the classes at a time; dz is rounded to
 * `type`, scaled by a power of two so that the largest |grad_loss| of a row with a label lies near the middle of the
 * type's range (grad_bias is summed before that). */
TBK_EXPORT int tbk_class_loss_backward_workspace(int64_t n_rows, int64_t width, int64_t classes, int32_t type,
                                               int32_t aligned, int32_t device, uint64_t *bytes);
TBK_EXPORT int tbk_class_loss_backward(const float *grad_loss, const void *x, int64_t ld_x, const void *weight,
                                       int64_t ld_weight, const void *bias, const void *labels, int32_t label_bytes,
                                       const float *lse, void *grad_x, int64_t ld_grad_x, void *grad_weight,
                                       int64_t ld_grad_weight, void *grad_bias, int64_t n_rows, int64_t width,
                                       int64_t classes, int32_t type, void *workspace, uint64_t workspace_bytes,
                                       int32_t device, void *stream);

/* Waits for a device and reads the status words of these kernels on it: TBK_ERR_DEVICE_WAIT if a bounded wait inside
 * one gave up since the last check, else TBK_OK.  The words are the device's, and reading clears them: of several
 * threads that use it, the first to ask learns of it.  What the calls since the last check wrote is not to be
 * trusted then. */
TBK_EXPORT int tbk_leaf_check_status(int32_t device);

#ifdef __cplusplus
}
#endif
#endif /* TBK_LEAF_H */
