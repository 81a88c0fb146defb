/* clid_dense.h -- C ABI of the dense operators in libclid_native.so: a layer of a decoder of ANY width (matrix product, bias,
 * activation, residual), the softmax cross entropy of a class head without its logits, and the class of each row.
 *
 * They serve what the fixed 11 -> 64 -> 1 kernels of clid_native.h refuse: Decoder.mlp / sem_label_prob of the reference
 * (model/decoder.py:58-95) at other widths, depths and output counts, and Mesher.query_points(query_sem=True)
 * (utils/mesher.py:38-163).
 *
 * Conventions as in clid_native.h: device pointers borrowed for the call, everything enqueued on `stream` (a hipStream_t of the
 * CURRENT device), nothing allocated, nothing synchronised, 0 or a negative CLID_E_* with clid_last_error().
 *   - a matrix is rows of `ld` elements (ld >= its columns), columns contiguous; weights are [n][k] as nn.Linear has them;
 *   - dtype (CLID_F32 / CLID_BF16 / CLID_F16) is that of x, w, bias, residual, y and of the gradients; sums, softmax statistics,
 *     losses and log-probabilities are fp32;
 *   - `ws` has at least clid_*_workspace() bytes, 256-byte aligned, and holds nothing between calls;
 *   - rows >= 0, k >= 1, n >= 1, each matrix at most 2^40 elements; rows < 2^31, k, n < 2^20.
 *
 * Workspaces grow with the rows where n or k is over 64 and there are more than 32 rows: copies of operands that are not 16-bit rows of
 * whole aligned 16 bytes (fp32: 6 bytes a value; the cross entropy always copies its rows); a layer's backward pass its dz (2 bytes a
 * value, fp32 6); a class head's statistics 12 bytes (label) or 8 (cross entropy) a row for every 32 or 64 classes.  The cross entropy's backward
 * pass holds dz of a piece of the classes: at most about 512 MB, but never under 256 classes, that is 512 bytes a row (fp32: 1536) from 1 M
 * rows (350 k) on, and with more than one piece 4 k bytes a row for dx's sums.  A product whose k is cut adds 4 bytes a result and part.
 */
#ifndef CLID_DENSE_H
#define CLID_DENSE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CLID_F32 0
#define CLID_BF16 1
#define CLID_F16 2

#define CLID_ACT_NONE 0
#define CLID_ACT_RELU 1
#define CLID_ACT_LEAKY_RELU 2 /* slope 0.01, torch.nn.functional.leaky_relu's default (model/decoder.py:66) */
#define CLID_ACT_GELU 3       /* z Phi(z), the erf form */
#define CLID_ACT_SILU 4       /* z / (1 + exp(-z)) */

/* y = act(x w^T + bias) + residual.  z_out (may be NULL): x w^T + bias for the backward pass, in fp32 or, where dtype has 16 bits, in
 * fp16 (also for bf16: a slope needs the bits more than the range) -- nearest, except that a non-zero z never becomes 0 and a finite
 * one never becomes infinite, so that its activation's slope stays the right one. */
typedef struct clid_linear_args {
  const void *x, *w, *bias, *residual; /* [rows][k], [n][k], [n] or NULL, [rows][n] or NULL */
  void *y, *z_out;                     /* [rows][n], [rows][n] or NULL (both dense: ld = n) */
  int64_t ldx, ldw, ldr;
  int64_t rows;
  int32_t k, n, dtype, act;
  void* ws;
  int64_t ws_bytes;
} clid_linear_args;
int64_t clid_linear_workspace(const clid_linear_args* a);
int clid_linear_fwd(const clid_linear_args* a, void* stream);

/* dz = dy act'(z) (relu: dy where not z <= 0, else 0), dx = dz w, dw = dz^T x, db = sum over rows of dz.  z (dense) is z_out of the forward call, or with
 * z_is_y (relu and leaky_relu without a residual) its y, whose sign is z's; NULL for CLID_ACT_NONE.  dx, dw, db: NULL where not wanted.
 * dz is rounded to dtype between the products (fp32: not at all). */
typedef struct clid_linear_bwd_args {
  const void *x, *w, *dy, *z;
  void *dx, *dw, *db; /* dense: [rows][k], [n][k], [n] */
  int64_t ldx, ldw, lddy;
  int64_t rows;
  int32_t k, n, dtype, act, z_is_y, reserved;
  void* ws;
  int64_t ws_bytes;
} clid_linear_bwd_args;
int64_t clid_linear_bwd_workspace(const clid_linear_bwd_args* a);
int clid_linear_bwd(const clid_linear_bwd_args* a, void* stream);

/* Softmax cross entropy of z = x w^T + bias against target, never storing z.  A row whose target is ignore_index has loss 0, no
 * gradient, and what its x holds (NaN, infinities) reaches nothing.  A target outside [0, n) that is not ignore_index makes its
 * row's loss NaN.
 *   saved     clid_ce_saved() bytes, 256-byte aligned: what the backward pass needs of the forward one (which rows count, their
 *             statistics; never z)
 *   loss_out  [1] (CLID_REDUCE_MEAN: the sum over the counted rows / their number, 0 if there are none; CLID_REDUCE_SUM) or
 *             [rows] (CLID_REDUCE_NONE) fp32
 * Backward: g is dL/dloss_out (fp32, one value or [rows]); saved as the forward call left it. */
#define CLID_REDUCE_NONE 0
#define CLID_REDUCE_MEAN 1
#define CLID_REDUCE_SUM 2
typedef struct clid_ce_args {
  const void *x, *w, *bias; /* [rows][k], [n][k], [n] or NULL */
  const int64_t* target;    /* [rows] */
  void* saved;
  float* loss_out;
  const float* g;     /* backward only */
  void *dx, *dw, *db; /* backward only, dense, NULL where not wanted */
  int64_t ldx, ldw;
  int64_t rows, ignore_index;
  int32_t k, n, dtype, reduction;
  void* ws;
  int64_t ws_bytes;
} clid_ce_args;
int64_t clid_ce_saved(const clid_ce_args* a);
int64_t clid_ce_workspace(const clid_ce_args* a);
int clid_ce_fwd(const clid_ce_args* a, void* stream);
int64_t clid_ce_bwd_workspace(const clid_ce_args* a);
int clid_ce_bwd(const clid_ce_args* a, void* stream);

/* label[m] = the lowest column of the largest z[m] (a NaN counts as largest), log_prob[m] = log softmax(z[m])[label[m]]. */
typedef struct clid_label_args {
  const void *x, *w, *bias;
  int64_t* label;  /* [rows] */
  float* log_prob; /* [rows] */
  int64_t ldx, ldw;
  int64_t rows;
  int32_t k, n, dtype, reserved;
  void* ws;
  int64_t ws_bytes;
} clid_label_args;
int64_t clid_label_workspace(const clid_label_args* a);
int clid_label_fwd(const clid_label_args* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif
