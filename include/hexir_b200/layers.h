/*
 * hexir_b200/layers.h -- kernel-level C ABI of the layers of a feed-forward
 * block on sm_100a: the linear with bias, activation and residual in its
 * epilogue, its gradients, and layer norm forward and backward.
 *
 * No reference counterpart: the reference's linear is f64 without an
 * epilogue (runtime/src/kernels/reference_kernels.c:3) and its dialect
 * declares the activations without lowering them
 * (include/hexir/Dialect/Hexir/IR/HexirOps.td:189-308).
 *
 * Conventions, as in kernels.h: every call takes the CUDA ordinal its device
 * pointers belong to and a CUstream (NULL = the legacy default stream), is
 * asynchronous, and returns HEXIR_ERROR_* with a message in
 * hexir_cuda_last_error(); hexir_cuda_synchronize reports kernel-side errors.
 * Tensors are row-major with a row stride (ld*, in elements, at least the row
 * length; 0 = dense).  Any strides and sizes are taken and pointers need only
 * their element's alignment; rows that start on 16-byte boundaries (pointer
 * and stride) run the TMA-fed kernels.  No call allocates device memory,
 * synchronises, or keeps state between calls, so all of them can be captured
 * into CUDA graphs and run on any streams at once; where scratch is needed
 * the caller passes it, and calls that may overlap pass different scratch.
 * Results do not depend on timing: every sum has a fixed order.
 *
 * An output may not overlap an input or another output, except that two may
 * be the same tensor (same pointer and stride) where one takes the other's
 * place row by row: y (dx) and residual, dz and dy, a norm's y and x, a
 * norm's dx and dy.  Inputs may overlap each other.
 *
 * The first of these calls on a device loads their device code, which a
 * stream capture does not allow: make one (of any size, an empty one will do)
 * before capturing.
 */
#ifndef HEXIR_B200_LAYERS_H
#define HEXIR_B200_LAYERS_H

#include <stddef.h>
#include <stdint.h>

#include "hexir_b200/kernels.h"
#include "hexir_runtime/status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define HEXIR_DTYPE_F64 0u
#define HEXIR_DTYPE_F32 1u
#define HEXIR_DTYPE_BF16 2u
#define HEXIR_DTYPE_F16 3u

/* Activations of the linear calls: none, relu (the kernel kind number of
 * hexir_runtime/program.h) or an elementwise HEXIR_ACTIVATION_* of kernels.h
 * (softmax, a row operation, is refused).  In f32 inside the kernels. */
#define HEXIR_ACTIVATION_NONE 0u
#define HEXIR_ACTIVATION_RELU 3u /* x > 0 ? x : 0 */

/* flags of the linear calls, for tests: which kernel runs (the call is
 * refused where that kernel cannot run it), over how many CTAs of a cluster
 * the sum is split (1, 2, 4 or 8; single, skinny, guarded), and the columns
 * of a tile (256 or 128 of a pair, 128 or 64 of a single CTA). */
#define HEXIR_LINEAR_FORCE_PAIR 0x100u    /* CTA pairs, 256-row tiles */
#define HEXIR_LINEAR_FORCE_SINGLE 0x200u  /* one CTA, 128-row tiles */
#define HEXIR_LINEAR_FORCE_SKINNY 0x400u  /* tokens as tile columns, m <= 64 */
#define HEXIR_LINEAR_FORCE_GUARDED 0x800u /* bounds-checked loads */
#define HEXIR_LINEAR_SPLIT(S) (((uint32_t)(S) & 0xFFu) << 16)
#define HEXIR_LINEAR_TILE(N) (((uint32_t)(N) / 16u & 0xFFu) << 24)

/* y = act(z) + residual with z = x . w + bias, for x [m][k], w [k][n],
 * bias [n], residual, preact and y [m][n], all of one type, bf16 or f16.
 * bias, residual and preact may be NULL; preact receives z rounded to the
 * type (what the gradient of act needs).  The products are summed in f32; z,
 * act(z) and the residual add stay f32 and y is rounded once.  k == 0 is an
 * empty sum; m == 0 or n == 0 writes nothing.
 *
 * Other types are refused (HEXIR_ERROR_UNIMPLEMENTED): f64 is
 * hexir_cuda_matmul_add_f64 and hexir_cuda_activation_f64, and the tensor
 * cores have no f32 product. */
typedef struct {
  uint32_t dtype, activation;
  uint32_t m, n, k, flags;
  const void *x, *w, *bias, *residual;
  void *preact, *y;
  uint64_t ldx, ldw, ldr, ldp, ldy;
} hexir_linear_call_t;
hexir_status_t hexir_cuda_linear(int ordinal, const hexir_linear_call_t *call,
                                 void *stream);

/* The gradient through the epilogue: dz = dy * act'(preact), rounded to the
 * type, and dbias[j] = sum over i of dz[i][j] as it was rounded, summed in
 * f32.  dy, preact and dz are [m][n] (bf16 or f16).  With
 * HEXIR_ACTIVATION_NONE preact is not read and dz may be NULL (dz is dy);
 * dbias may be NULL.  m == 0 gives a zero dbias.  act' at a corner is the
 * slope from the left (relu'(0) = 0), and at an infinity, which preact holds
 * where z is beyond the type's range, its limit.
 * workspace: hexir_cuda_grad_workspace(n, dtype) bytes, 16-byte aligned,
 * when dbias is wanted; its contents need no initial value. */
typedef struct {
  uint32_t dtype, activation;
  uint32_t m, n;
  const void *dy, *preact;
  void *dz, *dbias, *workspace;
  uint64_t workspace_bytes;
  uint64_t lddy, ldp, lddz;
} hexir_linear_output_grad_call_t;
hexir_status_t hexir_cuda_linear_output_grad(
    int ordinal, const hexir_linear_output_grad_call_t *call, void *stream);

/* dx = (dz . w^T) * act'(preact) + residual, for dz [m][n], w [k][n] (the
 * forward's w) and preact, residual, dx [m][k].  preact and activation are
 * those of the layer whose output x was: the product of its output's
 * gradient with its activation's slope gives that layer's dz.  With
 * HEXIR_ACTIVATION_NONE preact is not read.  residual may be NULL (the
 * gradient that reaches x around the layer). */
typedef struct {
  uint32_t dtype, activation;
  uint32_t m, n, k, flags;
  const void *dz, *w, *preact, *residual;
  void *dx;
  uint64_t lddz, ldw, ldp, ldr, lddx;
} hexir_linear_input_grad_call_t;
hexir_status_t hexir_cuda_linear_input_grad(
    int ordinal, const hexir_linear_input_grad_call_t *call, void *stream);

/* dw = x^T . dz, [k][n], for x [m][k] and dz [m][n]; m == 0 gives zeros. */
typedef struct {
  uint32_t dtype, reserved; /* reserved: 0 */
  uint32_t m, n, k, flags;
  const void *x, *dz;
  void *dw;
  uint64_t ldx, lddz, lddw;
} hexir_linear_weight_grad_call_t;
hexir_status_t hexir_cuda_linear_weight_grad(
    int ordinal, const hexir_linear_weight_grad_call_t *call, void *stream);

/* Which kernel a product would run on: *variant 1 = CTA pairs, 2 = single
 * CTAs, 3 = skinny, 4 = guarded, 0 = none (an empty output); *tile_n its tile's
 * columns, *split the CTAs that share one tile's sum.  op 0 = hexir_cuda_linear,
 * 1 = input_grad, 2 = weight_grad; m, n, k and flags as that call has them.
 * What else the choice depends on:
 *   aligned  the tensors all of whose rows start on 16-byte boundaries:
 *            HEXIR_LINEAR_ALIGNED_*, 1 for all and 0 for none;
 *   flags    with HEXIR_LINEAR_PLAN_PLAIN the answer is for a call without
 *            residual and without preactivations whose slope it takes;
 *            without it, for one that has either (weight_grad has none). */
#define HEXIR_LINEAR_ALIGNED_ALL 1
#define HEXIR_LINEAR_ALIGNED_FIRST 2  /* x; dz; x (in the order of op) */
#define HEXIR_LINEAR_ALIGNED_SECOND 4 /* w; w; dz */
#define HEXIR_LINEAR_ALIGNED_REST 8   /* outputs, residual, preactivations */
#define HEXIR_LINEAR_PLAN_PLAIN 0x1u
hexir_status_t hexir_cuda_linear_plan(int ordinal, uint32_t op, uint32_t m,
                                      uint32_t n, uint32_t k, int aligned,
                                      uint32_t flags, uint32_t *variant,
                                      uint32_t *tile_n, uint32_t *split);

/* Bytes of workspace the two calls that sum over rows need, for rows of
 * `cols` elements: 640 partial sums per column, f32 (f64 for f64). */
uint64_t hexir_cuda_grad_workspace(uint32_t cols, uint32_t dtype);

/* Layer norm of each row of x [rows][cols]:
 *   mean = sum x / cols, var = sum (x - mean)^2 / cols,
 *   rstd = 1 / sqrt(var + eps), y = (x - mean) * rstd * gamma + beta.
 * x, gamma, beta and y are of one type: f64, f32, bf16 or f16; gamma (1 if
 * NULL) and beta (0 if NULL) are [cols].  mean and rstd ([rows], f32, or f64
 * for f64; either may be NULL) are what the gradient needs.  Arithmetic in
 * f32 (f64 for f64); the variance is of the differences from the mean, not
 * of squares.  y may be x (same pointer and stride). */
typedef struct {
  uint32_t dtype, cols;
  uint64_t rows;
  double eps; /* >= 0 */
  const void *x, *gamma, *beta;
  void *y, *mean, *rstd;
  uint64_t ldx, ldy;
} hexir_layer_norm_call_t;
hexir_status_t hexir_cuda_layer_norm(int ordinal,
                                     const hexir_layer_norm_call_t *call,
                                     void *stream);

/* Its gradient.  With xhat = (x - mean) * rstd and g = dy * gamma:
 *   dx = rstd * (g - sum(g) / cols - xhat * sum(g * xhat) / cols) + residual
 *   dgamma[j] = sum over rows of dy * xhat,  dbeta[j] = sum over rows of dy.
 * residual ([rows][cols], may be NULL) is the gradient that reaches x around
 * the norm.  dx, dgamma and dbeta may each be NULL.  dx may be dy or residual
 * (same pointer and stride).  rows == 0 gives zero dgamma and dbeta.
 * workspace: hexir_cuda_grad_workspace(cols, dtype) bytes, 16-byte aligned,
 * when dgamma or dbeta is wanted. */
typedef struct {
  uint32_t dtype, cols;
  uint64_t rows;
  const void *dy, *x, *mean, *rstd, *gamma, *residual;
  void *dx, *dgamma, *dbeta, *workspace;
  uint64_t workspace_bytes;
  uint64_t lddy, ldx, ldr, lddx;
} hexir_layer_norm_grad_call_t;
hexir_status_t hexir_cuda_layer_norm_grad(
    int ordinal, const hexir_layer_norm_grad_call_t *call, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* HEXIR_B200_LAYERS_H */
