/*
 * layers_abi.h -- by-value argument blocks of the layer kernels (layers.cu),
 * shared with the host launcher (runtime/layers.cc).
 */
#ifndef HEXIR_B200_LAYERS_ABI_H
#define HEXIR_B200_LAYERS_ABI_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The three products of a linear layer, out[rows][cols] summed over depth:
 *   forward      x . w      a = x  (K-major),  b = w  (MN-major)
 *   input grad   dz . w^T   a = dz (K-major),  b = w  (K-major)
 *   weight grad  x^T . dz   a = x  (MN-major), b = dz (MN-major)
 * K-major: consecutive elements follow the summed index. */
#define HEXIR_PRODUCT_FORWARD 0
#define HEXIR_PRODUCT_INPUT_GRAD 1
#define HEXIR_PRODUCT_WEIGHT_GRAD 2

/* One stage holds 64 of the summed index (128 bytes, the swizzle's span). */
#define HEXIR_PRODUCT_BK 64
#define HEXIR_PRODUCT_BM 128 /* rows per CTA: the lanes of TMEM */
/* Slots of 1 KiB (32 rows x 16 columns) an epilogue warp fetches ahead into,
 * and one more for stores. */
#define HEXIR_EPILOGUE_SLOTS 6
#define HEXIR_EPILOGUE_BYTES(WARPS) ((WARPS) * (HEXIR_EPILOGUE_SLOTS + 1) * 1024)
/* CTA pair: 5 stages of A 16 KiB + B 16 KiB (each CTA holds half of the 256
 * columns), 4 warps of loads and MMA, 8 of epilogue. */
#define HEXIR_PAIR_STAGES 5
#define HEXIR_PAIR_STAGE_BYTES 32768
#define HEXIR_PAIR_THREADS 384
#define HEXIR_PAIR_SMEM_BYTES                           \
  (HEXIR_PAIR_STAGES * HEXIR_PAIR_STAGE_BYTES + 1024 + \
   HEXIR_EPILOGUE_BYTES(8))
/* Single CTAs: a load warp, an MMA warp and 8 epilogue warps, which are the
 * first of the 16 that load where loads are guarded. */
#define HEXIR_SINGLE_EPILOGUE_WARPS 8
#define HEXIR_SINGLE_THREADS (64 + HEXIR_SINGLE_EPILOGUE_WARPS * 32)
#define HEXIR_GUARDED_LOAD_WARPS 16
#define HEXIR_GUARDED_THREADS (64 + HEXIR_GUARDED_LOAD_WARPS * 32)
#define HEXIR_SINGLE_MAX_STAGES 12

typedef struct {
  void *out;
  void *preact_out;       /* forward: z, or null */
  const void *bias;       /* forward: [cols], or null */
  const void *residual;   /* or null */
  const void *slope_at;   /* input grad: the preactivations, or null */
  uint64_t ldo, ldp, ldr, lds;
  const void *a, *b;      /* guarded loads only */
  uint64_t lda, ldb;
  uint32_t rows, cols, depth;
  uint32_t activation;
  uint32_t is_f16;        /* f16, else bf16 */
  uint32_t vec;           /* epilogue rows on 16- (1) or 32-byte (2) boundaries */
  uint32_t tiles_m, tiles_n, group_m;
  uint32_t full_tiles;    /* pair: those not cut in two */
  uint32_t tile_n;        /* columns of a tile */
  uint32_t k_tiles;       /* ceil(depth / BK) */
  uint32_t split;
  uint32_t stages;        /* single: pipeline stages */
  uint32_t tmem_cols;     /* single: TMEM columns (a power of two >= 32) */
  uint32_t ring_bytes;    /* single: the stages, or the sums of a split tile */
  uint32_t tma_operands;  /* guarded: bit 0 a, bit 1 b come by TMA */
  uint64_t timeout_ns;
} hexir_product_args_t;

typedef struct {
  const void *dy, *preact;
  void *dz, *dbias;
  float *partials;        /* [parts][n] */
  uint64_t lddy, ldp, lddz;
  uint32_t m, n, activation, parts;
  uint32_t is_f16, vec;
  uint32_t rows_per_part, reserved;
} hexir_output_grad_args_t;

typedef struct {
  const void *x, *gamma, *beta;
  void *y, *mean, *rstd;
  uint64_t ldx, ldy, rows;
  double eps;
  uint32_t cols, reserved;
} hexir_layer_norm_args_t;

typedef struct {
  const void *dy, *x, *mean, *rstd, *gamma, *residual;
  void *dx, *dgamma, *dbeta;
  void *partials;         /* [parts][2][cols] f32 (f64) */
  uint64_t lddy, ldx, ldr, lddx, rows;
  uint32_t cols, parts;
} hexir_layer_norm_grad_args_t;

#ifdef __cplusplus
}
#endif
#endif /* HEXIR_B200_LAYERS_ABI_H */
