// linear_16.cu -- the products of a bf16 / f16 linear layer on the fifth
// generation tensor cores (include/hexir_b200/layers.h):
//
//   forward      z = x . w + bias, y = act(z) + residual
//   input grad   dx = (dz . w^T) * act'(z of the layer before) + residual
//   weight grad  dw = x^T . dz
//
// One out[rows][cols] = sum over depth each; what differs is which way the
// operands lie in memory (the MMA takes either) and the epilogue.  Tiles go
// from HBM to shared memory by TMA with the 128-byte swizzle, one thread
// issues tcgen05.mma, sums stay f32 in TMEM, and the epilogue warps read them
// from there and write the finished rows.
//
// Every wait is bounded (common.cuh): a wait that runs out sets the error
// word, its role stops, and the block still frees its TMEM and ends.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "activation_f32.cuh"
#include "common.cuh"
#include "layers_abi.h"
#include "linear_tiles.cuh"
#include "tcgen05.cuh"

using namespace hexir;

namespace {

typedef hexir_product_args_t Args;

constexpr uint32_t kBK = HEXIR_PRODUCT_BK;
constexpr uint32_t kBM = HEXIR_PRODUCT_BM;
constexpr uint32_t kABytes = kBM * 128u;  // a stage's A tile
constexpr uint32_t kBox = 8192u;          // an MN-major box: 64 x 64 elements

__device__ __forceinline__ float from_bits(uint16_t b, bool is_f16) {
  return is_f16 ? __half2float(__ushort_as_half(b))
                : __uint_as_float(static_cast<uint32_t>(b) << 16);
}
__device__ __forceinline__ uint16_t to_bits(float f, bool is_f16) {
  return is_f16 ? __half_as_ushort(__float2half_rn(f))
                : __bfloat16_as_ushort(__float2bfloat16_rn(f));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool is_f16) {
  if (is_f16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void unpack2(uint32_t w, float &lo, float &hi,
                                        bool is_f16) {
  if (is_f16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    lo = f.x;
    hi = f.y;
  } else {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  }
}

// 16 consecutive elements at p, of which the first `left` are the row's.
__device__ __forceinline__ void load16(const uint16_t *p, uint32_t left,
                                       bool vec, bool is_f16, float (&v)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (vec && left >= 8u * h + 8u) {
      const uint4 w = *reinterpret_cast<const uint4 *>(p + 8 * h);
      unpack2(w.x, v[8 * h], v[8 * h + 1], is_f16);
      unpack2(w.y, v[8 * h + 2], v[8 * h + 3], is_f16);
      unpack2(w.z, v[8 * h + 4], v[8 * h + 5], is_f16);
      unpack2(w.w, v[8 * h + 6], v[8 * h + 7], is_f16);
    } else {
#pragma unroll
      for (int i = 8 * h; i < 8 * h + 8; ++i)
        v[i] = static_cast<uint32_t>(i) < left ? from_bits(p[i], is_f16) : 0.0f;
    }
  }
}

__device__ __forceinline__ void store16(uint16_t *p, uint32_t left, bool vec,
                                        bool is_f16, const float (&v)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (vec && left >= 8u * h + 8u) {
      uint4 w;
      w.x = pack2(v[8 * h], v[8 * h + 1], is_f16);
      w.y = pack2(v[8 * h + 2], v[8 * h + 3], is_f16);
      w.z = pack2(v[8 * h + 4], v[8 * h + 5], is_f16);
      w.w = pack2(v[8 * h + 6], v[8 * h + 7], is_f16);
      *reinterpret_cast<uint4 *>(p + 8 * h) = w;
    } else {
#pragma unroll
      for (int i = 8 * h; i < 8 * h + 8; ++i)
        if (static_cast<uint32_t>(i) < left)
          p[i] = to_bits(v[i], is_f16);
    }
  }
}

// The epilogue of 16 consecutive columns of one row, from the f32 sums to
// the stored row; each stored value is rounded once.
template <int FORM>
__device__ __forceinline__ void finish16(const Args &p, float (&v)[16],
                                         uint32_t row, uint32_t col) {
  if (row >= p.rows || col >= p.cols)
    return;
  const uint32_t left = p.cols - col;
  const bool vec = p.vec != 0, f16 = p.is_f16 != 0;
  if (FORM == HEXIR_PRODUCT_FORWARD) {
    if (p.bias) {
      float b[16];
      load16(static_cast<const uint16_t *>(p.bias) + col, left, vec, f16, b);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        v[i] += b[i];
    }
    if (p.preact_out)
      store16(static_cast<uint16_t *>(p.preact_out) + row * p.ldp + col, left,
              vec, f16, v);
    act_f32(p.activation, v);
  }
  if (FORM == HEXIR_PRODUCT_INPUT_GRAD && p.slope_at) {
    float z[16];
    load16(static_cast<const uint16_t *>(p.slope_at) + row * p.lds + col, left,
           vec, f16, z);
    slope_f32(p.activation, z, v);
  }
  if (FORM != HEXIR_PRODUCT_WEIGHT_GRAD && p.residual) {
    float r[16];
    load16(static_cast<const uint16_t *>(p.residual) + row * p.ldr + col, left,
           vec, f16, r);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      v[i] += r[i];
  }
  store16(static_cast<uint16_t *>(p.out) + row * p.ldo + col, left, vec, f16, v);
}

// The same for one column of 16 consecutive rows (the skinny forward, whose
// tile is the transposed product: lanes are columns, so a warp's store of one
// row covers 32 consecutive columns).
__device__ __forceinline__ void finish_column16(const Args &p, float (&v)[16],
                                                uint32_t row, uint32_t col) {
  if (col >= p.cols || row >= p.rows)
    return;
  const bool f16 = p.is_f16 != 0;
  const uint32_t left = p.rows - row;
  if (p.bias) {
    const float b = from_bits(static_cast<const uint16_t *>(p.bias)[col], f16);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      v[i] += b;
  }
  if (p.preact_out) {
    uint16_t *z = static_cast<uint16_t *>(p.preact_out) + row * p.ldp + col;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (static_cast<uint32_t>(i) < left)
        z[i * p.ldp] = to_bits(v[i], f16);
  }
  act_f32(p.activation, v);
  if (p.residual) {
    const uint16_t *r =
        static_cast<const uint16_t *>(p.residual) + row * p.ldr + col;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (static_cast<uint32_t>(i) < left)
        v[i] += from_bits(r[i * p.ldr], f16);
  }
  uint16_t *y = static_cast<uint16_t *>(p.out) + row * p.ldo + col;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (static_cast<uint32_t>(i) < left)
      y[i * p.ldo] = to_bits(v[i], f16);
}

// Load `size` (a multiple of 64) of an operand's side and 64 of the summed
// index into a stage: one box for K-major rows, a box per 64 for MN-major.
template <bool MN, typename Load>
__device__ __forceinline__ void load_operand(uint8_t *dst, uint32_t size,
                                             uint32_t side, uint32_t k,
                                             Load load) {
  if (MN) {
    for (uint32_t b = 0; b < size / 64; ++b)
      load(dst + b * kBox, static_cast<int32_t>(side + b * 64),
           static_cast<int32_t>(k));
  } else {
    load(dst, static_cast<int32_t>(k), static_cast<int32_t>(side));
  }
}

// The four K = 16 steps of one stage.
template <int CG, bool A_MN, bool B_MN>
__device__ __forceinline__ void mma_stage(uint32_t tmem, uint32_t a, uint32_t b,
                                          uint32_t desc, bool first) {
  const uint64_t da = operand_desc<A_MN>(a), db = operand_desc<B_MN>(b);
#pragma unroll
  for (uint32_t s = 0; s < kBK / 16; ++s)
    mma_f16<CG>(tmem, da + s * operand_step<A_MN>(), db + s * operand_step<B_MN>(),
                desc, !first || s > 0);
}

__device__ __forceinline__ uint8_t *align1024(uint8_t *p) {
  return p + ((1024u - (smem_addr(p) & 1023u)) & 1023u);
}

// ------------------------------------------------------------- CTA pairs
//
// A persistent pair of CTAs computes 256 x tile_n tiles: each holds 128 rows
// of A, half of the columns of B and its own rows' sums in TMEM, so a stage
// costs half the shared-memory traffic per product of a single CTA's.  Two
// sets of sums alternate: the epilogue of one tile runs under the MMAs of the
// next.
template <int FORM>
__device__ __forceinline__ void product_pair(const CUtensorMap *map_a,
                                             const CUtensorMap *map_b,
                                             const Args &p) {
  constexpr bool A_MN = FORM == HEXIR_PRODUCT_WEIGHT_GRAD;
  constexpr bool B_MN = FORM != HEXIR_PRODUCT_INPUT_GRAD;
  constexpr uint32_t kStages = HEXIR_PAIR_STAGES;
  constexpr uint32_t kEpilogueWarps = 8;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStages], empty[kStages], sums_full[2], sums_empty[2];
  __shared__ uint32_t tmem_slot;
  uint8_t *ring = align1024(smem_raw);
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const uint32_t half_n = p.tile_n / 2;
  const uint32_t stage_bytes = kABytes + half_n * 128u;

  if (threadIdx.x == 0) {
    prefetch_tensormap(map_a);
    prefetch_tensormap(map_b);
    for (uint32_t s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (uint32_t s = 0; s < 2; ++s) {
      mbar_init(&sums_full[s], 1);
      mbar_init(&sums_empty[s], 2 * kEpilogueWarps);
    }
    fence_mbar_init();
  }
  if (warp == 2)
    tmem_alloc<2>(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers exist before anything arrives there
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  const uint32_t tiles = p.tiles_m * p.tiles_n;
  const uint32_t first = blockIdx.x / 2, step = gridDim.x / 2;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (uint32_t tile = first; tile < tiles && ok; tile += step) {
        uint32_t tm, tn;
        tile_of(tile, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
        const uint32_t row0 = tm * 2 * kBM + rank * kBM;
        const uint32_t col0 = tn * p.tile_n + rank * half_n;
        for (uint32_t kt = 0; kt < p.k_tiles; ++kt, ++it) {
          const uint32_t s = it % kStages;
          if (!mbar_wait_bounded(&empty[s], (it / kStages & 1u) ^ 1u,
                                 p.timeout_ns)) {
            ok = false;
            break;
          }
          if (rank == 0)
            mbar_arrive_expect_tx(&full[s], 2 * stage_bytes);
          uint8_t *dst = ring + s * HEXIR_PAIR_STAGE_BYTES;
          const uint32_t bar = cluster_addr(&full[s], 0);
          load_operand<A_MN>(dst, kBM, row0, kt * kBK,
                             [&](uint8_t *d, int32_t x, int32_t y) {
                               tma_load_2d_pair(d, map_a, x, y, bar);
                             });
          load_operand<B_MN>(dst + kABytes, half_n, col0, kt * kBK,
                             [&](uint8_t *d, int32_t x, int32_t y) {
                               tma_load_2d_pair(d, map_b, x, y, bar);
                             });
        }
      }
      // Given up: the copies in flight land before the block ends.
      if (!ok && rank == 0)
        for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
          mbar_wait_bounded(&full[i % kStages], i / kStages & 1u, p.timeout_ns);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t desc = mma_desc<A_MN, B_MN>(2 * kBM, p.tile_n, p.is_f16 != 0);
      uint32_t it = 0, t = 0;
      bool ok = true;
      for (uint32_t tile = first; tile < tiles && ok; tile += step, ++t) {
        const uint32_t set = t & 1u;
        if (!mbar_wait_bounded(&sums_empty[set], (t >> 1 & 1u) ^ 1u,
                               p.timeout_ns))
          break;
        tc_fence_after();
        for (uint32_t kt = 0; kt < p.k_tiles; ++kt, ++it) {
          const uint32_t s = it % kStages;
          if (!mbar_wait_bounded(&full[s], it / kStages & 1u, p.timeout_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_addr(ring + s * HEXIR_PAIR_STAGE_BYTES);
          mma_stage<2, A_MN, B_MN>(tmem + set * 256u, a, a + kABytes, desc,
                                   kt == 0);
          mma_commit_pair(&empty[s]);
        }
        if (ok)
          mma_commit_pair(&sums_full[set]);
      }
    }
  } else if (warp >= 4) {
    const uint32_t quarter = warp & 3u, side = (warp - 4) / 4;
    uint32_t t = 0;
    for (uint32_t tile = first; tile < tiles; tile += step, ++t) {
      uint32_t tm, tn;
      tile_of(tile, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
      const uint32_t row = tm * 2 * kBM + rank * kBM + quarter * 32 + lane;
      const uint32_t set = t & 1u;
      // The whole warp leaves together: its TMEM loads are warp-wide.
      if (!__all_sync(0xFFFFFFFFu,
                      mbar_wait_bounded(&sums_full[set], t >> 1 & 1u,
                                        4 * p.timeout_ns)))
        break;
      tc_fence_after();
      const uint32_t src = tmem + (quarter * 32u << 16) + set * 256u;
      for (uint32_t c = side * half_n; c < side * half_n + half_n; c += 16) {
        float v[16];
        __syncwarp();
        tmem_load16(src + c, v);
        finish16<FORM>(p, v, row, tn * p.tile_n + c);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive_cluster(cluster_addr(&sums_empty[set], 0));
    }
  }
  __syncthreads();
  __syncwarp();
  cluster_sync();  // nothing arrives at, or reads, a CTA that has ended
  if (warp == 2)
    tmem_free<2>(tmem, 512);
}

// ------------------------------------------------------------ single CTAs
//
// One 128 x tile_n tile per cluster of `split` CTAs, each summing its share
// of the depth.  With split > 1 every CTA leaves its sums in its own shared
// memory and, after a cluster barrier, adds up its share of the tile's
// columns over the cluster in rank order (the same order every time) and
// finishes them: no workspace and no second launch.
//
// SWAP (the forward of up to 64 tokens): the lanes are the weight's columns
// and the tile's columns the tokens, so a 128-row MMA multiplies weights
// instead of padding.
//
// GUARDED: rows that TMA cannot describe (a stride or base off 16 bytes).
// The epilogue warps load the operands with bounds checks, into the layout
// TMA would have written, and become the epilogue afterwards.

// One 16-byte chunk: 8 elements of row `major` from `minor` on, zero beyond
// the operand.
__device__ __forceinline__ uint4 guarded_chunk(const uint16_t *base, uint64_t ld,
                                               uint32_t major, uint32_t majors,
                                               uint32_t minor, uint32_t minors) {
  uint4 w = make_uint4(0, 0, 0, 0);
  if (major >= majors || minor >= minors)
    return w;
  const uint16_t *src = base + major * ld + minor;
  const uint32_t left = minors - minor;
  const uintptr_t at = reinterpret_cast<uintptr_t>(src);
  if (left >= 8 && (at & 15u) == 0)
    return *reinterpret_cast<const uint4 *>(src);
  uint32_t e[8];
  if (left >= 8 && (at & 3u) == 0) {
    const uint32_t *q = reinterpret_cast<const uint32_t *>(src);
    return make_uint4(q[0], q[1], q[2], q[3]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    e[i] = static_cast<uint32_t>(i) < left ? src[i] : 0u;
  w.x = e[0] | e[1] << 16;
  w.y = e[2] | e[3] << 16;
  w.z = e[4] | e[5] << 16;
  w.w = e[6] | e[7] << 16;
  return w;
}

// size x 64 of an operand (side from `side0`, summed index from k0) into the
// swizzled layout of a stage, by 128 threads.
template <bool MN>
__device__ __forceinline__ void guarded_operand(uint8_t *dst, const void *base,
                                                uint64_t ld, uint32_t size,
                                                uint32_t side0, uint32_t sides,
                                                uint32_t k0, uint32_t depth,
                                                uint32_t tid) {
  const uint16_t *src = static_cast<const uint16_t *>(base);
  const uint32_t chunks = size * 8;
#pragma unroll 4
  for (uint32_t i = tid; i < chunks; i += 128) {
    const uint32_t r = i / 8, c = i % 8;  // 128-byte row of the stage, chunk
    uint4 w;
    if (MN)
      w = guarded_chunk(src, ld, k0 + r % 64, depth, side0 + r / 64 * 64 + c * 8,
                        sides);
    else
      w = guarded_chunk(src, ld, side0 + r, sides, k0 + c * 8, depth);
    *reinterpret_cast<uint4 *>(dst + r * 128 + ((c ^ (r & 7u)) << 4)) = w;
  }
}

template <int FORM, bool GUARDED, bool SWAP>
__device__ __forceinline__ void product_single(const CUtensorMap *map_a,
                                               const CUtensorMap *map_b,
                                               const Args &p) {
  constexpr bool A_MN = SWAP || FORM == HEXIR_PRODUCT_WEIGHT_GRAD;
  constexpr bool B_MN = !SWAP && FORM != HEXIR_PRODUCT_INPUT_GRAD;
  constexpr uint32_t kMax = HEXIR_SINGLE_MAX_STAGES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMax], empty[kMax], done;
  __shared__ uint32_t tmem_slot;
  uint8_t *ring = align1024(smem_raw);
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = p.split > 1 ? cluster_ctarank() : 0;
  const uint32_t stages = p.stages;
  const uint32_t stage_bytes = kABytes + p.tile_n * 128u;

  if (threadIdx.x == 0) {
    if (!GUARDED) {
      prefetch_tensormap(map_a);
      prefetch_tensormap(map_b);
    }
    for (uint32_t s = 0; s < stages; ++s) {
      mbar_init(&full[s], GUARDED ? 128 : 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == 1)
    tmem_alloc<1>(&tmem_slot, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // The tile, and this CTA's share of its sum.
  uint32_t tm, tn;
  tile_of(blockIdx.x / p.split, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
  const uint32_t kt0 = static_cast<uint32_t>(
      static_cast<uint64_t>(p.k_tiles) * rank / p.split);
  const uint32_t kt1 = static_cast<uint32_t>(
      static_cast<uint64_t>(p.k_tiles) * (rank + 1) / p.split);
  const uint32_t lane0 = tm * kBM, col0 = tn * p.tile_n;
  bool ok = true;

  if (warp == 0) {
    if (!GUARDED && lane == 0) {
      uint32_t it = 0;
      for (uint32_t kt = kt0; kt < kt1; ++kt, ++it) {
        const uint32_t s = it % stages;
        if (!mbar_wait_bounded(&empty[s], (it / stages & 1u) ^ 1u,
                               p.timeout_ns)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[s], stage_bytes);
        uint8_t *dst = ring + s * stage_bytes;
        load_operand<A_MN>(dst, kBM, lane0, kt * kBK,
                           [&](uint8_t *d, int32_t x, int32_t y) {
                             tma_load_2d(d, map_a, x, y, &full[s]);
                           });
        load_operand<B_MN>(dst + kABytes, p.tile_n, col0, kt * kBK,
                           [&](uint8_t *d, int32_t x, int32_t y) {
                             tma_load_2d(d, map_b, x, y, &full[s]);
                           });
      }
      if (!ok)
        for (uint32_t i = it > stages ? it - stages : 0; i < it; ++i)
          mbar_wait_bounded(&full[i % stages], i / stages & 1u, p.timeout_ns);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t desc = mma_desc<A_MN, B_MN>(kBM, p.tile_n, p.is_f16 != 0);
      uint32_t it = 0;
      for (uint32_t kt = kt0; kt < kt1; ++kt, ++it) {
        const uint32_t s = it % stages;
        if (!mbar_wait_bounded(&full[s], it / stages & 1u, p.timeout_ns))
          break;
        tc_fence_after();
        const uint32_t a = smem_addr(ring + s * stage_bytes);
        mma_stage<1, A_MN, B_MN>(tmem, a, a + kABytes, desc, kt == kt0);
        mma_commit(&empty[s]);
      }
      mma_commit(&done);  // also after a wait that ran out: nothing in flight
    }
  } else {
    const uint32_t tid = threadIdx.x - 64;
    if (GUARDED) {
      uint32_t it = 0;
      for (uint32_t kt = kt0; kt < kt1; ++kt, ++it) {
        const uint32_t s = it % stages;
        if (!mbar_wait_bounded(&empty[s], (it / stages & 1u) ^ 1u, p.timeout_ns))
          break;
        uint8_t *dst = ring + s * stage_bytes;
        guarded_operand<A_MN>(dst, p.a, p.lda, kBM, lane0, p.rows, kt * kBK,
                              p.depth, tid);
        guarded_operand<B_MN>(dst + kABytes, p.b, p.ldb, p.tile_n, col0, p.cols,
                              kt * kBK, p.depth, tid);
        fence_async_smem();
        mbar_arrive(&full[s]);
      }
      __syncwarp();
    }
    ok = __all_sync(0xFFFFFFFFu,
                    mbar_wait_bounded(&done, 0, 4 * p.timeout_ns));
    tc_fence_after();
    const uint32_t quarter = warp & 3u;
    const uint32_t src = tmem + (quarter * 32u << 16);
    const uint32_t my = quarter * 32 + lane;
    float *sums = reinterpret_cast<float *>(ring);  // [tile_n][128], split > 1
    if (ok) {
      for (uint32_t c = 0; c < p.tile_n; c += 16) {
        float v[16];
        __syncwarp();
        if (kt1 > kt0) {
          tmem_load16(src + c, v);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            v[i] = 0.0f;
        }
        if (p.split > 1) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sums[(c + i) * kBM + my] = v[i];
        } else if (SWAP) {
          finish_column16(p, v, col0 + c, lane0 + my);
        } else {
          finish16<FORM>(p, v, lane0 + my, col0 + c);
        }
      }
    }
  }

  if (p.split > 1) {
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && ok) {
      const uint32_t my = (warp & 3u) * 32 + lane;
      const float *sums = reinterpret_cast<const float *>(ring);
      for (uint32_t c = rank * 16; c < p.tile_n; c += p.split * 16) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] = 0.0f;
        for (uint32_t r = 0; r < p.split; ++r) {
          const uint32_t from = cluster_addr(sums + c * kBM + my, r);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            v[i] += ld_cluster_f32(from + i * (kBM * 4u));
        }
        if (SWAP)
          finish_column16(p, v, col0 + c, lane0 + my);
        else
          finish16<FORM>(p, v, lane0 + my, col0 + c);
      }
    }
    __syncwarp();
    cluster_sync();  // the peers have read this CTA's sums
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<1>(tmem, p.tmem_cols);
  }
}

}  // namespace

#define PRODUCT_PAIR(NAME, FORM)                                              \
  extern "C" __global__ void __launch_bounds__(HEXIR_PAIR_THREADS, 1)         \
      __cluster_dims__(2, 1, 1)                                               \
          NAME(const __grid_constant__ CUtensorMap map_a,                     \
               const __grid_constant__ CUtensorMap map_b, const Args args) {  \
    product_pair<FORM>(&map_a, &map_b, args);                                 \
  }
#define PRODUCT_SINGLE(NAME, FORM, SWAP)                                      \
  extern "C" __global__ void __launch_bounds__(HEXIR_SINGLE_THREADS)          \
      NAME(const __grid_constant__ CUtensorMap map_a,                         \
           const __grid_constant__ CUtensorMap map_b, const Args args) {      \
    product_single<FORM, false, SWAP>(&map_a, &map_b, args);                  \
  }
#define PRODUCT_GUARDED(NAME, FORM)                                           \
  extern "C" __global__ void __launch_bounds__(HEXIR_SINGLE_THREADS)          \
      NAME(const Args args) {                                                 \
    product_single<FORM, true, false>(nullptr, nullptr, args);                \
  }

PRODUCT_PAIR(hexir_linear_16_pair, HEXIR_PRODUCT_FORWARD)
PRODUCT_PAIR(hexir_linear_16_input_grad_pair, HEXIR_PRODUCT_INPUT_GRAD)
PRODUCT_PAIR(hexir_linear_16_weight_grad_pair, HEXIR_PRODUCT_WEIGHT_GRAD)
PRODUCT_SINGLE(hexir_linear_16_single, HEXIR_PRODUCT_FORWARD, false)
PRODUCT_SINGLE(hexir_linear_16_input_grad_single, HEXIR_PRODUCT_INPUT_GRAD, false)
PRODUCT_SINGLE(hexir_linear_16_weight_grad_single, HEXIR_PRODUCT_WEIGHT_GRAD, false)
PRODUCT_SINGLE(hexir_linear_16_skinny, HEXIR_PRODUCT_FORWARD, true)
PRODUCT_GUARDED(hexir_linear_16_guarded, HEXIR_PRODUCT_FORWARD)
PRODUCT_GUARDED(hexir_linear_16_input_grad_guarded, HEXIR_PRODUCT_INPUT_GRAD)
PRODUCT_GUARDED(hexir_linear_16_weight_grad_guarded, HEXIR_PRODUCT_WEIGHT_GRAD)
