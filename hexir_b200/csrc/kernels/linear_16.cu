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
// The load and MMA warps run their loops converged and one lane issues: what
// the instructions take is then the same for the warp as far as the compiler
// can tell and goes to them without a detour.  Issued by one thread of its own,
// with a wait of ~100 cycles before each stage, the MMAs of a stage took 660
// cycles instead of 512.
//
// Every wait is bounded (tcgen05.cuh): a wait that runs out sets the error
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

// 16 bytes as 8 f32 and back.
__device__ __forceinline__ void unpack8(const uint4 &w, bool is_f16, float *v) {
  unpack2(w.x, v[0], v[1], is_f16);
  unpack2(w.y, v[2], v[3], is_f16);
  unpack2(w.z, v[4], v[5], is_f16);
  unpack2(w.w, v[6], v[7], is_f16);
}
__device__ __forceinline__ uint4 pack8(const float *v, bool is_f16) {
  return make_uint4(pack2(v[0], v[1], is_f16), pack2(v[2], v[3], is_f16),
                    pack2(v[4], v[5], is_f16), pack2(v[6], v[7], is_f16));
}

// -------------------------------------------------------------- epilogue
//
// An epilogue warp finishes 32 rows x 16 columns at a time: a lane has one
// row's 16 sums from TMEM, adds the bias, applies the activation (or the slope
// at the stored preactivations), adds the residual and stores.  What it reads
// besides (residual, preactivations) it fetches several such blocks ahead, into
// slots of its own in shared memory, while the main loop still runs: read when
// needed, each block waited for memory, which made the epilogue of a 256 x 256
// tile 26 k cycles long.
//
// Rows on 16-byte boundaries (p.vec) are fetched and stored a lane's row at a
// time, 16 bytes an access (stored 32 where they are on 32-byte boundaries, so
// that each access fills a sector); any others by the whole warp, two rows of 16
// elements an access, through the slots.

constexpr uint32_t kSlotBytes = 1024u;  // 32 rows x 32 bytes

// Where lane's row keeps its 16-byte half h: rows 4 apart swap halves, so that
// 8 lanes' accesses fall into different banks.
__device__ __forceinline__ uint32_t slot_at(uint32_t row, uint32_t h) {
  return row * 32u + ((h ^ (row >> 2 & 1u)) << 4);
}

__device__ __forceinline__ void copy_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Tensors an epilogue reads: the residual, then the preactivations.
template <int FORM>
__device__ __forceinline__ uint32_t epilogue_tensors(const Args &p) {
  return (FORM != HEXIR_PRODUCT_WEIGHT_GRAD && p.residual ? 1u : 0u) +
         (FORM == HEXIR_PRODUCT_INPUT_GRAD && p.slope_at ? 1u : 0u);
}

// Blocks fetched ahead: 6 of one tensor or 3 of two.
constexpr uint32_t kAhead1 = HEXIR_EPILOGUE_SLOTS, kAhead2 = HEXIR_EPILOGUE_SLOTS / 2;

__device__ __forceinline__ void fetch_tensor(const Args &p, const void *base,
                                             uint64_t ld, uint8_t *slot,
                                             uint32_t row0, uint32_t col,
                                             uint32_t lane) {
  const uint16_t *src = static_cast<const uint16_t *>(base);
  if (p.vec) {
    const uint32_t row = row0 + lane;
    if (row < p.rows) {
      src += row * ld + col;
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t c = col + 8 * h;
        if (c + 8 <= p.cols) {
          copy_async16(smem_addr(slot + slot_at(lane, h)), src + 8 * h);
        } else if (c < p.cols) {
          uint16_t e[8];
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i)
            e[i] = src[8 * h + min(i, p.cols - c - 1)];
          uint16_t *dst = reinterpret_cast<uint16_t *>(slot + slot_at(lane, h));
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i)
            dst[i] = e[i];
        }
      }
    }
  } else {
    const uint32_t c = lane % 16;
    const uint32_t col_in = min(col + c, p.cols - 1);
    uint16_t e[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      e[i] = src[min(row0 + 2 * i + lane / 16, p.rows - 1) * ld + col_in];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      *reinterpret_cast<uint16_t *>(slot + slot_at(2 * i + lane / 16, c / 8) +
                                    c % 8 * 2) = e[i];
  }
}

// Fetch the block at (row0, col) into `slot` (a slot per tensor); blocks
// outside the output fetch nothing.
template <int FORM>
__device__ __forceinline__ void fetch_block(const Args &p, uint8_t *slot,
                                            uint32_t row0, uint32_t col,
                                            uint32_t lane) {
  if (row0 >= p.rows || col >= p.cols)
    return;
  if (FORM != HEXIR_PRODUCT_WEIGHT_GRAD && p.residual) {
    fetch_tensor(p, p.residual, p.ldr, slot, row0, col, lane);
    slot += kSlotBytes;
  }
  if (FORM == HEXIR_PRODUCT_INPUT_GRAD && p.slope_at)
    fetch_tensor(p, p.slope_at, p.lds, slot, row0, col, lane);
}

__device__ __forceinline__ void read_slot(const uint8_t *slot, uint32_t lane,
                                          bool is_f16, float (&v)[16]) {
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h)
    unpack8(*reinterpret_cast<const uint4 *>(slot + slot_at(lane, h)), is_f16,
            v + 8 * h);
}

// Store a block's rows; `out` is a slot for rows off 16 bytes.
__device__ __forceinline__ void store_block(const Args &p, void *base, uint64_t ld,
                                            uint8_t *out, uint32_t row0,
                                            uint32_t col, uint32_t lane,
                                            const float (&v)[16]) {
  const bool f16 = p.is_f16 != 0;
  uint16_t *dst = static_cast<uint16_t *>(base);
  if (p.vec) {
    const uint32_t row = row0 + lane;
    if (row >= p.rows)
      return;
    dst += row * ld + col;
    if (p.vec == 2 && col + 16 <= p.cols) {
      const uint4 lo = pack8(v, f16), hi = pack8(v + 8, f16);
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                       dst),
                   "r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w), "r"(hi.x),
                   "r"(hi.y), "r"(hi.z), "r"(hi.w)
                   : "memory");
      return;
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t c = col + 8 * h;
      if (c + 8 <= p.cols) {
        *reinterpret_cast<uint4 *>(dst + 8 * h) = pack8(v + 8 * h, f16);
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (c + i < p.cols)
            dst[8 * h + i] = to_bits(v[8 * h + i], f16);
      }
    }
    return;
  }
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h)
    *reinterpret_cast<uint4 *>(out + slot_at(lane, h)) = pack8(v + 8 * h, f16);
  __syncwarp();
  const uint32_t c = lane % 16;
#pragma unroll
  for (uint32_t i = 0; i < 16; ++i) {
    const uint32_t r = 2 * i + lane / 16;
    if (row0 + r < p.rows && col + c < p.cols)
      dst[(row0 + r) * ld + col + c] = *reinterpret_cast<const uint16_t *>(
          out + slot_at(r, c / 8) + c % 8 * 2);
  }
  __syncwarp();
}

// Finish the block at (row0, col), whose tensors are in `slot`; each stored
// value is rounded once.  `bias` has the tile's bias in f32 from this block's
// column on.
template <int FORM>
__device__ __forceinline__ void finish_block(const Args &p, float (&v)[16],
                                             const float *bias,
                                             const uint8_t *slot, uint8_t *out,
                                             uint32_t row0, uint32_t col,
                                             uint32_t lane) {
  if (row0 >= p.rows || col >= p.cols)
    return;
  const bool f16 = p.is_f16 != 0;
  if (FORM == HEXIR_PRODUCT_FORWARD) {
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4 b = *reinterpret_cast<const float4 *>(bias + i);
        v[i] += b.x;
        v[i + 1] += b.y;
        v[i + 2] += b.z;
        v[i + 3] += b.w;
      }
    }
    if (p.preact_out)
      store_block(p, p.preact_out, p.ldp, out, row0, col, lane, v);
    act_f32(p.activation, v);
  }
  float r[16];
  if (FORM == HEXIR_PRODUCT_INPUT_GRAD && p.slope_at) {
    read_slot(slot + (p.residual ? kSlotBytes : 0u), lane, f16, r);
    slope_f32(p.activation, r, v);
  }
  if (FORM != HEXIR_PRODUCT_WEIGHT_GRAD && p.residual) {
    read_slot(slot, lane, f16, r);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      v[i] += r[i];
  }
  store_block(p, p.out, p.ldo, out, row0, col, lane, v);
}

// The bias of columns col0 .. col0 + count into a warp's own shared memory;
// zeros beyond the row.
__device__ __forceinline__ void stage_bias(const Args &p, float *bias, uint32_t col0,
                                           uint32_t count, uint32_t lane) {
  __syncwarp();
  for (uint32_t c = lane; c < count; c += 32)
    bias[c] = col0 + c < p.cols
                  ? from_bits(static_cast<const uint16_t *>(p.bias)[col0 + c],
                              p.is_f16 != 0)
                  : 0.0f;
  __syncwarp();
}

// A warp's blocks in order, fetched ahead of their use.
template <int FORM>
struct Ahead {
  const Args &p;
  uint8_t *slots;  // this warp's: kAhead1 slots, and one for stores
  uint32_t tensors, lane, depth, put = 0, got = 0;
  __device__ __forceinline__ Ahead(const Args &args, uint8_t *area, uint32_t lane_)
      : p(args), slots(area), tensors(epilogue_tensors<FORM>(args)), lane(lane_),
        depth(tensors == 2 ? kAhead2 : kAhead1) {}
  __device__ __forceinline__ uint8_t *out() const {
    return slots + kAhead1 * kSlotBytes;
  }
  __device__ __forceinline__ uint8_t *slot(uint32_t i) const {
    return slots + i * tensors * kSlotBytes;
  }
  // The next block to come (`exists`: there is one).
  __device__ __forceinline__ void fetch(uint32_t row0, uint32_t col, bool exists) {
    if (tensors) {
      if (exists)
        fetch_block<FORM>(p, slot(put), row0, col, lane);
      copies_commit();
      put = put + 1 == depth ? 0 : put + 1;
    }
  }
  // The oldest fetched block has arrived.
  __device__ __forceinline__ uint8_t *arrived() {
    if (tensors == 2)
      copies_wait<kAhead2 - 1>();
    else if (tensors == 1)
      copies_wait<kAhead1 - 1>();
    __syncwarp();
    uint8_t *at = slot(got);
    got = got + 1 == depth ? 0 : got + 1;
    return at;
  }
};

// Columns of 16 consecutive rows (the skinny forward, whose tile is the
// transposed product: lanes are columns, so a warp's access of one row covers
// 32 consecutive columns).  Rows past the last are read as the last, so that
// the loads need no branches and are in flight together.
__device__ __forceinline__ void finish_column16(const Args &p, float (&v)[16],
                                                uint32_t row, uint32_t col) {
  if (col >= p.cols || row >= p.rows)
    return;
  const bool f16 = p.is_f16 != 0;
  const uint32_t left = p.rows - row;
  uint16_t r[16];
  if (p.residual) {
    const uint16_t *src =
        static_cast<const uint16_t *>(p.residual) + row * p.ldr + col;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      r[i] = src[min(i, left - 1) * p.ldr];
  }
  if (p.bias) {
    const float b = from_bits(static_cast<const uint16_t *>(p.bias)[col], f16);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      v[i] += b;
  }
  if (p.preact_out) {
    uint16_t *z = static_cast<uint16_t *>(p.preact_out) + row * p.ldp + col;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      if (i < left)
        z[i * p.ldp] = to_bits(v[i], f16);
  }
  act_f32(p.activation, v);
  if (p.residual) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      v[i] += from_bits(r[i], f16);
  }
  uint16_t *y = static_cast<uint16_t *>(p.out) + row * p.ldo + col;
#pragma unroll
  for (uint32_t i = 0; i < 16; ++i)
    if (i < left)
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
// A pair's part of B: boxes of 64 in either layout, for tiles of two widths.
template <bool MN, typename Load>
__device__ __forceinline__ void load_boxes(uint8_t *dst, uint32_t size, uint32_t side,
                                           uint32_t k, Load load) {
  for (uint32_t b = 0; b < size / 64; ++b) {
    const int32_t at = static_cast<int32_t>(side + b * 64);
    if (MN)
      load(dst + b * kBox, at, static_cast<int32_t>(k));
    else
      load(dst + b * kBox, static_cast<int32_t>(k), at);
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
// next.  Where the tiles of the last turn would leave half of the pairs or more
// without work, they are cut in two (a half costs about 0.7 of a tile: 4096
// cubed 101.3 to 99.0 us, 2048 x 8192 x 2048 with gelu and z 57.4 to 55.8).
//
// A stage takes 512 cycles of the tensor pipe and is bound by it where the
// clock holds: 4096 cubed runs the pipe 82 % of the active cycles.  8192 cubed
// (816 us with bias and residual, 1.35 PFLOP/s) is bound by power.
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
  __shared__ alignas(16) float bias[kEpilogueWarps][128];
  uint8_t *ring = align1024(smem_raw);
  uint8_t *slots = ring + kStages * HEXIR_PAIR_STAGE_BYTES;
  const uint32_t warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x / 32, 0);
  const uint32_t lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();

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
  griddep_wait();  // nothing global is read or written before this
  griddep_launch_dependents();

  // The work: full_tiles tiles, then the halves (along the columns) of the rest.
  struct Item {
    uint32_t row0, col0, half_n;  // half_n: columns of B a CTA holds
  };
  const uint32_t items = 2 * p.tiles_m * p.tiles_n - p.full_tiles;
  auto item_of = [&](uint32_t i) {
    const uint32_t over = i < p.full_tiles ? 0 : i - p.full_tiles;
    uint32_t tm, tn;
    tile_of(i < p.full_tiles ? i : p.full_tiles + over / 2, p.tiles_m, p.tiles_n,
            p.group_m, tm, tn);
    const uint32_t half_n = p.tile_n / (i < p.full_tiles ? 2u : 4u);
    return Item{tm * 2 * kBM, tn * p.tile_n + (over & 1u) * (p.tile_n / 2), half_n};
  };
  const uint32_t first = blockIdx.x / 2, step = gridDim.x / 2;

  if (warp == 0) {
    const bool leader = elect_one();
    RingPlace at;
    uint32_t fills = 0;
    bool ok = true;
    for (uint32_t i = first; i < items && ok; i += step) {
      const Item item = item_of(i);
      const uint32_t row0 = item.row0 + rank * kBM;
      const uint32_t col0 = item.col0 + rank * item.half_n;
      for (uint32_t kt = 0; kt < p.k_tiles; ++kt, ++fills, at.next(kStages)) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_pipeline(&empty[at.stage],
                                                        at.parity ^ 1u, p.timeout_ns));
        if (!ok)
          break;
        if (leader) {
          if (rank == 0)
            mbar_arrive_expect_tx(&full[at.stage],
                                  2 * (kABytes + item.half_n * 128u));
          uint8_t *dst = ring + at.stage * HEXIR_PAIR_STAGE_BYTES;
          const uint32_t bar = cluster_addr(&full[at.stage], 0);
          load_operand<A_MN>(dst, kBM, row0, kt * kBK,
                             [&](uint8_t *d, int32_t x, int32_t y) {
                               tma_load_2d_pair(d, map_a, x, y, bar);
                             });
          load_boxes<B_MN>(dst + kABytes, item.half_n, col0, kt * kBK,
                           [&](uint8_t *d, int32_t x, int32_t y) {
                             tma_load_2d_pair(d, map_b, x, y, bar);
                           });
        }
        __syncwarp();
      }
    }
    // Given up: the copies in flight land before the block ends.
    if (!ok && rank == 0)
      for (uint32_t i = fills > kStages ? fills - kStages : 0; i < fills; ++i)
        mbar_wait_pipeline(&full[i % kStages], i / kStages & 1u, p.timeout_ns);
  } else if (warp == 1 && rank == 0) {
    const bool leader = elect_one();
    const uint32_t whole = mma_desc<A_MN, B_MN>(2 * kBM, p.tile_n, p.is_f16 != 0);
    const uint32_t part = mma_desc<A_MN, B_MN>(2 * kBM, p.tile_n / 2, p.is_f16 != 0);
    const uint32_t ring_addr = smem_addr(ring);
    RingPlace at;
    uint32_t t = 0;
    bool ok = true, ready = false;
    for (uint32_t i = first; i < items && ok; i += step, ++t) {
      const uint32_t set = t & 1u;
      const uint32_t desc = i < p.full_tiles ? whole : part;
      ok = __all_sync(0xFFFFFFFFu, mbar_wait_pipeline(&sums_empty[set],
                                                      (t >> 1 & 1u) ^ 1u,
                                                      p.timeout_ns));
      if (!ok)
        break;
      tc_fence_after();
      for (uint32_t kt = 0; kt < p.k_tiles; ++kt) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_pipeline(&full[at.stage], at.parity,
                                                        p.timeout_ns, ready));
        if (!ok)
          break;
        tc_fence_after();
        const uint32_t stage = at.stage;
        const uint32_t a = ring_addr + stage * HEXIR_PAIR_STAGE_BYTES;
        at.next(kStages);
        // The next stage's barrier is tried under this one's MMAs.
        ready = mbar_test(&full[at.stage], at.parity);
        if (leader) {
          mma_stage<2, A_MN, B_MN>(tmem + set * 256u, a, a + kABytes, desc, kt == 0);
          mma_commit_pair(&empty[stage]);
          if (kt + 1 == p.k_tiles)
            mma_commit_pair(&sums_full[set]);
        }
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    const uint32_t quarter = warp & 3u, side = (warp - 4) / 4;
    const uint32_t row_in = rank * kBM + quarter * 32;
    Ahead<FORM> ahead(p, slots + (warp - 4) * (kAhead1 + 1) * kSlotBytes, lane);
    // A warp takes its half of a tile's columns in blocks of 16.
    uint32_t next_item = first, next_block = 0;
    auto fetch_next = [&] {
      Item next = {0, 0, 16};
      if (next_item < items)
        next = item_of(next_item);
      ahead.fetch(next.row0 + row_in, next.col0 + side * next.half_n + next_block * 16,
                  next_item < items);
      if (++next_block >= next.half_n / 16) {
        next_block = 0;
        next_item += step;
      }
    };
    for (uint32_t i = 0; i < ahead.depth; ++i)
      fetch_next();
    uint32_t t = 0;
    for (uint32_t item_at = first; item_at < items; item_at += step, ++t) {
      const Item item = item_of(item_at);
      const uint32_t row0 = item.row0 + row_in, blocks = item.half_n / 16;
      const uint32_t set = t & 1u;
      if (FORM == HEXIR_PRODUCT_FORWARD && p.bias)
        stage_bias(p, bias[warp - 4], item.col0 + side * item.half_n, item.half_n, lane);
      // The whole warp leaves together: its TMEM loads are warp-wide.
      if (!__all_sync(0xFFFFFFFFu,
                      mbar_wait_pipeline(&sums_full[set], t >> 1 & 1u,
                                         4 * p.timeout_ns)))
        break;
      tc_fence_after();
      const uint32_t src = tmem + (quarter * 32u << 16) + set * 256u;
      for (uint32_t i = 0; i < blocks; ++i) {
        const uint32_t c = side * item.half_n + i * 16;
        float v[16];
        __syncwarp();
        tmem_load16(src + c, v);
        if (i + 1 == blocks) {
          // The sums are in registers: the next tile but one may begin.
          tc_fence_before();
          __syncwarp();
          if (lane == 0)
            mbar_arrive_cluster(cluster_addr(&sums_empty[set], 0));
        }
        uint8_t *slot = ahead.arrived();
        finish_block<FORM>(p, v, bias[warp - 4] + i * 16, slot, ahead.out(), row0,
                           item.col0 + c, lane);
        __syncwarp();
        fetch_next();
      }
    }
    copies_wait<0>();
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
// instead of padding.  Bound by the weight's stream from HBM: 8192 x 8192 with
// one token 24.7 us (134 MB, 0.83 of copy bandwidth).
//
// GUARDED: rows that TMA cannot describe (a stride or base off 16 bytes).
// The epilogue warps load the operands with bounds checks, into the layout
// TMA would have written, and become the epilogue afterwards.  An operand
// that TMA can describe still comes by TMA.

constexpr uint32_t kLoaders = HEXIR_GUARDED_LOAD_WARPS * 32;  // threads
constexpr uint32_t kChunks = kBM * 8 / kLoaders;  // of an operand's tile, a thread

// The two 16-byte blocks of memory that each of a stage's chunks (8 elements of
// a row, which may start anywhere) lies in, as loaded.
struct Blocks {
  uint4 lo[kChunks], hi[kChunks];
  uint32_t apart;  // bit i: chunk i is to be taken element by element
};

// A load that stays where it is written.  Not a non-coherent one: those want
// memory that nothing writes during the kernel, which begins, up to its
// griddep_wait, while the kernel before may still write the operands.
__device__ __forceinline__ uint4 load_now(uintptr_t at) {
  uint4 w;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
               : "l"(at)
               : "memory");
  return w;
}

// One thread's chunks of an operand's 128 x 64 tiles: chunk i is 8 elements of
// 128-byte row (i * 64 + warp / 8 * 32 + lane / 8 * 8 + warp % 8) of the stage.
// The chunks of a warp, in every tile, start at the same byte of a 16-byte
// block: their rows are 8 apart (and 64 elements or 64 values of the sum), and
// each of these is a multiple of 16 bytes whatever the stride.  So the words to
// shift by are the warp's, taken by a branch, and only halves are shifted by
// instructions.
//
// A k tile wholly inside the operand along the sum, whose blocks lie wholly
// inside the tensor's memory (from its first element to its last, gaps between
// rows included), needs no checks: chunks beyond the operand's side read the
// side's first instead, and what they leave in the sums is never stored.  In
// the others (the last k tiles, and the first at the tensor's start) every
// chunk is checked, and the few whose blocks reach outside the memory are taken
// element by element.
//
// A stage of two such operands takes 0.7 us, of one 0.5, by TMA 0.23; with
// checks in the loop, 8 warps and words shifted by selects it took 1.5, with
// every chunk checked 3.6.  What is left is shared-memory and L1 wavefronts
// (two loads and a store of every chunk) and the issue of some 15 instructions
// a chunk: 777 x 1001 x 1537 19.6 us, 2048 cubed off alignment 67.

__device__ __forceinline__ uintptr_t element_at(const void *p, uint64_t ld, bool mn,
                                                uint32_t s, uint32_t k) {
  return reinterpret_cast<uintptr_t>(p) + (mn ? k * ld + s : s * ld + k) * 2;
}

// One past an operand's last element.
__device__ __forceinline__ uintptr_t memory_end(const void *p, uint64_t ld, bool mn,
                                                uint32_t sides, uint32_t depth) {
  return depth ? element_at(p, ld, mn, sides - 1, depth - 1) + 2
               : reinterpret_cast<uintptr_t>(p);
}

// Leaves of the k tiles [inner0, inner1) those that need no checks of a tile
// that starts at side0: blocks from the one of its first element to 32 bytes
// past the start of its last lie in the memory.
__device__ __forceinline__ void keep_inner(const void *p, uint64_t ld, bool mn,
                                           uint32_t sides, uint32_t depth,
                                           uint32_t side0, uint32_t &inner0,
                                           uint32_t &inner1) {
  const uint64_t step = mn ? ld * (2 * kBK) : 2 * kBK;
  const uintptr_t low =
      element_at(p, ld, mn, side0, 0) & ~static_cast<uintptr_t>(15);
  const uintptr_t high =
      element_at(p, ld, mn, min(side0 + kBM, sides) - 1, kBK - 1) + 32;
  const uintptr_t end = memory_end(p, ld, mn, sides, depth);
  if (low < reinterpret_cast<uintptr_t>(p))
    inner0 = max(inner0, 1u);
  inner1 = min(inner1, depth / kBK);
  while (inner1 > inner0 && high + (inner1 - 1) * step > end)
    --inner1;
}

template <bool MN>
struct GuardedOperand {
  uintptr_t block[kChunks];     // of k tile 0
  uintptr_t first, last, safe;  // the tensor; its first whole block
  uint64_t step;                // bytes to the next k tile
  uint32_t depth;
  uint32_t shift;               // bytes into a block
  uint32_t side_counts;         // 4 bits a chunk: elements inside the side
  uint32_t k0, dst0;            // chunk 0: of the sum; byte in the stage

  __device__ __forceinline__ GuardedOperand(const void *p, uint64_t ld,
                                            uint32_t sides, uint32_t depth_,
                                            uint32_t side0, uint32_t warp,
                                            uint32_t lane)
      : depth(depth_) {
    const uint32_t row0 = warp / 8 * 32 + lane / 8 * 8 + warp % 8;
    const uint32_t column = lane % 8 * 8;
    first = reinterpret_cast<uintptr_t>(p);
    last = memory_end(p, ld, MN, sides, depth);
    safe = (first + 15) & ~static_cast<uintptr_t>(15);
    step = MN ? ld * (2 * kBK) : 2 * kBK;
    k0 = MN ? row0 : column;
    dst0 = row0 * 128 + ((lane % 8 ^ warp % 8) << 4);
    // Within a warp the major index is the same but for multiples of 8.
    const uint64_t major = (MN ? 0 : side0) + warp % 8;
    shift = static_cast<uint32_t>(first + major * ld * 2) & 15u;
    side_counts = 0;
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
      const uint32_t row = i * 64 + row0;
      uint32_t s = side0 + (MN ? i * 64 + column : row);
      const uint32_t n = s >= sides ? 0u : (MN ? min(8u, sides - s) : 8u);
      side_counts |= n << 4 * i;
      s = n ? s : side0;
      block[i] = element_at(p, ld, MN, s, MN ? row0 : column) &
                 ~static_cast<uintptr_t>(15);
    }
  }
  // Elements of chunk i that the operand has.
  __device__ __forceinline__ uint32_t count(uint32_t i, uint32_t kt) const {
    const uint32_t k = kt * kBK + k0;
    const uint32_t n = side_counts >> 4 * i & 15u;
    return k >= depth ? 0u : (MN ? n : min(n, depth - k));
  }

  // A k tile without checks: the blocks at `block`, which is on the tile.
  __device__ __forceinline__ void load_inner(Blocks &b) {
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
      b.lo[i] = load_now(block[i]);
      b.hi[i] = load_now(block[i] + 16);
      block[i] += step;
    }
  }
  __device__ __forceinline__ void load_checked(uint32_t kt, Blocks &b) const {
    b.apart = 0;
    const bool any = safe + 16 <= last;
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
      const uint32_t n = count(i, kt);
      const uintptr_t at = block[i] + kt * step;
      const bool two = shift + 2 * n > 16;
      const bool inside = at >= first && at + (two ? 32 : 16) <= last;
      b.apart |= static_cast<uint32_t>(n && !inside) << i;
      const bool use = n && inside;
      if (any) {
        b.lo[i] = load_now(use ? at : safe);
        b.hi[i] = load_now(use && two ? at + 16 : safe);
      }
    }
  }
  // The chunks, WORDS 32-bit words and possibly a half into their blocks.
  template <int WORDS>
  __device__ __forceinline__ void store_shifted(const Blocks &b, uint8_t *dst) const {
    const uint32_t half = (shift & 2u) * 8u;
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
      const uint32_t w[9] = {b.lo[i].x, b.lo[i].y, b.lo[i].z, b.lo[i].w, b.hi[i].x,
                             b.hi[i].y, b.hi[i].z, b.hi[i].w, 0};
      uint4 out;
      out.x = __funnelshift_r(w[WORDS], w[WORDS + 1], half);
      out.y = __funnelshift_r(w[WORDS + 1], w[WORDS + 2], half);
      out.z = __funnelshift_r(w[WORDS + 2], w[WORDS + 3], half);
      out.w = __funnelshift_r(w[WORDS + 3], w[WORDS + 4], half);
      *reinterpret_cast<uint4 *>(dst + i * (kLoaders * 16)) = out;
    }
  }
  // Into the stage, as TMA's 128-byte swizzle would have it.
  __device__ __forceinline__ void store_inner(const Blocks &b, uint8_t *stage,
                                              uint32_t words) const {
    // The rows of a thread's chunks are 64 apart, so they swizzle alike.
    uint8_t *dst = stage + dst0;
    if (words < 2) {
      if (words == 0)
        store_shifted<0>(b, dst);
      else
        store_shifted<1>(b, dst);
    } else if (words == 2) {
      store_shifted<2>(b, dst);
    } else {
      store_shifted<3>(b, dst);
    }
  }
  // Elements beyond the sum are 0.
  __device__ __forceinline__ void store_checked(uint32_t kt, const Blocks &b,
                                                uint8_t *stage) const {
    uint8_t *dst = stage + dst0;
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
      uint32_t w[8] = {b.lo[i].x, b.lo[i].y, b.lo[i].z, b.lo[i].w,
                       b.hi[i].x, b.hi[i].y, b.hi[i].z, b.hi[i].w};
#pragma unroll
      for (int j = 0; j < 6; ++j)
        w[j] = shift & 8u ? w[j + 2] : w[j];
#pragma unroll
      for (int j = 0; j < 5; ++j)
        w[j] = shift & 4u ? w[j + 1] : w[j];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = __funnelshift_r(w[j], w[j + 1], (shift & 2u) * 8u);
      const uint32_t n = count(i, kt);
      if (b.apart >> i & 1u) {
        const uint16_t *src =
            reinterpret_cast<const uint16_t *>(block[i] + kt * step + shift);
        uint32_t e[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
          e[j] = src[min(j, n - 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = e[2 * j] | e[2 * j + 1] << 16;
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        w[j] = n >= 2 * j + 2 ? w[j] : (n == 2 * j + 1 ? w[j] & 0xFFFFu : 0u);
      *reinterpret_cast<uint4 *>(dst + i * (kLoaders * 16)) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

template <int FORM, bool GUARDED, bool SWAP>
__device__ __forceinline__ void product_single(const CUtensorMap *map_a,
                                               const CUtensorMap *map_b,
                                               const Args &p) {
  constexpr bool A_MN = SWAP || FORM == HEXIR_PRODUCT_WEIGHT_GRAD;
  constexpr bool B_MN = !SWAP && FORM != HEXIR_PRODUCT_INPUT_GRAD;
  constexpr uint32_t kMax = HEXIR_SINGLE_MAX_STAGES;
  constexpr uint32_t kWarps = HEXIR_SINGLE_EPILOGUE_WARPS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMax], empty[kMax], done;
  __shared__ uint32_t tmem_slot;
  __shared__ alignas(16) float bias[SWAP ? 1 : kWarps][64];
  uint8_t *ring = align1024(smem_raw);
  uint8_t *slots = ring + p.ring_bytes;
  const uint32_t warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x / 32, 0);
  const uint32_t lane = threadIdx.x % 32;
  const uint32_t rank = p.split > 1 ? cluster_ctarank() : 0;
  const uint32_t stages = p.stages;
  const uint32_t b_bytes = p.tile_n * 128u;
  const uint32_t stage_bytes = kABytes + b_bytes;
  // Which operands come by TMA.
  const bool tma_a = !GUARDED || (p.tma_operands & 1u);
  const bool tma_b = !GUARDED || (p.tma_operands & 2u);
  const uint32_t tma_bytes = (tma_a ? kABytes : 0u) + (tma_b ? b_bytes : 0u);

  if (threadIdx.x == 0) {
    if (tma_a)
      prefetch_tensormap(map_a);
    if (tma_b)
      prefetch_tensormap(map_b);
    for (uint32_t s = 0; s < stages; ++s) {
      mbar_init(&full[s], (GUARDED ? kLoaders / 32 : 0u) + (tma_bytes ? 1u : 0u));
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
  griddep_wait();  // nothing global is read or written before this
  griddep_launch_dependents();

  // The tile, and this CTA's share of its sum.
  uint32_t tm, tn;
  tile_of(blockIdx.x / p.split, p.tiles_m, p.tiles_n, p.group_m, tm, tn);
  const uint32_t kt0 = static_cast<uint32_t>(
      static_cast<uint64_t>(p.k_tiles) * rank / p.split);
  const uint32_t kt1 = static_cast<uint32_t>(
      static_cast<uint64_t>(p.k_tiles) * (rank + 1) / p.split);
  const uint32_t lane0 = tm * kBM, col0 = tn * p.tile_n;
  // GUARDED: of these, [inner0, inner1) need no checks.  The others come first,
  // so that what checking needs is no longer there in the loop without checks.
  uint32_t inner0 = kt0, inner1 = kt1;
  if (GUARDED) {
    if (!tma_a)
      keep_inner(p.a, p.lda, A_MN, p.rows, p.depth, lane0, inner0, inner1);
    if (!tma_b)
      keep_inner(p.b, p.ldb, B_MN, p.cols, p.depth, col0, inner0, inner1);
    if (inner0 >= inner1)
      inner0 = inner1 = kt1;
  }
  const uint32_t head = inner0 - kt0, checked = head + (kt1 - inner1);
  auto nth_tile = [&](uint32_t i) {
    return !GUARDED || i < head ? kt0 + i
           : i < checked        ? inner1 + (i - head)
                                : inner0 + (i - checked);
  };
  // The epilogue warps: 32 lanes' rows, and every other block of 16 columns
  // (of the cluster's share of them, once the sums are joined).
  const uint32_t quarter = warp & 3u, side = warp >= 2 ? (warp - 2) / 4 : 0;
  const uint32_t row0 = lane0 + quarter * 32;
  const uint32_t blocks = p.tile_n / 16;
  const uint32_t block0 = rank * 2 + side, block_step = 2 * p.split;
  Ahead<FORM> ahead(p, slots + (warp >= 2 ? warp - 2 : 0) * (kAhead1 + 1) * kSlotBytes,
                    lane);
  uint32_t next_block = block0;
  auto fetch_next = [&] {
    ahead.fetch(row0, col0 + next_block * 16, next_block < blocks);
    next_block += block_step;
  };
  bool ok = true;

  if (warp == 0) {
    if (tma_bytes) {
      const bool leader = elect_one();
      RingPlace at;
      uint32_t fills = 0;
      for (; fills < kt1 - kt0; ++fills, at.next(stages)) {
        const uint32_t kt = nth_tile(fills);
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_pipeline(&empty[at.stage],
                                                        at.parity ^ 1u, p.timeout_ns));
        if (!ok)
          break;
        if (leader) {
          uint64_t *bar = &full[at.stage];
          mbar_arrive_expect_tx(bar, tma_bytes);
          uint8_t *dst = ring + at.stage * stage_bytes;
          if (tma_a)
            load_operand<A_MN>(dst, kBM, lane0, kt * kBK,
                               [&](uint8_t *d, int32_t x, int32_t y) {
                                 tma_load_2d(d, map_a, x, y, bar);
                               });
          if (tma_b)
            load_operand<B_MN>(dst + kABytes, p.tile_n, col0, kt * kBK,
                               [&](uint8_t *d, int32_t x, int32_t y) {
                                 tma_load_2d(d, map_b, x, y, bar);
                               });
        }
        __syncwarp();
      }
      // Given up: the copies in flight land before the block ends (with loads
      // beside them the phase may not complete: the wait is bounded).
      if (!ok)
        for (uint32_t i = fills > stages ? fills - stages : 0; i < fills; ++i)
          mbar_wait_pipeline(&full[i % stages], i / stages & 1u, p.timeout_ns);
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t desc = mma_desc<A_MN, B_MN>(kBM, p.tile_n, p.is_f16 != 0);
    const uint32_t ring_addr = smem_addr(ring);
    RingPlace at;
    bool ready = false;
    for (uint32_t kt = kt0; kt < kt1; ++kt) {
      if (!__all_sync(0xFFFFFFFFu, mbar_wait_pipeline(&full[at.stage], at.parity,
                                                      p.timeout_ns, ready)))
        break;
      tc_fence_after();
      const uint32_t stage = at.stage;
      const uint32_t a = ring_addr + stage * stage_bytes;
      at.next(stages);
      // The next stage's barrier is tried under this one's MMAs.
      ready = mbar_test(&full[at.stage], at.parity);
      if (leader) {
        mma_stage<1, A_MN, B_MN>(tmem, a, a + kABytes, desc, kt == kt0);
        mma_commit(&empty[stage]);
      }
      __syncwarp();
    }
    if (leader)
      mma_commit(&done);  // also after a wait that ran out: nothing in flight
  } else {
    if (!SWAP && warp < 2 + kWarps) {
      for (uint32_t i = 0; i < ahead.depth; ++i)
        fetch_next();
      if (FORM == HEXIR_PRODUCT_FORWARD && p.bias) {
        // Block i of this warp has bias[16 i ..].
        __syncwarp();
        for (uint32_t i = lane; i < blocks * 8; i += 32) {
          const uint32_t c = col0 + (block0 + i / 16 * block_step) * 16 + i % 16;
          bias[warp - 2][i] =
              block0 + i / 16 * block_step < blocks && c < p.cols
                  ? from_bits(static_cast<const uint16_t *>(p.bias)[c], p.is_f16 != 0)
                  : 0.0f;
        }
        __syncwarp();
      }
    }
    if (GUARDED) {
      GuardedOperand<A_MN> a(p.a, p.lda, p.rows, p.depth, lane0, warp - 2, lane);
      GuardedOperand<B_MN> b(p.b, p.ldb, p.cols, p.depth, col0, warp - 2, lane);
      RingPlace at;
      const uint32_t words_a = __shfl_sync(0xFFFFFFFFu, a.shift / 4, 0);
      const uint32_t words_b = __shfl_sync(0xFFFFFFFFu, b.shift / 4, 0);
      bool going = true;
      auto empty_stage = [&] {
        going = __all_sync(0xFFFFFFFFu, mbar_wait_pipeline(&empty[at.stage],
                                                           at.parity ^ 1u, p.timeout_ns));
        return ring + at.stage * stage_bytes;
      };
      auto filled = [&] {
        fence_async_smem();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&full[at.stage]);
        at.next(stages);
      };
      Blocks ra[2], rb[2];
#pragma unroll 1
      for (uint32_t i = 0; i < checked && going; ++i) {
        const uint32_t kt = nth_tile(i);
        if (!tma_a)
          a.load_checked(kt, ra[0]);
        if (!tma_b)
          b.load_checked(kt, rb[0]);
        uint8_t *dst = empty_stage();
        if (going) {
          if (!tma_a)
            a.store_checked(kt, ra[0], dst);
          if (!tma_b)
            b.store_checked(kt, rb[0], dst + kABytes);
          filled();
        }
      }
#pragma unroll
      for (uint32_t i = 0; i < kChunks; ++i) {
        a.block[i] += inner0 * a.step;
        b.block[i] += inner0 * b.step;
      }
      // The loads of one stage are in flight while the last one's are shifted
      // into place and stored.
      auto load = [&](Blocks &xa, Blocks &xb) {
        if (!tma_a)
          a.load_inner(xa);
        if (!tma_b)
          b.load_inner(xb);
      };
      auto settle = [&](const Blocks &xa, const Blocks &xb) {
        uint8_t *dst = empty_stage();
        if (going) {
          if (!tma_a)
            a.store_inner(xa, dst, words_a);
          if (!tma_b)
            b.store_inner(xb, dst + kABytes, words_b);
          filled();
        }
      };
      uint32_t left = inner1 - inner0;
      if (left)
        load(ra[0], rb[0]);
#pragma unroll 1
      while (left && going) {
        if (left > 1)
          load(ra[1], rb[1]);
        settle(ra[0], rb[0]);
        if (left == 1 || !going)
          break;
        if (left > 2)
          load(ra[0], rb[0]);
        settle(ra[1], rb[1]);
        left -= 2;
      }
      __syncwarp();
    }
  }

  const bool finishes = warp >= 2 && warp < 2 + kWarps;
  if (finishes) {
    ok = __all_sync(0xFFFFFFFFu,
                    mbar_wait_pipeline(&done, 0, 4 * p.timeout_ns));
    tc_fence_after();
    const uint32_t src = tmem + (quarter * 32u << 16);
    const uint32_t my = quarter * 32 + lane;
    // split > 1: this CTA's sums, [tile_n / 4][128] of 4.
    float4 *sums = reinterpret_cast<float4 *>(ring);
    if (ok) {
      for (uint32_t n = side; n < blocks; n += 2) {
        float v[16];
        __syncwarp();
        if (kt1 > kt0) {
          tmem_load16(src + n * 16, v);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            v[i] = 0.0f;
        }
        if (p.split > 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sums[(n * 4 + i) * kBM + my] =
                make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else if (SWAP) {
          finish_column16(p, v, col0 + n * 16, lane0 + my);
        } else {
          uint8_t *slot = ahead.arrived();
          finish_block<FORM>(p, v, bias[warp - 2] + n / 2 * 16, slot, ahead.out(),
                             row0, col0 + n * 16, lane);
          __syncwarp();
          fetch_next();
        }
      }
    }
  }

  if (p.split > 1) {
    __syncwarp();
    cluster_sync();
    if (finishes && ok) {
      const uint32_t my = quarter * 32 + lane;
      const float4 *sums = reinterpret_cast<const float4 *>(ring);
      uint32_t nth = 0;
      for (uint32_t n = block0; n < blocks; n += block_step, ++nth) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] = 0.0f;
#pragma unroll 2
        for (uint32_t r = 0; r < p.split; ++r) {
          const uint32_t from = cluster_addr(sums + n * 4 * kBM + my, r);
          float4 q[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            q[i] = ld_cluster_v4(from + i * (kBM * 16u));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[4 * i] += q[i].x;
            v[4 * i + 1] += q[i].y;
            v[4 * i + 2] += q[i].z;
            v[4 * i + 3] += q[i].w;
          }
        }
        if (SWAP) {
          finish_column16(p, v, col0 + n * 16, lane0 + my);
        } else {
          uint8_t *slot = ahead.arrived();
          finish_block<FORM>(p, v, bias[warp - 2] + nth * 16, slot, ahead.out(), row0,
                             col0 + n * 16, lane);
          __syncwarp();
          fetch_next();
        }
      }
    }
    __syncwarp();
    cluster_sync();  // the peers have read this CTA's sums
  }
  if (finishes)
    copies_wait<0>();
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
  extern "C" __global__ void __launch_bounds__(HEXIR_SINGLE_THREADS, 2)       \
      NAME(const __grid_constant__ CUtensorMap map_a,                         \
           const __grid_constant__ CUtensorMap map_b, const Args args) {      \
    product_single<FORM, false, SWAP>(&map_a, &map_b, args);                  \
  }
#define PRODUCT_GUARDED(NAME, FORM)                                           \
  extern "C" __global__ void __launch_bounds__(HEXIR_GUARDED_THREADS)         \
      NAME(const __grid_constant__ CUtensorMap map_a,                         \
           const __grid_constant__ CUtensorMap map_b, const Args args) {      \
    product_single<FORM, true, false>(&map_a, &map_b, args);                  \
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
