// layer_norm.cu -- layer norm and its gradient over the rows of a row-major
// tensor (include/hexir_b200/layers.h), and the elementwise gradient of a
// linear layer's epilogue with its column sums.
//
// A row is held in the registers of its threads (a warp's or a block's), so
// each pass reads its tensors once: forward x -> y, backward x, dy
// (, residual) -> dx.  Both are bound by HBM; rows longer than a block holds
// are read again from L2.  16384 x 4096, forward / gradient with its sums, and
// the share of the measured copy bandwidth: bf16 45.1 / 75.1 us (0.91 / 0.82),
// f32 85.6 / 134 (0.96 / 0.92), f64 190 / 261 (0.86 / 0.94).  The 16-bit gradient
// is as much bound by its conversions (issue slots 59 % busy at two blocks an
// SM; three, with their sums spilled, took 117 us).
//
// The gradients of gamma, beta and the bias are sums over rows: each block
// adds up its rows in registers and leaves one partial row in the caller's
// workspace, and a second kernel adds the partial rows in order.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "activation_f32.cuh"
#include "common.cuh"
#include "layers_abi.h"
#include "norm_ring.h"
#include "two.cuh"

using namespace hexir;

namespace {

// Storage types, the type they are computed in, and elements per 16 bytes.
template <typename T>
struct Real {
  typedef float type;
};
template <>
struct Real<double> {
  typedef double type;
};
template <typename T>
using real_t = typename Real<T>::type;

__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T narrow(real_t<T> v);
template <>
__device__ __forceinline__ double narrow<double>(double v) { return v; }
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// 16 bytes of a row.  widen_pack / narrow_pack convert whole words, two 16-bit
// elements at a time: element by element, the conversions were what bounded
// the 16-bit kernels (0.55 of copy bandwidth at 16384 x 4096, f32 0.92).
template <typename T>
struct Pack {
  static constexpr int kN = 16 / sizeof(T);
  uint4 w;
};

__device__ __forceinline__ void widen_pack(const Pack<double> &p,
                                           Two<double> (&f)[1]) {
  f[0] = {__hiloint2double(static_cast<int>(p.w.y), static_cast<int>(p.w.x)),
          __hiloint2double(static_cast<int>(p.w.w), static_cast<int>(p.w.z))};
}
__device__ __forceinline__ void widen_pack(const Pack<float> &p,
                                           Two<float> (&f)[2]) {
  f[0] = {__uint_as_float(p.w.x), __uint_as_float(p.w.y)};
  f[1] = {__uint_as_float(p.w.z), __uint_as_float(p.w.w)};
}
__device__ __forceinline__ void widen_pack(const Pack<__nv_bfloat16> &p,
                                           Two<float> (&f)[4]) {
  const uint32_t w[4] = {p.w.x, p.w.y, p.w.z, p.w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f[i] = {__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)};
}
__device__ __forceinline__ void widen_pack(const Pack<__half> &p,
                                           Two<float> (&f)[4]) {
  const uint32_t w[4] = {p.w.x, p.w.y, p.w.z, p.w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    f[i] = {v.x, v.y};
  }
}
__device__ __forceinline__ void narrow_pack(const Two<double> (&f)[1],
                                            Pack<double> &p) {
  p.w = make_uint4(__double2loint(f[0].x), __double2hiint(f[0].x),
                   __double2loint(f[0].y), __double2hiint(f[0].y));
}
__device__ __forceinline__ void narrow_pack(const Two<float> (&f)[2],
                                            Pack<float> &p) {
  p.w = make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y),
                   __float_as_uint(f[1].x), __float_as_uint(f[1].y));
}
__device__ __forceinline__ uint32_t bits2(const __nv_bfloat162 &h) {
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t bits2(const __half2 &h) {
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void narrow_pack(const Two<float> (&f)[4],
                                            Pack<__nv_bfloat16> &p) {
  p.w = make_uint4(bits2(__floats2bfloat162_rn(f[0].x, f[0].y)),
                   bits2(__floats2bfloat162_rn(f[1].x, f[1].y)),
                   bits2(__floats2bfloat162_rn(f[2].x, f[2].y)),
                   bits2(__floats2bfloat162_rn(f[3].x, f[3].y)));
}
__device__ __forceinline__ void narrow_pack(const Two<float> (&f)[4],
                                            Pack<__half> &p) {
  p.w = make_uint4(bits2(__floats2half2_rn(f[0].x, f[0].y)),
                   bits2(__floats2half2_rn(f[1].x, f[1].y)),
                   bits2(__floats2half2_rn(f[2].x, f[2].y)),
                   bits2(__floats2half2_rn(f[3].x, f[3].y)));
}

// Element j of a pack, for the packs at a row's ends.
template <typename T>
__device__ __forceinline__ T pack_get(const Pack<T> &p, int j) {
  T v[Pack<T>::kN];
  *reinterpret_cast<uint4 *>(v) = p.w;
  return v[j];
}

// How a row lies over its threads.
//   kWhole    16-byte packs tid, tid + TH, ... of a row that starts and ends on
//             16-byte boundaries;
//   kShifted  the same packs of memory, but the row starts `phase` elements
//             after a boundary: its first pack is filled from element `phase`
//             on (16-bit types and long f32 rows; every tensor of the call has
//             the same phase, and a thread's rows are a multiple of 8 apart so
//             that they share it);
//   kAny      single elements tid, tid + TH, ..., so that a warp's accesses
//             stay consecutive.
enum Layout { kWhole, kShifted, kAny };

// The packs at the ends of a shifted row, an element at a time.  They stand
// behind branches that a whole warp takes or not: as predicated instructions
// they were more than half of what every pack cost (410 instructions a warp
// and row of 16 elements a thread, 243 without), and as calls they made their
// warp wait for its loads in flight.
template <typename T>
__device__ __forceinline__ uint4 gather_pack(const T *row, uint32_t column,
                                             uint32_t cols) {
  constexpr int kN = Pack<T>::kN;
  T e[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j)
    e[j] = column + j < cols ? row[column + j] : narrow<T>(real_t<T>(0));
  return *reinterpret_cast<const uint4 *>(e);
}
template <typename T>
__device__ __forceinline__ void scatter_pack(T *row, uint32_t column,
                                             uint32_t cols, uint4 v) {
  constexpr int kN = Pack<T>::kN;
  T e[kN];
  *reinterpret_cast<uint4 *>(e) = v;
#pragma unroll
  for (int j = 0; j < kN; ++j)
    if (column + j < cols)
      row[column + j] = e[j];
}
// The elements of a tensor from its first to its last, gaps between rows
// included: what a load may touch.
struct Span {
  uintptr_t first, last;
  __device__ __forceinline__ bool holds16(const void *p) const {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return at >= first && at + 16 <= last;
  }
};
template <typename T>
__device__ __forceinline__ Span span_of(const T *p, uint64_t ld, uint64_t rows,
                                        uint32_t cols) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  return {at, at + ((rows - 1) * ld + cols) * sizeof(T)};
}

template <typename T, int TH, int NE, int LAYOUT>
struct Row {
  static constexpr int kN = Pack<T>::kN;
  static constexpr int kPacks = NE / kN;
  uint32_t tid, cols, phase;
  // Shifted rows, a bit per pack: whether it has elements of the row, whether
  // it has others too, and whether such a one is in this warp.
  uint32_t some_bits, cut_bits, warp_cut_bits;

  __device__ __forceinline__ Row(uint32_t tid_, uint32_t cols_, const void *row)
      : tid(tid_), cols(cols_), phase(0), some_bits(0), cut_bits(0),
        warp_cut_bits(0) {
    if (LAYOUT == kShifted) {
      phase = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        const uint32_t c = column(i, 0);
        const bool has = (i * TH + tid) * kN < cols + phase;
        some_bits |= static_cast<uint32_t>(has) << i;
        cut_bits |= static_cast<uint32_t>(has && (c >= cols || cols - c < kN)) << i;
      }
      warp_cut_bits = __reduce_or_sync(0xFFFFFFFFu, cut_bits);
    }
  }
  // Column of element j of pack i; wraps below 0 for the elements before the
  // row, so `column < cols` holds for the row's elements alone.
  __device__ __forceinline__ uint32_t column(int i, int j) const {
    return LAYOUT != kAny ? (i * TH + tid) * kN + j - phase
                          : (i * kN + j) * TH + tid;
  }
  __device__ __forceinline__ bool some(int i) const {
    return LAYOUT == kShifted ? (some_bits >> i & 1u) != 0 : column(i, 0) < cols;
  }
  __device__ __forceinline__ bool cut(int i) const {
    return LAYOUT == kShifted && (cut_bits >> i & 1u) != 0;
  }
  __device__ __forceinline__ bool warp_cut(int i) const {
    return LAYOUT == kShifted && (warp_cut_bits >> i & 1u) != 0;
  }
  // A cut pack with the elements outside the row (its neighbours' or the
  // gap's) zeroed.
  __device__ __forceinline__ uint4 inside(uint4 w, int i) const {
    const uint32_t c = column(i, 0);
    uint32_t m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (sizeof(T) == 2)
        m[j] = (c + 2 * j < cols ? 0xFFFFu : 0u) |
               (c + 2 * j + 1 < cols ? 0xFFFF0000u : 0u);
      else
        m[j] = c + static_cast<uint32_t>(j * 4 / sizeof(T)) < cols ? 0xFFFFFFFFu : 0u;
    }
    return make_uint4(w.x & m[0], w.y & m[1], w.z & m[2], w.w & m[3]);
  }
  // The row's packs; a cut one may carry its neighbours' elements until
  // clean() (which a load must not wait for).  `edge`: such a pack may reach
  // outside the tensor (norm_row_at_edge).
  __device__ __forceinline__ void load(const T *row, const Span &span, bool edge,
                                       Pack<T> (&v)[kPacks]) const {
#pragma unroll
    for (int i = 0; i < kPacks; ++i)
      v[i] = load_pack<true>(row, i, span, edge);
  }
  __device__ __forceinline__ void clean(Pack<T> (&v)[kPacks]) const {
#pragma unroll
    for (int i = 0; i < kPacks; ++i)
      if (warp_cut(i))
        v[i].w = inside(v[i].w, i);
  }
  __device__ __forceinline__ bool apart(const T *row, int i, const Span &span) const {
    return cut(i) && !span.holds16(row + static_cast<int32_t>(column(i, 0)));
  }
  // STREAM: read once, not kept in L1 (where gamma and beta are).
  template <bool STREAM>
  __device__ __forceinline__ Pack<T> load_pack(const T *row, int i,
                                               const Span &span, bool edge) const {
    Pack<T> v;
    v.w = make_uint4(0, 0, 0, 0);
    if (LAYOUT == kAny) {
      T e[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const uint32_t c = column(i, j);
        e[j] = c < cols ? row[c] : narrow<T>(real_t<T>(0));
      }
      v.w = *reinterpret_cast<const uint4 *>(e);
      return v;
    }
    const uint4 *at =
        reinterpret_cast<const uint4 *>(row + static_cast<int32_t>(column(i, 0)));
    if (LAYOUT == kShifted && edge && warp_cut(i)) {
      if (apart(row, i, span))
        v.w = gather_pack(row, column(i, 0), cols);
      else if (some(i))
        v.w = *at;
    } else if (some(i)) {
      v.w = STREAM ? __ldcs(at) : *at;
    }
    return v;
  }
  __device__ __forceinline__ void store(T *row, int i, const Pack<T> &v) const {
    if (LAYOUT == kAny) {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const uint32_t c = column(i, j);
        if (c < cols)
          row[c] = pack_get(v, j);
      }
      return;
    }
    uint4 *at = reinterpret_cast<uint4 *>(row + static_cast<int32_t>(column(i, 0)));
    if (warp_cut(i)) {
      if (cut(i))
        scatter_pack(row, column(i, 0), cols, v.w);
      else if (some(i))
        __stcs(at, v.w);
    } else if (some(i)) {
      __stcs(at, v.w);
    }
  }
  // Pack i of gamma or beta, which start at column 0: as the row's packs
  // lie.
  __device__ __forceinline__ Pack<T> parameter(const T *p, int i) const {
    if (LAYOUT != kShifted)
      return load_pack<false>(p, i, Span{}, false);
    Pack<T> v;
    v.w = gather_pack(p, column(i, 0), cols);
    return v;
  }
};

// Every thread of a row: all of the block's, or, where a block has several
// rows, of a named barrier per row.
template <int TH>
__device__ __forceinline__ void row_sync() {
  if (TH >= 256)
    __syncthreads();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.x / TH + 1), "n"(TH) : "memory");
}

// Sum over the TH threads of a row, in an order that depends on TH alone.
// `slot` holds a value per warp of the block (two for row_sum2); calls
// alternate between two slots, so one barrier per call is enough.
template <int TH, typename R>
__device__ __forceinline__ void row_sum(R &a, R *slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
  if (TH == 32)
    return;
  if (threadIdx.x % 32 == 0)
    slot[threadIdx.x / 32] = a;
  row_sync<TH>();
  slot += threadIdx.x / TH * (TH / 32);
  a = slot[0];
#pragma unroll
  for (int w = 1; w < TH / 32; ++w)
    a += slot[w];
}

template <int TH, typename R>
__device__ __forceinline__ void row_sum2(R &a, R &b, R *slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
    b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
  }
  if (TH == 32)
    return;
  if (threadIdx.x % 32 == 0) {
    slot[2 * (threadIdx.x / 32)] = a;
    slot[2 * (threadIdx.x / 32) + 1] = b;
  }
  row_sync<TH>();
  slot += threadIdx.x / TH * (2 * TH / 32);
  a = slot[0];
  b = slot[1];
#pragma unroll
  for (int w = 1; w < TH / 32; ++w) {
    a += slot[2 * w];
    b += slot[2 * w + 1];
  }
}

__device__ __forceinline__ float inv_sqrt(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inv_sqrt(double v) { return rsqrt(v); }

// Rows of up to TH * NE columns, several to a block of 256 threads where TH is
// less.
// Blocks are persistent and load their next row before they work on the
// present one, so that HBM is read while the row's sums and barriers run; the
// row stays packed in registers, which lets several blocks share an SM.
template <typename T, int TH, int NE, int LAYOUT>
__device__ __forceinline__ void norm_rows(const hexir_layer_norm_args_t &p) {
  typedef real_t<T> R;
  typedef Row<T, TH, NE, LAYOUT> Lay;
  constexpr int kN = Lay::kN, kPacks = Lay::kPacks;
  constexpr uint32_t kRows = TH < 256 ? 256 / TH : 1;
  __shared__ R slots[2][kRows * TH / 32];
  extern __shared__ uint4 copies[];  // gamma and beta as this block's rows lie
  const uint32_t tid = threadIdx.x % TH, group = threadIdx.x / TH;
  griddep_wait();  // nothing global is read or written before this
  griddep_launch_dependents();
  const R n = static_cast<R>(p.cols), inv_n = R(1) / n;
  const T *x_rows = static_cast<const T *>(p.x);
  const T *gamma = static_cast<const T *>(p.gamma);
  const T *beta = static_cast<const T *>(p.beta);
  const uint64_t step = (uint64_t)gridDim.x * kRows;
  uint64_t row = (uint64_t)blockIdx.x * kRows + group;
  if (row >= p.rows)
    return;
  const Lay lay(tid, p.cols, x_rows + row * p.ldx);
  const Span span = span_of(x_rows, p.ldx, p.rows, p.cols);
  Pack<T> x[kPacks], next[kPacks];
  lay.load(x_rows + row * p.ldx, span, norm_row_at_edge<kN>(row, p.rows, p.cols), x);
  // Shifted rows: gamma and beta as this row's packs lie, in shared memory.
  // Each thread reads back only what it writes here.
  uint4 *gamma_copy = copies + group * (2 * TH * kPacks);
  uint4 *beta_copy = gamma_copy + TH * kPacks;
  if (LAYOUT == kShifted) {
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      if (gamma)
        gamma_copy[i * TH + tid] = lay.parameter(gamma, i).w;
      if (beta)
        beta_copy[i * TH + tid] = lay.parameter(beta, i).w;
    }
  }
  for (;; row += step) {
    const bool more = row + step < p.rows;
    lay.clean(x);
    if (more)
      lay.load(x_rows + (row + step) * p.ldx, span,
               norm_row_at_edge<kN>(row + step, p.rows, p.cols), next);
    Two<R> sum2 = twice(R(0));
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      Two<R> f[kN / 2];
      widen_pack(x[i], f);
#pragma unroll
      for (int j = 0; j < kN / 2; ++j)
        sum2 = add(sum2, f[j]);
    }
    R sum = sum2.x + sum2.y;
    row_sum<TH>(sum, slots[0]);
    const R mean = sum / n;  // exact for a row of one small integer
    Two<R> m2 = twice(R(0));
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      if (LAYOUT != kAny && !lay.some(i))
        continue;
      Two<R> f[kN / 2];
      widen_pack(x[i], f);
#pragma unroll
      for (int j = 0; j < kN / 2; ++j)
        f[j] = add(f[j], twice(-mean));
      if (LAYOUT == kAny || lay.warp_cut(i)) {
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) {
          f[j].x = lay.column(i, 2 * j) < p.cols ? f[j].x : R(0);
          f[j].y = lay.column(i, 2 * j + 1) < p.cols ? f[j].y : R(0);
        }
      }
#pragma unroll
      for (int j = 0; j < kN / 2; ++j)
        m2 = fma(f[j], f[j], m2);
    }
    R var = m2.x + m2.y;
    row_sum<TH>(var, slots[1]);
    const R rstd = inv_sqrt(var * inv_n + static_cast<R>(p.eps));
    T *y = static_cast<T *>(p.y) + row * p.ldy;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      if (LAYOUT != kAny && !lay.some(i))
        continue;
      Two<R> f[kN / 2], q[kN / 2];
      Pack<T> v;
      widen_pack(x[i], f);
#pragma unroll
      for (int j = 0; j < kN / 2; ++j)
        f[j] = mul(add(f[j], twice(-mean)), twice(rstd));
      if (gamma) {
        if (LAYOUT == kShifted)
          v.w = gamma_copy[i * TH + tid];
        else
          v = lay.parameter(gamma, i);
        widen_pack(v, q);
#pragma unroll
        for (int j = 0; j < kN / 2; ++j)
          f[j] = mul(f[j], q[j]);
      }
      if (beta) {
        if (LAYOUT == kShifted)
          v.w = beta_copy[i * TH + tid];
        else
          v = lay.parameter(beta, i);
        widen_pack(v, q);
#pragma unroll
        for (int j = 0; j < kN / 2; ++j)
          f[j] = add(f[j], q[j]);
      }
      narrow_pack(f, v);
      lay.store(y, i, v);
    }
    if (tid == 0) {
      if (p.mean)
        static_cast<R *>(p.mean)[row] = mean;
      if (p.rstd)
        static_cast<R *>(p.rstd)[row] = rstd;
    }
    if (!more)
      return;
#pragma unroll
    for (int i = 0; i < kPacks; ++i)
      x[i] = next[i];
  }
}

// Longer rows: three passes, the later two from L2.
template <typename T>
__device__ __forceinline__ void norm_rows_wide(const hexir_layer_norm_args_t &p) {
  typedef real_t<T> R;
  constexpr int TH = 512;
  griddep_wait();
  griddep_launch_dependents();
  __shared__ R slots[2][2 * TH / 32];
  const R n = static_cast<R>(p.cols), inv_n = R(1) / n;
  const T *gamma = static_cast<const T *>(p.gamma);
  const T *beta = static_cast<const T *>(p.beta);
  for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(p.x) + row * p.ldx;
    T *y = static_cast<T *>(p.y) + row * p.ldy;
    R sum = 0, m2 = 0;
    for (uint64_t c = threadIdx.x; c < p.cols; c += TH)
      sum += widen(x[c]);
    row_sum<TH>(sum, slots[0]);
    const R mean = sum / n;  // exact for a row of one small integer
    for (uint64_t c = threadIdx.x; c < p.cols; c += TH) {
      const R d = widen(x[c]) - mean;
      m2 += d * d;
    }
    row_sum<TH>(m2, slots[1]);
    const R rstd = inv_sqrt(m2 * inv_n + static_cast<R>(p.eps));
    for (uint64_t c = threadIdx.x; c < p.cols; c += TH) {
      R v = (widen(x[c]) - mean) * rstd;
      if (gamma)
        v *= widen(gamma[c]);
      if (beta)
        v += widen(beta[c]);
      y[c] = narrow<T>(v);
    }
    if (threadIdx.x == 0) {
      if (p.mean)
        static_cast<R *>(p.mean)[row] = mean;
      if (p.rstd)
        static_cast<R *>(p.rstd)[row] = rstd;
    }
    __syncthreads();  // every thread has read the slots
  }
}

// cp.async of `bytes` (4, 8 or 16) from global to shared memory.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src) {
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src),
                 "n"(BYTES)
                 : "memory");
}

// The gradient; block b takes rows b * kRows on, every kRows * grid, and leaves
// its sums of dy * xhat and dy in partial row b.
//
// The rows to come (x, dy and the residual) are copied into a ring of DEPTH
// rows in shared memory.  Every thread zeroes, copies and reads its own places
// alone (norm_ring.h), so the ring needs no barrier, and the registers hold the
// column sums instead of rows in flight (with one row ahead in registers, two
// blocks fit an SM and the loads' latency was 5 of 9 cycles between
// instructions).
template <typename T, int TH, int NE, int LAYOUT, int DEPTH>
__device__ __forceinline__ void norm_grad_rows(
    const hexir_layer_norm_grad_args_t &p) {
  typedef real_t<T> R;
  typedef Row<T, TH, NE, LAYOUT> Lay;
  constexpr int kN = Lay::kN, kPacks = Lay::kPacks;
  constexpr uint32_t kRows = TH < 256 ? 256 / TH : 1;
  constexpr uint32_t kBlock = kRows * TH;
  constexpr uint32_t kTensor = kPacks * kBlock;  // packs of a tensor's rows
  __shared__ R slots[2][kRows * 2 * TH / 32];
  extern __shared__ uint4 ring[];  // [DEPTH][tensors][kPacks][kBlock]
  const uint32_t tid = threadIdx.x % TH, group = threadIdx.x / TH;
  griddep_wait();  // nothing global is read or written before this
  griddep_launch_dependents();
  const R inv_n = R(1) / static_cast<R>(p.cols);
  const T *x_rows = static_cast<const T *>(p.x);
  const T *dy_rows = static_cast<const T *>(p.dy);
  const T *res_rows = p.dx ? static_cast<const T *>(p.residual) : nullptr;
  const R *means = static_cast<const R *>(p.mean);
  const R *rstds = static_cast<const R *>(p.rstd);
  const uint64_t step = (uint64_t)gridDim.x * kRows;
  uint64_t row = (uint64_t)blockIdx.x * kRows + group;
  const Lay lay(tid, p.cols, x_rows + row * p.ldx);
  const uint32_t tensors = res_rows ? 3 : 2;
  // Rows of single elements: the ring holds them one by one.
  constexpr bool kSingles = LAYOUT == kAny && sizeof(T) >= 4;
  // Element j of this thread's pack `pack` of the ring; with j = 0, the pack
  // itself where the ring holds packs.
  auto ring_at = [&](uint32_t pack, uint32_t j) {
    return reinterpret_cast<T *>(ring) +
           NormRing<kN, kBlock, kSingles>::at(pack, j, threadIdx.x);
  };

  Two<R> dgamma[NE / 2], dbeta[NE / 2];
#pragma unroll
  for (int i = 0; i < NE / 2; ++i)
    dgamma[i] = dbeta[i] = twice(R(0));
  Pack<T> g[kPacks];
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    if (!p.gamma) {
      Two<R> one[kN / 2];
#pragma unroll
      for (int j = 0; j < kN / 2; ++j)
        one[j] = twice(R(1));
      narrow_pack(one, g[i]);
    } else {
      g[i] = lay.parameter(static_cast<const T *>(p.gamma), i);
    }
  }
  // The places that no copy fills are 0, and those alone are zeroed: nothing
  // orders a plain store before a copy to the same place.  (16-bit single
  // elements are stored as whole packs, zeros included.)
  for (uint32_t s = 0; s < DEPTH * tensors; ++s) {
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      const uint32_t pack = s * kPacks + i;
      if (kSingles) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (lay.column(i, j) >= p.cols)
            *ring_at(pack, j) = narrow<T>(R(0));
      } else if (LAYOUT != kAny && !lay.some(i)) {
        *reinterpret_cast<uint4 *>(ring_at(pack, 0)) = make_uint4(0, 0, 0, 0);
      }
    }
  }

  auto fetch = [&](uint64_t at, uint32_t stage) {
    if (at < p.rows) {
      const bool edge = LAYOUT == kShifted && norm_row_at_edge<kN>(at, p.rows, p.cols);
      const T *src[3] = {x_rows + at * p.ldx, dy_rows + at * p.lddy,
                         res_rows ? res_rows + at * p.ldr : nullptr};
      const Span spans[3] = {span_of(x_rows, p.ldx, p.rows, p.cols),
                             span_of(dy_rows, p.lddy, p.rows, p.cols),
                             span_of(res_rows, p.ldr, p.rows, p.cols)};
#pragma unroll
      for (uint32_t t = 0; t < 3; ++t) {
        if (t == 2 && !res_rows)
          break;
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
          const uint32_t at_pack = (stage * tensors + t) * kPacks + i;
          uint4 *dst = reinterpret_cast<uint4 *>(ring_at(at_pack, 0));
          if (kSingles) {
#pragma unroll
            for (int j = 0; j < kN; ++j) {
              const uint32_t c = lay.column(i, j);
              if (c < p.cols)
                copy_async<sizeof(T) >= 4 ? sizeof(T) : 4>(
                    smem_addr(ring_at(at_pack, j)), src[t] + c);
            }
          } else if (LAYOUT == kAny) {
            *dst = lay.template load_pack<true>(src[t], i, spans[t], false).w;
          } else {
            const T *from = src[t] + static_cast<int32_t>(lay.column(i, 0));
            if (edge && lay.warp_cut(i)) {
              if (lay.apart(src[t], i, spans[t]))
                *dst = gather_pack(src[t], lay.column(i, 0), p.cols);
              else if (lay.some(i))
                copy_async<16>(smem_addr(dst), from);
            } else if (lay.some(i)) {
              copy_async<16>(smem_addr(dst), from);
            }
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto place = [&](uint32_t stage, uint32_t t, int i) {
    Pack<T> v;
    const uint32_t at_pack = (stage * tensors + t) * kPacks + i;
    if (kSingles) {
      T e[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j)
        e[j] = *ring_at(at_pack, j);
      v.w = *reinterpret_cast<const uint4 *>(e);
    } else {
      v.w = *reinterpret_cast<const uint4 *>(ring_at(at_pack, 0));
    }
    if (lay.warp_cut(i))
      v.w = lay.inside(v.w, i);
    return v;
  };

#pragma unroll
  for (uint32_t s = 0; s + 1 < DEPTH; ++s)
    fetch(row + s * step, s);
  R mean = 0, rstd = 0;
  if (row < p.rows) {
    mean = means[row];
    rstd = rstds[row];
  }
  uint32_t turn = 0, stage = 0;
  for (; row < p.rows; row += step, turn ^= 1u) {
    fetch(row + (DEPTH - 1) * step, stage == 0 ? DEPTH - 1 : stage - 1);
    R next_mean = 0, next_rstd = 0;
    if (row + step < p.rows) {
      next_mean = means[row + step];
      next_rstd = rstds[row + step];
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
    // Elements outside the row have dy = 0.  b multiplies g by rstd before x -
    // mean, because mean * rstd may be beyond the type's range, where 0 times
    // the xhat of such an element would be NaN; g * rstd is not where dx is not.
    // (Masked instead, rows off 16 bytes took 5 to 14 % longer; this, 0 to 2 %.)
    Two<R> a2 = twice(R(0)), b2 = a2;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      Two<R> fx[kN / 2], fd[kN / 2], fg[kN / 2];
      widen_pack(place(stage, 0, i), fx);
      widen_pack(place(stage, 1, i), fd);
      widen_pack(g[i], fg);
#pragma unroll
      for (int j = 0; j < kN / 2; ++j) {
        const Two<R> from_mean = add(fx[j], twice(-mean));
        Two<R> &dg = dgamma[i * kN / 2 + j], &db = dbeta[i * kN / 2 + j];
        dg = fma(fd[j], mul(from_mean, twice(rstd)), dg);
        db = add(db, fd[j]);
        const Two<R> gd = mul(fd[j], fg[j]);
        a2 = add(a2, gd);
        b2 = fma(mul(gd, twice(rstd)), from_mean, b2);
      }
    }
    if (p.dx) {
      R a = a2.x + a2.y, b = b2.x + b2.y;
      row_sum2<TH>(a, b, slots[turn]);
      // rstd (g - a - xhat b), with xhat = (x - mean) rstd, as a polynomial
      // in g and x - mean.
      const R ca = -a * inv_n * rstd, cb = -b * inv_n * rstd * rstd;
      T *dx = static_cast<T *>(p.dx) + row * p.lddx;
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        if (LAYOUT != kAny && !lay.some(i))
          continue;
        Two<R> fx[kN / 2], fd[kN / 2], fg[kN / 2];
        widen_pack(place(stage, 0, i), fx);
        widen_pack(place(stage, 1, i), fd);
        widen_pack(g[i], fg);
#pragma unroll
        for (int j = 0; j < kN / 2; ++j)
          fx[j] = fma(mul(fd[j], fg[j]), twice(rstd),
                      fma(add(fx[j], twice(-mean)), twice(cb), twice(ca)));
        if (res_rows) {
          widen_pack(place(stage, 2, i), fd);
#pragma unroll
          for (int j = 0; j < kN / 2; ++j)
            fx[j] = add(fx[j], fd[j]);
        }
        Pack<T> out;
        narrow_pack(fx, out);
        lay.store(dx, i, out);
      }
    }
    mean = next_mean;
    rstd = next_rstd;
    stage = stage + 1 == DEPTH ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!p.partials)
    return;
  R *part = static_cast<R *>(p.partials) + (uint64_t)blockIdx.x * 2 * p.cols;
  // Whole rows in 16-byte stores (a warp's 4-byte stores would each touch 32
  // sectors); single elements lie next to each other across a warp.
  if (kRows == 1 && LAYOUT == kWhole) {
    constexpr int kV = 16 / sizeof(R);
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      if (!lay.some(i))
        continue;
#pragma unroll
      for (int j = 0; j < kN; j += kV) {
        R *at = part + lay.column(i, j);
        Pack<R> v;
        Two<R> f[kV / 2];
#pragma unroll
        for (int e = 0; e < kV / 2; ++e)
          f[e] = dgamma[(i * kN + j) / 2 + e];
        narrow_pack(f, v);
        *reinterpret_cast<uint4 *>(at) = v.w;
#pragma unroll
        for (int e = 0; e < kV / 2; ++e)
          f[e] = dbeta[(i * kN + j) / 2 + e];
        narrow_pack(f, v);
        *reinterpret_cast<uint4 *>(at + p.cols) = v.w;
      }
    }
    return;
  }
  if (kRows == 1 && LAYOUT == kAny) {
#pragma unroll
    for (int i = 0; i < kPacks; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const uint32_t c = lay.column(i, j);
        if (c < p.cols) {
          part[c] = half_of(dgamma[(i * kN + j) / 2], j);
          part[(uint64_t)p.cols + c] = half_of(dbeta[(i * kN + j) / 2], j);
        }
      }
    return;
  }
  // The block's rows may differ in phase, and a shifted row's packs are not
  // whole 16 bytes of sums: the sums meet in the ring's place, by their place
  // in the row's packs.
  static_assert(DEPTH * sizeof(T) >= sizeof(R), "the ring holds the sums");
  R(*joined)[2][TH * NE] = reinterpret_cast<R(*)[2][TH * NE]>(ring);
  __shared__ uint32_t phases[kRows];
  __syncthreads();
  if (tid == 0)
    phases[group] = lay.phase;
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    if (LAYOUT == kAny) {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const uint32_t at = (i * kN + j) * TH + tid;
        joined[group][0][at] = half_of(dgamma[(i * kN + j) / 2], j);
        joined[group][1][at] = half_of(dbeta[(i * kN + j) / 2], j);
      }
    } else {
      constexpr int kV = 16 / sizeof(R);
#pragma unroll
      for (int j = 0; j < kN; j += kV) {
        const uint32_t at = (i * TH + tid) * kN + j;
        Pack<R> v;
        Two<R> f[kV / 2];
#pragma unroll
        for (int e = 0; e < kV / 2; ++e)
          f[e] = dgamma[(i * kN + j) / 2 + e];
        narrow_pack(f, v);
        *reinterpret_cast<uint4 *>(&joined[group][0][at]) = v.w;
#pragma unroll
        for (int e = 0; e < kV / 2; ++e)
          f[e] = dbeta[(i * kN + j) / 2 + e];
        narrow_pack(f, v);
        *reinterpret_cast<uint4 *>(&joined[group][1][at]) = v.w;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 2; ++which)
    for (uint32_t c = threadIdx.x; c < p.cols; c += kBlock) {
      R s = 0;
#pragma unroll
      for (uint32_t w = 0; w < kRows; ++w)
        s += joined[w][which][c + phases[w]];
      part[(uint64_t)which * p.cols + c] = s;
    }
}

// Longer rows: dx in three passes (the later two from L2); dgamma and dbeta
// by norm_grad_columns.
template <typename T>
__device__ __forceinline__ void norm_grad_rows_wide(
    const hexir_layer_norm_grad_args_t &p) {
  typedef real_t<T> R;
  constexpr int TH = 512;
  griddep_wait();
  griddep_launch_dependents();
  __shared__ R slots[2][2 * TH / 32];
  const R inv_n = R(1) / static_cast<R>(p.cols);
  const T *gamma = static_cast<const T *>(p.gamma);
  uint32_t turn = 0;
  for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1u) {
    const T *x = static_cast<const T *>(p.x) + row * p.ldx;
    const T *dy = static_cast<const T *>(p.dy) + row * p.lddy;
    const R mean = static_cast<const R *>(p.mean)[row];
    const R rstd = static_cast<const R *>(p.rstd)[row];
    R a = 0, b = 0;
    for (uint64_t c = threadIdx.x; c < p.cols; c += TH) {
      const R gd = widen(dy[c]) * (gamma ? widen(gamma[c]) : R(1));
      a += gd;
      b += gd * ((widen(x[c]) - mean) * rstd);
    }
    row_sum2<TH>(a, b, slots[turn]);
    a *= inv_n;
    b *= inv_n;
    T *dx = static_cast<T *>(p.dx) + row * p.lddx;
    const T *res = static_cast<const T *>(p.residual);
    for (uint64_t c = threadIdx.x; c < p.cols; c += TH) {
      const R gd = widen(dy[c]) * (gamma ? widen(gamma[c]) : R(1));
      R v = rstd * (gd - a - (widen(x[c]) - mean) * rstd * b);
      if (res)
        v += widen(res[row * p.ldr + c]);
      dx[c] = narrow<T>(v);
    }
  }
}

// dgamma and dbeta partials of 32 columns x the rows of part blockIdx.y.
template <typename T>
__device__ __forceinline__ void norm_grad_columns(
    const hexir_layer_norm_grad_args_t &p) {
  typedef real_t<T> R;
  __shared__ R joined[8][32][2];
  griddep_wait();
  griddep_launch_dependents();
  const uint64_t c = (uint64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const uint32_t lane = threadIdx.x / 32;
  R dgamma = 0, dbeta = 0;
  if (c < p.cols) {
    for (uint64_t row = (uint64_t)blockIdx.y * 8 + lane; row < p.rows;
         row += (uint64_t)p.parts * 8) {
      const R d = widen(static_cast<const T *>(p.dy)[row * p.lddy + c]);
      const R x = widen(static_cast<const T *>(p.x)[row * p.ldx + c]);
      dgamma += d * ((x - static_cast<const R *>(p.mean)[row]) *
                     static_cast<const R *>(p.rstd)[row]);
      dbeta += d;
    }
  }
  joined[lane][threadIdx.x % 32][0] = dgamma;
  joined[lane][threadIdx.x % 32][1] = dbeta;
  __syncthreads();
  if (lane < 2 && c < p.cols) {
    R s = 0;
    for (int w = 0; w < 8; ++w)
      s += joined[w][threadIdx.x % 32][lane];
    static_cast<R *>(p.partials)[((uint64_t)blockIdx.y * 2 + lane) * p.cols + c] = s;
  }
}

// out[c] = sum over parts of partials[part * stride + c]: 32 interleaved runs,
// each in part order, joined in order.
template <typename T>
__device__ __forceinline__ void column_sums(const real_t<T> *partials,
                                            uint64_t stride, uint32_t parts,
                                            T *out, uint64_t cols) {
  typedef real_t<T> R;
  __shared__ R joined[32][33];
  const uint32_t lane = threadIdx.x % 32, run = threadIdx.x / 32;
  const uint64_t c = (uint64_t)blockIdx.x * 32 + lane;
  R s = 0;
  if (c < cols) {
#pragma unroll 4
    for (uint32_t i = run; i < parts; i += 32)
      s += partials[i * stride + c];
  }
  joined[run][lane] = s;
  __syncthreads();
  // Warp w adds up column w, lane by lane in a fixed tree.
  s = joined[lane][run];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  const uint64_t mine = (uint64_t)blockIdx.x * 32 + run;
  if (lane == 0 && mine < cols)
    out[mine] = narrow<T>(s);
}

// dgamma (blockIdx.y == 0) and dbeta (1) from the partial rows.
template <typename T>
__device__ __forceinline__ void norm_grad_join(
    const hexir_layer_norm_grad_args_t &p) {
  T *out = static_cast<T *>(blockIdx.y ? p.dbeta : p.dgamma);
  griddep_wait();
  griddep_launch_dependents();
  if (out)
    column_sums<T>(static_cast<const real_t<T> *>(p.partials) +
                       (uint64_t)blockIdx.y * p.cols,
                   2ull * p.cols, p.parts, out, p.cols);
}

// dz = dy * act'(z) and the sums of dz over the rows of part blockIdx.y, for
// 256 columns: a warp covers a row's 256 columns (8 per lane), the 8 warps
// take the part's rows in turn, 4 of them in flight at a time (with one, the
// loads' latency left HBM at 0.4 of its rate).
template <typename T>
__device__ __forceinline__ void output_grad(const hexir_output_grad_args_t &p) {
  constexpr uint32_t kRows = 4;
  __shared__ float joined[8][256];
  griddep_wait();  // nothing global is read or written before this
  griddep_launch_dependents();
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t col = blockIdx.x * 256 + lane * 8;
  const uint32_t left = col < p.n ? p.n - col : 0;
  const bool whole = p.vec && left >= 8;
  const T *dy = static_cast<const T *>(p.dy) + col;
  const T *z = static_cast<const T *>(p.preact) + col;
  T *dz = static_cast<T *>(p.dz) + col;
  const uint32_t row0 = blockIdx.y * p.rows_per_part;
  const uint32_t rows = row0 < p.m ? min(p.rows_per_part, p.m - row0) : 0;
  Two<float> sum[4] = {{0, 0}, {0, 0}, {0, 0}, {0, 0}};
  if (left) {
    for (uint32_t i = warp; i < rows; i += 8 * kRows) {
      Pack<T> g[kRows], at[kRows];
#pragma unroll
      for (uint32_t r = 0; r < kRows; ++r) {
        // Rows past the part are read as its last and not used.
        const uint64_t row = row0 + min(i + 8 * r, rows - 1);
        if (whole) {
          g[r].w = __ldcs(reinterpret_cast<const uint4 *>(dy + row * p.lddy));
          if (p.activation)
            at[r].w = __ldcs(reinterpret_cast<const uint4 *>(z + row * p.ldp));
        } else {
          T e[8], f[8];
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j) {
            e[j] = dy[row * p.lddy + min(j, left - 1)];
            f[j] = p.activation ? z[row * p.ldp + min(j, left - 1)] : e[j];
          }
          g[r].w = *reinterpret_cast<const uint4 *>(e);
          at[r].w = *reinterpret_cast<const uint4 *>(f);
        }
      }
#pragma unroll
      for (uint32_t r = 0; r < kRows; ++r) {
        if (i + 8 * r >= rows)
          break;
        const uint64_t row = row0 + i + 8 * r;
        Two<float> v[4], s[4];
        if (p.activation) {
          widen_pack(g[r], v);
          widen_pack(at[r], s);
          slope_f32(p.activation, reinterpret_cast<const float(&)[8]>(s),
                    reinterpret_cast<float(&)[8]>(v));
          narrow_pack(v, g[r]);
        }
        if (p.dz) {
          if (whole) {
            *reinterpret_cast<uint4 *>(dz + row * p.lddz) = g[r].w;
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (static_cast<uint32_t>(j) < left)
                dz[row * p.lddz + j] = pack_get(g[r], j);
          }
        }
        widen_pack(g[r], v);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sum[j] = add(sum[j], v[j]);
      }
    }
  }
  if (!p.partials)
    return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    joined[warp][j * 32 + lane] = half_of(sum[j / 2], j);
  __syncthreads();
  float s = joined[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < 8; ++w)
    s += joined[w][threadIdx.x];
  const uint64_t c = blockIdx.x * 256ull + (threadIdx.x % 32) * 8 + threadIdx.x / 32;
  if (c < p.n)
    p.partials[(uint64_t)blockIdx.y * p.n + c] = s;
}

template <typename T>
__device__ __forceinline__ void output_grad_join(
    const hexir_output_grad_args_t &p) {
  griddep_wait();
  griddep_launch_dependents();
  column_sums<T>(p.partials, p.n, p.parts, static_cast<T *>(p.dbias), p.n);
}

}  // namespace

// Kernels by threads per row, elements per thread and layout (w whole, h
// shifted, s any); MINB blocks share an SM, DEPTH rows the gradient's ring.
#define NORM(SUFFIX, T, TH, NE, MODE, LAYOUT, MINB)                            \
  extern "C" __global__ void __launch_bounds__(TH < 256 ? 256 : TH, MINB)      \
      hexir_layer_norm_##SUFFIX##_##MODE##TH##x##NE(                           \
          const hexir_layer_norm_args_t args) {                                \
    norm_rows<T, TH, NE, LAYOUT>(args);                                        \
  }
#define NORM_GRAD(SUFFIX, T, TH, NE, MODE, LAYOUT, MINB, DEPTH)                \
  extern "C" __global__ void __launch_bounds__(TH < 256 ? 256 : TH, MINB)      \
      hexir_layer_norm_grad_##SUFFIX##_##MODE##TH##x##NE(                      \
          const hexir_layer_norm_grad_args_t args) {                           \
    norm_grad_rows<T, TH, NE, LAYOUT, DEPTH>(args);                            \
  }

#define NORMS(SUFFIX, T)                                                       \
  extern "C" __global__ void __launch_bounds__(512)                            \
      hexir_layer_norm_##SUFFIX##_wide(const hexir_layer_norm_args_t args) {   \
    norm_rows_wide<T>(args);                                                   \
  }                                                                            \
  extern "C" __global__ void __launch_bounds__(512)                            \
      hexir_layer_norm_grad_##SUFFIX##_wide(                                   \
          const hexir_layer_norm_grad_args_t args) {                           \
    norm_grad_rows_wide<T>(args);                                              \
  }                                                                            \
  extern "C" __global__ void __launch_bounds__(256)                            \
      hexir_layer_norm_grad_##SUFFIX##_columns(                                \
          const hexir_layer_norm_grad_args_t args) {                           \
    norm_grad_columns<T>(args);                                                \
  }                                                                            \
  extern "C" __global__ void __launch_bounds__(1024)                           \
      hexir_layer_norm_grad_##SUFFIX##_join(                                   \
          const hexir_layer_norm_grad_args_t args) {                           \
    norm_grad_join<T>(args);                                                   \
  }

#define NORMS_16(SUFFIX, T)                                                    \
  NORMS(SUFFIX, T)                                                             \
  NORM(SUFFIX, T, 32, 8, w, kWhole, 5)                                         \
  NORM(SUFFIX, T, 32, 16, w, kWhole, 3)                                        \
  NORM(SUFFIX, T, 32, 24, w, kWhole, 2)                                        \
  NORM(SUFFIX, T, 32, 32, w, kWhole, 2)                                        \
  NORM(SUFFIX, T, 128, 16, w, kWhole, 4)                                       \
  NORM(SUFFIX, T, 256, 16, w, kWhole, 4)                                       \
  NORM(SUFFIX, T, 256, 24, w, kWhole, 2)                                       \
  NORM(SUFFIX, T, 256, 32, w, kWhole, 2)                                       \
  NORM(SUFFIX, T, 512, 32, w, kWhole, 1)                                       \
  NORM(SUFFIX, T, 32, 8, h, kShifted, 5)                                       \
  NORM(SUFFIX, T, 32, 16, h, kShifted, 3)                                      \
  NORM(SUFFIX, T, 64, 16, h, kShifted, 3)                                      \
  NORM(SUFFIX, T, 128, 16, h, kShifted, 4)                                     \
  NORM(SUFFIX, T, 256, 16, h, kShifted, 3)                                     \
  NORM(SUFFIX, T, 320, 16, h, kShifted, 2)                                     \
  NORM(SUFFIX, T, 384, 16, h, kShifted, 2)                                     \
  NORM(SUFFIX, T, 512, 16, h, kShifted, 2)                                     \
  NORM(SUFFIX, T, 1024, 16, h, kShifted, 1)                                    \
  NORM(SUFFIX, T, 32, 32, s, kAny, 2)                                          \
  NORM(SUFFIX, T, 256, 16, s, kAny, 3)                                         \
  NORM(SUFFIX, T, 512, 32, s, kAny, 1)                                         \
  NORM_GRAD(SUFFIX, T, 32, 8, w, kWhole, 2, 6)                                 \
  NORM_GRAD(SUFFIX, T, 32, 16, w, kWhole, 2, 4)                                \
  NORM_GRAD(SUFFIX, T, 64, 16, w, kWhole, 2, 4)                                \
  NORM_GRAD(SUFFIX, T, 128, 16, w, kWhole, 2, 3)                               \
  NORM_GRAD(SUFFIX, T, 256, 16, w, kWhole, 2, 3)                               \
  NORM_GRAD(SUFFIX, T, 384, 16, w, kWhole, 1, 4)                               \
  NORM_GRAD(SUFFIX, T, 512, 16, w, kWhole, 1, 3)                               \
  NORM_GRAD(SUFFIX, T, 1024, 16, w, kWhole, 1, 2)                              \
  NORM_GRAD(SUFFIX, T, 32, 8, h, kShifted, 2, 6)                               \
  NORM_GRAD(SUFFIX, T, 32, 16, h, kShifted, 2, 4)                              \
  NORM_GRAD(SUFFIX, T, 64, 16, h, kShifted, 2, 4)                              \
  NORM_GRAD(SUFFIX, T, 128, 16, h, kShifted, 2, 4)                             \
  NORM_GRAD(SUFFIX, T, 256, 16, h, kShifted, 2, 4)                             \
  NORM_GRAD(SUFFIX, T, 384, 16, h, kShifted, 1, 4)                             \
  NORM_GRAD(SUFFIX, T, 512, 16, h, kShifted, 1, 3)                             \
  NORM_GRAD(SUFFIX, T, 1024, 16, h, kShifted, 1, 2)                            \
  NORM_GRAD(SUFFIX, T, 32, 32, s, kAny, 1, 2)                                  \
  NORM_GRAD(SUFFIX, T, 1024, 16, s, kAny, 1, 2)

NORMS_16(bf16, __nv_bfloat16)
NORMS_16(f16, __half)

NORMS(f32, float)
NORM(f32, float, 32, 8, w, kWhole, 5)
NORM(f32, float, 32, 16, w, kWhole, 3)
NORM(f32, float, 32, 32, w, kWhole, 2)
NORM(f32, float, 128, 16, w, kWhole, 3)
NORM(f32, float, 256, 16, w, kWhole, 3)
NORM(f32, float, 512, 16, w, kWhole, 2)
NORM(f32, float, 1024, 16, w, kWhole, 1)
NORM(f32, float, 256, 8, h, kShifted, 4)
NORM(f32, float, 320, 8, h, kShifted, 3)
NORM(f32, float, 512, 8, h, kShifted, 2)
NORM(f32, float, 640, 8, h, kShifted, 1)
NORM(f32, float, 512, 16, h, kShifted, 1)
NORM(f32, float, 1024, 16, h, kShifted, 1)
NORM(f32, float, 32, 8, s, kAny, 5)
NORM(f32, float, 32, 16, s, kAny, 3)
NORM(f32, float, 128, 8, s, kAny, 4)
NORM(f32, float, 320, 8, s, kAny, 3)
NORM(f32, float, 512, 8, s, kAny, 2)
NORM(f32, float, 512, 16, s, kAny, 1)
NORM(f32, float, 1024, 16, s, kAny, 1)
NORM_GRAD(f32, float, 32, 8, w, kWhole, 2, 4)
NORM_GRAD(f32, float, 64, 8, w, kWhole, 2, 4)
NORM_GRAD(f32, float, 128, 8, w, kWhole, 2, 4)
NORM_GRAD(f32, float, 256, 8, w, kWhole, 2, 4)
NORM_GRAD(f32, float, 512, 8, w, kWhole, 1, 3)
NORM_GRAD(f32, float, 512, 16, w, kWhole, 1, 2)
NORM_GRAD(f32, float, 256, 8, h, kShifted, 2, 4)
NORM_GRAD(f32, float, 320, 8, h, kShifted, 2, 4)
NORM_GRAD(f32, float, 512, 8, h, kShifted, 1, 3)
NORM_GRAD(f32, float, 640, 8, h, kShifted, 1, 2)
NORM_GRAD(f32, float, 512, 16, h, kShifted, 1, 2)
NORM_GRAD(f32, float, 64, 8, s, kAny, 2, 4)
NORM_GRAD(f32, float, 128, 8, s, kAny, 2, 4)
NORM_GRAD(f32, float, 320, 8, s, kAny, 2, 4)
NORM_GRAD(f32, float, 512, 8, s, kAny, 1, 3)
NORM_GRAD(f32, float, 512, 16, s, kAny, 1, 2)

NORMS(f64, double)
NORM(f64, double, 32, 8, w, kWhole, 3)
NORM(f64, double, 64, 8, w, kWhole, 3)
NORM(f64, double, 128, 8, w, kWhole, 3)
NORM(f64, double, 256, 8, w, kWhole, 3)
NORM(f64, double, 512, 8, w, kWhole, 1)
NORM(f64, double, 512, 16, w, kWhole, 1)
NORM(f64, double, 32, 8, s, kAny, 3)
NORM(f64, double, 64, 8, s, kAny, 3)
NORM(f64, double, 192, 8, s, kAny, 3)
NORM(f64, double, 256, 8, s, kAny, 3)
NORM(f64, double, 512, 8, s, kAny, 1)
NORM(f64, double, 512, 16, s, kAny, 1)
NORM_GRAD(f64, double, 32, 8, w, kWhole, 2, 3)
NORM_GRAD(f64, double, 64, 8, w, kWhole, 2, 3)
NORM_GRAD(f64, double, 128, 8, w, kWhole, 2, 3)
NORM_GRAD(f64, double, 256, 8, w, kWhole, 2, 3)
NORM_GRAD(f64, double, 512, 8, w, kWhole, 1, 2)
NORM_GRAD(f64, double, 32, 8, s, kAny, 1, 3)
NORM_GRAD(f64, double, 64, 8, s, kAny, 2, 3)
NORM_GRAD(f64, double, 192, 8, s, kAny, 2, 3)
NORM_GRAD(f64, double, 256, 8, s, kAny, 2, 3)
NORM_GRAD(f64, double, 512, 8, s, kAny, 1, 2)

#define OUTPUT_GRAD(SUFFIX, T)                                                 \
  extern "C" __global__ void __launch_bounds__(256)                            \
      hexir_linear_output_grad_##SUFFIX(const hexir_output_grad_args_t args) { \
    output_grad<T>(args);                                                      \
  }                                                                            \
  extern "C" __global__ void __launch_bounds__(1024)                           \
      hexir_linear_output_grad_##SUFFIX##_join(                                \
          const hexir_output_grad_args_t args) {                               \
    output_grad_join<T>(args);                                                 \
  }

OUTPUT_GRAD(bf16, __nv_bfloat16)
OUTPUT_GRAD(f16, __half)
