// layer_norm.cu -- layer norm and its gradient over the rows of a row-major
// tensor (include/hexir_b200/layers.h), and the elementwise gradient of a
// linear layer's epilogue with its column sums.
//
// A row is held in the registers of its threads (a warp's or a block's), so
// each pass reads its tensors once: forward x -> y, backward x, dy
// (, residual) -> dx.  Both are bound by HBM; rows longer than a block holds
// are read again from L2.
//
// The gradients of gamma, beta and the bias are sums over rows: each block
// adds up its rows in registers and leaves one partial row in the caller's
// workspace, and a second kernel adds the partial rows in order.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "activation_f32.cuh"
#include "common.cuh"
#include "layers_abi.h"

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

template <typename T>
struct alignas(16) Pack {
  static constexpr int kN = 16 / sizeof(T);
  T v[kN];
};

// Which columns a thread of `TH` holds: with 16-byte aligned rows, packs
// tid, tid + TH, ...; otherwise single elements tid, tid + TH, ..., so that a
// warp's loads stay consecutive either way.
template <typename T, int TH>
__device__ __forceinline__ uint32_t column(int pack, int j, uint32_t tid,
                                           bool vec) {
  constexpr int kN = Pack<T>::kN;
  return vec ? (pack * TH + tid) * kN + j : (pack * kN + j) * TH + tid;
}

// NE elements of a row in packs; columns past the end give `fill`.
template <typename T, int TH, int NE>
__device__ __forceinline__ void load_row(const T *row, uint32_t cols,
                                         uint32_t tid, bool vec, T fill,
                                         Pack<T> (&v)[NE / Pack<T>::kN]) {
  constexpr int kN = Pack<T>::kN;
#pragma unroll
  for (int i = 0; i < NE / kN; ++i) {
    const uint32_t c0 = column<T, TH>(i, 0, tid, true);
    if (vec && c0 + kN <= cols) {
      v[i] = *reinterpret_cast<const Pack<T> *>(row + c0);
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const uint32_t c = column<T, TH>(i, j, tid, vec);
        v[i].v[j] = c < cols ? row[c] : fill;
      }
    }
  }
}

template <typename T, int TH, int NE>
__device__ __forceinline__ void store_row(T *row, uint32_t cols, uint32_t tid,
                                          bool vec,
                                          const Pack<T> (&v)[NE / Pack<T>::kN]) {
  constexpr int kN = Pack<T>::kN;
#pragma unroll
  for (int i = 0; i < NE / kN; ++i) {
    const uint32_t c0 = column<T, TH>(i, 0, tid, true);
    if (vec && c0 + kN <= cols) {
      *reinterpret_cast<Pack<T> *>(row + c0) = v[i];
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const uint32_t c = column<T, TH>(i, j, tid, vec);
        if (c < cols)
          row[c] = v[i].v[j];
      }
    }
  }
}

// Sums of two values over the TH threads of a row, in an order that depends
// on TH alone.  `slot` holds 2 * TH / 32 values; calls alternate between two
// slots, so one barrier per call is enough.
template <int TH, typename R>
__device__ __forceinline__ void row_sum2(R &a, R &b, R *slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
    b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
  }
  if (TH == 32)
    return;
  constexpr int kWarps = TH / 32;
  const uint32_t warp = threadIdx.x / 32;
  if (threadIdx.x % 32 == 0) {
    slot[2 * warp] = a;
    slot[2 * warp + 1] = b;
  }
  __syncthreads();
  a = slot[0];
  b = slot[1];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    a += slot[2 * w];
    b += slot[2 * w + 1];
  }
}

__device__ __forceinline__ float inv_sqrt(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

// Rows of up to TH * NE columns; TH == 32: a warp per row, 8 rows per block.
template <typename T, int TH, int NE>
__device__ __forceinline__ void norm_rows(const hexir_layer_norm_args_t &p) {
  typedef real_t<T> R;
  constexpr int kN = Pack<T>::kN;
  constexpr uint32_t kRows = TH == 32 ? 8 : 1;
  __shared__ R slots[2][TH == 32 ? 1 : 2 * TH / 32];
  const uint32_t tid = TH == 32 ? threadIdx.x % 32 : threadIdx.x;
  const bool vec = p.vec != 0;
  const R n = static_cast<R>(p.cols);
  for (uint64_t row = (uint64_t)blockIdx.x * kRows +
                      (TH == 32 ? threadIdx.x / 32 : 0);
       row < p.rows; row += (uint64_t)gridDim.x * kRows) {
    Pack<T> x[NE / kN];
    load_row<T, TH, NE>(static_cast<const T *>(p.x) + row * p.ldx, p.cols, tid,
                        vec, narrow<T>(R(0)), x);
    R sum = 0, none = 0;
#pragma unroll
    for (int i = 0; i < NE / kN; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j)
        sum += widen(x[i].v[j]);
    row_sum2<TH>(sum, none, slots[0]);
    const R mean = sum / n;
    R m2 = 0;
#pragma unroll
    for (int i = 0; i < NE / kN; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const R d = widen(x[i].v[j]) - mean;
        m2 += column<T, TH>(i, j, tid, vec) < p.cols ? d * d : R(0);
      }
    row_sum2<TH>(m2, none, slots[1]);
    const R rstd = inv_sqrt(m2 / n + static_cast<R>(p.eps));
    Pack<T> g[NE / kN], b[NE / kN];
    if (p.gamma)
      load_row<T, TH, NE>(static_cast<const T *>(p.gamma), p.cols, tid, vec,
                          narrow<T>(R(0)), g);
    if (p.beta)
      load_row<T, TH, NE>(static_cast<const T *>(p.beta), p.cols, tid, vec,
                          narrow<T>(R(0)), b);
#pragma unroll
    for (int i = 0; i < NE / kN; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        R v = (widen(x[i].v[j]) - mean) * rstd;
        if (p.gamma)
          v *= widen(g[i].v[j]);
        if (p.beta)
          v += widen(b[i].v[j]);
        x[i].v[j] = narrow<T>(v);
      }
    store_row<T, TH, NE>(static_cast<T *>(p.y) + row * p.ldy, p.cols, tid, vec, x);
    if (tid == 0) {
      if (p.mean)
        static_cast<R *>(p.mean)[row] = mean;
      if (p.rstd)
        static_cast<R *>(p.rstd)[row] = rstd;
    }
  }
}

// Longer rows: three passes, the later two from L2.
template <typename T>
__device__ __forceinline__ void norm_rows_wide(const hexir_layer_norm_args_t &p) {
  typedef real_t<T> R;
  constexpr int TH = 512;
  __shared__ R slots[2][2 * TH / 32];
  const R n = static_cast<R>(p.cols);
  const T *gamma = static_cast<const T *>(p.gamma);
  const T *beta = static_cast<const T *>(p.beta);
  for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(p.x) + row * p.ldx;
    T *y = static_cast<T *>(p.y) + row * p.ldy;
    R sum = 0, none = 0, m2 = 0;
    for (uint64_t c = threadIdx.x; c < p.cols; c += TH)
      sum += widen(x[c]);
    row_sum2<TH>(sum, none, slots[0]);
    const R mean = sum / n;
    for (uint64_t c = threadIdx.x; c < p.cols; c += TH) {
      const R d = widen(x[c]) - mean;
      m2 += d * d;
    }
    row_sum2<TH>(m2, none, slots[1]);
    const R rstd = inv_sqrt(m2 / n + static_cast<R>(p.eps));
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

// The gradient; block b takes rows b, b + grid, ... (by warps for TH == 32)
// and leaves its sums of dy * xhat and dy in partial row b.
template <typename T, int TH, int NE>
__device__ __forceinline__ void norm_grad_rows(
    const hexir_layer_norm_grad_args_t &p) {
  typedef real_t<T> R;
  constexpr int kN = Pack<T>::kN;
  constexpr uint32_t kRows = TH == 32 ? 8 : 1;
  __shared__ R slots[2][TH == 32 ? 1 : 2 * TH / 32];
  __shared__ R joined[TH == 32 ? 8 * 32 * 2 : 1];
  const uint32_t tid = TH == 32 ? threadIdx.x % 32 : threadIdx.x;
  const bool vec = p.vec != 0;
  const R inv_n = R(1) / static_cast<R>(p.cols);
  R dgamma[NE], dbeta[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i)
    dgamma[i] = dbeta[i] = 0;
  Pack<T> g[NE / kN];
  if (p.gamma) {
    load_row<T, TH, NE>(static_cast<const T *>(p.gamma), p.cols, tid, vec,
                        narrow<T>(R(0)), g);
  } else {
#pragma unroll
    for (int i = 0; i < NE / kN; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j)
        g[i].v[j] = narrow<T>(R(1));
  }
  uint32_t turn = 0;
  for (uint64_t row = (uint64_t)blockIdx.x * kRows +
                      (TH == 32 ? threadIdx.x / 32 : 0);
       row < p.rows; row += (uint64_t)gridDim.x * kRows, turn ^= 1u) {
    Pack<T> x[NE / kN], dy[NE / kN];
    load_row<T, TH, NE>(static_cast<const T *>(p.x) + row * p.ldx, p.cols, tid,
                        vec, narrow<T>(R(0)), x);
    load_row<T, TH, NE>(static_cast<const T *>(p.dy) + row * p.lddy, p.cols,
                        tid, vec, narrow<T>(R(0)), dy);
    const R mean = static_cast<const R *>(p.mean)[row];
    const R rstd = static_cast<const R *>(p.rstd)[row];
    R a = 0, b = 0;  // columns past the end have dy = 0
#pragma unroll
    for (int i = 0; i < NE / kN; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const R xhat = (widen(x[i].v[j]) - mean) * rstd;
        const R d = widen(dy[i].v[j]);
        const R gd = d * widen(g[i].v[j]);
        a += gd;
        b += gd * xhat;
        dgamma[i * kN + j] += d * xhat;
        dbeta[i * kN + j] += d;
      }
    if (p.dx) {
      row_sum2<TH>(a, b, slots[turn]);
      a *= inv_n;
      b *= inv_n;
      Pack<T> r[NE / kN];
      if (p.residual)
        load_row<T, TH, NE>(static_cast<const T *>(p.residual) + row * p.ldr,
                            p.cols, tid, vec, narrow<T>(R(0)), r);
#pragma unroll
      for (int i = 0; i < NE / kN; ++i)
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          const R xhat = (widen(x[i].v[j]) - mean) * rstd;
          const R gd = widen(dy[i].v[j]) * widen(g[i].v[j]);
          R v = rstd * (gd - a - xhat * b);
          if (p.residual)
            v += widen(r[i].v[j]);
          x[i].v[j] = narrow<T>(v);
        }
      store_row<T, TH, NE>(static_cast<T *>(p.dx) + row * p.lddx, p.cols, tid,
                           vec, x);
    }
  }
  if (!p.partials)
    return;
  R *part = static_cast<R *>(p.partials) + (uint64_t)blockIdx.x * 2 * p.cols;
  if (TH != 32) {
#pragma unroll
    for (int i = 0; i < NE / kN; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const uint32_t c = column<T, TH>(i, j, tid, vec);
        if (c < p.cols) {
          part[c] = dgamma[i * kN + j];
          part[(uint64_t)p.cols + c] = dbeta[i * kN + j];
        }
      }
    return;
  }
  // Join the 8 warps' sums, one element of every lane at a time.
  const uint32_t warp = threadIdx.x / 32;
#pragma unroll
  for (int i = 0; i < NE / kN; ++i)
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      joined[(warp * 32 + tid) * 2] = dgamma[i * kN + j];
      joined[(warp * 32 + tid) * 2 + 1] = dbeta[i * kN + j];
      __syncthreads();
      const uint32_t c = column<T, TH>(i, j, tid, vec);
      if (warp < 2 && c < p.cols) {
        R s = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w)
          s += joined[(w * 32 + tid) * 2 + warp];
        part[(uint64_t)warp * p.cols + c] = s;
      }
      __syncthreads();
    }
}

// Longer rows: dx in three passes (the later two from L2); dgamma and dbeta
// by norm_grad_columns.
template <typename T>
__device__ __forceinline__ void norm_grad_rows_wide(
    const hexir_layer_norm_grad_args_t &p) {
  typedef real_t<T> R;
  constexpr int TH = 512;
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

// out[c] = sum over parts of partials[part * stride + c], in part order within
// each of 8 interleaved runs, the runs joined in order.
template <typename T>
__device__ __forceinline__ void column_sums(const real_t<T> *partials,
                                            uint64_t stride, uint32_t parts,
                                            T *out, uint64_t cols) {
  typedef real_t<T> R;
  __shared__ R joined[8][32];
  const uint64_t c = (uint64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const uint32_t lane = threadIdx.x / 32;
  R s = 0;
  if (c < cols)
    for (uint32_t i = lane; i < parts; i += 8)
      s += partials[i * stride + c];
  joined[lane][threadIdx.x % 32] = s;
  __syncthreads();
  if (lane == 0 && c < cols) {
    for (int w = 1; w < 8; ++w)
      s += joined[w][threadIdx.x];
    out[c] = narrow<T>(s);
  }
}

// dgamma (blockIdx.y == 0) and dbeta (1) from the partial rows.
template <typename T>
__device__ __forceinline__ void norm_grad_join(
    const hexir_layer_norm_grad_args_t &p) {
  T *out = static_cast<T *>(blockIdx.y ? p.dbeta : p.dgamma);
  griddep_wait();
  if (out)
    column_sums<T>(static_cast<const real_t<T> *>(p.partials) +
                       (uint64_t)blockIdx.y * p.cols,
                   2ull * p.cols, p.parts, out, p.cols);
}

// dz = dy * act'(z) and the sums of dz over the rows of part blockIdx.y, for
// 256 columns: a warp covers a row's 256 columns (8 per lane), the 8 warps
// take the part's rows in turn.
template <typename T>
__device__ __forceinline__ void output_grad(const hexir_output_grad_args_t &p) {
  __shared__ float joined[8][256];
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t col = blockIdx.x * 256 + lane * 8;
  const uint32_t left = col < p.n ? p.n - col : 0;
  const bool whole = p.vec && left >= 8;
  const T *dy = static_cast<const T *>(p.dy) + col;
  const T *z = static_cast<const T *>(p.preact) + col;
  T *dz = static_cast<T *>(p.dz) + col;
  const uint32_t row0 = blockIdx.y * p.rows_per_part;
  const uint32_t rows = row0 < p.m ? min(p.rows_per_part, p.m - row0) : 0;
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (left) {
    for (uint32_t i = warp; i < rows; i += 8) {
      const uint64_t row = row0 + i;
      Pack<T> g, at;
      if (whole) {
        g = *reinterpret_cast<const Pack<T> *>(dy + row * p.lddy);
        if (p.activation)
          at = *reinterpret_cast<const Pack<T> *>(z + row * p.ldp);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = static_cast<uint32_t>(j) < left;
          g.v[j] = in ? dy[row * p.lddy + j] : narrow<T>(0.0f);
          at.v[j] = in && p.activation ? z[row * p.ldp + j] : narrow<T>(0.0f);
        }
      }
      if (p.activation) {
        float v[8], s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = widen(g.v[j]);
          s[j] = widen(at.v[j]);
        }
        slope_f32(p.activation, s, v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          g.v[j] = narrow<T>(v[j]);
      }
      if (p.dz) {
        if (whole) {
          *reinterpret_cast<Pack<T> *>(dz + row * p.lddz) = g;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (static_cast<uint32_t>(j) < left)
              dz[row * p.lddz + j] = g.v[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        sum[j] += widen(g.v[j]);
    }
  }
  if (!p.partials)
    return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    joined[warp][j * 32 + lane] = sum[j];
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
  column_sums<T>(p.partials, p.n, p.parts, static_cast<T *>(p.dbias), p.n);
}

}  // namespace

#define NORM(SUFFIX, T, TH, NE)                                                \
  extern "C" __global__ void __launch_bounds__(TH == 32 ? 256 : TH)            \
      hexir_layer_norm_##SUFFIX##_##TH##x##NE(                                 \
          const hexir_layer_norm_args_t args) {                                \
    norm_rows<T, TH, NE>(args);                                                \
  }                                                                            \
  extern "C" __global__ void __launch_bounds__(TH == 32 ? 256 : TH)            \
      hexir_layer_norm_grad_##SUFFIX##_##TH##x##NE(                            \
          const hexir_layer_norm_grad_args_t args) {                           \
    norm_grad_rows<T, TH, NE>(args);                                           \
  }

#define NORMS(SUFFIX, T)                                                       \
  NORM(SUFFIX, T, 32, 8)                                                       \
  NORM(SUFFIX, T, 32, 16)                                                      \
  NORM(SUFFIX, T, 32, 32)                                                      \
  NORM(SUFFIX, T, 256, 8)                                                      \
  NORM(SUFFIX, T, 256, 16)                                                     \
  NORM(SUFFIX, T, 512, 16)                                                     \
  NORM(SUFFIX, T, 1024, 16)                                                    \
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
  extern "C" __global__ void __launch_bounds__(256)                            \
      hexir_layer_norm_grad_##SUFFIX##_join(                                   \
          const hexir_layer_norm_grad_args_t args) {                           \
    norm_grad_join<T>(args);                                                   \
  }

NORMS(f64, double)
NORMS(f32, float)
NORMS(bf16, __nv_bfloat16)
NORMS(f16, __half)

#define OUTPUT_GRAD(SUFFIX, T)                                                 \
  extern "C" __global__ void __launch_bounds__(256)                            \
      hexir_linear_output_grad_##SUFFIX(const hexir_output_grad_args_t args) { \
    output_grad<T>(args);                                                      \
  }                                                                            \
  extern "C" __global__ void __launch_bounds__(256)                            \
      hexir_linear_output_grad_##SUFFIX##_join(                                \
          const hexir_output_grad_args_t args) {                               \
    output_grad_join<T>(args);                                                 \
  }

OUTPUT_GRAD(bf16, __nv_bfloat16)
OUTPUT_GRAD(f16, __half)
