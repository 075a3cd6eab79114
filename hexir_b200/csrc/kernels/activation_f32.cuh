// activation_f32.cuh -- the activations and their slopes in f32, for the
// epilogues of the 16-bit products and the elementwise gradient.  The forms
// keep relative accuracy where 1 - t or 1 + erf would cancel; results are
// rounded to bf16 or f16 (by up to 2^-8, 2^-11 of the value) after them.
//
// Exponentials and reciprocals are the hardware's approximations (a few 2^-24
// of the value): with expf, erfcf and IEEE divides the gelu of a 256 x 256 tile
// took longer than the 32 k tiles of its sum.
#pragma once

#include <stdint.h>

#include "launch_abi.h"
#include "two.cuh"

namespace hexir {

constexpr uint32_t kActRelu = 3u;

// 2^x, and e^x; subnormal results are kept.
__device__ __forceinline__ float exp2_near(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp_near(float x) {
  return exp2_near(1.4426950408889634f * x);
}
// 1 / x for x >= 1 (0 from 2^126 on).
__device__ __forceinline__ float inverse_near(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// e^x - 1 for x <= 0: where the difference would cancel, its Taylor polynomial
// (the next term is below 2e-7 of the value).
__device__ __forceinline__ float expm1_near(float x) {
  float p = 1.0f / 5040.0f;
  p = ::fmaf(p, x, 1.0f / 720.0f);
  p = ::fmaf(p, x, 1.0f / 120.0f);
  p = ::fmaf(p, x, 1.0f / 24.0f);
  p = ::fmaf(p, x, 1.0f / 6.0f);
  p = ::fmaf(p, x, 0.5f);
  p = ::fmaf(p, x, 1.0f) * x;
  // Both, and a choice: as a branch around each it took twice the time.
  const float e = exp_near(x) - 1.0f;
  float y;
  asm("{\n\t.reg .pred q;\n\tsetp.gt.f32 q, %3, 0fBF000000;\n\t"
      "selp.f32 %0, %1, %2, q;\n\t}"
      : "=f"(y)
      : "f"(p), "f"(e), "f"(x));
  return y;
}
// x > 0 ? x : y, as a choice.
__device__ __forceinline__ float above_zero(float x, float y) {
  float r;
  asm("{\n\t.reg .pred q;\n\tsetp.gt.f32 q, %1, 0f00000000;\n\t"
      "selp.f32 %0, %1, %2, q;\n\t}"
      : "=f"(r)
      : "f"(x), "f"(y));
  return r;
}

// 1 / (1 + e^-z), from e^-|z| so that nothing overflows.
__device__ __forceinline__ float sigmoid_near(float z) {
  const float u = exp_near(-fabsf(z)), r = inverse_near(1.0f + u);
  return z >= 0.0f ? r : (z < 0.0f ? u * r : z);  // NaN stays
}

// The normal distribution function Phi(z) = erfc(-z / sqrt 2) / 2 and
// e^(-z^2 / 2), two at a time.  For u = |z| / sqrt 2, erfc(u) / 2 =
// t P(t) e^(-u^2) with t = 1 / (1 + u / 2): P is smooth on the whole half
// line, and its polynomial of degree 8 (least maximal relative error on
// t in [1/6, 1], by reweighted least squares in extended precision) is within
// 4.3e-8 of it.  Where t is below 1/6 (|z| > 14.1, without bound), e^(-z^2 / 2)
// is below 2^-144, the last bits of f32's smallest numbers, or 0, and P, which
// stays between 0.14 and 0.17, does not matter.  Above 0, Phi(z) = 1 - Phi(-z).
__device__ __forceinline__ void normal_cdf(const Two<float> &z, Two<float> &phi,
                                           Two<float> &e) {
  const Two<float> t = {
      inverse_near(::fmaf(0.35355339059327376f, fabsf(z.x), 1.0f)),
      inverse_near(::fmaf(0.35355339059327376f, fabsf(z.y), 1.0f))};
  Two<float> p = twice(-0.02954281121492386f);
  p = fma(p, t, twice(0.14232470095157623f));
  p = fma(p, t, twice(-0.24366994202136993f));
  p = fma(p, t, twice(0.1391056925058365f));
  p = fma(p, t, twice(-0.013357238844037056f));
  p = fma(p, t, twice(0.10136011987924576f));
  p = fma(p, t, twice(0.12154816091060638f));
  p = fma(p, t, twice(0.1411880999803543f));
  p = fma(p, t, twice(0.1410430818796157f));
  const Two<float> x = mul(mul(z, z), twice(-0.72134752044448170f));
  e = {exp2_near(x.x), exp2_near(x.y)};
  const Two<float> h = mul(mul(p, t), e);
  phi = {z.x < 0.0f ? h.x : 1.0f - h.x, z.y < 0.0f ? h.y : 1.0f - h.y};
}

// tanh(softplus(z)) = w / d; with u = e^-|z|: w = u (u + 2), d = w + 2 for
// z <= 0, w = 1 + 2u, d = 1 + 2u + 2u^2 above.
__device__ __forceinline__ void mish_parts(float z, float &u, float &w, float &d) {
  u = exp_near(-fabsf(z));
  w = z > 0.0f ? ::fmaf(2.0f, u, 1.0f) : u * (u + 2.0f);
  d = z > 0.0f ? ::fmaf(2.0f * u, u, w) : w + 2.0f;
}

// v[i] = act(v[i]); the switch is outside the loops (act is the same for the
// whole launch).
template <int N>
__device__ __forceinline__ void act_f32(uint32_t act, float (&v)[N]) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = v[i] > 0.0f ? v[i] : 0.0f;
      break;
    case HEXIR_ACT_LEAKY_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = v[i] > 0.0f ? v[i] : (float)HEXIR_LEAKY_RELU_ALPHA * v[i];
      break;
    case HEXIR_ACT_ELU:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = above_zero(v[i], expm1_near(v[i]));
      break;
    case HEXIR_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = sigmoid_near(v[i]);
      break;
    case HEXIR_ACT_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = tanhf(v[i]);
      break;
    case HEXIR_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const Two<float> z = {v[i], v[i + 1]};
        Two<float> phi, e;
        normal_cdf(z, phi, e);
        const Two<float> y = mul(z, phi);
        v[i] = y.x;
        v[i + 1] = y.y;
      }
      break;
    case HEXIR_ACT_SWISH:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] *= sigmoid_near(v[i]);
      break;
    case HEXIR_ACT_MISH:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float u, w, d;
        mish_parts(v[i], u, w, d);
        v[i] *= w * inverse_near(d);
      }
      break;
    default:
      break;
  }
}

// z with magnitudes above 128 made 128, as a factor of something that is 0 to f32
// from |z| = 105 on (and NaN for NaN).  An infinity, which a z beyond its type's
// range is stored as, would make that product NaN.  One instruction: bounded by
// a minimum and a maximum, the elementwise gradient took 6 to 14 % longer (gelu
// 8192 x 8192 88 us before, 93 with two, 91 with one; the products' epilogues
// are not slowed down by it).
__device__ __forceinline__ float factor_near(float z) {
  float r;
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(128.0f));
  return r;
}

// g[i] *= act'(z[i]).
template <int N>
__device__ __forceinline__ void slope_f32(uint32_t act, const float (&z)[N],
                                          float (&g)[N]) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < N; ++i)
        g[i] = z[i] > 0.0f ? g[i] : 0.0f * g[i];
      break;
    case HEXIR_ACT_LEAKY_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i)
        g[i] = z[i] > 0.0f ? g[i] : (float)HEXIR_LEAKY_RELU_ALPHA * g[i];
      break;
    case HEXIR_ACT_ELU:
#pragma unroll
      for (int i = 0; i < N; ++i)
        g[i] *= z[i] > 0.0f ? 1.0f : exp_near(z[i]);
      break;
    case HEXIR_ACT_SIGMOID:  // s (1 - s) = u / (1 + u)^2, u = e^-|z|
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = exp_near(-fabsf(z[i])), r = inverse_near(1.0f + u);
        g[i] *= u * r * r;
      }
      break;
    case HEXIR_ACT_TANH:  // sech^2 = 4u / (1 + u)^2, u = e^-2|z|
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = exp_near(-2.0f * fabsf(z[i])), r = inverse_near(1.0f + u);
        g[i] *= 4.0f * u * r * r;
      }
      break;
    case HEXIR_ACT_GELU:  // Phi(z) + z e^(-z^2 / 2) / sqrt(2 pi)
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const Two<float> at = {z[i], z[i + 1]};
        Two<float> phi, e;
        normal_cdf(at, phi, e);
        const Two<float> factor = {factor_near(z[i]), factor_near(z[i + 1])};
        const Two<float> s =
            fma(mul(factor, e), twice(0.39894228040143268f), phi);
        g[i] *= s.x;
        g[i + 1] *= s.y;
      }
      break;
    case HEXIR_ACT_SWISH:  // s (1 + z (1 - s)), 1 - s being sigmoid(-z)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = exp_near(-fabsf(z[i])), r = inverse_near(1.0f + u);
        const float s = z[i] > 0.0f ? r : u * r, c = z[i] > 0.0f ? u * r : r;
        g[i] *= s * ::fmaf(factor_near(z[i]), c, 1.0f);
      }
      break;
    case HEXIR_ACT_MISH:
      // t + z (1 - t^2) s with t = tanh(softplus(z)) = w / d, s = sigmoid(z):
      // (1 - t^2) s is 4 u^2 (1 + u) / d^2 for z > 0, 4 u (1 + u) / d^2 below.
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float u, w, d;
        mish_parts(z[i], u, w, d);
        const float r = inverse_near(d);
        const float c = 4.0f * u * (1.0f + u) * (z[i] > 0.0f ? u : 1.0f);
        g[i] *= ::fmaf(factor_near(z[i]) * c * r, r, w * r);
      }
      break;
    default:
      break;
  }
}

}  // namespace hexir
