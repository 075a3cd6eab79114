// activation_f32.cuh -- the activations and their slopes in f32, for the
// epilogues of the 16-bit products and the elementwise gradient.  The forms
// keep relative accuracy where 1 - t or 1 + erf would cancel; results are
// rounded to bf16 or f16 (by up to 2^-8, 2^-11 of the value) after them.
#pragma once

#include <stdint.h>

#include "launch_abi.h"

namespace hexir {

constexpr uint32_t kActNone = 0u;
constexpr uint32_t kActRelu = 3u;

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
        v[i] = v[i] > 0.0f ? v[i] : expm1f(v[i]);
      break;
    case HEXIR_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = 1.0f / (1.0f + expf(-v[i]));
      break;
    case HEXIR_ACT_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = tanhf(v[i]);
      break;
    case HEXIR_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = 0.5f * v[i] * erfcf(-0.70710678118654752f * v[i]);
      break;
    case HEXIR_ACT_SWISH:
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = v[i] / (1.0f + expf(-v[i]));
      break;
    case HEXIR_ACT_MISH:
      // tanh(softplus(x)) = w / (w + 2), w = u (u + 2), u = e^x; for x > 0
      // with u = e^-x: (1 + 2u) / (1 + 2u + 2u^2).
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = v[i], u = expf(-fabsf(x));
        const float w = x > 0.0f ? fmaf(2.0f, u, 1.0f) : u * (u + 2.0f);
        const float d = x > 0.0f ? fmaf(2.0f * u, u, w) : w + 2.0f;
        v[i] = x * (w / d);
      }
      break;
    default:
      break;
  }
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
        g[i] = z[i] > 0.0f ? g[i] : expf(z[i]) * g[i];
      break;
    case HEXIR_ACT_SIGMOID:  // s (1 - s) = u / (1 + u)^2, u = e^-|z|
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = expf(-fabsf(z[i])), d = 1.0f + u;
        g[i] *= u / (d * d);
      }
      break;
    case HEXIR_ACT_TANH:  // sech^2 = 4u / (1 + u)^2, u = e^-2|z|
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = expf(-2.0f * fabsf(z[i])), d = 1.0f + u;
        g[i] *= 4.0f * u / (d * d);
      }
      break;
    case HEXIR_ACT_GELU:  // Phi(z) + z phi(z)
#pragma unroll
      for (int i = 0; i < N; ++i)
        g[i] *= 0.5f * erfcf(-0.70710678118654752f * z[i]) +
                z[i] * (0.39894228040143268f * expf(-0.5f * z[i] * z[i]));
      break;
    case HEXIR_ACT_SWISH:  // s (1 + z (1 - s))
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float s = 1.0f / (1.0f + expf(-z[i]));
        g[i] *= s * fmaf(z[i], 1.0f - s, 1.0f);
      }
      break;
    case HEXIR_ACT_MISH:
      // t + z (1 - t^2) s with t = tanh(softplus(z)), s = sigmoid(z); with u
      // and the quotient w / d of the activation, (1 - t^2) s is
      // 4 u^2 (1 + u) / d^2 for z > 0 and 4 u (1 + u) / d^2 otherwise.
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = z[i], u = expf(-fabsf(x));
        const float w = x > 0.0f ? fmaf(2.0f, u, 1.0f) : u * (u + 2.0f);
        const float d = x > 0.0f ? fmaf(2.0f * u, u, w) : w + 2.0f;
        const float c = 4.0f * u * (1.0f + u) * (x > 0.0f ? u : 1.0f);
        g[i] *= w / d + x * (c / (d * d));
      }
      break;
    default:
      break;
  }
}

}  // namespace hexir
