// gated_act.cuh -- the gated layer's activations and their derivatives.
#pragma once
#include <cuda_bf16.h>

#include "../../include/mx_matmul.h"

namespace mx {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// 1 / y and x / y to 2 units in the last place, without the slow path of an
// exact division; y is 1 or more here, and from 2^126 on the result is 0.
__device__ __forceinline__ float ratio(float x, float y) { return __fdividef(x, y); }

template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == MX_ACT_SILU) return ratio(z, 1.0f + expf(-z));
  if constexpr (ACT == MX_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  if constexpr (ACT == MX_ACT_GELU_TANH)
    return 0.5f * z * (1.0f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
  if constexpr (ACT == MX_ACT_RELU) return z > 0.0f ? z : 0.0f;
  if constexpr (ACT == MX_ACT_SIGMOID) return ratio(1.0f, 1.0f + expf(-z));
  return z;
}
template <int ACT>
__device__ __forceinline__ void act_grad_of(float z, float& a, float& da) {
  if constexpr (ACT == MX_ACT_SILU) {
    const float s = ratio(1.0f, 1.0f + expf(-z));
    a = z * s;
    da = s * (1.0f + z * (1.0f - s));
  } else if constexpr (ACT == MX_ACT_GELU) {
    const float c = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
    a = z * c;
    da = c + z * expf(-0.5f * z * z) * 0.39894228040143268f;
  } else if constexpr (ACT == MX_ACT_GELU_TANH) {
    const float k = 0.79788456080286536f;
    const float t = tanhf(k * (z + 0.044715f * z * z * z));
    a = 0.5f * z * (1.0f + t);
    da = 0.5f * (1.0f + t) + 0.5f * z * (1.0f - t * t) * k * (1.0f + 0.134145f * z * z);
  } else if constexpr (ACT == MX_ACT_RELU) {
    a = z > 0.0f ? z : 0.0f;
    da = z > 0.0f ? 1.0f : 0.0f;
  } else {
    a = ratio(1.0f, 1.0f + expf(-z));
    da = a * (1.0f - a);
  }
}

// The activation is chosen once for N values, not for each: a choice inside an
// unrolled loop repeats every activation's code N times, which the instruction
// cache does not hold.
template <int ACT, int N>
__device__ __forceinline__ void gate_n(float (&g)[N], const float (&u)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) g[i] = act_of<ACT>(g[i]) * u[i];
}
// g = act(g) * u
template <int N>
__device__ __forceinline__ void gate(int act, float (&g)[N], const float (&u)[N]) {
  switch (act) {
    case MX_ACT_SILU: gate_n<MX_ACT_SILU>(g, u); return;
    case MX_ACT_GELU: gate_n<MX_ACT_GELU>(g, u); return;
    case MX_ACT_GELU_TANH: gate_n<MX_ACT_GELU_TANH>(g, u); return;
    case MX_ACT_RELU: gate_n<MX_ACT_RELU>(g, u); return;
    default: gate_n<MX_ACT_SIGMOID>(g, u);
  }
}
template <int ACT, int N>
__device__ __forceinline__ void gate_grad_n(const float (&d)[N], float (&g)[N], float (&u)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float a, da;
    act_grad_of<ACT>(g[i], a, da);
    g[i] = d[i] * u[i] * da;
    u[i] = d[i] * a;
  }
}
// (g, u) = (d * u * act'(g), d * act(g))
template <int N>
__device__ __forceinline__ void gate_grad(int act, const float (&d)[N], float (&g)[N],
                                          float (&u)[N]) {
  switch (act) {
    case MX_ACT_SILU: gate_grad_n<MX_ACT_SILU>(d, g, u); return;
    case MX_ACT_GELU: gate_grad_n<MX_ACT_GELU>(d, g, u); return;
    case MX_ACT_GELU_TANH: gate_grad_n<MX_ACT_GELU_TANH>(d, g, u); return;
    case MX_ACT_RELU: gate_grad_n<MX_ACT_RELU>(d, g, u); return;
    default: gate_grad_n<MX_ACT_SIGMOID>(d, g, u);
  }
}

}  // namespace mx
