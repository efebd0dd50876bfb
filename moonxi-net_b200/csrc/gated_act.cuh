// gated_act.cuh -- the gated layer's activations and their derivatives.
#pragma once
#include <cuda_bf16.h>

#include "../../include/mx_matmul.h"

namespace mx {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ float act_value(int act, float z) {
  switch (act) {
    case MX_ACT_SILU: return z / (1.0f + expf(-z));
    case MX_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case MX_ACT_GELU_TANH:
      return 0.5f * z * (1.0f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
    case MX_ACT_RELU: return z > 0.0f ? z : 0.0f;
    default: return 1.0f / (1.0f + expf(-z));
  }
}
__device__ __forceinline__ void act_grad(int act, float z, float& a, float& da) {
  switch (act) {
    case MX_ACT_SILU: {
      const float s = 1.0f / (1.0f + expf(-z));
      a = z * s;
      da = s * (1.0f + z * (1.0f - s));
      return;
    }
    case MX_ACT_GELU: {
      const float c = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
      a = z * c;
      da = c + z * expf(-0.5f * z * z) * 0.39894228040143268f;
      return;
    }
    case MX_ACT_GELU_TANH: {
      const float k = 0.79788456080286536f;
      const float t = tanhf(k * (z + 0.044715f * z * z * z));
      a = 0.5f * z * (1.0f + t);
      da = 0.5f * (1.0f + t) + 0.5f * z * (1.0f - t * t) * k * (1.0f + 0.134145f * z * z);
      return;
    }
    case MX_ACT_RELU:
      a = z > 0.0f ? z : 0.0f;
      da = z > 0.0f ? 1.0f : 0.0f;
      return;
    default:
      a = 1.0f / (1.0f + expf(-z));
      da = a * (1.0f - a);
  }
}

}  // namespace mx
