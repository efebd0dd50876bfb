// gated.cu -- the gated linear layer and its gradients.
//
//   [g | u] = x op(w) + bias,  h = act(g) * u
//   dpre = [dh * u * act'(g) | dh * act(g)],  dx = dpre op(w)^T,
//   dw = x^T dpre (w stored [K,2F]) or dpre^T x ([2F,K]),  dbias = sum_rows dpre
#include <algorithm>
#include <cmath>

#include <cuda_bf16.h>

#include "mx_internal.h"
#include "mx_ptx.cuh"

namespace mx {
namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// act(z) and, for the backward pass, act'(z).
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

// One thread an output; 32 x 32 tiles of the operands in shared memory.
// C(m, n) = sum_k A(m, k) B(k, n), any strides.
template <typename TA, typename TB, typename TC, bool GATED>
__global__ void __launch_bounds__(1024) tile_kernel(const TA* a, int64_t am, int64_t ak,
                                                    const TB* b, int64_t bk, int64_t bn,
                                                    const TB* bias, TC* c, float* pre, int M,
                                                    int N, int K, int act) {
  __shared__ float sa[32][33], sb[32][33], su[32][33];
  const int tx = threadIdx.x, ty = threadIdx.y;
  const int m = blockIdx.y * 32 + ty, n = blockIdx.x * 32 + tx;
  float g = 0.0f, u = 0.0f;
  for (int k0 = 0; k0 < K; k0 += 32) {
    sa[ty][tx] = m < M && k0 + tx < K ? to_f(a[m * am + (k0 + tx) * ak]) : 0.0f;
    sb[ty][tx] = n < N && k0 + ty < K ? to_f(b[(k0 + ty) * bk + n * bn]) : 0.0f;
    if (GATED) su[ty][tx] = n < N && k0 + ty < K ? to_f(b[(k0 + ty) * bk + (n + N) * bn]) : 0.0f;
    __syncthreads();
    for (int k = 0; k < 32; ++k) {
      g += sa[ty][k] * sb[k][tx];
      if (GATED) u += sa[ty][k] * su[k][tx];
    }
    __syncthreads();
  }
  if (m >= M || n >= N) return;
  if (GATED) {
    if (bias) {
      g += to_f(bias[n]);
      u += to_f(bias[N + n]);
    }
    if (pre) {
      pre[static_cast<int64_t>(m) * 2 * N + n] = g;
      pre[static_cast<int64_t>(m) * 2 * N + N + n] = u;
    }
    g = act_value(act, g) * u;
  }
  put(c + static_cast<int64_t>(m) * N + n, g);
}

template <typename T>
__global__ void __launch_bounds__(256) dpre_kernel(const T* dh, const float* pre, float* dpre,
                                                   int64_t n, int F, int act) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t m = i / F, f = i - m * F;
    float a, da;
    act_grad(act, pre[m * 2 * F + f], a, da);
    const float d = to_f(dh[i]);
    dpre[m * 2 * F + f] = d * pre[m * 2 * F + F + f] * da;
    dpre[m * 2 * F + F + f] = d * a;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) colsum_kernel(const float* x, T* out, int rows, int cols) {
  __shared__ float sh[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  float s = 0.0f;
  if (c < cols)
    for (int64_t r = warp; r < rows; r += 8) s += x[r * cols + c];
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < cols) {
    s = 0.0f;
    for (int i = 0; i < 8; ++i) s += sh[i][lane];
    put(out + c, s);
  }
}

template <typename T>
int fwd(const GatedArgs& a, cudaStream_t s) {
  const dim3 grid((a.F + 31) / 32, (a.M + 31) / 32);
  const int64_t bk = a.tw ? 1 : 2ll * a.F, bn = a.tw ? a.K : 1;
  tile_kernel<T, T, T, true><<<grid, dim3(32, 32), 0, s>>>(
      static_cast<const T*>(a.x), a.K, 1, static_cast<const T*>(a.w), bk, bn,
      static_cast<const T*>(a.bias), static_cast<T*>(a.h), a.pre, a.M, a.F, a.K, a.act);
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

template <typename T>
int bwd(Context* ctx, const GatedArgs& a, cudaStream_t s) {
  const int F2 = 2 * a.F;
  float* dpre = static_cast<float*>(a.ws);
  const int64_t n = static_cast<int64_t>(a.M) * a.F;
  dpre_kernel<T><<<static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, ctx->num_sms * 8)), 256,
                   0, s>>>(static_cast<const T*>(a.dh), a.pre, dpre, n, a.F, a.act);
  const dim3 th(32, 32);
  const T* w = static_cast<const T*>(a.w);
  const T* x = static_cast<const T*>(a.x);
  if (a.dx) {
    const dim3 grid((a.K + 31) / 32, (a.M + 31) / 32);
    tile_kernel<float, T, T, false><<<grid, th, 0, s>>>(
        dpre, F2, 1, w, a.tw ? a.K : 1, a.tw ? 1 : F2, nullptr, static_cast<T*>(a.dx), nullptr,
        a.M, a.K, F2, 0);
  }
  if (a.dw && !a.tw) {
    const dim3 grid((F2 + 31) / 32, (a.K + 31) / 32);
    tile_kernel<T, float, T, false><<<grid, th, 0, s>>>(x, 1, a.K, dpre, F2, 1, nullptr,
                                                       static_cast<T*>(a.dw), nullptr, a.K, F2,
                                                       a.M, 0);
  } else if (a.dw) {
    const dim3 grid((a.K + 31) / 32, (F2 + 31) / 32);
    tile_kernel<float, T, T, false><<<grid, th, 0, s>>>(dpre, 1, F2, x, a.K, 1, nullptr,
                                                       static_cast<T*>(a.dw), nullptr, F2, a.K,
                                                       a.M, 0);
  }
  if (a.dbias)
    colsum_kernel<T><<<(F2 + 31) / 32, 256, 0, s>>>(dpre, static_cast<T*>(a.dbias), a.M, F2);
  note_launches(4);
  return cuda_status(cudaGetLastError());
}

}  // namespace

size_t gated_workspace_bytes(const Context* ctx, const GatedArgs& a, bool backward) {
  (void)ctx;
  return backward ? static_cast<size_t>(a.M) * 2 * a.F * sizeof(float) : 0;
}

int gated_fwd(Context* ctx, const GatedArgs& a, cudaStream_t s) {
  (void)ctx;
  return a.dtype == MX_BF16 ? fwd<__nv_bfloat16>(a, s) : fwd<float>(a, s);
}

int gated_bwd(Context* ctx, const GatedArgs& a, cudaStream_t s) {
  return a.dtype == MX_BF16 ? bwd<__nv_bfloat16>(ctx, a, s) : bwd<float>(ctx, a, s);
}

}  // namespace mx
