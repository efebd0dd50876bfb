// norm_ops.cu -- layer norm over the last dimension, forward and backward.
//
//   mean = sum(x) / C,  rstd = 1 / sqrt(sum((x - mean)^2) / C + eps)
//   xhat = (x - mean) * rstd,  y = xhat * weight + bias
//   with a = dy * weight:  dx = rstd * (a - mean(a) - xhat * mean(a * xhat))
//   dweight = sum over rows of dy * xhat,  dbias = sum over rows of dy
//
// x, y, dy, dx are float32 or bfloat16, weight, bias and their gradients
// float32 (the framework keeps its parameters in float32); every sum is held
// in float32.  All of it is bound by the bytes of the rows: a row is read once
// into registers, the two moments are taken there (mean first, then the
// centred squares: no cancellation at a large mean), and it is written once.
// The backward pass keeps each thread's columns of dweight and dbias in
// registers over all the rows of its block; the blocks' partial sums are added
// in a fixed order by a second, small kernel, so results repeat bit for bit.
#include <algorithm>

#include <cuda_bf16.h>

#include "../../include/mx_matmul.h"
#include "mx_internal.h"
#include "mx_ptx.cuh"

namespace mx {
namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// V consecutive values; V > 1: one 16-byte access.
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f(*p);
  } else {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y);
      v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // bf16 is the upper half of a float32
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// float32 parameters at the same columns (V values; 16-byte loads when V > 1)
template <int V>
__device__ __forceinline__ void load_par(const float* p, int c, float (&v)[V], float none) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = none;
  } else if constexpr (V == 1) {
    v[0] = __ldg(p + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 t = __ldg(reinterpret_cast<const float4*>(p + c + i));
      v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    }
  }
}

// Sums of N values over the TPR threads of a row, given to all of them, in a
// fixed order.  TPR = 32: the row is a warp's.  Otherwise the block's: `buf`
// holds two sets of N floats a warp, used in turn, so that one barrier a sum is
// enough (whoever writes a set again has passed the barrier of the sum between,
// which its readers reach after reading).
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float* buf, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    float* b = buf + turn * N * W;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) b[i * W + (threadIdx.x >> 5)] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = b[i * W + (threadIdx.x & (W - 1))];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  }
}

// Rows in flight of a block: a thread copies its own 16-byte pieces of the next
// rows to its own places in shared memory (no other thread reads them, so no
// barrier), and takes them into registers when their turn comes.
constexpr int kRingBytes = 200 * 1024;  // of an SM, over its blocks
__host__ __device__ constexpr int block_threads(int tpr) { return tpr == 32 ? 128 : tpr; }
// Blocks an SM is given: 768 threads forward (one tensor), 512 backward (two,
// and the columns' sums in registers).
__host__ __device__ constexpr int blocks_per_sm(int tpr, int tensors) {
  const int n = (tensors == 1 ? 768 : 512) / block_threads(tpr);
  return n < 1 ? 1 : n;
}
__host__ __device__ constexpr int ring_rows(int tpr, int e, int size, int tensors) {
  const int d = kRingBytes / blocks_per_sm(tpr, tensors) / (block_threads(tpr) * e * size * tensors);
  return d < 1 ? 1 : d > 4 ? 4 : d;
}
__host__ __device__ constexpr int ring_bytes(int tpr, int e, int size, int tensors, int v) {
  return v == 1 ? 0 : ring_rows(tpr, e, size, tensors) * block_threads(tpr) * e * size * tensors;
}
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}

struct NormFwd {
  const void* x;
  const float* w;
  const float* b;
  void* y;
  float* mean;
  float* rstd;
  int64_t ldx, ldy;
  int rows, cols;
  float eps;
};

// Rows of up to TPR * E values, in registers: a thread holds E / V groups of V
// consecutive columns.  A block takes rows blockIdx.x, + gridDim.x, ...
// (TPR = 32: four at a time, one a warp).
template <typename T, int TPR, int E, int V>
__global__ void __launch_bounds__(block_threads(TPR), blocks_per_sm(TPR, 1)) norm_fwd_kernel(const NormFwd p) {
  constexpr int NV = E / V, D = ring_rows(TPR, E, sizeof(T), 1), BLOCK = block_threads(TPR);
  extern __shared__ uint4 ring[];  // [D][NV][BLOCK]
  __shared__ __align__(16) float buf[TPR > 32 ? 2 * 2 * TPR / 32 : 1];
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t step = TPR == 32 ? gridDim.x * 4ll : gridDim.x;
  int64_t row = TPR == 32 ? blockIdx.x * 4ll + (threadIdx.x >> 5) : blockIdx.x;
  const float inv_n = 1.0f / static_cast<float>(p.cols);
  auto fetch = [&](int64_t r, int slot) {
    if constexpr (V > 1) {
      if (r < p.rows) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + t) * V;
          if (c < p.cols) copy16(ring + (slot * NV + i) * BLOCK + threadIdx.x, x + c);
        }
      }
      cp_async_commit();
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(row + d * step, d);
  float w[NV][V], b[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V;
    if (c < p.cols) {
      load_par<V>(p.w, c, w[i], 1.0f);
      load_par<V>(p.b, c, b[i], 0.0f);
    }
  }
  int slot = 0, turn = 0;
  for (; row < p.rows; row += step) {
    float v[NV][V];
    float s[1] = {0.0f};
    if constexpr (V > 1) cp_async_wait<D - 1>();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < p.cols) {
        if constexpr (V > 1)
          load_vec<T, V>(reinterpret_cast<const T*>(ring + (slot * NV + i) * BLOCK + threadIdx.x), v[i]);
        else
          load_vec<T, V>(static_cast<const T*>(p.x) + row * p.ldx + c, v[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) s[0] += v[i][j];
      }
    }
    fetch(row + D * step, slot);
    slot = slot + 1 == D ? 0 : slot + 1;
    row_sum<TPR>(s, buf, turn);
    const float mean = s[0] * inv_n;
    // The centred values' own mean is what rounding left of it: it is taken off
    // the values and off the variance, so a mean far above the deviation costs
    // no more than the rounding of x itself.
    float q[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * TPR + t) * V < p.cols)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[i][j] -= mean;
          q[0] += v[i][j];
          q[1] += v[i][j] * v[i][j];
        }
    row_sum<TPR>(q, buf, turn);
    const float rest = q[0] * inv_n;
    const float var = q[1] * inv_n - rest * rest;
    const float rstd = rsqrtf((var < 0.0f ? 0.0f : var) + p.eps);  // NaN stays NaN
    if (t == 0) {
      if (p.mean) p.mean[row] = mean + rest;
      if (p.rstd) p.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(p.y) + row * p.ldy;
    const float shift = rest * rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < p.cols) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = (v[i][j] * rstd - shift) * w[i][j] + b[i][j];
        store_vec<T, V>(y + c, v[i]);
      }
    }
  }
}

// Rows longer than the registers of a block hold: three passes over the row,
// the second and third from the caches.
template <typename T>
__global__ void __launch_bounds__(1024) norm_fwd_long_kernel(const NormFwd p) {
  __shared__ __align__(16) float buf[2 * 2 * 32];
  int turn = 0;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  float s[1] = {0.0f};
  for (int c = threadIdx.x; c < p.cols; c += 1024) s[0] += to_f(x[c]);
  row_sum<1024>(s, buf, turn);
  const float mean = s[0] / static_cast<float>(p.cols);
  float q[2] = {0.0f, 0.0f};
  for (int c = threadIdx.x; c < p.cols; c += 1024) {
    const float d = to_f(x[c]) - mean;
    q[0] += d;
    q[1] += d * d;
  }
  row_sum<1024>(q, buf, turn);
  const float n = static_cast<float>(p.cols), rest = q[0] / n;
  const float var = q[1] / n - rest * rest;
  const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + p.eps);  // NaN stays NaN
  if (threadIdx.x == 0) {
    if (p.mean) p.mean[row] = mean + rest;
    if (p.rstd) p.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(p.y) + row * p.ldy;
  for (int c = threadIdx.x; c < p.cols; c += 1024)
    y[c] = from_f<T>((to_f(x[c]) - mean - rest) * rstd * (p.w ? p.w[c] : 1.0f) + (p.b ? p.b[c] : 0.0f));
}

struct NormBwd {
  const void* dy;
  const void* x;
  const float* w;
  const float* mean;
  const float* rstd;
  void* dx;
  float* part;  // [blocks][2][cols]: each block's sums of dweight and dbias
  int64_t lddy, ldx, lddx;
  int rows, cols;
};

// Rows as in norm_fwd_kernel; TPR = 32: the four warps' sums meet in shared
// memory at the end.
template <typename T, int TPR, int E, int V>
__global__ void __launch_bounds__(block_threads(TPR), blocks_per_sm(TPR, 2)) norm_bwd_kernel(const NormBwd p) {
  constexpr int NV = E / V, D = ring_rows(TPR, E, sizeof(T), 2), BLOCK = block_threads(TPR);
  extern __shared__ uint4 ring[];  // [D][2][NV][BLOCK]
  __shared__ __align__(16) float buf[TPR > 32 ? 2 * 2 * TPR / 32 : 4 * 32 * E];
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int warp = threadIdx.x >> 5;
  const float inv_c = 1.0f / static_cast<float>(p.cols);
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) w[i][j] = dw[i][j] = db[i][j] = 0.0f;
    if (c < p.cols) load_par<V>(p.w, c, w[i], 1.0f);
  }
  const int64_t step = TPR == 32 ? gridDim.x * 4ll : gridDim.x;
  int64_t row = TPR == 32 ? blockIdx.x * 4ll + warp : blockIdx.x;
  auto fetch = [&](int64_t r, int slot) {
    if constexpr (V > 1) {
      if (r < p.rows) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx;
        const T* dy = static_cast<const T*>(p.dy) + r * p.lddy;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + t) * V;
          if (c < p.cols) {
            copy16(ring + (slot * 2 * NV + i) * BLOCK + threadIdx.x, x + c);
            copy16(ring + (slot * 2 * NV + NV + i) * BLOCK + threadIdx.x, dy + c);
          }
        }
      }
      cp_async_commit();
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(row + d * step, d);
  int slot = 0, turn = 0;
  float next_mean = 0.0f, next_rstd = 0.0f;  // a row ahead, like the rows
  if (row < p.rows) {
    next_mean = __ldg(p.mean + row);
    next_rstd = __ldg(p.rstd + row);
  }
  for (; row < p.rows; row += step) {
    const float mean = next_mean, rstd = next_rstd;
    if (row + step < p.rows) {
      next_mean = __ldg(p.mean + row + step);
      next_rstd = __ldg(p.rstd + row + step);
    }
    float xh[NV][V], a[NV][V];
    float s[2] = {0.0f, 0.0f};
    if constexpr (V > 1) cp_async_wait<D - 1>();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < p.cols) {
        if constexpr (V > 1) {
          load_vec<T, V>(reinterpret_cast<const T*>(ring + (slot * 2 * NV + i) * BLOCK + threadIdx.x), xh[i]);
          load_vec<T, V>(reinterpret_cast<const T*>(ring + (slot * 2 * NV + NV + i) * BLOCK + threadIdx.x), a[i]);
        } else {
          load_vec<T, V>(static_cast<const T*>(p.x) + row * p.ldx + c, xh[i]);
          load_vec<T, V>(static_cast<const T*>(p.dy) + row * p.lddy + c, a[i]);
        }
      }
    }
    fetch(row + D * step, slot);
    slot = slot + 1 == D ? 0 : slot + 1;
    // (x - mean) * rstd in one operation: the product's rounding is that of the
    // saved mean once more
    const float shift = -mean * rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * TPR + t) * V < p.cols)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          xh[i][j] = fmaf(xh[i][j], rstd, shift);
          dw[i][j] += a[i][j] * xh[i][j];
          db[i][j] += a[i][j];
          a[i][j] *= w[i][j];
          s[0] += a[i][j];
          s[1] += a[i][j] * xh[i][j];
        }
    row_sum<TPR>(s, buf, turn);
    // rstd * (a - mean(a) - xhat * mean(a * xhat))
    const float k1 = -rstd * (s[0] * inv_c), k2 = -rstd * (s[1] * inv_c);
    if (p.dx) {
      T* dx = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * V;
        if (c < p.cols) {
#pragma unroll
          for (int j = 0; j < V; ++j) a[i][j] = fmaf(a[i][j], rstd, fmaf(xh[i][j], k2, k1));
          store_vec<T, V>(dx + c, a[i]);
        }
      }
    }
  }
  if (!p.part) return;
  float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.cols;
  if constexpr (TPR == 32) {
    // the four warps' sums, in their order
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          buf[warp * 32 * E + (i * 32 + t) * V + j] = k ? db[i][j] : dw[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < p.cols; c += 128)
        out[k * p.cols + c] = (buf[c] + buf[32 * E + c]) + (buf[2 * 32 * E + c] + buf[3 * 32 * E + c]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < p.cols)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          out[c + j] = dw[i][j];
          out[p.cols + c + j] = db[i][j];
        }
    }
  }
}

// Long rows: dx in two passes over the row; the columns' sums are a kernel of
// their own (norm_cols_kernel), since no block holds a row's columns.
template <typename T>
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(const NormBwd p) {
  __shared__ __align__(16) float buf[2 * 2 * 32];
  int turn = 0;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
  T* dx = static_cast<T*>(p.dx) + row * p.lddx;
  const float mean = p.mean[row], rstd = p.rstd[row];
  float s[2] = {0.0f, 0.0f};
  for (int c = threadIdx.x; c < p.cols; c += 1024) {
    const float a = to_f(dy[c]) * (p.w ? p.w[c] : 1.0f);
    s[0] += a;
    s[1] += a * ((to_f(x[c]) - mean) * rstd);
  }
  row_sum<1024>(s, buf, turn);
  const float inv_c = 1.0f / static_cast<float>(p.cols);
  const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
  for (int c = threadIdx.x; c < p.cols; c += 1024) {
    const float a = to_f(dy[c]) * (p.w ? p.w[c] : 1.0f);
    dx[c] = from_f<T>(rstd * (a - c1 - (to_f(x[c]) - mean) * rstd * c2));
  }
}
template <typename T>
__global__ void __launch_bounds__(256) norm_cols_kernel(const NormBwd p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.cols) return;
  const int64_t per = (static_cast<int64_t>(p.rows) + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per, r1 = r0 + per < p.rows ? r0 + per : p.rows;
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = to_f(static_cast<const T*>(p.dy)[r * p.lddy + c]);
    dw += g * ((to_f(static_cast<const T*>(p.x)[r * p.ldx + c]) - p.mean[r]) * p.rstd[r]);
    db += g;
  }
  float* out = p.part + static_cast<int64_t>(blockIdx.y) * 2 * p.cols;
  out[c] = dw;
  out[p.cols + c] = db;
}

// Small problems in one launch: the first row_blocks blocks make dx, a warp a
// row, in two passes over it (the second from L1); the others sum 32 columns of
// dweight and dbias each over all rows, reading x and dy once more, from L2.
constexpr int kSmallWarps = 16;
template <typename T, int V>
__global__ void __launch_bounds__(32 * kSmallWarps) norm_bwd_small_kernel(const NormBwd p, float* dw, float* db,
                                                             int row_blocks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) < row_blocks) {
    const int64_t row = blockIdx.x * static_cast<int64_t>(kSmallWarps) + warp;
    if (row >= p.rows) return;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    T* dx = static_cast<T*>(p.dx) + row * p.lddx;
    const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    float s[2] = {0.0f, 0.0f};
    int turn = 0;
#pragma unroll 4
    for (int c = lane * V; c < p.cols; c += 32 * V) {
      float xv[V], a[V], w[V];
      load_vec<T, V>(x + c, xv);
      load_vec<T, V>(dy + c, a);
      load_par<V>(p.w, c, w, 1.0f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        a[j] *= w[j];
        s[0] += a[j];
        s[1] += a[j] * ((xv[j] - mean) * rstd);
      }
    }
    row_sum<32>(s, nullptr, turn);
    const float inv_c = 1.0f / static_cast<float>(p.cols);
    const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
#pragma unroll 4
    for (int c = lane * V; c < p.cols; c += 32 * V) {
      float xv[V], a[V], w[V];
      load_vec<T, V>(x + c, xv);
      load_vec<T, V>(dy + c, a);
      load_par<V>(p.w, c, w, 1.0f);
#pragma unroll
      for (int j = 0; j < V; ++j)
        a[j] = rstd * (a[j] * w[j] - c1 - (xv[j] - mean) * rstd * c2);
      store_vec<T, V>(dx + c, a);
    }
    return;
  }
  __shared__ float sh[2][kSmallWarps][33];
  const int64_t c = (blockIdx.x - row_blocks) * 32ll + lane;
  float sw = 0.0f, sb = 0.0f;
  if (c < p.cols) {
    const T* dy = static_cast<const T*>(p.dy) + c;
    const T* x = static_cast<const T*>(p.x) + c;
    for (int r0 = warp; r0 < p.rows; r0 += 8 * kSmallWarps) {
      T g[8], xv[8];
      float mean[8], rstd[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // past the last row: the last one, not added
        const int64_t r = min(r0 + i * kSmallWarps, p.rows - 1);
        g[i] = dy[r * p.lddy];
        xv[i] = x[r * p.ldx];
        mean[i] = p.mean[r];
        rstd[i] = p.rstd[r];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + i * kSmallWarps < p.rows) {
          sw += to_f(g[i]) * ((to_f(xv[i]) - mean[i]) * rstd[i]);
          sb += to_f(g[i]);
        }
    }
  }
  sh[0][warp][lane] = sw;
  sh[1][warp][lane] = sb;
  __syncthreads();
  if (warp < 2 && c < p.cols) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kSmallWarps; ++i) s += sh[warp][i][lane];
    float* out = warp == 0 ? dw : db;
    if (out) out[c] = s;
  }
}

// out[c] = the sum over `blocks` partial rows; column c < cols goes to dw, the
// rest to db.  A block takes 32 columns, its warps a share of the rows each; the
// order is fixed.
constexpr int kFinishWarps = 32;
__global__ void __launch_bounds__(32 * kFinishWarps) norm_finish_kernel(
    const float* __restrict__ part, int blocks, int cols, float* dw, float* db) {
  __shared__ float sh[kFinishWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t width = 2ll * cols, c = blockIdx.x * 32ll + lane;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int r = warp; r < blocks; r += kFinishWarps) s += part[r * width + c];
  }
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < width) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < kFinishWarps; ++i) s += sh[i][lane];
    if (c < cols) {
      if (dw) dw[c] = s;
    } else if (db) {
      db[c - cols] = s;
    }
  }
}

// Columns up to which a row is held in registers.
constexpr int kNormRegCols = 16384;

// Blocks of a pass over rows: as many as fit on the SMs at a time.
int row_blocks(int rows, int cols, int per_sm, int num_sms) {
  const int at_once = cols <= 512 ? 4 : 1;  // rows of a block
  return std::max(1, std::min(per_sm * num_sms, (rows + at_once - 1) / at_once));
}

template <typename T, int TPR, int E, int V>
cudaError_t run_fwd(const NormFwd& p, int num_sms, cudaStream_t s) {
  constexpr int kBytes = ring_bytes(TPR, E, sizeof(T), 1, V);
  auto kern = norm_fwd_kernel<T, TPR, E, V>;
  static SmemOptIn opt_in;
  cudaError_t e = kBytes > 32768 ? opt_in.ensure(kern, kBytes) : cudaSuccess;
  if (e != cudaSuccess) return e;
  kern<<<row_blocks(p.rows, p.cols, blocks_per_sm(TPR, 1), num_sms), block_threads(TPR), kBytes,
         s>>>(p);
  return cudaGetLastError();
}
template <typename T, int V>
cudaError_t launch_fwd(const NormFwd& p, int num_sms, cudaStream_t s) {
  const int c = p.cols;
  if (c <= 256) return run_fwd<T, 32, 8, V>(p, num_sms, s);
  if (c <= 512) return run_fwd<T, 32, 16, V>(p, num_sms, s);
  if (c <= 1024) return run_fwd<T, 64, 16, V>(p, num_sms, s);
  if (c <= 2048) return run_fwd<T, 128, 16, V>(p, num_sms, s);
  if (c <= 4096) return run_fwd<T, 256, 16, V>(p, num_sms, s);
  if (c <= 8192) return run_fwd<T, 512, 16, V>(p, num_sms, s);
  return run_fwd<T, 1024, 16, V>(p, num_sms, s);
}

template <typename T, int TPR, int E, int V>
cudaError_t run_bwd(const NormBwd& p, int blocks, cudaStream_t s) {
  constexpr int kBytes = ring_bytes(TPR, E, sizeof(T), 2, V);
  auto kern = norm_bwd_kernel<T, TPR, E, V>;
  static SmemOptIn opt_in;
  cudaError_t e = kBytes > 32768 ? opt_in.ensure(kern, kBytes) : cudaSuccess;
  if (e != cudaSuccess) return e;
  kern<<<blocks, block_threads(TPR), kBytes, s>>>(p);
  return cudaGetLastError();
}
template <typename T, int V>
cudaError_t launch_bwd(const NormBwd& p, int blocks, cudaStream_t s) {
  const int c = p.cols;
  if (c <= 256) return run_bwd<T, 32, 8, V>(p, blocks, s);
  if (c <= 512) return run_bwd<T, 32, 16, V>(p, blocks, s);
  if (c <= 1024) return run_bwd<T, 64, 16, V>(p, blocks, s);
  if (c <= 2048) return run_bwd<T, 128, 16, V>(p, blocks, s);
  if (c <= 4096) return run_bwd<T, 256, 16, V>(p, blocks, s);
  if (c <= 8192) return run_bwd<T, 512, 16, V>(p, blocks, s);
  return run_bwd<T, 1024, 16, V>(p, blocks, s);
}

// Blocks of the backward pass (rows of partial sums).
int bwd_blocks(int rows, int cols, int num_sms) {
  if (cols > kNormRegCols) return std::min(64, (rows + 63) / 64);  // row ranges of norm_cols
  const int tpr = cols <= 512 ? 32 : cols <= 1024 ? 64 : cols <= 2048 ? 128 : cols <= 4096 ? 256
                : cols <= 8192 ? 512 : 1024;
  return row_blocks((rows + 1) / 2, cols, blocks_per_sm(tpr, 2), num_sms);
}

// Small enough for norm_bwd_small_kernel, whose columns' blocks walk down all
// rows and whose warps walk along theirs.  Float32, one launch against two, us:
// 64 x 257 2.7 / 5.1, 512 x 1024 4.9 / 8.6, 1000 x 257 8.2 / 6.9 (and a launch
// less for the host, 4 us); 256 x 2048 8.0 / 6.6, 128 x 4096 13.4 / 7.0.
bool bwd_small(int rows, int cols) { return rows <= 1024 && cols <= 1024; }

bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) == 0; }

}  // namespace

size_t layer_norm_bwd_scratch_bytes(const Context* ctx, int rows, int cols) {
  if (rows <= 0 || cols <= 0 || bwd_small(rows, cols)) return 0;
  return static_cast<size_t>(bwd_blocks(rows, cols, ctx->num_sms)) * 2 * cols * sizeof(float);
}

int layer_norm_fwd(Context* ctx, int dtype, const void* x, int64_t ldx, const float* w,
                   const float* b, void* y, int64_t ldy, float* mean, float* rstd, int rows,
                   int cols, float eps, cudaStream_t s) {
  if (rows <= 0) return kOk;
  const int n = ctx->num_sms;
  const NormFwd p{x, w, b, y, mean, rstd, ldx, ldy, rows, cols, eps};
  const int vec = dtype == MX_BF16 ? 8 : 4;
  const bool v16 = cols % vec == 0 && ldx % vec == 0 && ldy % vec == 0 && aligned16(x) &&
                   aligned16(y) && aligned16(w) && aligned16(b);
  cudaError_t e;
  if (cols > kNormRegCols) {
    if (dtype == MX_BF16) norm_fwd_long_kernel<__nv_bfloat16><<<rows, 1024, 0, s>>>(p);
    else norm_fwd_long_kernel<float><<<rows, 1024, 0, s>>>(p);
    e = cudaGetLastError();
  } else if (dtype == MX_BF16) {
    e = v16 ? launch_fwd<__nv_bfloat16, 8>(p, n, s) : launch_fwd<__nv_bfloat16, 1>(p, n, s);
  } else {
    e = v16 ? launch_fwd<float, 4>(p, n, s) : launch_fwd<float, 1>(p, n, s);
  }
  note_launches(1);
  return cuda_status(e);
}

int layer_norm_bwd(Context* ctx, int dtype, const void* dy, int64_t lddy, const void* x,
                   int64_t ldx, const float* w, const float* mean, const float* rstd, void* dx,
                   int64_t lddx, float* dw, float* db, int rows, int cols, void* scratch,
                   size_t scratch_bytes, cudaStream_t s) {
  const bool sums = dw || db;
  if (rows <= 0) {  // an empty sum is zero
    cudaError_t e = dw ? cudaMemsetAsync(dw, 0, sizeof(float) * cols, s) : cudaSuccess;
    if (e == cudaSuccess && db) e = cudaMemsetAsync(db, 0, sizeof(float) * cols, s);
    return cuda_status(e);
  }
  const int vec = dtype == MX_BF16 ? 8 : 4;
  const bool v16 = cols % vec == 0 && ldx % vec == 0 && lddy % vec == 0 && aligned16(x) &&
                   aligned16(dy) && aligned16(w) && (!dx || (lddx % vec == 0 && aligned16(dx)));
  if (bwd_small(rows, cols)) {
    const NormBwd p{dy, x, w, mean, rstd, dx, nullptr, lddy, ldx, lddx, rows, cols};
    const int rb = dx ? (rows + kSmallWarps - 1) / kSmallWarps : 0, grid = rb + (sums ? (cols + 31) / 32 : 0);
    if (grid == 0) return kOk;
    if (dtype == MX_BF16) {
      if (v16) norm_bwd_small_kernel<__nv_bfloat16, 8><<<grid, 32 * kSmallWarps, 0, s>>>(p, dw, db, rb);
      else norm_bwd_small_kernel<__nv_bfloat16, 1><<<grid, 32 * kSmallWarps, 0, s>>>(p, dw, db, rb);
    } else {
      if (v16) norm_bwd_small_kernel<float, 4><<<grid, 32 * kSmallWarps, 0, s>>>(p, dw, db, rb);
      else norm_bwd_small_kernel<float, 1><<<grid, 32 * kSmallWarps, 0, s>>>(p, dw, db, rb);
    }
    note_launches(1);
    return cuda_status(cudaGetLastError());
  }
  if (sums && (!scratch || scratch_bytes < layer_norm_bwd_scratch_bytes(ctx, rows, cols)))
    return kErrInvalid;
  const int blocks = bwd_blocks(rows, cols, ctx->num_sms);
  const NormBwd p{dy, x, w, mean, rstd, dx, sums ? static_cast<float*>(scratch) : nullptr,
                  lddy, ldx, lddx, rows, cols};
  cudaError_t e = cudaSuccess;
  if (cols > kNormRegCols) {
    if (dx) {
      if (dtype == MX_BF16) norm_bwd_long_kernel<__nv_bfloat16><<<rows, 1024, 0, s>>>(p);
      else norm_bwd_long_kernel<float><<<rows, 1024, 0, s>>>(p);
      note_launches(1);
      e = cudaGetLastError();
    }
    if (e == cudaSuccess && sums) {
      const dim3 grid((cols + 255) / 256, blocks);
      if (dtype == MX_BF16) norm_cols_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
      else norm_cols_kernel<float><<<grid, 256, 0, s>>>(p);
      note_launches(1);
      e = cudaGetLastError();
    }
  } else {
    e = dtype == MX_BF16 ? (v16 ? launch_bwd<__nv_bfloat16, 8>(p, blocks, s)
                                : launch_bwd<__nv_bfloat16, 1>(p, blocks, s))
                         : (v16 ? launch_bwd<float, 4>(p, blocks, s)
                                : launch_bwd<float, 1>(p, blocks, s));
    note_launches(1);
  }
  if (e == cudaSuccess && sums) {
    norm_finish_kernel<<<static_cast<unsigned>((2ll * cols + 31) / 32), 32 * kFinishWarps, 0, s>>>(static_cast<const float*>(scratch),
                                                           blocks, cols, dw, db);
    note_launches(1);
    e = cudaGetLastError();
  }
  return cuda_status(e);
}

}  // namespace mx
