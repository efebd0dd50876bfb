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
//
// Measured, with the copy rate of such sizes in mind (64 MB bf16: 5.4 TB/s):
// 8192 x 4096 bf16 25.5 us forward (134 MB, 5.3 TB/s), 42 us backward (201 MB,
// 4.8 TB/s; 16384 rows 69 us, 5.8 TB/s: a row's two sums wait for one another, the
// registers leave room for two blocks an SM, and every block has 32 KB of partial
// sums to write, which the finish reads in 5 us); float32 39 and 61 us (kernels
// alone, on overwritten caches, the L2 keeping part of what they write).
//
// The registers that the blocks leave (80 a thread forward, 128 backward) hold a
// row's values; of the 54 kernels 14 spill 4 to 28 bytes a thread to local memory
// beside them, most of them of rows off 16 bytes.
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
// fixed order.  TPR = 32: the row is a warp's.  Otherwise the row is the
// block's, or (rows > 1) that of the block's group-th TPR threads, which have a
// named barrier of their own.  `buf` holds two sets of N floats a warp of the
// row, used in turn, so that one barrier a sum is enough (whoever writes a set
// again has passed the barrier of the sum between, which its readers reach
// after reading).
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float* buf, int& turn, int rows = 1,
                                        int group = 0) {
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
      for (int i = 0; i < N; ++i) b[i * W + (threadIdx.x % TPR >> 5)] = s[i];
    if (rows == 1) {
      __syncthreads();
    } else {
      __syncwarp();  // the barrier is an instruction of whole warps
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
    }
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
// Threads of a block: forward a row's (or four rows' of a warp each), backward
// 256 (or a longer row's), so that few blocks have partial sums to write.
__host__ __device__ constexpr int block_threads(int tpr, int tensors) {
  return tensors == 1 ? (tpr == 32 ? 128 : tpr) : tpr < 256 ? 256 : tpr;
}
// Blocks an SM is given: 768 threads forward (one tensor), 512 backward (two,
// and the columns' sums in registers).
__host__ __device__ constexpr int blocks_per_sm(int tpr, int tensors) {
  const int n = (tensors == 1 ? 768 : 512) / block_threads(tpr, tensors);
  return n < 1 ? 1 : n;
}
__host__ __device__ constexpr int ring_rows(int tpr, int e, int size, int tensors) {
  const int d = kRingBytes / blocks_per_sm(tpr, tensors) /
                (block_threads(tpr, tensors) * e * size * tensors);
  return d < 1 ? 1 : d > 4 ? 4 : d;
}
__host__ __device__ constexpr int ring_bytes(int tpr, int e, int size, int tensors, int v) {
  return v == 1 ? 0
                : ring_rows(tpr, e, size, tensors) * block_threads(tpr, tensors) * e * size * tensors;
}
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}

// Two float32 in a register pair, one instruction for both (fma.rn.f32x2 and
// its kin): the backward pass has ten operations a value (8192 x 1024 bf16: 13.3
// us against 14.2 one at a time, 65536 x 256: 21.4 against 23.7).
using Pair = uint64_t;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(Pair p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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
__global__ void __launch_bounds__(block_threads(TPR, 1), blocks_per_sm(TPR, 1)) norm_fwd_kernel(const NormFwd p) {
  constexpr int NV = E / V, D = ring_rows(TPR, E, sizeof(T), 1), BLOCK = block_threads(TPR, 1);
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

// A block takes ROWS rows at a time, TPR threads each; the rows' sums of dweight
// and dbias meet in shared memory at the end.
template <typename T, int TPR, int E, int V>
__global__ void __launch_bounds__(block_threads(TPR, 2), blocks_per_sm(TPR, 2)) norm_bwd_kernel(const NormBwd p) {
  constexpr int NV = E / V, D = ring_rows(TPR, E, sizeof(T), 2), BLOCK = block_threads(TPR, 2);
  constexpr int ROWS = BLOCK / TPR;
  extern __shared__ uint4 ring[];  // [D][2][NV][BLOCK]
  __shared__ __align__(16) float buf[ROWS > 1 ? BLOCK * E : 2 * 2 * TPR / 32];
  grid_trigger();
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  float* sums = buf + (ROWS > 1 ? group * (2 * 2 * TPR / 32) : 0);
  const float inv_c = 1.0f / static_cast<float>(p.cols);
  // value e = i * V + j of a thread is column (i * TPR + t) * V + j; past the
  // last column all of it is zero
  Pair w[E / 2], dw[E / 2], db[E / 2];
  {
    float v[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = 0.0f;
      if (c < p.cols) load_par<V>(p.w, c, v[i], 1.0f);
    }
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      w[e / 2] = pair(v[e / V][e % V], v[(e + 1) / V][(e + 1) % V]);
      dw[e / 2] = db[e / 2] = pair(0.0f, 0.0f);
    }
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + group;
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
  // The rows' statistics, 32 rows of the block at a time, one a lane: a load a
  // row would be waited for at every row.
  float lane_mean = 0.0f, lane_rstd = 0.0f;
  for (int n = 0; row < p.rows; row += step, ++n) {
    if ((n & 31) == 0) {
      const int64_t r = row + (threadIdx.x & 31) * step;
      if (r < p.rows) {
        lane_mean = __ldg(p.mean + r);
        lane_rstd = __ldg(p.rstd + r);
      }
    }
    const float mean = __shfl_sync(0xffffffffu, lane_mean, n & 31);
    const float rstd = __shfl_sync(0xffffffffu, lane_rstd, n & 31);
    Pair xh[E / 2], a[E / 2];
    if constexpr (V > 1) cp_async_wait<D - 1>();
    {
      float xv[NV][V], g[NV][V];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          xv[i][j] = mean;  // past the last column: xhat is zero
          g[i][j] = 0.0f;
        }
        if (c < p.cols) {
          if constexpr (V > 1) {
            load_vec<T, V>(reinterpret_cast<const T*>(ring + (slot * 2 * NV + i) * BLOCK + threadIdx.x), xv[i]);
            load_vec<T, V>(reinterpret_cast<const T*>(ring + (slot * 2 * NV + NV + i) * BLOCK + threadIdx.x), g[i]);
          } else {
            load_vec<T, V>(static_cast<const T*>(p.x) + row * p.ldx + c, xv[i]);
            load_vec<T, V>(static_cast<const T*>(p.dy) + row * p.lddy + c, g[i]);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        xh[e / 2] = pair(xv[e / V][e % V], xv[(e + 1) / V][(e + 1) % V]);
        a[e / 2] = pair(g[e / V][e % V], g[(e + 1) / V][(e + 1) % V]);
      }
    }
    fetch(row + D * step, slot);
    slot = slot + 1 == D ? 0 : slot + 1;
    // (x - mean) * rstd, and not x * rstd - mean * rstd in one operation: that
    // would round mean * rstd, which is all there is in a row without deviation,
    // and overflow where this does not
    const Pair r2 = pair(rstd, rstd), shift = pair(-mean, -mean);
    Pair s0 = pair(0.0f, 0.0f), s1 = s0;
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      xh[e] = mul2(add2(xh[e], shift), r2);
      dw[e] = fma2(a[e], xh[e], dw[e]);
      db[e] = add2(db[e], a[e]);
      a[e] = mul2(a[e], w[e]);
      s0 = add2(s0, a[e]);
      s1 = fma2(a[e], xh[e], s1);
    }
    float s[2], hi[2];
    unpair(s0, s[0], hi[0]);
    unpair(s1, s[1], hi[1]);
    s[0] += hi[0];
    s[1] += hi[1];
    row_sum<TPR>(s, sums, turn, ROWS, group);
    // rstd * (a - mean(a) - xhat * mean(a * xhat))
    const float k1 = -rstd * (s[0] * inv_c), k2 = -rstd * (s[1] * inv_c);
    if (p.dx) {
      T* dx = static_cast<T*>(p.dx) + row * p.lddx;
      const Pair k1p = pair(k1, k1), k2p = pair(k2, k2);
      float v[NV][V];
#pragma unroll
      for (int e = 0; e < E; e += 2)
        unpair(fma2(a[e / 2], r2, fma2(xh[e / 2], k2p, k1p)), v[e / V][e % V],
               v[(e + 1) / V][(e + 1) % V]);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * V;
        if (c < p.cols) store_vec<T, V>(dx + c, v[i]);
      }
    }
  }
  float dwf[NV][V], dbf[NV][V];
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    unpair(dw[e / 2], dwf[e / V][e % V], dwf[(e + 1) / V][(e + 1) % V]);
    unpair(db[e / 2], dbf[e / V][e % V], dbf[(e + 1) / V][(e + 1) % V]);
  }
  if (!p.part) return;
  float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.cols;
  if constexpr (ROWS > 1) {
    // the rows' sums, in their order
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          buf[group * TPR * E + (i * TPR + t) * V + j] = k ? dbf[i][j] : dwf[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < p.cols; c += BLOCK) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) sum += buf[r * TPR * E + c];
        out[k * p.cols + c] = sum;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < p.cols)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          out[c + j] = dwf[i][j];
          out[p.cols + c + j] = dbf[i][j];
        }
    }
  }
}

// Long rows: dx in two passes over the row; the columns' sums are a kernel of
// their own (norm_cols_kernel), since no block holds a row's columns.
template <typename T, int V>
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(const NormBwd p) {
  __shared__ __align__(16) float buf[2 * 2 * 32];
  int turn = 0;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
  T* dx = static_cast<T*>(p.dx) + row * p.lddx;
  const float mean = p.mean[row], rstd = p.rstd[row];
  float s[2] = {0.0f, 0.0f};
#pragma unroll 2
  for (int c = threadIdx.x * V; c < p.cols; c += 1024 * V) {
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
  row_sum<1024>(s, buf, turn);
  const float inv_c = 1.0f / static_cast<float>(p.cols);
  const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
#pragma unroll 2
  for (int c = threadIdx.x * V; c < p.cols; c += 1024 * V) {
    float xv[V], a[V], w[V];
    load_vec<T, V>(x + c, xv);
    load_vec<T, V>(dy + c, a);
    load_par<V>(p.w, c, w, 1.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = rstd * (a[j] * w[j] - c1 - (xv[j] - mean) * rstd * c2);
    store_vec<T, V>(dx + c, a);
  }
}
// A block: 256 * V columns, a range of rows.
template <typename T, int V>
__global__ void __launch_bounds__(256) norm_cols_kernel(const NormBwd p) {
  grid_trigger();
  const int64_t c = (blockIdx.x * 256ll + threadIdx.x) * V;
  if (c >= p.cols) return;
  const int64_t per = (static_cast<int64_t>(p.rows) + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per, r1 = r0 + per < p.rows ? r0 + per : p.rows;
  float dw[V], db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) dw[j] = db[j] = 0.0f;
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    float xv[V], g[V];
    load_vec<T, V>(static_cast<const T*>(p.x) + r * p.ldx + c, xv);
    load_vec<T, V>(static_cast<const T*>(p.dy) + r * p.lddy + c, g);
    const float mean = __ldg(p.mean + r), rstd = __ldg(p.rstd + r);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      dw[j] += g[j] * ((xv[j] - mean) * rstd);
      db[j] += g[j];
    }
  }
  float* out = p.part + static_cast<int64_t>(blockIdx.y) * 2 * p.cols;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    out[c + j] = dw[j];
    out[p.cols + c + j] = db[j];
  }
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
  grid_wait();
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

// Columns up to which a row is held in registers.  (Backward, 2048 x 16384
// bf16: 137 us with the columns' sums of 1024 threads partly in local memory, 93
// us in two passes.)
constexpr int kFwdCols = 16384, kBwdCols = 8192;

// Blocks of a pass over rows, at_once each: as many as fit on the SMs at a time.
int row_blocks(int rows, int at_once, int per_sm, int num_sms) {
  return std::max(1, std::min(per_sm * num_sms, (rows + at_once - 1) / at_once));
}

template <typename T, int TPR, int E, int V>
cudaError_t run_fwd(const NormFwd& p, int num_sms, cudaStream_t s) {
  constexpr int kBytes = ring_bytes(TPR, E, sizeof(T), 1, V);
  auto kern = norm_fwd_kernel<T, TPR, E, V>;
  static SmemOptIn opt_in;
  cudaError_t e = kBytes > 32768 ? opt_in.ensure(kern, kBytes) : cudaSuccess;
  if (e != cudaSuccess) return e;
  const int at_once = block_threads(TPR, 1) / TPR;
  kern<<<row_blocks(p.rows, at_once, blocks_per_sm(TPR, 1), num_sms), block_threads(TPR, 1), kBytes,
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
  kern<<<blocks, block_threads(TPR, 2), kBytes, s>>>(p);
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
  return run_bwd<T, 512, 16, V>(p, blocks, s);
}

template <typename T, int V>
cudaError_t launch_long(const NormBwd& p, int blocks, cudaStream_t s) {
  if (p.dx) {
    norm_bwd_long_kernel<T, V><<<p.rows, 1024, 0, s>>>(p);
    note_launches(1);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  if (p.part) {
    norm_cols_kernel<T, V><<<dim3((p.cols + 256 * V - 1) / (256 * V), blocks), 256, 0, s>>>(p);
    note_launches(1);
  }
  return cudaGetLastError();
}

// Blocks of the backward pass (rows of partial sums).
int bwd_blocks(int rows, int cols, int num_sms) {
  if (cols > kBwdCols) return std::min(64, (rows + 63) / 64);  // row ranges of norm_cols
  const int tpr = cols <= 512 ? 32 : cols <= 1024 ? 64 : cols <= 2048 ? 128 : cols <= 4096 ? 256 : 512;
  return row_blocks((rows + 1) / 2, block_threads(tpr, 2) / tpr, blocks_per_sm(tpr, 2), num_sms);
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
  if (cols > kFwdCols) {
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
  if (cols > kBwdCols) {
    e = dtype == MX_BF16 ? (v16 ? launch_long<__nv_bfloat16, 8>(p, blocks, s)
                                : launch_long<__nv_bfloat16, 1>(p, blocks, s))
                         : (v16 ? launch_long<float, 4>(p, blocks, s)
                                : launch_long<float, 1>(p, blocks, s));
  } else {
    e = dtype == MX_BF16 ? (v16 ? launch_bwd<__nv_bfloat16, 8>(p, blocks, s)
                                : launch_bwd<__nv_bfloat16, 1>(p, blocks, s))
                         : (v16 ? launch_bwd<float, 4>(p, blocks, s)
                                : launch_bwd<float, 1>(p, blocks, s));
    note_launches(1);
  }
  if (e == cudaSuccess && sums) {
    note_launches(1);
    e = launch_after(norm_finish_kernel, static_cast<unsigned>((2ll * cols + 31) / 32),
                     32 * kFinishWarps, 0, s, true, static_cast<const float*>(scratch), blocks, cols,
                     dw, db);
  }
  return cuda_status(e);
}

}  // namespace mx
