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
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
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

// Sums of N values over the TPR threads of a row, given to all of them.  The
// order is fixed.  TPR = 32: the row is a warp's.  Otherwise the block's, and
// `buf` holds N floats a warp.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();  // the last sum's readers are done
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) buf[i * W + warp] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = lane < W ? buf[i * W + lane] : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      s[i] = t;
    }
  }
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
// consecutive columns.  TPR = 32: four rows a block, one a warp.
template <typename T, int TPR, int E, int V>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) norm_fwd_kernel(const NormFwd p) {
  constexpr int NV = E / V;
  __shared__ float buf[TPR > 32 ? 2 * TPR / 32 : 1];
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = TPR == 32 ? blockIdx.x * 4ll + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  float v[NV][V];
  float s[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V;
    if (c < p.cols) {
      load_vec<T, V>(x + c, v[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += v[i][j];
    }
  }
  row_sum<TPR>(s, buf);
  const float n = static_cast<float>(p.cols);
  const float mean = s[0] / n;
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
  row_sum<TPR>(q, buf);
  const float rest = q[0] / n;
  const float var = q[1] / n - rest * rest;
  const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + p.eps);  // NaN stays NaN
  if (t == 0) {
    if (p.mean) p.mean[row] = mean + rest;
    if (p.rstd) p.rstd[row] = rstd;
  }
  T* y = static_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V;
    if (c < p.cols) {
      float w[V], b[V];
      load_par<V>(p.w, c, w, 1.0f);
      load_par<V>(p.b, c, b, 0.0f);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = (v[i][j] - rest) * rstd * w[j] + b[j];
      store_vec<T, V>(y + c, v[i]);
    }
  }
}

// Rows longer than the registers of a block hold: three passes over the row,
// the second and third from the caches.
template <typename T>
__global__ void __launch_bounds__(1024) norm_fwd_long_kernel(const NormFwd p) {
  __shared__ float buf[2 * 32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  float s[1] = {0.0f};
  for (int c = threadIdx.x; c < p.cols; c += 1024) s[0] += to_f(x[c]);
  row_sum<1024>(s, buf);
  const float mean = s[0] / static_cast<float>(p.cols);
  float q[2] = {0.0f, 0.0f};
  for (int c = threadIdx.x; c < p.cols; c += 1024) {
    const float d = to_f(x[c]) - mean;
    q[0] += d;
    q[1] += d * d;
  }
  row_sum<1024>(q, buf);
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

// A block takes rows blockIdx.x, + gridDim.x, ... (TPR = 32: four at a time,
// one a warp, whose sums meet in shared memory at the end).
template <typename T, int TPR, int E, int V>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) norm_bwd_kernel(const NormBwd p) {
  constexpr int NV = E / V;
  __shared__ float buf[TPR > 32 ? 2 * TPR / 32 : 4 * 32 * E];
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
  for (int64_t row = TPR == 32 ? blockIdx.x * 4ll + warp : blockIdx.x; row < p.rows; row += step) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    float xh[NV][V], a[NV][V];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < p.cols) {
        load_vec<T, V>(x + c, xh[i]);
        load_vec<T, V>(dy + c, a[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * TPR + t) * V < p.cols)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          xh[i][j] = (xh[i][j] - mean) * rstd;
          dw[i][j] += a[i][j] * xh[i][j];
          db[i][j] += a[i][j];
          a[i][j] *= w[i][j];
          s[0] += a[i][j];
          s[1] += a[i][j] * xh[i][j];
        }
    row_sum<TPR>(s, buf);
    const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
    if (p.dx) {
      T* dx = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * V;
        if (c < p.cols) {
#pragma unroll
          for (int j = 0; j < V; ++j) a[i][j] = rstd * (a[i][j] - c1 - xh[i][j] * c2);
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
  __shared__ float buf[2 * 32];
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
  row_sum<1024>(s, buf);
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

// out[c] = the sum over `blocks` partial rows; column c < cols goes to dw, the
// rest to db.  A block takes 32 columns, its eight warps an eighth of the rows
// each; the order is fixed.
__global__ void __launch_bounds__(256) norm_finish_kernel(const float* __restrict__ part,
                                                          int blocks, int cols, float* dw,
                                                          float* db) {
  __shared__ float sh[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t width = 2ll * cols, c = blockIdx.x * 32ll + lane;
  float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
  if (c < width) {
    int r = warp;
    for (; r + 24 < blocks; r += 32) {
      s0 += part[r * width + c];
      s1 += part[(r + 8) * width + c];
      s2 += part[(r + 16) * width + c];
      s3 += part[(r + 24) * width + c];
    }
    for (; r < blocks; r += 8) s0 += part[r * width + c];
  }
  sh[warp][lane] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  if (warp == 0 && c < width) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sh[i][lane];
    if (c < cols) {
      if (dw) dw[c] = s;
    } else if (db) {
      db[c - cols] = s;
    }
  }
}

// Columns up to which a row is held in registers.
constexpr int kNormRegCols = 16384;

template <typename T, int V>
cudaError_t launch_fwd(const NormFwd& p, cudaStream_t s) {
  const int c = p.cols;
  if (c <= 256) norm_fwd_kernel<T, 32, 8, V><<<(p.rows + 3) / 4, 128, 0, s>>>(p);
  else if (c <= 1024) norm_fwd_kernel<T, 32, 32, V><<<(p.rows + 3) / 4, 128, 0, s>>>(p);
  else if (c <= 2048) norm_fwd_kernel<T, 128, 16, V><<<p.rows, 128, 0, s>>>(p);
  else if (c <= 4096) norm_fwd_kernel<T, 256, 16, V><<<p.rows, 256, 0, s>>>(p);
  else if (c <= 8192) norm_fwd_kernel<T, 512, 16, V><<<p.rows, 512, 0, s>>>(p);
  else norm_fwd_kernel<T, 1024, 16, V><<<p.rows, 1024, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int V>
cudaError_t launch_bwd(const NormBwd& p, int blocks, cudaStream_t s) {
  const int c = p.cols;
  if (c <= 256) norm_bwd_kernel<T, 32, 8, V><<<blocks, 128, 0, s>>>(p);
  else if (c <= 1024) norm_bwd_kernel<T, 32, 32, V><<<blocks, 128, 0, s>>>(p);
  else if (c <= 2048) norm_bwd_kernel<T, 128, 16, V><<<blocks, 128, 0, s>>>(p);
  else if (c <= 4096) norm_bwd_kernel<T, 256, 16, V><<<blocks, 256, 0, s>>>(p);
  else if (c <= 8192) norm_bwd_kernel<T, 512, 16, V><<<blocks, 512, 0, s>>>(p);
  else norm_bwd_kernel<T, 1024, 16, V><<<blocks, 1024, 0, s>>>(p);
  return cudaGetLastError();
}

// Blocks of the backward pass (rows of partial sums).
int bwd_blocks(int rows, int cols, int num_sms) {
  if (cols > kNormRegCols) return std::min(64, (rows + 63) / 64);  // row ranges of norm_cols
  const int threads = cols <= 2048 ? 128 : cols <= 4096 ? 256 : cols <= 8192 ? 512 : 1024;
  const int per_block = cols <= 1024 ? 4 : 1;  // rows at a time
  const int fit = std::max(1, 512 / threads) * num_sms;
  return std::max(1, std::min(fit, (rows + 2 * per_block - 1) / (2 * per_block)));
}

bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) == 0; }

}  // namespace

size_t layer_norm_bwd_scratch_bytes(const Context* ctx, int rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return static_cast<size_t>(bwd_blocks(rows, cols, ctx->num_sms)) * 2 * cols * sizeof(float);
}

int layer_norm_fwd(Context* ctx, int dtype, const void* x, int64_t ldx, const float* w,
                   const float* b, void* y, int64_t ldy, float* mean, float* rstd, int rows,
                   int cols, float eps, cudaStream_t s) {
  (void)ctx;
  if (rows <= 0) return kOk;
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
    e = v16 ? launch_fwd<__nv_bfloat16, 8>(p, s) : launch_fwd<__nv_bfloat16, 1>(p, s);
  } else {
    e = v16 ? launch_fwd<float, 4>(p, s) : launch_fwd<float, 1>(p, s);
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
  if (sums && (!scratch || scratch_bytes < layer_norm_bwd_scratch_bytes(ctx, rows, cols)))
    return kErrInvalid;
  const int blocks = bwd_blocks(rows, cols, ctx->num_sms);
  const NormBwd p{dy, x, w, mean, rstd, dx, sums ? static_cast<float*>(scratch) : nullptr,
                  lddy, ldx, lddx, rows, cols};
  const int vec = dtype == MX_BF16 ? 8 : 4;
  const bool v16 = cols % vec == 0 && ldx % vec == 0 && lddy % vec == 0 && aligned16(x) &&
                   aligned16(dy) && aligned16(w) && (!dx || (lddx % vec == 0 && aligned16(dx)));
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
    norm_finish_kernel<<<static_cast<unsigned>((2ll * cols + 31) / 32), 256, 0, s>>>(static_cast<const float*>(scratch),
                                                           blocks, cols, dw, db);
    note_launches(1);
    e = cudaGetLastError();
  }
  return cuda_status(e);
}

}  // namespace mx
