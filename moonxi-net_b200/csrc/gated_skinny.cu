// gated_skinny.cu -- the gated linear layer for a few rows (single tokens).
//
// One to four rows read every weight once and do one to four multiply-adds with
// it: bound by the weights' bytes.  One row of 4096 x 2 x 8192 bfloat16 (134
// MB, a floor of 20.5 us): 23.3 us here with w [K,2F] and 24.8 us with w
// [2F,K], 43 us on the tensor-core kernel, whose pipeline has no second tile to
// hide its start and end behind; four rows 32 us with w [K,2F] against 42.
// float32: 44 us for one row, a floor of 41.  A warp reads 512 consecutive
// bytes of a row of w, products and sums stay in float32, and one launch does
// it all:
//   w stored [K,2F]: a lane owns 16 bytes of the gate's columns and the same of
//     the other projection's and walks down K; the eight warps of a block and
//     the blocks of a cluster split K, and the partial sums meet in
//     (distributed) shared memory, added in a fixed order.  Few columns leave
//     SMs without a block: there 8 lanes read a row, 4 rows a warp (4096 x 2 x
//     1024: 18.5 -> 12.3 us; 1024 x 2 x 4096 would go 12.3 -> 16.4);
//   w stored [2F,K]: a warp owns one or two pairs of rows and the lanes split K.
//     Each value of x is converted once a warp, which costs what three rows of
//     long K gain (4096 x 2 x 8192, M = 3: 55 us, tensor cores 43; K = 1024, F
//     = 4096: 14 and 18): those go to the tensor cores.
// Rows that do not start on 16 bytes are read as pairs of aligned pieces that a
// shift joins: 4095 x 2 x 8191 bfloat16, M = 1: 41 us with w [K,2F] and 55 with
// [2F,K], 92 where they are packed for the tensor cores first.
#include <algorithm>

#include "gated_act.cuh"
#include "mx_internal.h"
#include "mx_ptx.cuh"
#include "mx_unaligned.cuh"

namespace mx {
namespace {

using bf16 = __nv_bfloat16;
constexpr int kWarps = 8;

struct Skinny {
  const void* x;
  const void* w;
  const void* bias;
  void* h;
  float* pre;
  int M, K, F, act;
  int k_per;  // [K,2F]: rows of K of one block of a cluster
};

template <typename T>
__host__ __device__ constexpr int vec_of() { return 16 / static_cast<int>(sizeof(T)); }

template <typename T, int V>
__device__ __forceinline__ void unpack(const uint4 r, float (&x)[V]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// weights are read once: past L1, first out of L2
__device__ __forceinline__ uint4 stream16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

template <typename T>
__device__ __forceinline__ void finish(const Skinny& p, int m, int f, float g, float u) {
  if (p.bias) {
    g += to_f(static_cast<const T*>(p.bias)[f]);
    u += to_f(static_cast<const T*>(p.bias)[p.F + f]);
  }
  if (p.pre) {
    const int64_t up = (p.F + 7) & ~7ll;  // pre's halves are padded to 8
    p.pre[m * 2 * up + f] = g;
    p.pre[m * 2 * up + up + f] = u;
  }
  float ga[1] = {g}, ua[1] = {u};
  gate(p.act, ga, ua);
  put(static_cast<T*>(p.h) + static_cast<int64_t>(m) * p.F + f, ga[0]);
}

// w [K,2F].  A cluster owns 32 * V columns of each half; its blocks split K.
// x of row k in rows m .. of the block's chunk, [k][MT].
template <int MT>
__device__ __forceinline__ void load_x(const float* p, float (&x)[MT]) {
  if constexpr (MT == 1) {
    x[0] = *p;
  } else if constexpr (MT == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x; x[1] = v.y;
  } else {
#pragma unroll
    for (int m = 0; m < MT; m += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + m);
      x[m] = v.x; x[m + 1] = v.y; x[m + 2] = v.z; x[m + 3] = v.w;
    }
  }
}

// LW lanes read a row's columns and 32 / LW of the warp's lanes share them, each
// with rows of its own.
template <typename T, int MT, bool ANY, int LW>
__global__ void __launch_bounds__(32 * kWarps, 2) skinny_nn_kernel(const Skinny p, int cluster) {
  constexpr int V = vec_of<T>(), COLS = LW * V, R = 32 / LW, U = ANY ? (MT == 4 ? 2 : 4) : MT == 1 ? 8 : 4;
  constexpr int kChunk = 1024;  // rows of K whose x a block holds
  __shared__ __align__(16) float xs[kChunk][MT];
  __shared__ __align__(16) float red[kWarps][2][COLS];
  __shared__ __align__(16) float part[MT][2][COLS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % cluster;
  const int64_t f0 = static_cast<int64_t>(blockIdx.x / cluster) * COLS;
  const int col = lane % LW * V;
  const int64_t f = f0 + col;
  const bool in = f < p.F;  // what a last group has past column F is not stored
  const T* w = static_cast<const T*>(p.w) + f;
  const int64_t ld = 2ll * p.F;
  const T* lo = static_cast<const T*>(p.w);
  const T* hi = lo + p.K * ld;
  const int k_end = min(p.K, (rank + 1) * p.k_per);
  float g[MT][V], u[MT][V];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < V; ++i) g[m][i] = u[m][i] = 0.0f;
  for (int k0 = rank * p.k_per; k0 < k_end; k0 += kChunk) {
    const int n = min(kChunk, k_end - k0);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m)
      for (int k = threadIdx.x; k < n; k += 32 * kWarps)
        xs[k][m] = m < p.M ? to_f(static_cast<const T*>(p.x)[static_cast<int64_t>(m) * p.K + k0 + k])
                           : 0.0f;
    __syncthreads();
    if (!in) continue;
    for (int k = (warp * R + lane / LW) * U; k < n; k += kWarps * R * U) {
      uint4 a[U], b[U];
      const T* first = w + (k0 + k) * ld;
      if constexpr (!ANY) {
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (k + i < n) {
            a[i] = stream16(first + i * ld);
            b[i] = stream16(first + i * ld + p.F);
          }
      } else if (k + U <= n && pieces_inside(first, first + (U - 1) * ld + p.F, lo, hi)) {
        Piece pa[U], pb[U];  // all but the first and the last rows
#pragma unroll
        for (int i = 0; i < U; ++i) {
          pa[i] = load_piece(first + i * ld);
          pb[i] = load_piece(first + i * ld + p.F);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
          a[i] = shift_piece(pa[i], first + i * ld);
          b[i] = shift_piece(pb[i], first + i * ld + p.F);
        }
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (k + i < n) {
            a[i] = load16_any(first + i * ld, lo, hi);
            b[i] = load16_any(first + i * ld + p.F, lo, hi);
          }
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k + i < n) {
          float wa[V], wb[V];
          unpack<T>(a[i], wa);
          unpack<T>(b[i], wb);
          float xv[MT];
          load_x<MT>(xs[k + i], xv);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < V; ++j) {
              g[m][j] += xv[m] * wa[j];
              u[m][j] += xv[m] * wb[j];
            }
        }
    }
  }
  // the eight warps' sums, in their order, row by row
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m > 0) __syncthreads();
#pragma unroll
    for (int o = LW; o < 32; o *= 2)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        g[m][j] += __shfl_xor_sync(0xffffffffu, g[m][j], o);
        u[m][j] += __shfl_xor_sync(0xffffffffu, u[m][j], o);
      }
    if (lane < LW) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        red[warp][0][col + j] = g[m][j];
        red[warp][1][col + j] = u[m][j];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * COLS; c += 32 * kWarps) {
      float s = 0.0f;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) s += (&red[v][0][0])[c];
      (&part[m][0][0])[c] = s;
    }
  }
  // the cluster's blocks each finish a share of the columns
  if (cluster > 1) cluster_sync();
  else __syncthreads();
  const int share = COLS / cluster;
  for (int i = threadIdx.x; i < share * MT; i += 32 * kWarps) {
    const int m = i / share, c = rank * share + i % share;
    if (m >= p.M || f0 + c >= p.F) continue;
    float gs = 0.0f, us = 0.0f;
    if (cluster == 1) {
      gs = part[m][0][c];
      us = part[m][1][c];
    } else {
      for (int r = 0; r < cluster; ++r) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(&part[m][0][c], r)));
        gs += v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(&part[m][1][c], r)));
        us += v;
      }
    }
    finish<T>(p, m, static_cast<int>(f0 + c), gs, us);
  }
  if (cluster > 1) cluster_sync();  // no block leaves while its sums are read
}

// w [2F,K].  A warp makes FW columns of h for all rows, so that x is unpacked
// once for 2 FW products.
template <typename T, int MT, bool ANY, int FW>
__global__ void __launch_bounds__(32 * kWarps, 2) skinny_nt_kernel(const Skinny p) {
  constexpr int V = vec_of<T>(), U = (MT == 1 ? 8 : 4) / FW / (ANY ? 2 : 1);
  const int lane = threadIdx.x & 31;
  const int64_t f = (blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5)) * FW;
  if (f >= p.F) return;
  const T* wg[FW];
  const T* wu[FW];
#pragma unroll
  for (int c = 0; c < FW; ++c) {  // past the last column: the last one again
    const int64_t fc = f + c < p.F ? f + c : p.F - 1;
    wg[c] = static_cast<const T*>(p.w) + fc * p.K;
    wu[c] = static_cast<const T*>(p.w) + (fc + p.F) * p.K;
  }
  const T* x = static_cast<const T*>(p.x);
  const T* lo = static_cast<const T*>(p.w);
  const T* hi = lo + 2ll * p.F * p.K;
  const T* x_end = x + static_cast<int64_t>(p.M) * p.K;
  float g[FW][MT], u[FW][MT];
#pragma unroll
  for (int c = 0; c < FW; ++c)
#pragma unroll
    for (int m = 0; m < MT; ++m) g[c][m] = u[c][m] = 0.0f;
  for (int64_t k0 = lane * V; k0 < p.K; k0 += 32 * V * U) {
    uint4 a[U][FW], b[U][FW];
    if constexpr (!ANY) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k0 + i * 32 * V < p.K)
#pragma unroll
          for (int c = 0; c < FW; ++c) {
            a[i][c] = stream16(wg[c] + k0 + i * 32 * V);
            b[i][c] = stream16(wu[c] + k0 + i * 32 * V);
          }
    } else if (pieces_inside(wg[0] + k0, wu[FW - 1] + k0 + (U - 1) * 32 * V, lo, hi)) {
      Piece pa[U][FW], pb[U][FW];  // past a row's end: the next row's
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int c = 0; c < FW; ++c) {
          pa[i][c] = load_piece(wg[c] + k0 + i * 32 * V);
          pb[i][c] = load_piece(wu[c] + k0 + i * 32 * V);
        }
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int c = 0; c < FW; ++c) {
          a[i][c] = shift_piece(pa[i][c], wg[c]);
          b[i][c] = shift_piece(pb[i][c], wu[c]);
        }
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k0 + i * 32 * V < p.K)
#pragma unroll
          for (int c = 0; c < FW; ++c) {
            a[i][c] = load16_any(wg[c] + k0 + i * 32 * V, lo, hi);
            b[i][c] = load16_any(wu[c] + k0 + i * 32 * V, lo, hi);
          }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t k = k0 + i * 32 * V;
      if (k < p.K) {
        float wa[FW][V], wb[FW][V];
#pragma unroll
        for (int c = 0; c < FW; ++c) {
          unpack<T>(a[i][c], wa[c]);
          unpack<T>(b[i][c], wb[c]);
          if (ANY) {  // past the row's end is the next one
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (k + j >= p.K) wa[c][j] = wb[c][j] = 0.0f;
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (m < p.M) {
            float xv[V];
            const T* row = x + static_cast<int64_t>(m) * p.K + k;
            unpack<T>(ANY ? load16_any(row, x, x_end) : __ldg(reinterpret_cast<const uint4*>(row)), xv);
            if (ANY) {
#pragma unroll
              for (int j = 0; j < V; ++j)
                if (k + j >= p.K) xv[j] = 0.0f;
            }
#pragma unroll
            for (int c = 0; c < FW; ++c)
#pragma unroll
              for (int j = 0; j < V; ++j) {
                g[c][m] += xv[j] * wa[c][j];
                u[c][m] += xv[j] * wb[c][j];
              }
          }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int c = 0; c < FW; ++c)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        g[c][m] += __shfl_xor_sync(0xffffffffu, g[c][m], o);
        u[c][m] += __shfl_xor_sync(0xffffffffu, u[c][m], o);
      }
#pragma unroll
  for (int c = 0; c < FW; ++c)
#pragma unroll
    for (int m = 0; m < MT; ++m)  // a lane for each output
      if (lane == c * MT + m && m < p.M && f + c < p.F)
        finish<T>(p, m, static_cast<int>(f + c), g[c][m], u[c][m]);
}

template <typename T, int MT, bool ANY, int FW>
cudaError_t launch_nt(const Skinny& p, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>((p.F + kWarps * FW - 1) / (kWarps * FW));
  skinny_nt_kernel<T, MT, ANY, FW><<<blocks, 32 * kWarps, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int MT, bool ANY, int LW>
cudaError_t launch_nn(const Context* ctx, Skinny p, cudaStream_t s) {
  constexpr int COLS = LW * vec_of<T>();
  const int groups = (p.F + COLS - 1) / COLS;
  // blocks that share a group's K: about two blocks an SM, at least 64 of K each
  int cluster = 1;
  while (cluster < 8 && groups * cluster < 2 * ctx->num_sms && p.K >= 128 * cluster) cluster *= 2;
  p.k_per = (p.K + cluster - 1) / cluster;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(groups) * cluster);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, skinny_nn_kernel<T, MT, ANY, LW>, p, cluster);
}

template <typename T, int MT, bool ANY>
cudaError_t launch(const Context* ctx, const Skinny& p, bool tw, cudaStream_t s) {
  if (tw) {
    if constexpr (MT > 1) {
      // two columns a warp where that leaves a block an SM
      if (p.F >= 2 * kWarps * ctx->num_sms) return launch_nt<T, MT, ANY, 2>(p, s);
    }
    return launch_nt<T, MT, ANY, 1>(p, s);
  }
  // 512 bytes of a row a warp where clusters of eight then fill the machine
  if (p.F >= 32 * vec_of<T>() * (ctx->num_sms / 16)) return launch_nn<T, MT, ANY, 32>(ctx, p, s);
  return launch_nn<T, MT, ANY, 8>(ctx, p, s);
}

template <typename T, bool ANY>
cudaError_t launch_rows(const Context* ctx, const Skinny& p, bool tw, cudaStream_t s) {
  if (p.M == 1) return launch<T, 1, ANY>(ctx, p, tw, s);
  if (p.M == 2) return launch<T, 2, ANY>(ctx, p, tw, s);
  return launch<T, 4, ANY>(ctx, p, tw, s);
}

}  // namespace

bool gated_skinny_applies(const GatedArgs& a) {
  return !a.strict && a.M >= 1 && a.M <= 4 && a.K >= 1 &&
         !(a.tw && a.dtype == MX_BF16 && a.M > 2 && a.K >= 2048);
}

int gated_skinny_fwd(Context* ctx, const GatedArgs& a, cudaStream_t s) {
  const Skinny p{a.x, a.w, a.bias, a.h, a.pre, a.M, a.K, a.F, a.act, 0};
  // 16-byte pieces of w (and, for w [2F,K], of x) that start on 16 bytes
  const int v = a.dtype == MX_BF16 ? 8 : 4;
  const bool any = (a.tw ? a.K : a.F) % v != 0 || (reinterpret_cast<uintptr_t>(a.w) & 15u) != 0 ||
                   (a.tw && (reinterpret_cast<uintptr_t>(a.x) & 15u) != 0);
  const bool tw = a.tw != 0;
  const cudaError_t e =
      a.dtype == MX_BF16
          ? (any ? launch_rows<bf16, true>(ctx, p, tw, s) : launch_rows<bf16, false>(ctx, p, tw, s))
          : (any ? launch_rows<float, true>(ctx, p, tw, s) : launch_rows<float, false>(ctx, p, tw, s));
  note_launches(1);
  return cuda_status(e);
}

}  // namespace mx
