// gated.cu -- the gated linear layer and its gradients.
//
//   [g | u] = x op(w) + bias,  h = act(g) * u
//   dpre = [dh * u * act'(g) | dh * act(g)],  dx = dpre op(w)^T,
//   dw = x^T dpre (w stored [K,2F]) or dpre^T x ([2F,K]),  dbias = sum_rows dpre
//
// The products are those of gemm_bf16.cu (the forward one with the activation
// in its epilogue), read in the layout in which x, w and dpre are stored; a
// float32 tensor goes in as three bfloat16 copies, and a bfloat16 one whose
// rows TMA cannot address (not a multiple of 16 bytes) as one padded copy.
// Small float32 products stay on the exact SIMT kernels.  dpre is one pass over
// dh and the saved [g | u] that also sums dbias; it is rounded to bfloat16 once
// (bfloat16 tensors: an operand of the tensor cores' bfloat16 products.  Half a
// step, 2^-8 of a value at most, as much as dx and dw themselves are rounded by,
// and independent of it: 2.3e-3 of their norm together, where a dpre in float32
// leaves 1.7e-3 and asks for a second product of its rest) or split in three.
#include <algorithm>
#include <cmath>

#include "gated_act.cuh"
#include "mx_internal.h"
#include "mx_ptx.cuh"
#include "mx_unaligned.cuh"

namespace mx {
namespace {

using bf16 = __nv_bfloat16;

// The bfloat16 copies (NC of them, see gemm_bf16.cu) of 8 values.
template <int NC>
__device__ __forceinline__ void store_copies(const float (&x)[8], bf16* dst, int64_t copy) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(r[2 * i], r[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
      if (c + 1 < NC) {  // exact: the difference has fewer bits than r
        r[2 * i] -= __uint_as_float(w[i] << 16);
        r[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
      }
    }
    *reinterpret_cast<uint4*>(dst + c * copy) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The copies of 8 values a lane of consecutive lanes (`lanes`, from 0 on), of
// which `left` exist, to a row that starts `shift` elements behind 16 bytes: a
// lane stores the aligned piece that ends in its own values, with the last ones
// of the lane before it.  Ends are stored one by one.
template <int NC>
__device__ __forceinline__ void store_shifted(float (&x)[8], bf16* dst, int64_t copy, int shift,
                                              int left, uint32_t lanes) {
  const int lane = threadIdx.x & 31;
  const bool next = lane < 31 && (lanes >> (lane + 1) & 1) != 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint32_t w[8];  // the lane before's, then its own
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[4 + i] = *reinterpret_cast<const uint32_t*>(&h);
      if (c + 1 < NC) {
        x[2 * i] -= __uint_as_float(w[4 + i] << 16);
        x[2 * i + 1] -= __uint_as_float(w[4 + i] & 0xffff0000u);
      }
      w[i] = __shfl_up_sync(lanes, w[4 + i], 1);
    }
    bf16* to = dst + c * copy;
    if (left == 8 && (lane > 0 || shift == 0)) {
      // elements 8 - shift .. 15 - shift of the sixteen
      uint32_t v[5];
      const int word = (8 - shift) >> 1;
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        v[i] = 0;
#pragma unroll
        for (int j = 0; j <= 4; ++j)
          if (word == j && i + j < 8) v[i] = w[i + j];
      }
      const uint32_t bits = (shift & 1) * 16;
      *reinterpret_cast<uint4*>(to - shift) =
          make_uint4(__funnelshift_r(v[0], v[1], bits), __funnelshift_r(v[1], v[2], bits),
                     __funnelshift_r(v[2], v[3], bits), __funnelshift_r(v[3], v[4], bits));
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {  // the lane before's last and its own first
        const bool mine = i < 8 ? lane > 0 && i >= 8 - shift : i - 8 < left && i - 8 < 8 - shift;
        if (mine) to[i - 8] = __ushort_as_bfloat16(static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1))));
      }
    }
    if (!next) {  // nobody else stores its last
#pragma unroll
      for (int i = 1; i < 8; ++i)
        if (i >= 8 - shift && i < left)
          to[i] = __ushort_as_bfloat16(static_cast<uint16_t>(w[4 + (i >> 1)] >> (16 * (i & 1))));
    }
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8(const bf16* p, float (&x)[8]) {
  const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <typename T>
__device__ __forceinline__ void load8_any(const T* p, const T* lo, const T* hi, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const uint4 a = load16_any(p, lo, hi), b = load16_any(p + 4, lo, hi);
    x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y);
    x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
    x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y);
    x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
  } else {
    const uint4 r = load16_any(p, lo, hi);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// What the products need before they start, in one launch: up to two matrices
// packed and, for the backward pass, dpre made with dbias's partial sums.
// Blocks are given to the jobs in turn.
//
// Packing: copies of a row-major [rows][cols] matrix with rows of ldd elements
// (a multiple of 8): columns below `split` at 0, the others from `up` on, zeros
// between.  A thread makes 8 columns of every by-th row.
struct PackJob {
  const void* src;
  bf16* dst;
  int64_t ldd, copy;
  int rows, cols, split, up;
  int vec;     // rows start on 16 bytes, and nothing is moved
  int bx, by;  // blocks across columns and rows
};
struct Dpre {
  const void* dh;
  const float* pre;
  void* out;      // OUT 1, 3: bfloat16 copies; 0: float32
  int64_t ldo, copy;
  float* part;    // [row blocks][2F], or null
  int rows, F, act, per;  // per: rows of a block
  int vec;        // dh's rows and the output's halves start on 16 bytes
  int bx, by;     // blocks across columns and rows (0: no dpre)
};
struct Prep {
  Dpre dpre;
  PackJob pack[2];
  int packs;
};

template <typename T, int NC>
__device__ __forceinline__ void pack_block(const PackJob& p, int block) {
  const int64_t d = (block % p.bx * 256ll + threadIdx.x) * 8;
  if (d >= p.ldd) return;
  const T* src = static_cast<const T*>(p.src);
  int64_t r = block / p.bx;
  if (p.vec) {
    for (; r + p.by < p.rows; r += 2 * p.by) {  // two rows in flight
      float x[8], y[8];
      load8(src + r * p.cols + d, x);
      load8(src + (r + p.by) * p.cols + d, y);
      store_copies<NC>(x, p.dst + r * p.ldd + d, p.copy);
      store_copies<NC>(y, p.dst + (r + p.by) * p.ldd + d, p.copy);
    }
    if (r < p.rows) {
      float x[8];
      load8(src + r * p.cols + d, x);
      store_copies<NC>(x, p.dst + r * p.ldd + d, p.copy);
    }
    return;
  }
  // the source's column of d, and how many of the eight are there
  const int64_t c = d < p.up ? d : p.split + (d - p.up);
  const int64_t end = d < p.up ? p.split : p.cols;
  const int n = static_cast<int>(end - c < 8 ? end - c : 8);
  const T* hi = src + static_cast<int64_t>(p.rows) * p.cols;
  for (; r < p.rows; r += p.by) {
    float x[8];
    load8_any(src + r * p.cols + c, src, hi, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? x[i] : 0.0f;
    store_copies<NC>(x, p.dst + r * p.ldd + d, p.copy);
  }
}

// dpre: 256 columns of both halves, `per` rows, the eight warps a row at a
// time, a lane 8 columns.  Bound by the bytes: with bfloat16 tensors 10 read
// and 4 written a value of h (8192 x 8192: 174 us, 0.83 of the copy rate;
// four blocks an SM instead of three 181).
template <typename T, int OUT>
__device__ __forceinline__ void dpre_block(const Dpre& p, int block, float (&sh)[8][8][33]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cb = block % p.bx, rb = block / p.bx;
  const int64_t f = (cb * 32ll + lane) * 8, up = (p.F + 7) & ~7ll;
  const int64_t r0 = rb * static_cast<int64_t>(p.per);
  const int64_t r1 = r0 + p.per < p.rows ? r0 + p.per : p.rows;
  float sg[8], su[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sg[i] = su[i] = 0.0f;
  const uint32_t lanes = __ballot_sync(0xffffffffu, f < p.F);
  if (f < p.F) {
    const int left = static_cast<int>(p.F - f < 8 ? p.F - f : 8);
    for (int64_t r = r0 + warp; r < r1; r += 8) {
      const T* dh = static_cast<const T*>(p.dh) + r * p.F + f;
      const float* pre = p.pre + r * 2 * up + f;
      float d[8], g[8], u[8];
      if (p.vec) {
        load8(dh, d);
      } else {
        load8_any(dh, static_cast<const T*>(p.dh),
                  static_cast<const T*>(p.dh) + static_cast<int64_t>(p.rows) * p.F, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = i < left ? d[i] : 0.0f;
      }
      load8(pre, g);  // pre's rows are padded
      load8(pre + up, u);
      gate_grad(p.act, d, g, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sg[i] += g[i];
        su[i] += u[i];
      }
      if constexpr (OUT == 0) {
        float* out = static_cast<float*>(p.out) + r * p.ldo + f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) {
            out[i] = g[i];
            out[p.F + i] = u[i];
          }
      } else {
        bf16* out = static_cast<bf16*>(p.out) + r * p.ldo + f;
        if (p.vec) {
          store_copies<OUT>(g, out, p.copy);
          store_copies<OUT>(u, out + p.F, p.copy);
        } else {
          store_shifted<OUT>(g, out, p.copy, 0, left, lanes);
          store_shifted<OUT>(u, out + p.F, p.copy, static_cast<int>(p.F & 7), left, lanes);
        }
      }
    }
  }
  if (!p.part) return;
  float* part = p.part + rb * 2ll * p.F;
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // the eight warps' sums, in their order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) sh[warp][i][lane] = h ? su[i] : sg[i];
    __syncthreads();
    const int64_t c = cb * 256ll + threadIdx.x;
    if (c < p.F) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += sh[w][threadIdx.x & 7][threadIdx.x >> 3];
      part[h * static_cast<int64_t>(p.F) + c] = s;
    }
  }
}

template <typename T, int NC, bool DPRE>
__global__ void __launch_bounds__(256) prep_kernel(const __grid_constant__ Prep p) {
  grid_trigger();
  int block = blockIdx.x;
  if constexpr (DPRE) {
    __shared__ float sh[8][8][33];
    if (block < p.dpre.bx * p.dpre.by) {
      dpre_block<T, NC>(p.dpre, block, sh);
      return;
    }
    block -= p.dpre.bx * p.dpre.by;
  }
  if constexpr (NC > 0) {
    const int first = p.packs > 0 ? p.pack[0].bx * p.pack[0].by : 0;
    if (block < first) pack_block<T, NC>(p.pack[0], block);
    else if (p.packs > 1) pack_block<T, NC>(p.pack[1], block - first);
  }
}

// dbias = the row blocks' sums, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) dbias_kernel(const float* part, T* out, int blocks,
                                                    int64_t width) {
  __shared__ float sh[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  float s = 0.0f;
  if (c < width)
    for (int r = warp; r < blocks; r += 8) s += part[r * width + c];
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < width) {
    s = 0.0f;
    for (int i = 0; i < 8; ++i) s += sh[i][lane];
    put(out + c, s);
  }
}

// h and pre from the SIMT product's [M][2F] (bias included); without one, K = 0,
// [g | u] is the bias.
template <typename T>
__global__ void __launch_bounds__(256) gate_kernel(const float* gu, const T* bias, float* pre, T* h,
                                                   int64_t n, int F, int act) {
  const int64_t up = (F + 7) & ~7ll;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t m = i / F, f = i - m * F;
    float g[1], u[1];
    if (gu) {
      g[0] = gu[m * 2 * F + f];
      u[0] = gu[m * 2 * F + F + f];
    } else {
      g[0] = bias ? to_f(bias[f]) : 0.0f;
      u[0] = bias ? to_f(bias[F + f]) : 0.0f;
    }
    if (pre) {
      pre[m * 2 * up + f] = g[0];
      pre[m * 2 * up + up + f] = u[0];
    }
    gate(act, g, u);
    put(h + i, g[0]);
  }
}

int64_t pad8(int64_t n) { return (n + 7) & ~7ll; }
size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }
bool aligned16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) == 0; }
unsigned grid_for(int64_t n, int num_sms) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((n + 255) / 256, num_sms * 8)));
}

// Pieces of the workspace, 256-byte aligned.  With a null base it measures.
struct Carver {
  uint8_t* base;
  size_t used = 0;
  template <typename P>
  P* take(size_t bytes) {
    P* p = base ? reinterpret_cast<P*>(base + used) : nullptr;
    used += align256(bytes);
    return p;
  }
};

// float32 products on the tensor cores: above 24 rows, where the matrices are
// not tiny.  Measured (forward + backward, us, SIMT / tensor cores): M = 33, K x
// F = 784 x 1000: 116 / 54, 32 x 32: 28 / 35; M = 128, 32 x 32: 41 / 38; M =
// 24, 4096 x 8192: 548 / 587; M = 512, 1024 x 4096: 554 / 187.
bool tensor_f32(const GatedArgs& a) {
  if (a.exact || a.tensor) return a.tensor && !a.exact;
  return a.M > 24 && (a.M >= 128 || static_cast<int64_t>(a.K) * a.F >= 16384);
}
int copies_of(const GatedArgs& a) { return a.dtype == MX_BF16 ? 1 : 3; }
bool tensor_path(const GatedArgs& a) { return a.dtype == MX_BF16 || tensor_f32(a); }

// A packed copy of a [rows][cols] matrix, or (bfloat16 that TMA can address)
// the matrix itself.  `halves`: columns from cols / 2 on start at a multiple
// of 8.
struct Packed {
  bool direct;
  int64_t ld, up, copy;
};
Packed packed_of(const GatedArgs& a, const void* src, int rows, int64_t cols, bool halves) {
  Packed p;
  const int64_t half = cols / 2;
  p.direct = a.dtype == MX_BF16 && cols % 8 == 0 && aligned16(src) && (!halves || half % 8 == 0);
  p.ld = halves ? 2 * pad8(half) : pad8(cols);
  p.up = halves ? pad8(half) : p.ld;
  p.copy = static_cast<int64_t>(rows) * p.ld;
  return p;
}
size_t packed_bytes(const GatedArgs& a, const Packed& p) {
  return p.direct ? 0 : static_cast<size_t>(copies_of(a)) * p.copy * 2;
}
// Adds a matrix to what a launch packs, unless it is read as it is; its operand.
Bf16Operand add_pack(Prep& prep, const void* src, int rows, int64_t cols, const Packed& p,
                     bool halves, bf16* dst) {
  Bf16Operand o;
  o.copy = p.copy;
  o.ld = p.ld;
  o.base = p.direct ? src : dst;
  if (p.direct) return o;
  const int split = static_cast<int>(halves ? cols / 2 : cols);
  const bool vec = cols == p.ld && (!halves || p.up == split) && aligned16(src);
  prep.pack[prep.packs++] = PackJob{src, dst, p.ld, p.copy, rows, static_cast<int>(cols), split,
                                    static_cast<int>(p.up), vec ? 1 : 0,
                                    static_cast<int>((p.ld / 8 + 255) / 256), std::min((rows + 1) / 2, 2048)};
  return o;
}
// OUT: as in Dpre; without dpre 1 or 3, the copies of a packed matrix.
template <typename T, int OUT, bool DPRE>
cudaError_t run_prep(const Prep& p, cudaStream_t s) {
  int blocks = DPRE ? p.dpre.bx * p.dpre.by : 0;
  for (int i = 0; i < p.packs; ++i) blocks += p.pack[i].bx * p.pack[i].by;
  if (blocks == 0) return cudaSuccess;
  prep_kernel<T, OUT, DPRE><<<blocks, 256, 0, s>>>(p);
  note_launches(1);
  return cudaGetLastError();
}

// An exact SIMT product on scratch of its own (no workspace or counters of the
// context, so calls on different streams may overlap).
GemmArgs simt_args(const GatedArgs& a, const void* x, const void* w, float* c, int M, int K, int N,
                   int ta, int tb, const void* bias) {
  GemmArgs g;
  g.a = static_cast<const float*>(x);
  g.b = static_cast<const float*>(w);
  g.c = c;
  g.M = M; g.K = K; g.N = N;
  g.ta = ta; g.tb = tb;
  g.lda = ta ? M : K;
  g.ldb = tb ? K : N;
  g.ldc = N;
  g.bias = static_cast<const float*>(bias);
  g.strict = a.strict ? 1 : 0;
  return g;
}
size_t simt_scratch(const Context* ctx, GemmArgs g) {
  size_t need = 0;
  for (uintptr_t off : {0, 4}) {  // aligned and not: the plans differ
    g.a = reinterpret_cast<const float*>(off);
    g.b = reinterpret_cast<const float*>(off);
    need = std::max(need, simt_gemm_scratch_bytes(ctx, g));
  }
  return need;
}
int simt_product(Context* ctx, const GemmArgs& g, void* scratch, size_t bytes, cudaStream_t s) {
  Context local = *ctx;
  local.counters = nullptr;  // arrival counters come from the scratch
  return skinny_applies(g) ? skinny_gemm(&local, g, s, scratch, bytes)
                           : simt_gemm_launch(&local, g, s, static_cast<float*>(scratch), bytes);
}

// The three products' workspaces, laid out alike for the size query and the
// call.
struct FwdWork {
  Packed x, w;
  bf16 *xp, *wp;
  void* split;      // scratch of a split product
  size_t split_bytes;
  float* pre;       // SIMT: [g | u]
  void* scratch;
  size_t scratch_bytes, bytes;
};
FwdWork fwd_work(const Context* ctx, const GatedArgs& a) {
  FwdWork w{};
  Carver c{static_cast<uint8_t*>(a.ws)};
  if (tensor_path(a)) {
    // a size query knows no pointers: room for copies of unaligned tensors
    const bool asked = !a.x;
    const void* off = reinterpret_cast<const void*>(uintptr_t{1});
    w.x = packed_of(a, asked ? off : a.x, a.M, a.K, false);
    w.w = a.tw ? packed_of(a, asked ? off : a.w, 2 * a.F, a.K, false)
               : packed_of(a, asked ? off : a.w, a.K, 2ll * a.F, true);
    w.xp = c.take<bf16>(packed_bytes(a, w.x));
    w.wp = c.take<bf16>(packed_bytes(a, w.w));
    Bf16Gemm g;
    g.gated = true;
    g.copies = copies_of(a);
    g.M = a.M; g.N = a.F; g.K = a.K;
    w.split_bytes = bf16_gemm_scratch_bytes(ctx, &g, 1);
    w.split = c.take<void>(w.split_bytes);
  } else {
    w.pre = c.take<float>(static_cast<size_t>(a.M) * 2 * a.F * sizeof(float));
    w.scratch_bytes = simt_scratch(
        ctx, simt_args(a, nullptr, nullptr, nullptr, a.M, a.K, 2 * a.F, 0, a.tw, nullptr));
    w.scratch = c.take<void>(w.scratch_bytes);
  }
  w.bytes = c.used;
  return w;
}

template <typename T>
int fwd(Context* ctx, const GatedArgs& a, cudaStream_t s) {
  const int64_t n = static_cast<int64_t>(a.M) * a.F;
  if (a.K == 0) {
    gate_kernel<T><<<grid_for(n, ctx->num_sms), 256, 0, s>>>(
        nullptr, static_cast<const T*>(a.bias), a.pre, static_cast<T*>(a.h), n, a.F, a.act);
    note_launches(1);
    return cuda_status(cudaGetLastError());
  }
  if (gated_skinny_applies(a)) return gated_skinny_fwd(ctx, a, s);
  const FwdWork w = fwd_work(ctx, a);
  if (w.bytes > a.ws_bytes) return kErrInvalid;
  if (!tensor_path(a)) {
    const GemmArgs g = simt_args(a, a.x, a.w, w.pre, a.M, a.K, 2 * a.F, 0, a.tw, a.bias);
    const int rc = simt_product(ctx, g, w.scratch, w.scratch_bytes, s);
    if (rc != kOk) return rc;
    gate_kernel<T><<<grid_for(n, ctx->num_sms), 256, 0, s>>>(w.pre, nullptr, a.pre,
                                                             static_cast<T*>(a.h), n, a.F, a.act);
    note_launches(1);
    return cuda_status(cudaGetLastError());
  }
  Bf16Gemm g;
  Prep prep{};
  g.a = add_pack(prep, a.x, a.M, a.K, w.x, false, w.xp);
  g.b = a.tw ? add_pack(prep, a.w, 2 * a.F, a.K, w.w, false, w.wp)
             : add_pack(prep, a.w, a.K, 2ll * a.F, w.w, true, w.wp);
  const cudaError_t e = run_prep<T, sizeof(T) == 2 ? 1 : 3, false>(prep, s);
  if (e != cudaSuccess) return cuda_status(e);
  g.a.kmajor = true;
  g.b.kmajor = a.tw != 0;
  g.b2 = g.b;
  g.b2.base = static_cast<const bf16*>(g.b.base) + (a.tw ? a.F * g.b.ld : w.w.direct ? a.F : w.w.up);
  g.gated = true;
  g.copies = copies_of(a);
  g.M = a.M; g.N = a.F; g.K = a.K;
  g.out = a.h;
  g.ldc = a.F;
  g.bias = a.bias;
  g.pre = a.pre;
  g.act = a.act;
  return bf16_gemm(ctx, &g, 1, w.split, nullptr, prep.packs > 0, s);
}

struct BwdWork {
  Packed x, w;
  bf16 *xp, *wp;
  void* dpre;
  int64_t ldp, copy;
  float* part;
  int row_blocks, per;
  void* split;      // scratch of split products
  size_t split_bytes;
  void* scratch;
  size_t scratch_bytes, bytes;
};
// The backward products' shapes: dx = dpre op(w)^T, then dw.
void bwd_shapes(const GatedArgs& a, Bf16Gemm (&g)[2]) {
  g[0].copies = g[1].copies = copies_of(a);
  g[0].M = a.M; g[0].N = a.K; g[0].K = 2 * a.F;
  g[1].M = a.tw ? 2 * a.F : a.K; g[1].N = a.tw ? a.K : 2 * a.F; g[1].K = a.M;
}
BwdWork bwd_work(const Context* ctx, const GatedArgs& a) {
  BwdWork w{};
  Carver c{static_cast<uint8_t*>(a.ws)};
  // rows of a block of dpre's: at least 16, and one round of three blocks an SM
  // (1000 x 2736: 12.1 us, in two or three rounds 13.5; 4096 x 2736: 37.0, 38.7 and
  // 40.9; 8192 x 8192: 174 and 171)
  const int col_blocks = (a.F + 255) / 256;
  const int want = std::max(1, 3 * ctx->num_sms / col_blocks);
  w.per = std::max(16, (a.M + want - 1) / want);
  w.row_blocks = (a.M + w.per - 1) / w.per;
  w.part = c.take<float>(static_cast<size_t>(w.row_blocks) * 2 * a.F * sizeof(float));
  if (tensor_path(a)) {
    const int nc = copies_of(a);
    w.ldp = pad8(2ll * a.F);
    w.copy = w.ldp * a.M;
    w.dpre = c.take<void>(static_cast<size_t>(nc) * w.copy * 2);
    const bool asked = !a.pre;
    const void* off = reinterpret_cast<const void*>(uintptr_t{1});
    w.x = packed_of(a, asked ? off : a.x, a.M, a.K, false);
    w.w = a.tw ? packed_of(a, asked ? off : a.w, 2 * a.F, a.K, false)
               : packed_of(a, asked ? off : a.w, a.K, 2ll * a.F, false);
    w.xp = c.take<bf16>(packed_bytes(a, w.x));
    w.wp = c.take<bf16>(packed_bytes(a, w.w));
    // the larger of what the call's products may need: both, or one of them
    Bf16Gemm g[2];
    bwd_shapes(a, g);
    w.split_bytes = std::max({bf16_gemm_scratch_bytes(ctx, g, 2), bf16_gemm_scratch_bytes(ctx, g, 1),
                              bf16_gemm_scratch_bytes(ctx, g + 1, 1)});
    w.split = c.take<void>(w.split_bytes);
  } else {
    w.ldp = 2ll * a.F;
    w.dpre = c.take<void>(static_cast<size_t>(a.M) * w.ldp * sizeof(float));
    const GemmArgs dx = simt_args(a, nullptr, nullptr, nullptr, a.M, 2 * a.F, a.K, 0, !a.tw, nullptr);
    const GemmArgs dw = a.tw ? simt_args(a, nullptr, nullptr, nullptr, 2 * a.F, a.M, a.K, 1, 0, nullptr)
                             : simt_args(a, nullptr, nullptr, nullptr, a.K, a.M, 2 * a.F, 1, 0, nullptr);
    w.scratch_bytes = std::max(simt_scratch(ctx, dx), simt_scratch(ctx, dw));
    w.scratch = c.take<void>(w.scratch_bytes);
  }
  w.bytes = c.used;
  return w;
}

template <typename T>
int bwd(Context* ctx, const GatedArgs& a, cudaStream_t s) {
  const BwdWork w = bwd_work(ctx, a);
  if (w.bytes > a.ws_bytes) return kErrInvalid;
  const bool tensor = tensor_path(a);
  const int F2 = 2 * a.F;
  Prep prep{};
  prep.dpre = Dpre{a.dh, a.pre, w.dpre, w.ldp, w.copy, a.dbias ? w.part : nullptr, a.M, a.F, a.act,
                   w.per, a.F % 8 == 0 && aligned16(a.dh) ? 1 : 0, (a.F + 255) / 256, w.row_blocks};
  Bf16Operand x, wt;
  cudaError_t e;
  if (!tensor) {
    e = run_prep<float, 0, true>(prep, s);
  } else {
    if (a.dx)
      wt = a.tw ? add_pack(prep, a.w, F2, a.K, w.w, false, w.wp)
                : add_pack(prep, a.w, a.K, F2, w.w, false, w.wp);
    if (a.dw) x = add_pack(prep, a.x, a.M, a.K, w.x, false, w.xp);
    e = run_prep<T, sizeof(T) == 2 ? 1 : 3, true>(prep, s);
  }
  const bool products = tensor && (a.dx || a.dw);
  if (e == cudaSuccess && a.dbias && !products) {  // else with what follows them
    dbias_kernel<T><<<(F2 + 31) / 32, 256, 0, s>>>(w.part, static_cast<T*>(a.dbias), w.row_blocks, F2);
    note_launches(1);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return cuda_status(e);
  if (!tensor) {
    int rc = kOk;
    if (a.dx)
      rc = simt_product(ctx, simt_args(a, w.dpre, a.w, static_cast<float*>(a.dx), a.M, F2, a.K, 0,
                                       !a.tw, nullptr), w.scratch, w.scratch_bytes, s);
    if (rc == kOk && a.dw)
      rc = simt_product(ctx, a.tw ? simt_args(a, w.dpre, a.x, static_cast<float*>(a.dw), F2, a.M,
                                              a.K, 1, 0, nullptr)
                                  : simt_args(a, a.x, w.dpre, static_cast<float*>(a.dw), a.K, a.M,
                                              F2, 1, 0, nullptr),
                        w.scratch, w.scratch_bytes, s);
    return rc;
  }
  Bf16Operand d;
  d.base = w.dpre;
  d.copy = w.copy;
  d.ld = w.ldp;
  Bf16Gemm g[2];
  bwd_shapes(a, g);
  g[0].a = d;
  g[0].b = wt;
  g[0].a.kmajor = true;
  g[0].b.kmajor = !a.tw;
  g[0].out = a.dx;
  g[0].ldc = a.K;
  g[1].a = a.tw ? d : x;
  g[1].b = a.tw ? x : d;
  g[1].a.kmajor = g[1].b.kmajor = false;
  g[1].out = a.dw;
  g[1].ldc = g[1].N;
  if (!products) return kOk;
  const Bf16ColumnSum sum{w.part, a.dbias, w.row_blocks, F2};
  return bf16_gemm(ctx, a.dx ? g : g + 1, a.dx && a.dw ? 2 : 1, w.split, a.dbias ? &sum : nullptr, true, s);
}

}  // namespace

size_t gated_workspace_bytes(const Context* ctx, const GatedArgs& a, bool backward) {
  GatedArgs q = a;
  q.ws = nullptr;
  q.x = q.w = nullptr;  // the size does not depend on the tensors' alignment
  q.pre = nullptr;
  if (!backward && (a.K == 0 || gated_skinny_applies(a))) return 0;
  return backward ? bwd_work(ctx, q).bytes : fwd_work(ctx, q).bytes;
}

int gated_fwd(Context* ctx, const GatedArgs& a, cudaStream_t s) {
  return a.dtype == MX_BF16 ? fwd<bf16>(ctx, a, s) : fwd<float>(ctx, a, s);
}

int gated_bwd(Context* ctx, const GatedArgs& a, cudaStream_t s) {
  return a.dtype == MX_BF16 ? bwd<bf16>(ctx, a, s) : bwd<float>(ctx, a, s);
}

}  // namespace mx
