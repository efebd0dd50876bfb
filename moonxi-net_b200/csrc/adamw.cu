// adamw.cu -- one AdamW step over many tensors in one launch, its two moments
// held in float32 or in 8 bits, as square-root codes or as floating-point values.
//
//   g' = clip * g                         clip = max_norm / ||g|| when above it
//   m  = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2
//   p  = (1 - lr wd) p - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit states: 256 consecutive values of a tensor share one float32, the
// largest magnitude among them (top, at least 2^-120).  The first moment is
// held as signed codes c for (c / 127)^2 top with c's sign, the second as
// unsigned codes c for sqrt(v) = (c / 255)^2 top; the code is the nearest one
// in the root, except that the first moment's codes below 0.5 / (1 -
// sqrt(b1)) + 1 are rounded towards zero: a step without gradient shrinks
// such a code by less than half, and the nearest one would keep a value whose
// gradients have stopped moving for ever (codes up to 9, 0.5 % of the block's
// largest, for b1 = 0.9).  The square gives values near the largest fine steps (0.8 % of
// sqrt(v)) and still reaches 1.5e-5 of it; holding sqrt(v) halves the range of
// exponents that v spans.  A sqrt(v) above zero keeps a code above zero (a
// vanished v would blow the step up), and since `top` itself is not rounded,
// moments that decay together decay exactly.  The step itself
// uses this step's float32 moments, before they are rounded.  A moment that is
// not finite makes its block's scale, and so the whole block, NaN.
//
// Nearest codes lose a change of one value against its block's largest by less
// than half a step.  Without gradient no v code below 0.5 / (1 - b2^(1/4)) falls (39
// of 255 for b2 = 0.95, 66 for 0.97, all of them for 0.999), and a first moment
// under a constant gradient settles at 0.23, 0.33 and 0.38 of its true value where
// that is 0.4, 0.9 and 1.6 % of the block's largest, at 0.65 to 0.74 where it is 2
// to 5 % (b1 = 0.9; rounded to nearest 0.45, 0.50, 0.60).  So there is a
// second rounding, DITHER: up or down by a number made from the step and the
// value's place, with the chance that makes the stored moment (m, and v itself)
// right on the average.  It follows at any decay rates, at the price of noise: a
// v of code c is off by a deviation of sqrt(2 / c) or so for b2 = 0.999.  Small m
// then need no rounding towards zero: they die out by chance.
//
// 8-bit floating-point states (e4m3, three bits of mantissa): m and sqrt(v) as
// such values times a power of two, the same for 256 of them, which takes the
// largest magnitude (at least 2^-119) into [128, 256).  The nearest value is kept;
// what is not zero stays above zero (2^-9 before the power of two).  Neighbours are
// up to 1/8 apart, so that a nearest v never falls where sqrt(b2) is above 31/32;
// DITHER is there for these states too (and keeps v alone above zero).  A factor
// that is infinite marks a block with a moment that is not finite.  The step is
// that of 32-bit states, bit for bit the one of elementwise float32 operations,
// since a value near the middle of two falls by its last bit.
//
// Bound by the bytes: 28 B a value with float32 gradients and states, 16 B
// with 8-bit states (14 B with bf16 gradients).  A warp takes 256 values,
// 8 a lane in 16-byte accesses, so an 8-bit block is one warp's and its
// maximum one warp reduction.  201 M values with bf16 gradients and copies, 16 B each,
// a floor of 492 us: codes 544, e4m3 587; rounded by DITHER, whose numbers and
// neighbours then bound the step, 684 and 792.
#include <algorithm>
#include <cmath>

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "../../include/mx_matmul.h"
#include "mx_internal.h"
#include "mx_ptx.cuh"

namespace mx {
namespace {

constexpr int kQBlock = 256;           // values of one scale, of one warp
constexpr int kWarps = 8;
constexpr int kPerWarp = 1;            // 256-value blocks of a warp
constexpr int kChunk = kPerWarp * kWarps * kQBlock;  // values of one block

enum : uint32_t { kGradBf16 = 1, kVec = 2 };

// How the moments are held.
enum Kind { kF32, kRoot, kE4m3 };

struct Tensor {
  float* p;
  const void* g;
  void* m;
  void* v;
  float* ms;            // 8-bit states: the blocks' scales
  float* vs;
  __nv_bfloat16* copy;  // bf16 copy of the new values, or null
  int64_t n;
  float keep;           // 1 - lr * weight_decay
  uint32_t flags;
};

// The tensors of one launch, by value: nothing to upload, and a captured
// launch holds its own table.  first[i]: the first chunk of tensor i.
template <int CAP>
struct Table {
  Tensor t[CAP];
  int64_t first[CAP + 1];
  int count;
};

struct Hyper {
  float b1, omb1, b2, omb2, eps, step_size, inv_root;  // see adamw_one
  float down;             // 8-bit first moments: codes below it are rounded down
  uint32_t step;          // of the dither
  const float* scalars;   // device: {step_size, inv_root, step} instead, or null
  const float* norm;      // device: the gradients' norm, or null (no clipping)
  float max_norm;
};

template <int CAP>
__device__ __forceinline__ int find_tensor(const Table<CAP>& tb, int64_t chunk) {
  int lo = 0, hi = tb.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tb.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// To 2 units in the last place, values below 2^-126 as zeros.
__device__ __forceinline__ float fast_sqrt(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The new m, v and p of one value; returns sqrt(v).  32-bit and e4m3 moments:
// every operation rounded by itself, as the elementwise form of the step computes
// it.  Root codes: fused, with the approximate root and quotient (2 units in
// the last place, far below what the codes round away): 544 us for 201 M values
// against 590 with exact ones, 492 of bytes.
template <Kind KIND>
__device__ __forceinline__ float adamw_one(float& p, float g, float& m, float& v, float keep,
                                           const Hyper& h) {
  if constexpr (KIND == kRoot) {
    m = fmaf(m, h.b1, g * h.omb1);
    v = fmaf(v, h.b2, g * g * h.omb2);
    const float root = fast_sqrt(v);
    p = fmaf(p, keep, -(m * h.step_size) * fast_rcp(fmaf(root, h.inv_root, h.eps)));
    return root;
  }
  m = __fadd_rn(__fmul_rn(m, h.b1), __fmul_rn(g, h.omb1));
  v = __fadd_rn(__fmul_rn(v, h.b2), __fmul_rn(__fmul_rn(g, g), h.omb2));
  const float root = __fsqrt_rn(v);
  const float denom = __fadd_rn(__fmul_rn(root, h.inv_root), h.eps);
  p = __fsub_rn(__fmul_rn(p, keep), __fdiv_rn(__fmul_rn(m, h.step_size), denom));
  return root;
}

// 32 bits for the dither from a step and a place: multiplications by 2^32 over the
// golden ratio, and shifts that bring the upper bits down.  (Means, variances and
// the correlations between places, steps and both halves are those of random
// numbers to within 3 deviations of 2^20 places and 40 steps.)
__device__ __forceinline__ uint32_t scatter(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x9e3779b1u;
  x = (x ^ (x >> 15)) * 0x9e3779b1u;
  return x ^ (x >> 16);
}
// Whether 16 of them are below the chance part / whole.
__device__ __forceinline__ bool below(uint32_t bits, float part, float whole) {
  return (static_cast<float>(bits & 0xffffu) + 0.5f) * whole < part * 65536.0f;
}

// 8 values of a lane, those past `left` not touched.
__device__ __forceinline__ void load8(const float* p, bool vec, int left, float (&x)[8]) {
  if (vec && left >= 8) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < left ? p[i] : 0.0f;
  }
}
__device__ __forceinline__ void store8(float* p, bool vec, int left, const float (&x)[8]) {
  if (vec && left >= 8) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = x[i];
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool vec, int left, float (&x)[8]) {
  if (vec && left >= 8) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < left ? __bfloat162float(p[i]) : 0.0f;
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, bool vec, int left, const float (&x)[8]) {
  if (vec && left >= 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = __float2bfloat16_rn(x[i]);
  }
}

// What 8 codes of a block with the largest magnitude `top` stand for: the
// first moment, or (SIGNED false) the root of the second.  A byte is made a
// float32 by putting it under the exponent of 2^23.
template <bool SIGNED>
__device__ __forceinline__ void decode_words(const uint32_t (&w)[2], float top, float (&x)[8]) {
  const float unit = top * (SIGNED ? 1.0f / 16129.0f : 1.0f / 65025.0f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t word = SIGNED ? w[i >> 2] ^ 0x80808080u : w[i >> 2];
    const float c = __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440 + (i & 3))) -
                    (SIGNED ? 8388736.0f : 8388608.0f);
    x[i] = c * fabsf(c) * unit;
  }
}
// 8 bytes of a lane, those past `left` not touched (read as zeros).
__device__ __forceinline__ void load_bytes8(const uint8_t* q, bool vec, int left, uint32_t (&w)[2]) {
  w[0] = w[1] = 0;
  if (vec && left >= 8) {
    const uint2 r = *reinterpret_cast<const uint2*>(q);
    w[0] = r.x;
    w[1] = r.y;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) w[i >> 2] |= static_cast<uint32_t>(q[i]) << (8 * (i & 3));
  }
}
__device__ __forceinline__ void store_bytes8(uint8_t* q, bool vec, int left, const uint32_t (&w)[2]) {
  if (vec && left >= 8) {
    *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) q[i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
  }
}
template <bool SIGNED>
__device__ __forceinline__ void decode8(const uint8_t* q, float top, bool vec, int left,
                                        float (&x)[8]) {
  uint32_t w[2];
  load_bytes8(q, vec, left, w);
  decode_words<SIGNED>(w, top, x);
}
// The warp's largest magnitude, at least 2^-120; NaN if a value is not finite.
// As integers, magnitudes keep their order, with infinity and NaN above all.
template <bool SIGNED>
__device__ __forceinline__ float block_top(const float (&x)[8]) {
  uint32_t top = 0x03800000u;  // 2^-120
#pragma unroll
  for (int i = 0; i < 8; ++i)
    top = max(top, SIGNED ? __float_as_uint(x[i]) & 0x7fffffffu : __float_as_uint(x[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  return __uint_as_float(top >= 0x7f800000u ? 0x7fc00000u : top);
}
// The codes: c = round(sqrt(|x| / top) most), rounded by adding 1.5 * 2^23,
// which leaves it in the low byte; signed ones below `down` are floor(c + 1/64),
// so that a value that stays as it is keeps its code.  The root's last bit does
// not matter here.  (most^2 / top would pass float32 from a top of 2^-112 down,
// and infinity times a zero is no zero; 1 / top is at most 2^120.)
// DITHER: the two codes k and k + 1 around c stand for k^2 and (k + 1)^2 (m), or k^4
// and (k + 1)^4 (v).
template <bool SIGNED, bool DITHER>
__device__ __forceinline__ void encode8(uint8_t* q, float top, float down, bool vec, int left,
                                        const float (&x)[8], const uint32_t (&bits)[8]) {
  constexpr float kMost = SIGNED ? 127.0f : 255.0f;
  const float inv = __fdiv_rn(1.0f, top);
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float c = fast_sqrt(fabsf(x[i]) * inv) * kMost;
    if constexpr (DITHER) {
      const float k = fminf(floorf(c), kMost - 1.0f);  // the largest is the last code
      const float a = SIGNED ? c * c : c * c * c * c, lo = SIGNED ? k * k : k * k * k * k;
      const float k1 = k + 1.0f, hi = SIGNED ? k1 * k1 : k1 * k1 * k1 * k1;
      c = below(bits[i] >> (SIGNED ? 0 : 16), a - lo, hi - lo) ? k1 : k;
      if (SIGNED) c = copysignf(c, x[i]);
      else if (x[i] > 0.0f) c = fmaxf(c, 1.0f);
    } else if (SIGNED) c = copysignf(c < down ? fmaxf(c - 0.484375f, 0.0f) : c, x[i]);
    else if (x[i] > 0.0f) c = fmaxf(c, 1.0f);
    b[i] = __float_as_uint(c + 12582912.0f);
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040),
                       __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
  store_bytes8(q, vec, left, w);
}

// The power of two that takes the warp's largest magnitude, at least 2^-119, into
// [128, 256); infinity if a value is not finite.
__device__ __forceinline__ float block_power(const float (&x)[8]) {
  uint32_t top = 0x04000000u;  // 2^-119
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top) & 0x7f800000u;
  return __uint_as_float(top == 0x7f800000u ? top : top - (7u << 23));
}
// What 8 e4m3 values times `power` stand for (exact).
__device__ __forceinline__ void decode8_e4m3(const uint8_t* q, float power, bool vec, int left,
                                             float (&x)[8]) {
  uint32_t w[2];
  load_bytes8(q, vec, left, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h(__nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3));
    const float2 f = __half22float2(h);
    x[2 * i] = f.x * power;
    x[2 * i + 1] = f.y * power;
  }
}
// DITHER: the two values around y, q apart, are chosen between for m itself, or
// (SIGNED false) for the square that sqrt(v) stands for.
template <bool SIGNED, bool DITHER>
__device__ __forceinline__ void encode8_e4m3(uint8_t* q, float power, bool vec, int left,
                                             const float (&x)[8], const uint32_t (&bits)[8]) {
  const float inv = __fdiv_rn(1.0f, power);  // exact; 0 where power is infinite
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = x[i] * inv;
    if constexpr (DITHER) {
      const float a = fabsf(y[i]);
      if (a < 256.0f) {  // else it is not finite
        const uint32_t w = __float_as_uint(a);
        const bool normal = a >= 0.015625f;  // 2^-6
        const float step = normal ? __uint_as_float((w & 0x7f800000u) - (3u << 23)) : 0.001953125f;
        const float lo = normal ? __uint_as_float(w & 0xfff00000u) : floorf(a * 512.0f) * 0.001953125f;
        const float rest = a - lo;
        const bool up = SIGNED ? below(bits[i], rest, step)
                               : below(bits[i] >> 16, rest * (a + lo), step * (2.0f * lo + step));
        float r = up ? lo + step : lo;
        if (!SIGNED && a > 0.0f) r = fmaxf(r, 0.001953125f);
        y[i] = copysignf(r, y[i]);
      }
    } else if (y[i] != 0.0f && fabsf(y[i]) < 0.001953125f) y[i] = copysignf(0.001953125f, y[i]);
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i >> 1] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(
                     make_float2(y[2 * i], y[2 * i + 1]), __NV_SATFINITE, __NV_E4M3))
                 << (16 * (i & 1));
  store_bytes8(q, vec, left, w);
}

// The step of 256 values, a warp's; VEC: all of them are there, 16-byte
// aligned (8-bit states 8-byte).
template <Kind KIND, bool DITHER, bool VEC>
__device__ __forceinline__ void adamw_block(const Tensor& t, const Hyper& h, float clip,
                                            int64_t block) {
  const int lane = threadIdx.x & 31;
  const int64_t at = block * kQBlock + lane * 8;
  const int64_t rest = t.n - at;
  const int left = VEC ? 8 : rest >= 8 ? 8 : rest > 0 ? static_cast<int>(rest) : 0;
  float p[8], g[8], m[8], v[8];
  load8(t.p + at, VEC, left, p);
  if (t.flags & kGradBf16) load8(static_cast<const __nv_bfloat16*>(t.g) + at, VEC, left, g);
  else load8(static_cast<const float*>(t.g) + at, VEC, left, g);
  if constexpr (KIND != kF32) {
    const uint8_t* mq = static_cast<const uint8_t*>(t.m) + at;
    const uint8_t* vq = static_cast<const uint8_t*>(t.v) + at;
    if constexpr (KIND == kRoot) {
      decode8<true>(mq, t.ms[block], VEC, left, m);
      decode8<false>(vq, t.vs[block], VEC, left, v);
    } else {
      decode8_e4m3(mq, t.ms[block], VEC, left, m);
      decode8_e4m3(vq, t.vs[block], VEC, left, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], v[i]);
  } else {
    load8(static_cast<const float*>(t.m) + at, VEC, left, m);
    load8(static_cast<const float*>(t.v) + at, VEC, left, v);
  }
  if (h.norm) {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = __fmul_rn(g[i], clip);
  }
  float root[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) root[i] = adamw_one<KIND>(p[i], g[i], m[i], v[i], t.keep, h);
  store8(t.p + at, VEC, left, p);
  if (t.copy) store8(t.copy + at, VEC, left, p);
  if constexpr (KIND != kF32) {
    uint8_t* mq = static_cast<uint8_t*>(t.m) + at;
    uint8_t* vq = static_cast<uint8_t*>(t.v) + at;
    float sm, sv;
    uint32_t bits[8] = {};
    if constexpr (DITHER) {
      const uint32_t key = scatter(h.step * 0x9e3779b9u + 1u);
      const uint32_t place = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * kQBlock + lane * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) bits[i] = scatter((place + i) ^ key);
    }
    if constexpr (KIND == kRoot) {
      sm = block_top<true>(m);
      sv = block_top<false>(root);
      encode8<true, DITHER>(mq, sm, h.down, VEC, left, m, bits);
      encode8<false, DITHER>(vq, sv, 0.0f, VEC, left, root, bits);
    } else {
      sm = block_power(m);
      sv = block_power(root);
      encode8_e4m3<true, DITHER>(mq, sm, VEC, left, m, bits);
      encode8_e4m3<false, DITHER>(vq, sv, VEC, left, root, bits);
    }
    __syncwarp();  // every lane has read the old scales
    if (lane == 0) {
      t.ms[block] = sm;
      t.vs[block] = sv;
    }
  } else {
    store8(static_cast<float*>(t.m) + at, VEC, left, m);
    store8(static_cast<float*>(t.v) + at, VEC, left, v);
  }
}

template <int CAP, Kind KIND, bool DITHER>
__global__ void __launch_bounds__(32 * kWarps) adamw_kernel(const __grid_constant__ Table<CAP> tb,
                                                            const Hyper hy) {
  const int ti = find_tensor(tb, blockIdx.x);
  const Tensor t = tb.t[ti];
  Hyper h = hy;
  if (h.scalars) {
    h.step_size = h.scalars[0];
    h.inv_root = h.scalars[1];
    h.step = __float_as_uint(h.scalars[2]);
  }
  float clip = 1.0f;
  if (h.norm) {
    const float nv = *h.norm;
    if (nv > h.max_norm) clip = __fdiv_rn(h.max_norm, nv);
  }
  const int64_t first = (blockIdx.x - tb.first[ti]) * (kChunk / kQBlock) + (threadIdx.x >> 5);
#pragma unroll
  for (int k = 0; k < kPerWarp; ++k) {
    const int64_t block = first + k * kWarps;
    if (block * kQBlock >= t.n) return;  // the whole warp
    if ((t.flags & kVec) && (block + 1) * kQBlock <= t.n) adamw_block<KIND, DITHER, true>(t, h, clip, block);
    else adamw_block<KIND, DITHER, false>(t, h, clip, block);
  }
}

// The values that 8-bit codes stand for, rounded to bf16: the first moment, or
// (SIGNED false) the second.  A warp makes kValues blocks, whose loads are all on
// their way before the first is used: 3 bytes a value (201M values: 91 us, the copy
// rate; one block a warp: 115).
constexpr int kValues = 4;
template <bool SIGNED>
__device__ __forceinline__ void store_values(__nv_bfloat16* out, bool vec, int left, float (&x)[8]) {
  if (!SIGNED)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(x[i], x[i]);
  store8(out, vec, left, x);
}
template <bool SIGNED>
__global__ void __launch_bounds__(32 * kWarps) adamw_values_kernel(const uint8_t* q,
                                                                   const float* scale, int64_t n,
                                                                   __nv_bfloat16* out, bool vec) {
  const int lane = threadIdx.x & 31;
  const int64_t first = (blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5)) * kValues;
  if (vec && (first + kValues) * kQBlock <= n) {
    uint32_t w[kValues][2];
    float top[kValues];
#pragma unroll
    for (int k = 0; k < kValues; ++k) {
      const uint2 r = __ldg(reinterpret_cast<const uint2*>(q + (first + k) * kQBlock) + lane);
      w[k][0] = r.x;
      w[k][1] = r.y;
      top[k] = __ldg(scale + first + k);
    }
#pragma unroll
    for (int k = 0; k < kValues; ++k) {
      float x[8];
      decode_words<SIGNED>(w[k], top[k], x);
      store_values<SIGNED>(out + (first + k) * kQBlock + lane * 8, true, 8, x);
    }
    return;
  }
  for (int k = 0; k < kValues; ++k) {
    const int64_t at = (first + k) * kQBlock + lane * 8;
    if (at >= n) return;
    const int left = n - at >= 8 ? 8 : static_cast<int>(n - at);
    float x[8];
    decode8<SIGNED>(q + at, scale[first + k], vec, left, x);
    store_values<SIGNED>(out + at, vec, left, x);
  }
}

// Sum of squares of the gradients of one launch's tensors: block b's sum of
// its chunks goes to part[b]; the order is fixed.
template <int CAP>
__global__ void __launch_bounds__(32 * kWarps) grad_norm_kernel(const __grid_constant__ Table<CAP> tb,
                                                                float* part) {
  __shared__ float sh[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float s = 0.0f;
  for (int64_t c = blockIdx.x; c < tb.first[tb.count]; c += gridDim.x) {
    const int ti = find_tensor(tb, c);
    const Tensor& t = tb.t[ti];
#pragma unroll
    for (int k = 0; k < kPerWarp; ++k) {
      const int64_t at = (c - tb.first[ti]) * kChunk + (k * 32 * kWarps + threadIdx.x) * 8;
      const int64_t rest = t.n - at;
      const int left = rest >= 8 ? 8 : rest > 0 ? static_cast<int>(rest) : 0;
      float g[8];
      if (t.flags & kGradBf16)
        load8(static_cast<const __nv_bfloat16*>(t.g) + at, t.flags & kVec, left, g);
      else
        load8(static_cast<const float*>(t.g) + at, t.flags & kVec, left, g);
      float q = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) q += g[i] * g[i];
      s += q;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sh[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kWarps; ++i) s += sh[i];
    part[blockIdx.x] = s;
  }
}

// One block: the norm of `n` partial sums of squares, and the step's scalars
// from a step number on the device.  Either may be off.
__global__ void __launch_bounds__(256) adamw_prelude_kernel(const float* part, int n, float* norm,
                                                            float* norm_out, int32_t* step,
                                                            float* scalars, double lr, double b1,
                                                            double b2) {
  __shared__ float sh[256];
  if (norm) {
    float s = 0.0f;
    for (int i = threadIdx.x; i < n; i += 256) s += part[i];
    sh[threadIdx.x] = s;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
      if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      *norm = sqrtf(sh[0]);
      if (norm_out) *norm_out = *norm;
    }
  }
  if (scalars && threadIdx.x == 32) {
    const int32_t t = *step + 1;
    *step = t;
    scalars[0] = static_cast<float>(lr / (1.0 - pow(b1, static_cast<double>(t))));
    scalars[1] = static_cast<float>(1.0 / sqrt(1.0 - pow(b2, static_cast<double>(t))));
    scalars[2] = __uint_as_float(static_cast<uint32_t>(t));
  }
}

constexpr int kNormBlocks = 592;  // partial sums of a launch: four blocks an SM

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

bool aligned(const void* a, unsigned to) { return (reinterpret_cast<uintptr_t>(a) & (to - 1)) == 0; }

template <int CAP>
void fill(Table<CAP>& tb, const mx_adamw_tensor* ts, int count, int bits, double lr) {
  tb.count = 0;
  int64_t at = 0;
  for (int i = 0; i < count; ++i) {
    const mx_adamw_tensor& a = ts[i];
    if (a.n == 0) continue;
    Tensor& t = tb.t[tb.count];
    t.p = a.param;
    t.g = a.grad;
    t.m = a.m;
    t.v = a.v;
    t.ms = a.m_scale;
    t.vs = a.v_scale;
    t.copy = static_cast<__nv_bfloat16*>(a.copy_bf16);
    t.n = a.n;
    t.keep = static_cast<float>(1.0 - lr * a.weight_decay);
    const unsigned sa = bits & 8 ? 8 : 16;
    t.flags = (a.grad_type == MX_BF16 ? kGradBf16 : 0u) |
              (aligned(a.param, 16) && aligned(a.grad, 16) && aligned(a.m, sa) &&
                       aligned(a.v, sa) && aligned(a.copy_bf16, 16)
                   ? kVec : 0u);
    tb.first[tb.count++] = at;
    at += chunks_of(a.n);
  }
  tb.first[tb.count] = at;
}

template <int CAP>
cudaError_t launch_norm(const mx_adamw_tensor* ts, int count, int bits, float* part, int* blocks,
                        cudaStream_t s) {
  Table<CAP> tb;
  fill(tb, ts, count, bits, 0.0);
  *blocks = static_cast<int>(std::min<int64_t>(tb.first[tb.count], kNormBlocks));
  if (*blocks == 0) return cudaSuccess;
  grad_norm_kernel<CAP><<<*blocks, 32 * kWarps, 0, s>>>(tb, part);
  note_launches(1);
  return cudaGetLastError();
}

template <int CAP>
cudaError_t launch_step(const mx_adamw_tensor* ts, int count, int bits, double lr, const Hyper& h,
                        cudaStream_t s) {
  Table<CAP> tb;
  fill(tb, ts, count, bits, lr);
  const int64_t chunks = tb.first[tb.count];
  if (chunks == 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>(chunks);
  auto kern = adamw_kernel<CAP, kF32, false>;
  const bool dither = (bits & MX_ADAMW_DITHER) != 0;
  if (bits & MX_ADAMW_E4M3)
    kern = dither ? adamw_kernel<CAP, kE4m3, true> : adamw_kernel<CAP, kE4m3, false>;
  else if (bits & 8)
    kern = dither ? adamw_kernel<CAP, kRoot, true> : adamw_kernel<CAP, kRoot, false>;
  kern<<<grid, 32 * kWarps, 0, s>>>(tb, h);
  note_launches(1);
  return cudaGetLastError();
}

// Tensors of one launch.  A kernel's parameters hold up to 32 KB; the small
// table keeps a call on a few tensors at a quarter of a page.
constexpr int kSmallTable = 16, kLargeTable = 320;
static_assert(sizeof(Table<kLargeTable>) + sizeof(Hyper) <= 32764, "kernel parameters");

}  // namespace

size_t adamw_scratch_bytes(int count, int clip) {
  const int64_t launches = (std::max(count, 1) + kLargeTable - 1) / kLargeTable;
  return (4 + (clip ? launches * kNormBlocks : 0)) * sizeof(float);
}

int adamw_check(const mx_adamw_tensor* ts, int count, int bits) {
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const mx_adamw_tensor& a = ts[i];
    if (i % kLargeTable == 0) chunks = 0;  // a launch's
    if (a.n < 0 || (a.grad_type != MX_F32 && a.grad_type != MX_BF16)) return kErrInvalid;
    if (a.n == 0) continue;
    if (!a.param || !a.grad || !a.m || !a.v) return kErrInvalid;
    if ((bits & 8) && (!a.m_scale || !a.v_scale)) return kErrInvalid;
    chunks += chunks_of(a.n);
    if (chunks > 0x7fffffff) return kErrUnsupported;  // blocks of one launch
  }
  return kOk;
}

int adamw_step(const mx_adamw_tensor* ts, int count, int bits, double lr, double b1, double b2,
               double eps, int64_t step, int32_t* step_dev, double max_norm, float* norm_out,
               void* scratch, cudaStream_t s) {
  float* sc = static_cast<float*>(scratch);  // [0] norm, [1..3] scalars, [4..] partial sums
  float* part = sc + 4;
  const bool clip = max_norm > 0.0;
  int parts = 0;
  cudaError_t e = cudaSuccess;
  if (clip)
    for (int i = 0; i < count && e == cudaSuccess; i += kLargeTable) {
      const int k = std::min(kLargeTable, count - i);
      int blocks = 0;
      e = k <= kSmallTable ? launch_norm<kSmallTable>(ts + i, k, bits, part + parts, &blocks, s)
                           : launch_norm<kLargeTable>(ts + i, k, bits, part + parts, &blocks, s);
      parts += blocks;
    }
  if (e == cudaSuccess && (clip || step_dev)) {
    adamw_prelude_kernel<<<1, 256, 0, s>>>(part, parts, clip ? sc : nullptr, norm_out, step_dev,
                                           step_dev ? sc + 1 : nullptr, lr, b1, b2);
    note_launches(1);
    e = cudaGetLastError();
  }
  Hyper h;
  h.b1 = static_cast<float>(b1);
  h.omb1 = static_cast<float>(1.0 - b1);
  h.b2 = static_cast<float>(b2);
  h.omb2 = static_cast<float>(1.0 - b2);
  h.eps = static_cast<float>(eps);
  h.down = static_cast<float>(0.5 / (1.0 - std::sqrt(b1)) + 1.0);
  h.step = static_cast<uint32_t>(step);
  const double t = static_cast<double>(step);
  h.step_size = step_dev ? 0.0f : static_cast<float>(lr / (1.0 - std::pow(b1, t)));
  h.inv_root = step_dev ? 0.0f : static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(b2, t)));
  h.scalars = step_dev ? sc + 1 : nullptr;
  h.norm = clip ? sc : nullptr;
  h.max_norm = static_cast<float>(max_norm);
  for (int i = 0; i < count && e == cudaSuccess; i += kLargeTable) {
    const int k = std::min(kLargeTable, count - i);
    e = k <= kSmallTable ? launch_step<kSmallTable>(ts + i, k, bits, lr, h, s)
                         : launch_step<kLargeTable>(ts + i, k, bits, lr, h, s);
  }
  return cuda_status(e);
}

int adamw_state_values(const void* q, const float* scale, int64_t n, int is_signed, void* out,
                       cudaStream_t s) {
  if (n <= 0) return kOk;
  constexpr int64_t kEach = static_cast<int64_t>(kWarps) * kValues * kQBlock;
  const int64_t blocks = (n + kEach - 1) / kEach;
  if (blocks > 0x7fffffff) return kErrUnsupported;
  const bool vec = aligned(q, 8) && aligned(out, 16);
  const uint8_t* c = static_cast<const uint8_t*>(q);
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  if (is_signed)
    adamw_values_kernel<true><<<static_cast<unsigned>(blocks), 32 * kWarps, 0, s>>>(c, scale, n, o, vec);
  else
    adamw_values_kernel<false><<<static_cast<unsigned>(blocks), 32 * kWarps, 0, s>>>(c, scale, n, o, vec);
  note_launches(1);
  return cuda_status(cudaGetLastError());
}

}  // namespace mx
