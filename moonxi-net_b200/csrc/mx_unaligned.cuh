// mx_unaligned.cuh -- 16 bytes from any element of a matrix.
//
// A row of odd length starts anywhere.  Eight bfloat16 (four float32) from such a
// place are the overlap of two aligned 16-byte pieces: two wide loads, the second
// of which is the neighbouring lane's first and comes from L1, and a shift by
// whole words and a half, against eight loads of an element each.
#pragma once
#include <cstdint>

namespace mx {

struct Piece {
  uint4 x, y;  // the aligned 16 bytes that p points into, and the next
};

// Both pieces lie in the matrix where p - 16 bytes and p + 32 bytes do.
template <typename T>
__device__ __forceinline__ Piece load_piece(const T* p) {
  const uint4* a =
      reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15));
  return {__ldg(a), __ldg(a + 1)};
}

template <typename T>
__device__ __forceinline__ uint4 shift_piece(const Piece& q, const T* p) {
  const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
  uint32_t w0 = q.x.x, w1 = q.x.y, w2 = q.x.z, w3 = q.x.w, w4 = q.y.x, w5 = q.y.y, w6 = q.y.z;
  if (off & 8) {
    w0 = w2; w1 = w3; w2 = w4; w3 = w5; w4 = w6; w5 = q.y.w;
  }
  if (off & 4) {
    w0 = w1; w1 = w2; w2 = w3; w3 = w4; w4 = w5;
  }
  const uint32_t bits = (off & 3) * 8;
  return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits),
                    __funnelshift_r(w2, w3, bits), __funnelshift_r(w3, w4, bits));
}

// Whether load_piece may read at every element of [first, last].
template <typename T>
__device__ __forceinline__ bool pieces_inside(const T* first, const T* last, const T* lo,
                                              const T* hi) {
  return reinterpret_cast<uintptr_t>(first) >= reinterpret_cast<uintptr_t>(lo) + 16 &&
         reinterpret_cast<uintptr_t>(last) + 32 <= reinterpret_cast<uintptr_t>(hi);
}

// The 16 bytes at p, which points into the matrix [lo, hi), near its ends too:
// what lies past hi is zero.
template <typename T>
__device__ __forceinline__ uint4 load16_any(const T* p, const T* lo, const T* hi) {
  if (pieces_inside(p, p, lo, hi)) return shift_piece(load_piece(p), p);
  constexpr int N = 16 / sizeof(T);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (p + i < hi) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(p + i));
      } else {
        w[i >> 1] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(p + i)))
                     << (16 * (i & 1));
      }
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace mx
