// gemm_bf16.cu -- tcgen05 GEMM on bfloat16 operands for sm_100a, with the gated
// layer's epilogue; float32 operands as three bfloat16 copies.
//
// One copy: C = A B, fp32 accumulators in TMEM, rounded once on the way out.
// Three copies: x = x0 + x1 + x2 with x0 = bf16(x), x1 = bf16(x - x0), x2 =
// bf16(x - x0 - x1), 24 bits of mantissa between them.  The products whose
// factors' indexes sum to 2 or less are accumulated (the others are below
// 2^-24 of the result), six MMAs for one multiply-add: 1/6 of the bf16 rate.
// The tensor core truncates its accumulator at every MMA, about 2e-8 of the
// result each and always towards zero (measured: a 3xTF32 product of K = 1024
// left in one accumulator is off by 7e-6).  So a stage's six products go from
// the smallest to the largest, few MMAs meet a full accumulator, and after
// every stage, 64 of K, the epilogue warps add the accumulator to float32
// registers with rounding: 2e-7 for 512 x 1024 x 8192 where SGEMM has 9e-7.
// (Four stages of 32 of K: 60 us for that product against 45 when every stage
// is added up, the epilogue's rate, and 48 us and 6e-7 when every second is.)
//
// CTA pairs (cta_group::2): a pair computes a 256 x 256 tile, each CTA holding
// 128 rows of A, 128 columns of B and its 128 x 256 half of the accumulator:
// 32 KB of loads a CTA for 64 of K where a single CTA's 128 x 256 tile loads
// 48 KB, which is what keeps the L2 from being the bound.  Gated: the even
// CTA's 128 columns of B are the gate's, the odd one's the other projection's,
// so an accumulator row holds g and u of the same 128 outputs and the epilogue
// has both.
//
// Persistent, 320 threads: warp 0 one lane issues TMA loads (128-byte swizzle,
// both operands in their stored layout, K- or MN-major) into a ring of stages;
// warp 1 of the even CTA one lane issues the MMAs for the pair; warps 2-9 read
// the accumulator (32 lanes x 32 columns at a time) and store each thread's 32
// columns of a row in 32-byte pieces, whole sectors.  They stay off the shared
// memory, which the MMAs' operand reads and the TMA writes fill between them: a
// transpose there took the forward product of 8192 x 4096 x 2 x 8192 from 0.81
// to 1.6 ms.  Only where the output's rows are not 16-byte aligned do they
// transpose through padded shared memory, to store whole rows of odd width
// (pre and the partial tiles have padded rows).  Two accumulators: a tile's epilogue runs
// beside the next tile's (three copies: the next stage's) MMAs.
// Few tiles and a long K: the K range is split over the pairs, fp32 partial
// tiles go to scratch and a second kernel adds them in order.
// Every mbarrier wait is bounded (mx::wait_bar), as in gemm_tc.cu.
#include <algorithm>
#include <type_traits>

#include "gated_act.cuh"
#include "mx_internal.h"
#include "mx_ptx.cuh"

namespace mx {
namespace {

constexpr int kTile = 256;             // rows and columns of a pair's tile
constexpr int kHalf = 128;             // ... of one CTA's operand tiles
constexpr int kBK = 64;                // a stage's depth: 128 bytes of bf16
constexpr int kOpBytes = kHalf * kBK * 2;  // an operand tile
constexpr int kThreads = 320;
constexpr int kTmemCols = 512;
constexpr int kTrFloats = 32 * 33;     // a warp's transpose buffer

template <int NC>
struct Cfg {
  static constexpr int kStages = NC == 3 ? 2 : 6;
  static constexpr int kStageBytes = 2 * NC * kOpBytes;
  static constexpr int kSmem = kStages * kStageBytes + 8 * kTrFloats * 4 + 256 + 1024;
};
static_assert(Cfg<1>::kSmem <= 232448 && Cfg<3>::kSmem <= 232448, "shared memory of an SM");

template <int NC>
struct Maps {
  CUtensorMap a[NC];
  CUtensorMap b[2][NC];  // by the CTA's rank in the pair
};

struct Params {
  void* out;
  const void* bias;
  float* pre;
  float* parts;     // [splits][M][ldp] when the K range is split
  int* status;
  int64_t ldc;
  uint64_t timeout_ns;
  int M, N, K;
  int tiles_m, tiles_n, tiles;
  int splits, kb_per;  // k-blocks of a split
  int act;
  int64_t ldp;         // row of parts: pad8(N), gated twice that, like pre
  int vec;             // bytes of a store to out: 32, 16, or 0 (rows unaligned)
};

// Bands of 8 tiles of rows, column by column inside a band: the pairs that run
// at one time share rows of A and columns of B in L2.
__device__ __forceinline__ void tile_at(const Params& p, int t, int& tm, int& tn) {
  constexpr int G = 8;
  const int band = t / (G * p.tiles_n);
  const int gm = min(G, p.tiles_m - band * G);
  const int r = t - band * G * p.tiles_n;
  tm = band * G + r % gm;
  tn = r / gm;
}

// A 128 x 64 tile of one copy: one box of 64 k x 128 rows, or two of 64 rows x
// 64 k.
template <bool KMAJOR>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint32_t bar,
                                          int r0, int k0) {
  if (KMAJOR) {
    tma_load_2d_pair(dst, map, bar, k0, r0);
  } else {
    tma_load_2d_pair(dst, map, bar, r0, k0);
    tma_load_2d_pair(dst + kOpBytes / 2, map, bar, r0 + 64, k0);
  }
}

// The 16-deep slice j of a tile.  K-major: 128-byte rows, groups of 8 rows
// 1024 bytes apart, a slice 32 bytes on.  MN-major: chunks of 64 columns 8 KB
// apart, groups of 8 k 1024 bytes apart, a slice two groups on.
template <bool KMAJOR>
__device__ __forceinline__ uint64_t slice_desc(uint32_t addr, int j) {
  return KMAJOR ? sdesc_kmajor(addr + j * 32, 1024, 2)
                : sdesc_mnmajor(addr + j * 2048, kOpBytes / 2, 1024, 2);
}

__device__ __forceinline__ int64_t pad8(int64_t n) { return (n + 7) & ~7ll; }

// 32 consecutive values of a row in stores of BYTES; `left` columns remain, and
// a store that begins before the last of them may end after it.
template <int BYTES>
__device__ __forceinline__ void store_row(float* p, const float (&v)[32], int left) {
#pragma unroll
  for (int i = 0; i < 32; i += BYTES / 4)
    if (i < left) {
      if constexpr (BYTES == 32) {
        uint32_t r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = __float_as_uint(v[i + j]);
        st_global_32b(p + i, r);
      } else {
        *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
}
template <int BYTES>
__device__ __forceinline__ void store_row(__nv_bfloat16* p, const float (&v)[32], int left) {
#pragma unroll
  for (int i = 0; i < 32; i += BYTES / 2)
    if (i < left) {
      uint32_t r[8];
#pragma unroll
      for (int j = 0; j < BYTES / 4; ++j) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[i + 2 * j], v[i + 2 * j + 1]);
        r[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
      if constexpr (BYTES == 32) st_global_32b(p + i, r);
      else *reinterpret_cast<uint4*>(p + i) = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

template <int NC, bool AK, bool BKM, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    bf16_gemm_kernel(const __grid_constant__ Maps<NC> maps, const Params p) {
  using T = typename std::conditional<NC == 1, __nv_bfloat16, float>::type;
  using C = Cfg<NC>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* tr = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(tr + 8 * kTrFloats);  // the even CTA's are used
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + 2;  // the even CTA's are used
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      bar_init(&full[s], 1);
      bar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      bar_init(&acc_full[a], 1);
      bar_init(&acc_empty[a], 16);  // eight epilogue warps of each CTA
    }
    bar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    for (int i = 0; i < NC; ++i) {
      tma_prefetch_desc(&maps.a[i]);
      tma_prefetch_desc(&maps.b[rank][i]);
    }
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_kb = (p.K + kBK - 1) / kBK;
  const int jobs = p.tiles * p.splits;  // job j: split j / tiles of tile j % tiles

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t armed = 0, armed_parity = 0;  // bit s: a copy was issued, and its phase
      bool ok = true;
      for (int j = pair; ok && j < jobs; j += pairs) {
        int tm, tn;
        tile_at(p, j % p.tiles, tm, tn);
        const int kb0 = j / p.tiles * p.kb_per, kb1 = min(num_kb, kb0 + p.kb_per);
        const int m0 = tm * kTile + rank * kHalf;
        const int n0 = GATED ? tn * kHalf : tn * kTile + rank * kHalf;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_bar(&empty[stage], phase ^ 1, abort_flag, p.status, p.timeout_ns, 401)) {
            ok = false;
            break;
          }
          uint8_t* base = smem + stage * C::kStageBytes;
          if (rank == 0) bar_arrive_expect_tx(&full[stage], 2 * C::kStageBytes);
          armed |= 1u << stage;
          armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
          const uint32_t bar = cluster_addr(&full[stage], 0);
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            load_tile<AK>(base + i * kOpBytes, &maps.a[i], bar, m0, kb * kBK);
            load_tile<BKM>(base + (NC + i) * kOpBytes, &maps.b[rank][i], bar, n0, kb * kBK);
          }
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // Every copy has landed before the CTA can exit.  The even CTA's
      // barriers count both CTAs' copies and the pair exits together; when
      // waits gave up, the odd CTA also lets its own copies finish by time.
      if (rank == 0) {
        for (int s = 0; s < C::kStages; ++s)
          if (armed >> s & 1) drain_wait(&full[s], armed_parity >> s & 1, p.status, 407);
      } else if (!ok || *abort_flag) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 10000000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_bf16(kTile, kTile, !AK, !BKM);
      int stage = 0;
      uint32_t phase = 0;
      int seg = 0;  // accumulators used so far
      bool ok = true;
      auto take_acc = [&]() {
        const int acc = seg & 1;
        if (!wait_bar(&acc_empty[acc], (seg >> 1 & 1) ^ 1, abort_flag, p.status, p.timeout_ns, 402))
          return false;
        tc_fence_after();
        return true;
      };
      for (int j = pair; ok && j < jobs; j += pairs) {
        const int kb0 = j / p.tiles * p.kb_per, kb1 = min(num_kb, kb0 + p.kb_per);
        if (NC == 1) ok = take_acc();
        uint32_t accumulate = 0;
        for (int kb = kb0; ok && kb < kb1; ++kb) {
          if (NC == 3) {
            ok = take_acc();
            if (!ok) break;
            accumulate = 0;
          }
          if (!wait_bar(&full[stage], phase, abort_flag, p.status, p.timeout_ns, 403)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * C::kStageBytes);
          const uint32_t sb = sa + NC * kOpBytes;
          const uint32_t d = tmem_base + (seg & 1) * kTile;
          if (NC == 1) {
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              mma_f16_pair(d, slice_desc<AK>(sa, k), slice_desc<BKM>(sb, k), idesc, accumulate);
              accumulate = 1;
            }
          } else {
            // from the smallest products to the largest
            constexpr int pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
            for (int q = 0; q < 6; ++q)
#pragma unroll
              for (int k = 0; k < kBK / 16; ++k) {
                mma_f16_pair(d, slice_desc<AK>(sa + pa[q] * kOpBytes, k),
                             slice_desc<BKM>(sb + pb[q] * kOpBytes, k), idesc, accumulate);
                accumulate = 1;
              }
          }
          tc_commit_both(&empty[stage]);
          if (NC == 3) {
            tc_commit_both(&acc_full[seg & 1]);
            ++seg;
          }
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if (NC == 1) {
          tc_commit_both(&acc_full[seg & 1]);
          ++seg;
        }
      }
      tc_commit_pair(drain);  // every MMA is done before TMEM is released
      drain_wait(drain, 0, p.status, 408);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int group = warp & 3;         // the TMEM lanes that this warp may read
    const int half = (warp - 2) >> 2;   // which half of the columns it takes
    const uint32_t lanes = tmem_base + (static_cast<uint32_t>(group * 32) << 16);
    float* tw = tr + (warp - 2) * kTrFloats;
    int seg = 0;
    bool ok = true;
    // 32 columns of this warp's rows in accumulator `acc`
    auto load32 = [&](int acc, int col, uint32_t (&r)[32]) {
      tmem_ld_32cols(lanes + acc * kTile + col, r);
      tmem_wait_ld();
    };
    // a block of `out`: 32 columns of this warp's rows, lane = row
    auto store_out = [&](T* out, int64_t row0, int rows, int col0, const float (&v)[32]) {
      T* dst = out + (row0 + lane) * p.ldc + col0;
      const int left = p.N - col0;
      if (p.vec == 32) {
        if (lane < rows) store_row<32>(dst, v, left);
      } else if (p.vec == 16) {
        if (lane < rows) store_row<16>(dst, v, left);
      } else {
        // unaligned rows: through shared memory, a row at a time
        __syncwarp();  // the last block's reads are done
#pragma unroll
        for (int i = 0; i < 32; ++i) tw[lane * 33 + i] = v[i];
        __syncwarp();
        dst = out + row0 * p.ldc + col0 + lane;
        if (lane < left)
#pragma unroll 4
          for (int i = 0; i < rows; ++i) {
            put(dst, tw[i * 33 + lane]);
            dst += p.ldc;
          }
      }
    };
    auto wait_acc = [&]() {
      if (!wait_bar(&acc_full[seg & 1], seg >> 1 & 1, abort_flag, p.status, p.timeout_ns, 404))
        return false;
      tc_fence_after();
      return true;
    };
    auto free_acc = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive_cluster(cluster_addr(&acc_empty[seg & 1], 0));
      ++seg;
    };
    for (int j = pair; ok && j < jobs; j += pairs) {
      int tm, tn;
      tile_at(p, j % p.tiles, tm, tn);
      const int split = j / p.tiles;
      const int kb0 = split * p.kb_per, kb1 = min(num_kb, kb0 + p.kb_per);
      const int row0 = tm * kTile + rank * kHalf + group * 32;
      const int rows = min(32, p.M - row0);  // may be below 1
      // where this warp's block q of 32 columns is in the accumulator
      auto col_of = [&](int q) {
        return GATED ? (q & 1) * kHalf + half * 64 + (q >> 1) * 32 : half * kHalf + q * 32;
      };
      float acc[NC == 3 ? 4 : 1][32];
      if (NC == 3) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[q % (NC == 3 ? 4 : 1)][i] = 0.0f;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = wait_acc();
          if (!ok) break;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t r[32];
            load32(seg & 1, col_of(q), r);
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[q % (NC == 3 ? 4 : 1)][i] += __uint_as_float(r[i]);
          }
          free_acc();
        }
      } else {
        ok = wait_acc();
      }
      if (!ok) break;
      // block q of this warp, lane = row
      auto block = [&](int q, float (&v)[32]) {
        if (NC == 3) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = acc[q % (NC == 3 ? 4 : 1)][i];
        } else {
          uint32_t r[32];
          load32(seg & 1, col_of(q), r);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        }
      };
      // (one copy: the loops stay rolled, the instruction cache holds one body)
      const bool mine = lane < rows;
      if constexpr (GATED) {
#pragma unroll(NC == 3 ? 2 : 1)
        for (int q = 0; q < 4; q += 2) {
          const int col0 = tn * kHalf + half * 64 + (q >> 1) * 32;
          const int left = p.N - col0;
          float g[32], u[32];
          block(q, g);
          block(q + 1, u);
          if (left <= 0) continue;
          if (p.bias && !p.parts) {
            const T* bias = static_cast<const T*>(p.bias) + col0;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < left) {
                g[i] += to_f(bias[i]);
                u[i] += to_f(bias[p.N + i]);
              }
          }
          float* pre = p.parts ? p.parts + static_cast<int64_t>(split) * p.M * p.ldp : p.pre;
          if (pre && mine) {
            pre += static_cast<int64_t>(row0 + lane) * p.ldp + col0;
            store_row<32>(pre, g, left);
            store_row<32>(pre + p.ldp / 2, u, left);
          }
          if (!p.parts) {
            gate(p.act, g, u);
            store_out(static_cast<T*>(p.out), row0, rows, col0, g);
          }
        }
      } else {
#pragma unroll(NC == 3 ? 4 : 1)
        for (int q = 0; q < 4; ++q) {
          const int col0 = tn * kTile + col_of(q);
          float v[32];
          block(q, v);
          if (col0 >= p.N) continue;
          if (p.parts) {
            if (mine)
              store_row<32>(p.parts + (static_cast<int64_t>(split) * p.M + row0 + lane) * p.ldp + col0,
                            v, p.N - col0);
          } else {
            store_out(static_cast<T*>(p.out), row0, rows, col0, v);
          }
        }
      }
      if (NC == 1) free_acc();
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer reads neither this TMEM nor these barriers any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// The sum of a split product's parts, in order; gated: bias and activation too.
// A thread takes four columns.
template <typename T, bool GATED>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
  const int64_t quads = pad8(p.N) / 4, n = p.M * quads, part = p.M * p.ldp;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t m = i / quads;
    const int c = static_cast<int>(i - m * quads) * 4;
    const float* src = p.parts + m * p.ldp + c;
    float g[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < p.splits; ++s) {
      const float4 a = *reinterpret_cast<const float4*>(src + s * part);
      g[0] += a.x; g[1] += a.y; g[2] += a.z; g[3] += a.w;
      if (GATED) {
        const float4 b = *reinterpret_cast<const float4*>(src + s * part + p.ldp / 2);
        u[0] += b.x; u[1] += b.y; u[2] += b.z; u[3] += b.w;
      }
    }
    if (GATED) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (p.bias && c + j < p.N) {
          g[j] += to_f(static_cast<const T*>(p.bias)[c + j]);
          u[j] += to_f(static_cast<const T*>(p.bias)[p.N + c + j]);
        }
      if (p.pre) {
        *reinterpret_cast<float4*>(p.pre + m * p.ldp + c) = make_float4(g[0], g[1], g[2], g[3]);
        *reinterpret_cast<float4*>(p.pre + m * p.ldp + p.ldp / 2 + c) =
            make_float4(u[0], u[1], u[2], u[3]);
      }
      gate(p.act, g, u);
    }
    T* out = static_cast<T*>(p.out) + m * p.ldc + c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < p.N) put(out + j, g[j]);
  }
}

struct Plan {
  int tiles_m, tiles_n, tiles, splits, kb_per, pairs;
};
Plan plan_of(const Context* ctx, int M, int N, int K, bool gated, int copies) {
  Plan q;
  const int width = gated ? kHalf : kTile;
  q.tiles_m = (M + kTile - 1) / kTile;
  q.tiles_n = (N + width - 1) / width;
  q.tiles = q.tiles_m * q.tiles_n;
  const int num_kb = std::max(1, (K + kBK - 1) / kBK);
  const int pairs = std::max(1, ctx->tc_sms() / 2);
  // Split K when whole tiles leave more than half of the pairs idle, into
  // pieces of at least 512 of K (three copies: 128, six times the work).
  const int least = copies == 3 ? 2 : 8;
  q.splits = 1;
  if (2 * q.tiles <= pairs) q.splits = std::max(1, std::min(pairs / q.tiles, num_kb / least));
  q.kb_per = (num_kb + q.splits - 1) / q.splits;
  q.splits = (num_kb + q.kb_per - 1) / q.kb_per;
  q.pairs = std::min(pairs, q.tiles * q.splits);
  return q;
}

bool operand_map(CUtensorMap* m, const Bf16Operand& o, int copy, int rows, int K) {
  const void* base = static_cast<const __nv_bfloat16*>(o.base) + copy * o.copy;
  return o.kmajor ? make_tmap_bf16(m, base, K, rows, o.ld * 2, kBK, kHalf)
                  : make_tmap_bf16(m, base, rows, K, o.ld * 2, 64, kBK);
}

template <int NC, bool AK, bool BKM, bool GATED>
int launch(Context* ctx, const Bf16Gemm& g, cudaStream_t s) {
  using T = typename std::conditional<NC == 1, __nv_bfloat16, float>::type;
  const Plan q = plan_of(ctx, g.M, g.N, g.K, GATED, NC);
  Maps<NC> maps;
  for (int i = 0; i < NC; ++i)
    if (!operand_map(&maps.a[i], g.a, i, g.M, g.K) ||
        !operand_map(&maps.b[0][i], g.b, i, g.N, g.K) ||
        !operand_map(&maps.b[1][i], GATED ? g.b2 : g.b, i, g.N, g.K))
      return kErrUnsupported;
  Params p{};
  p.out = g.out;
  p.bias = g.bias;
  p.pre = g.pre;
  p.parts = q.splits > 1 ? g.parts : nullptr;
  p.status = ctx->status;
  p.ldc = g.ldc;
  p.timeout_ns = ctx->timeout_ns;
  p.M = g.M; p.N = g.N; p.K = g.K;
  p.tiles_m = q.tiles_m; p.tiles_n = q.tiles_n; p.tiles = q.tiles;
  p.splits = q.splits; p.kb_per = q.kb_per;
  p.act = g.act;
  if (q.splits > 1 && !g.parts) return kErrInvalid;
  auto out_on = [&](int bytes) {
    const int n = bytes / static_cast<int>(sizeof(T));
    return g.N % n == 0 && g.ldc % n == 0 && (reinterpret_cast<uintptr_t>(g.out) & (bytes - 1)) == 0;
  };
  p.vec = out_on(32) ? 32 : out_on(16) ? 16 : 0;
  p.ldp = ((static_cast<int64_t>(g.N) + 7) & ~7ll) * (GATED ? 2 : 1);
  if (((reinterpret_cast<uintptr_t>(g.pre) | reinterpret_cast<uintptr_t>(p.parts)) & 31u) != 0)
    return kErrInvalid;
  auto kern = bf16_gemm_kernel<NC, AK, BKM, GATED>;
  static SmemOptIn opt_in;
  cudaError_t e = opt_in.ensure(kern, Cfg<NC>::kSmem);
  if (e != cudaSuccess) return cuda_status(e);
  kern<<<2 * q.pairs, kThreads, Cfg<NC>::kSmem, s>>>(maps, p);
  note_launches(1);
  e = cudaGetLastError();
  if (e == cudaSuccess && q.splits > 1) {
    const int64_t n = static_cast<int64_t>(g.M) * (p.ldp / (GATED ? 8 : 4));
    join_kernel<T, GATED><<<static_cast<unsigned>(std::min<int64_t>((n + 255) / 256,
                                                                    ctx->num_sms * 16)),
                            256, 0, s>>>(p);
    note_launches(1);
    e = cudaGetLastError();
  }
  return cuda_status(e);
}

template <int NC>
int dispatch(Context* ctx, const Bf16Gemm& g, cudaStream_t s) {
  if (g.gated)
    return g.b.kmajor ? launch<NC, true, true, true>(ctx, g, s)
                      : launch<NC, true, false, true>(ctx, g, s);
  if (!g.a.kmajor) return launch<NC, false, false, false>(ctx, g, s);
  return g.b.kmajor ? launch<NC, true, true, false>(ctx, g, s)
                    : launch<NC, true, false, false>(ctx, g, s);
}

}  // namespace

size_t bf16_gemm_scratch_bytes(const Context* ctx, int M, int N, int K, bool gated, int copies) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan q = plan_of(ctx, M, N, K, gated, copies);
  const size_t row = (static_cast<size_t>(N) + 7) / 8 * 8 * (gated ? 2 : 1);
  return q.splits > 1 ? static_cast<size_t>(q.splits) * M * row * sizeof(float) : 0;
}

// Layouts: A K-major with B of either kind, or both MN-major (not gated).
int bf16_gemm(Context* ctx, const Bf16Gemm& g, cudaStream_t s) {
  if (g.M <= 0 || g.N <= 0 || g.K <= 0 || (!g.a.kmajor && (g.b.kmajor || g.gated)))
    return kErrInvalid;
  return g.copies == 3 ? dispatch<3>(ctx, g, s) : dispatch<1>(ctx, g, s);
}

}  // namespace mx
