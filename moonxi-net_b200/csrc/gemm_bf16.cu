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
// left in one accumulator is off by 7e-6).  So a k-block's six products go
// from the smallest to the largest, few MMAs meet a full accumulator, and after
// every k-block, 64 of K, the epilogue warps add the accumulator to float32
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
// One copy's MMAs still wait for the L2 (with half of the loads left out a
// forward product of 8192 x 4096 x 2 x 8192 took 770 us instead of 939, its
// gradients 1332 instead of 1708).  So where enough rows are left a job is 512 of
// them: two tiles of A share one of B, 48 KB a CTA for 1024 cycles of MMAs
// instead of 64, both accumulators are one job's, and the epilogue of one runs
// beside the other's last and the next job's first MMAs.  833 and 1473 us.  A
// short K with a pre-activation to store has more of its epilogue to hide than
// that: 4096 x 1000 x 2 x 2736 with pre, 62 us in tiles of 256 rows, 71 in 512.
// The plan's costs decide.
//
// One launch takes one product or two (a backward pass's dx and dw, which do not
// need each other): the second's tiles follow the first's, so the two share
// the waves of tiles and pay one start and one end.
//
// Persistent, 320 threads: warp 0 one lane issues TMA loads (128-byte swizzle,
// both operands in their stored layout, K- or MN-major) into a ring of slots;
// warp 1 of the even CTA one lane issues the MMAs for the pair; warps 2-9 read
// the accumulator (32 lanes x 32 columns at a time) and store each thread's 32
// columns of a row in 32-byte pieces, whole sectors.  They stay off the shared
// memory, which the MMAs' operand reads and the TMA writes fill between them: a
// transpose there took the forward product of 8192 x 4096 x 2 x 8192 from 0.81
// to 1.6 ms.  Only where the output's rows are not 16-byte aligned do they
// transpose through padded shared memory, to store whole rows of odd width
// (pre and the partial tiles have padded rows).  Two accumulators: a tile's epilogue runs
// beside the next tile's (three copies: the next k-block's) MMAs.
// Few tiles and a long K: the K range is split over the pairs, fp32 partial
// tiles go to scratch and a second kernel adds them in order.  (Added up by the
// last warp to arrive at its part of a tile instead, a product of 33 x 2 x 1000
// x 784 took 39 us against 12 and 4: few warps, each waiting for one part after
// the other.)
// Every mbarrier wait is bounded (mx::wait_bar), as in gemm_tc.cu.
//
// Registers: 320 threads get 168 each.  Three copies' epilogue holds 128 sums and
// the 32 values that it adds to them, and spills 84 to 96 bytes a thread to local
// memory (100 to 212 read back); one copy's kernels spill nothing.
#include <algorithm>
#include <array>
#include <type_traits>

#include "gated_act.cuh"
#include "mx_internal.h"
#include "mx_ptx.cuh"

namespace mx {
namespace {

constexpr int kTile = 256;             // rows and columns of a pair's tile
constexpr int kHalf = 128;             // ... of one CTA's operand tiles
constexpr int kBK = 64;                // a k-block: 128 bytes of bf16
constexpr int kOpBytes = kHalf * kBK * 2;  // an operand tile
constexpr int kThreads = 320;
constexpr int kTmemCols = 512;
constexpr int kTrFloats = 32 * 33;     // a warp's transpose buffer

// The ring.  One copy: a slot is a k-block, SUB tiles of A and one of B.  Three
// copies: a slot is one copy's tiles of A and B, a k-block takes three slots,
// from the smallest copy to the largest, which is the order in which the
// products give them back, so the next k-block but one begins to load after a
// third of this one's MMAs.
// VEC (the outputs' rows start on 16 bytes): no transpose buffers.
template <int NC, bool VEC, int SUB>
struct Ring {
  static constexpr int kSlots = SUB == 2 ? 4 : 6;
  static constexpr int kSlotBytes = (SUB + 1) * kOpBytes;
  static constexpr int kTranspose = VEC ? 0 : 8 * kTrFloats;
  static constexpr int kSmem = kSlots * kSlotBytes + kTranspose * 4 + 256 + 1024;
  static_assert(kSmem <= 232448, "shared memory of an SM");
};

// One product of a launch.
struct Problem {
  void* out;
  const void* bias;
  float* pre;
  float* parts;     // [splits][M][ldp] when the K range is split
  int64_t ldc;
  int64_t ldp;      // row of parts: pad8(N), gated twice that, like pre
  int M, N, K;
  int tiles_m, tiles_n, tiles;
  int splits, kb_per;  // k-blocks of a split
  int act;
  int vec;          // bytes of a store to out: 32 or 16 (0: rows unaligned, not VEC)
  int a_kmajor, b_kmajor;
};
template <int NC>
struct Launch {
  CUtensorMap a[2][NC];     // by problem
  CUtensorMap b[2][2][NC];  // by problem, by the CTA's rank in the pair
  Problem p[2];
  int* status;
  uint64_t timeout_ns;
  int jobs0, jobs1;         // of each problem
  int fill;                 // see Queue
  int sub;                  // tiles of 256 rows of a job
};

// The jobs of a pair, in order.  The first product's go round the pairs; where
// its last round leaves pairs idle, each of these takes `fill` jobs of the
// second product, and the rest of them go round again.
struct Queue {
  int c, pairs, short0;  // short0: pairs from here on miss the first's last round
  int q, j, extra;
  template <int NC>
  __device__ __forceinline__ void init(const Launch<NC>& L, int pair, int n) {
    c = pair;
    pairs = n;
    short0 = L.jobs0 % n;
    q = 0;
    j = c;
    extra = L.fill > 0 && c >= short0 ? L.fill : 0;
  }
  // The next job: its problem and number; false at the end.
  template <int NC>
  __device__ __forceinline__ bool next(const Launch<NC>& L, int& problem, int& job) {
    if (q == 0) {
      if (j < L.jobs0) {
        problem = 0;
        job = j;
        j += pairs;
        return true;
      }
      q = 1;
      j = c - short0;  // the fill, then the rounds
    }
    problem = 1;
    if (extra > 0) {
      job = j;
      j += pairs - short0;
      if (--extra == 0) q = 2;
      return true;
    }
    if (q < 3) {
      j = L.fill * (pairs - short0) + c;
      q = 3;
    }
    job = j;
    j += pairs;
    return job < L.jobs1;
  }
};

// Job j of problem q: split j / tiles of tile j % tiles; k-blocks [kb0, kb1).
struct Job {
  int q, tm, tn, split, tile, kb0, kb1;
};
template <int NC>
__device__ __forceinline__ Job job_at(const Launch<NC>& L, int q, int j) {
  Job r;
  r.q = q;
  const Problem& p = L.p[q];
  r.split = j / p.tiles;
  r.tile = j - r.split * p.tiles;
  // Bands of tiles of 2048 rows, column by column inside a band: the pairs that
  // run at one time share rows of A and columns of B in L2.
  const int G = 8 / L.sub;
  const int band = r.tile / (G * p.tiles_n);
  const int gm = min(G, p.tiles_m - band * G);
  const int i = r.tile - band * G * p.tiles_n;
  r.tm = band * G + i % gm;
  r.tn = i / gm;
  r.kb0 = r.split * p.kb_per;
  r.kb1 = min((p.K + kBK - 1) / kBK, r.kb0 + p.kb_per);
  return r;
}

// A 128 x 64 tile of one copy: one box of 64 k x 128 rows, or two of 64 rows x
// 64 k.
__device__ __forceinline__ void load_tile(bool kmajor, uint8_t* dst, const CUtensorMap* map,
                                          uint32_t bar, int r0, int k0) {
  if (kmajor) {
    tma_load_2d_pair(dst, map, bar, k0, r0);
  } else {
    tma_load_2d_pair(dst, map, bar, r0, k0);
    tma_load_2d_pair(dst + kOpBytes / 2, map, bar, r0 + 64, k0);
  }
}

// Operand tiles as the MMA reads them.  K-major: 128-byte rows, groups of 8
// rows 1024 bytes apart, a 16-deep slice 32 bytes on.  MN-major: chunks of 64
// columns 8 KB apart, groups of 8 k 1024 bytes apart, a slice two groups on.
struct TileDesc {
  uint64_t base;   // the descriptor of address 0
  uint32_t slice;  // bytes from a slice to the next
  __device__ __forceinline__ explicit TileDesc(bool kmajor)
      : base(kmajor ? sdesc_kmajor(0, 1024, 2) : sdesc_mnmajor(0, kOpBytes / 2, 1024, 2)),
        slice(kmajor ? 32 : 2048) {}
  __device__ __forceinline__ uint64_t at(uint32_t addr, int j) const {
    return base | static_cast<uint64_t>(((addr + j * slice) & 0x3FFFFu) >> 4);
  }
};

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

template <int NC, bool GATED, bool VEC, int SUB>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    bf16_gemm_kernel(const __grid_constant__ Launch<NC> L) {
  using T = typename std::conditional<NC == 1, __nv_bfloat16, float>::type;
  static_assert(NC == 1 || SUB == 1, "three copies' accumulators are added up");
  constexpr int kSlots = Ring<NC, VEC, SUB>::kSlots, kSlotBytes = Ring<NC, VEC, SUB>::kSlotBytes;
  constexpr int kB = SUB * kOpBytes;  // B's tile in a slot
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* tr = reinterpret_cast<float*>(smem + kSlots * kSlotBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(tr + Ring<NC, VEC, SUB>::kTranspose);  // the even CTA's are used
  uint64_t* empty = full + kSlots;
  uint64_t* acc_full = empty + kSlots;
  uint64_t* acc_empty = acc_full + 2;  // the even CTA's are used
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
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
      tma_prefetch_desc(&L.a[0][i]);
      tma_prefetch_desc(&L.b[0][rank][i]);
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
  grid_trigger();
  grid_wait();
  Queue queue;
  queue.init(L, pair, pairs);
  int prob, number;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int slot = 0;
      uint32_t phase = 0;
      uint32_t armed = 0, armed_parity = 0;  // bit s: a copy was issued, and its phase
      bool ok = true;
      while (ok && queue.next(L, prob, number)) {
        const Job r = job_at(L, prob, number);
        const bool ak = L.p[r.q].a_kmajor, bk = L.p[r.q].b_kmajor;
        const int m0 = r.tm * SUB * kTile + rank * kHalf;
        const int n0 = GATED ? r.tn * kHalf : r.tn * kTile + rank * kHalf;
        for (int kb = r.kb0; ok && kb < r.kb1; ++kb) {
#pragma unroll
          for (int i = NC - 1; i >= 0; --i) {
            if (!wait_bar(&empty[slot], phase ^ 1, abort_flag, L.status, L.timeout_ns, 401)) {
              ok = false;
              break;
            }
            uint8_t* base = smem + slot * kSlotBytes;
            if (rank == 0) bar_arrive_expect_tx(&full[slot], 2 * kSlotBytes);
            armed |= 1u << slot;
            armed_parity = (armed_parity & ~(1u << slot)) | (phase << slot);
            const uint32_t bar = cluster_addr(&full[slot], 0);
#pragma unroll
            for (int u = 0; u < SUB; ++u)
              load_tile(ak, base + u * kOpBytes, &L.a[r.q][i], bar, m0 + u * kTile, kb * kBK);
            load_tile(bk, base + kB, &L.b[r.q][rank][i], bar, n0, kb * kBK);
            if (++slot == kSlots) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
      }
      // Every copy has landed before the CTA can exit.  The even CTA's
      // barriers count both CTAs' copies and the pair exits together; when
      // waits gave up, the odd CTA also lets its own copies finish by time.
      if (rank == 0) {
        for (int s = 0; s < kSlots; ++s)
          if (armed >> s & 1) drain_wait(&full[s], armed_parity >> s & 1, L.status, 407);
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
      int slot = 0;
      uint32_t phase = 0;
      int seg = 0;  // accumulators used so far
      bool ok = true;
      auto take_acc = [&](int n) {
        if (!wait_bar(&acc_empty[n & 1], (n >> 1 & 1) ^ 1, abort_flag, L.status, L.timeout_ns, 402))
          return false;
        tc_fence_after();
        return true;
      };
      auto wait_slot = [&](int n, uint32_t parity) {
        if (!wait_bar(&full[n], parity, abort_flag, L.status, L.timeout_ns, 403)) return false;
        tc_fence_after();
        return true;
      };
      auto advance = [&](int& n, uint32_t& parity, int by) {
        n += by;
        if (n == kSlots) {
          n = 0;
          parity ^= 1;
        }
      };
      while (ok && queue.next(L, prob, number)) {
        const Job r = job_at(L, prob, number);
        const bool ak = L.p[r.q].a_kmajor, bk = L.p[r.q].b_kmajor;
        const uint32_t idesc = idesc_bf16(kTile, kTile, !ak, !bk);
        const TileDesc da(ak), db(bk);
        // the k-block's product of the operand tiles at sa and sb into
        // accumulator n
        auto product = [&](int n, uint32_t sa, uint32_t sb, bool first) {
          const uint32_t d = tmem_base + (n & 1) * kTile;
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            mma_f16_pair(d, da.at(sa, k), db.at(sb, k), idesc, first && k == 0 ? 0 : 1);
        };
        if constexpr (NC == 3) {
          for (int kb = r.kb0; ok && kb < r.kb1; ++kb) {
            ok = take_acc(seg);
            // copy i is in slot + 2 - i (six slots: a k-block does not wrap)
#pragma unroll
            for (int i = 0; ok && i < 3; ++i) ok = wait_slot(slot + i, phase);
            if (!ok) break;
            const uint32_t s0 = smem_u32(smem + slot * kSlotBytes);
            auto copies = [&](int ca, int cb, bool first) {
              product(seg, s0 + (2 - ca) * kSlotBytes, s0 + (2 - cb) * kSlotBytes + kB, first);
            };
            // from the smallest products to the largest
            copies(2, 0, true);
            copies(0, 2, false);
            tc_commit_both(&empty[slot]);
            copies(1, 1, false);
            copies(1, 0, false);
            copies(0, 1, false);
            tc_commit_both(&empty[slot + 1]);
            copies(0, 0, false);
            tc_commit_both(&empty[slot + 2]);
            tc_commit_both(&acc_full[seg & 1]);
            ++seg;
            advance(slot, phase, 3);
          }
        } else if constexpr (SUB == 1) {
          ok = take_acc(seg);
          for (int kb = r.kb0; ok && kb < r.kb1; ++kb) {
            ok = wait_slot(slot, phase);
            if (!ok) break;
            const uint32_t sa = smem_u32(smem + slot * kSlotBytes);
            product(seg, sa, sa + kB, kb == r.kb0);
            tc_commit_both(&empty[slot]);
            advance(slot, phase, 1);
          }
          if (!ok) break;
          tc_commit_both(&acc_full[seg & 1]);
          ++seg;
        } else {
          // The first accumulator's products of a ring's worth of k-blocks run
          // while the epilogue still reads the second.
          const int ahead = min(kSlots, r.kb1 - r.kb0);
          ok = take_acc(seg);
          int n = slot;
          uint32_t parity = phase;
          for (int i = 0; ok && i < ahead; ++i) {
            ok = wait_slot(n, parity);
            if (!ok) break;
            const uint32_t sa = smem_u32(smem + n * kSlotBytes);
            product(seg, sa, sa + kB, i == 0);
            advance(n, parity, 1);
          }
          if (ok && r.kb0 + ahead == r.kb1) tc_commit_both(&acc_full[seg & 1]);
          ok = ok && take_acc(seg + 1);
          for (int i = 0; ok && i < ahead; ++i) {
            const uint32_t sa = smem_u32(smem + slot * kSlotBytes);
            product(seg + 1, sa + kOpBytes, sa + kB, i == 0);
            tc_commit_both(&empty[slot]);
            advance(slot, phase, 1);
          }
          for (int kb = r.kb0 + ahead; ok && kb < r.kb1; ++kb) {
            ok = wait_slot(slot, phase);
            if (!ok) break;
            const uint32_t sa = smem_u32(smem + slot * kSlotBytes);
            product(seg, sa, sa + kB, false);
            if (kb + 1 == r.kb1) tc_commit_both(&acc_full[seg & 1]);
            product(seg + 1, sa + kOpBytes, sa + kB, false);
            tc_commit_both(&empty[slot]);
            advance(slot, phase, 1);
          }
          if (!ok) break;
          tc_commit_both(&acc_full[(seg + 1) & 1]);
          seg += 2;
        }
      }
      tc_commit_pair(drain);  // every MMA is done before TMEM is released
      drain_wait(drain, 0, L.status, 408);
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
    // 32 columns of this warp's rows in accumulator `acc`.  The lanes part where
    // rows end and where an activation branches; the load wants them together.
    auto load32 = [&](int acc, int col, uint32_t (&r)[32]) {
      __syncwarp();
      tmem_ld_32cols(lanes + acc * kTile + col, r);
      tmem_wait_ld();
    };
    auto wait_acc = [&]() {
      // one lane polls
      int got = 0;
      if (lane == 0)
        got = wait_bar(&acc_full[seg & 1], seg >> 1 & 1, abort_flag, L.status, L.timeout_ns, 404);
      got = __shfl_sync(0xffffffffu, got, 0);
      tc_fence_after();
      return got != 0;
    };
    auto free_acc = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive_cluster(cluster_addr(&acc_empty[seg & 1], 0));
      ++seg;
    };
    // where this warp's block q of 32 columns is in the accumulator (gated: the
    // gate's for even q, the other projection's for odd)
    auto col_of = [&](int q) {
      return GATED ? (q & 1) * kHalf + half * 64 + (q >> 1) * 32 : half * kHalf + q * 32;
    };
    while (ok && queue.next(L, prob, number)) {
      const Job r = job_at(L, prob, number);
      const Problem& p = L.p[r.q];
#pragma unroll 1
      for (int sub = 0; ok && sub < SUB; ++sub) {
      const int row0 = (r.tm * SUB + sub) * kTile + rank * kHalf + group * 32;
      const int rows = min(32, p.M - row0);  // may be below 1
      const bool mine = lane < rows;
      const int64_t row = row0 + lane;
      // the first column of blocks q (and q + 1 when gated) in the output
      auto out_col = [&](int q) {
        return GATED ? r.tn * kHalf + half * 64 + (q >> 1) * 32 : r.tn * kTile + col_of(q);
      };
      // a block of `out`: 32 columns of this warp's rows, lane = row
      auto store_out = [&](int col0, const float (&v)[32]) {
        T* dst = static_cast<T*>(p.out) + row * p.ldc + col0;
        const int left = p.N - col0;
        if (VEC) {
          if (!mine) return;
          if (p.vec == 32) store_row<32>(dst, v, left);
          else store_row<16>(dst, v, left);
        } else {
          // unaligned rows: through shared memory, a row at a time
          __syncwarp();  // the last block's reads are done
#pragma unroll
          for (int i = 0; i < 32; ++i) tw[lane * 33 + i] = v[i];
          __syncwarp();
          dst = static_cast<T*>(p.out) + static_cast<int64_t>(row0) * p.ldc + col0 + lane;
          if (lane < left)
#pragma unroll 4
            for (int i = 0; i < rows; ++i) {
              put(dst, tw[i * 33 + lane]);
              dst += p.ldc;
            }
        }
      };
      // a complete block (gated: two) into the outputs
      auto finish = [&](int q, float (&g)[32], float (&u)[32]) {
        const int col0 = out_col(q), left = p.N - col0;
        if (left <= 0) return;
        if constexpr (GATED) {
          if (p.bias) {
            const T* bias = static_cast<const T*>(p.bias) + col0;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < left) {
                g[i] += to_f(bias[i]);
                u[i] += to_f(bias[p.N + i]);
              }
          }
          if (p.pre && mine) {
            float* pre = p.pre + row * p.ldp + col0;
            store_row<32>(pre, g, left);
            store_row<32>(pre + p.ldp / 2, u, left);
          }
          gate(p.act, g, u);
        }
        store_out(col0, g);
      };
      // a block of this split's part
      auto park = [&](int q, const float (&g)[32], const float (&u)[32]) {
        const int col0 = out_col(q), left = p.N - col0;
        if (left <= 0 || !mine) return;
        float* dst = p.parts + (static_cast<int64_t>(r.split) * p.M + row) * p.ldp + col0;
        store_row<32>(dst, g, left);
        if (GATED) store_row<32>(dst + p.ldp / 2, u, left);
      };
      constexpr int kStep = GATED ? 2 : 1;
      if constexpr (NC == 3) {
        float acc[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[q][i] = 0.0f;
        for (int kb = r.kb0; kb < r.kb1; ++kb) {
          ok = wait_acc();
          if (!ok) break;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t t[32];
            load32(seg & 1, col_of(q), t);
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[q][i] += __uint_as_float(t[i]);
          }
          free_acc();
        }
        if (!ok) break;
#pragma unroll
        for (int q = 0; q < 4; q += kStep) {
          if (p.splits > 1) park(q, acc[q], acc[(q + 1) & 3]);
          else finish(q, acc[q], acc[(q + 1) & 3]);
        }
      } else {
        ok = wait_acc();
        if (!ok) break;
        // (rolled: the instruction cache holds one body)
#pragma unroll 1
        for (int q = 0; q < 4; q += kStep) {
          uint32_t t[32];
          float g[32], u[32];
          load32(seg & 1, col_of(q), t);
#pragma unroll
          for (int i = 0; i < 32; ++i) g[i] = __uint_as_float(t[i]);
          if (GATED) load32(seg & 1, col_of(q + 1), t);
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = GATED ? __uint_as_float(t[i]) : 0.0f;
          if (p.splits > 1) park(q, g, u);
          else finish(q, g, u);
        }
        free_acc();
      }
      }
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

// What follows the products, in one launch: the sums of split products' parts,
// in order (gated: bias and activation too), four columns a thread; and a
// column sum over rows of partial sums (dbias), 32 columns a block.
struct Tail {
  Problem p[2];
  int blocks[2];      // of each product's sum (0: not split)
  const float* part;  // [rows][width]
  void* sum;
  int rows, width;
};
template <typename T, bool GATED>
__device__ __forceinline__ void join_block(const Problem& p, int block, int blocks) {
  const int64_t quads = pad8(p.N) / 4, n = p.M * quads, part = p.M * p.ldp;
  for (int64_t i = block * 256ll + threadIdx.x; i < n; i += blocks * 256ll) {
    const int64_t m = i / quads;
    const int c = static_cast<int>(i - m * quads) * 4;
    const float* src = p.parts + m * p.ldp + c;
    float g[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
      const float4 a = __ldcg(reinterpret_cast<const float4*>(src + s * part));
      g[0] += a.x; g[1] += a.y; g[2] += a.z; g[3] += a.w;
      if (GATED) {
        const float4 b = __ldcg(reinterpret_cast<const float4*>(src + s * part + p.ldp / 2));
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
template <typename T, bool GATED>
__global__ void __launch_bounds__(256) tail_kernel(const __grid_constant__ Tail t) {
  grid_wait();
  int block = blockIdx.x;
  if (block < t.blocks[0]) {
    join_block<T, GATED>(t.p[0], block, t.blocks[0]);
    return;
  }
  if constexpr (!GATED) {
    block -= t.blocks[0];
    if (block < t.blocks[1]) {
      join_block<T, false>(t.p[1], block, t.blocks[1]);
      return;
    }
    block -= t.blocks[1];
    __shared__ float sh[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = block * 32ll + lane;
    float s = 0.0f;
    if (c < t.width)
#pragma unroll 4
      for (int r = warp; r < t.rows; r += 8) s += t.part[static_cast<int64_t>(r) * t.width + c];
    sh[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < t.width) {
      s = 0.0f;
      for (int i = 0; i < 8; ++i) s += sh[i][lane];
      put(static_cast<T*>(t.sum) + c, s);
    }
  }
}

struct Plan {
  int tiles_m = 0, tiles_n = 0, tiles = 0, num_kb = 0, splits = 1, kb_per = 0;
  size_t part_bytes = 0;
  int jobs() const { return tiles * splits; }
};
struct Plans {
  Plan p[2];
  int pairs = 0, sub = 1;
  bool vec = true, save = false;  // the outputs' rows start on 16 bytes; pre is stored
  bool split() const { return p[0].splits > 1 || p[1].splits > 1; }
};

void set_splits(Plan& q, int want) {
  q.kb_per = (q.num_kb + want - 1) / want;
  q.splits = (q.num_kb + q.kb_per - 1) / q.kb_per;
}

// A job's cost in cycles, as measured: a k-block (one copy, 256 rows: 512
// cycles of MMAs, which wait for L2; 512 rows: 1024; three copies: 3072), and a
// start and an epilogue, which runs beside the next job's MMAs (512 rows: only
// beside a ring's worth of them, so what it stores counts for more); a split job
// has the partial tile's way through memory on top.
int64_t job_cost(const Plans& pl, int i, int copies) {
  const Plan& q = pl.p[i];
  const bool tall = pl.sub == 2;
  const int kb = copies == 3 ? 3400 : tall ? 1160 : 700;
  int ends = copies == 3 ? 3400 : tall ? 7000 : 4200;
  if (copies == 1 && pl.save) ends += tall ? 13000 : 3800;
  if (copies == 1 && !pl.vec) ends += tall ? 14000 : 5000;
  return static_cast<int64_t>(q.kb_per) * kb + ends * (q.splits > 1 ? 2 : 1);
}
// Queue's fill: what the first product's last round leaves to the pairs that
// miss it.
int fill_of(const Plans& pl, int pairs, int copies) {
  const int shorter = pairs - pl.p[0].jobs() % pairs;
  if (shorter == pairs || pl.p[1].jobs() == 0) return 0;
  return static_cast<int>(std::min<int64_t>(job_cost(pl, 0, copies) / job_cost(pl, 1, copies),
                                            pl.p[1].jobs() / shorter));
}
// The longest queue of a pair (queues differ only where a product's last round
// ends), and the launch that adds split products up.
int64_t makespan(const Plans& pl, int pairs, int copies) {
  const int64_t c0 = job_cost(pl, 0, copies);
  const int64_t c1 = pl.p[1].jobs() > 0 ? job_cost(pl, 1, copies) : 0;
  const int j0 = pl.p[0].jobs(), r = j0 % pairs, fill = fill_of(pl, pairs, copies);
  const int rest = pl.p[1].jobs() - (fill > 0 ? fill * (pairs - r) : 0);
  const int at[3] = {0, r, rest % pairs};
  int64_t worst = 0;
  for (int c : at) {
    const int n0 = (j0 - c + pairs - 1) / pairs;
    const int n1 = (c >= r ? fill : 0) + (rest - c + pairs - 1) / pairs;
    worst = std::max(worst, n0 * c0 + n1 * c1);
  }
  return worst + (pl.split() ? 6000 : 0);
}

void set_tiles(Plans& pl, const Bf16Gemm* g, int count, int sub) {
  pl.sub = sub;
  for (int i = 0; i < count; ++i) {
    Plan& q = pl.p[i];
    const int width = g[i].gated ? kHalf : kTile;
    q.tiles_m = (g[i].M + sub * kTile - 1) / (sub * kTile);
    q.tiles_n = (g[i].N + width - 1) / width;
    q.tiles = q.tiles_m * q.tiles_n;
    q.num_kb = std::max(1, (g[i].K + kBK - 1) / kBK);
    q.kb_per = q.num_kb;
    q.splits = 1;
  }
}

// Tiles of 256 rows: whole ones where they fill the machine; otherwise the
// split counts, the longer product's first, with the shortest longest queue.
// Sizes alone decide, and with them the scratch.
Plans make_plan(const Bf16Gemm* g, int count, int pairs) {
  Plans pl;
  const int copies = g[0].copies;
  set_tiles(pl, g, count, 1);
  const int least = copies == 3 ? 2 : 8;  // k-blocks of a split
  const int longer = pl.p[1].num_kb > pl.p[0].num_kb ? 1 : 0;
  if (pl.p[0].tiles + pl.p[1].tiles < 3 * pairs) {
    for (int n = 0; n < count; ++n) {
      Plan& q = pl.p[n == 0 ? longer : 1 - longer];
      int best = 1;
      int64_t cost = makespan(pl, pairs, copies);
      for (int want = 2; want <= 16 && q.num_kb / want >= least; ++want) {
        set_splits(q, want);
        const int64_t c = makespan(pl, pairs, copies);
        if (c < cost) {
          best = want;
          cost = c;
        }
      }
      set_splits(q, best);
    }
  }
  for (int i = 0; i < count; ++i) {
    Plan& q = pl.p[i];
    const size_t row = (static_cast<size_t>(g[i].N) + 7) / 8 * 8 * (g[i].gated ? 2 : 1);
    if (q.splits > 1)
      q.part_bytes = (static_cast<size_t>(q.splits) * g[i].M * row * sizeof(float) + 255) & ~size_t{255};
  }
  pl.pairs = std::min(pairs, pl.p[0].jobs() + pl.p[1].jobs());
  return pl;
}

// A plan depends on nothing but its key.  A backward call asks for the same few
// plans eleven times (its workspace's size, the check of it, the launch), which
// took 3 us of the host's 28 for 33 x 784 x 2 x 1000.
Plans plan_of(const Context* ctx, const Bf16Gemm* g, int count) {
  using Key = std::array<int, 10>;
  struct Entry {
    Key key{};
    Plans plans;
  };
  static thread_local Entry kept[8];
  static thread_local unsigned turn = 0;
  const int pairs = std::max(1, ctx->tc_sms() / 2);
  const Bf16Gemm& h = g[count - 1];
  const Key key{pairs, count, g[0].copies, g[0].gated, g[0].M, g[0].N, g[0].K, h.M, h.N, h.K};
  for (const Entry& e : kept)
    if (e.key == key) return e.plans;
  Entry& e = kept[turn++ % 8];
  e.plans = make_plan(g, count, pairs);
  e.key = key;
  return e.plans;
}

// The plan of a launch: tiles of 512 rows (one copy, no scratch) where those are
// sooner done.  vec: the outputs' rows start on 16 bytes; save: pre is stored.
Plans launch_plan(const Context* ctx, const Bf16Gemm* g, int count, bool vec, bool save) {
  Plans pl = plan_of(ctx, g, count);
  pl.vec = vec;
  pl.save = save;
  if (g[0].copies != 1) return pl;
  const int pairs = std::max(1, ctx->tc_sms() / 2);
  Plans tall;
  tall.vec = vec;
  tall.save = save;
  set_tiles(tall, g, count, 2);
  if (makespan(tall, pairs, 1) >= makespan(pl, pairs, 1)) return pl;
  tall.pairs = std::min(pairs, tall.p[0].jobs() + tall.p[1].jobs());
  return tall;
}

bool operand_map(CUtensorMap* m, const Bf16Operand& o, int copy, int rows, int K) {
  const void* base = static_cast<const __nv_bfloat16*>(o.base) + copy * o.copy;
  return o.kmajor ? make_tmap_bf16(m, base, K, rows, o.ld * 2, kBK, kHalf)
                  : make_tmap_bf16(m, base, rows, K, o.ld * 2, 64, kBK);
}

template <int NC, bool GATED>
int launch(Context* ctx, const Bf16Gemm* g, int count, void* scratch, const Bf16ColumnSum* sum,
           bool after, cudaStream_t s) {
  using T = typename std::conditional<NC == 1, __nv_bfloat16, float>::type;
  auto out_on = [&](const Bf16Gemm& q, int bytes) {
    const int n = bytes / static_cast<int>(sizeof(T));
    return q.N % n == 0 && q.ldc % n == 0 && (reinterpret_cast<uintptr_t>(q.out) & (bytes - 1)) == 0;
  };
  const bool vec = out_on(g[0], 16) && (count == 1 || out_on(g[1], 16));
  const Plans pl = launch_plan(ctx, g, count, vec, GATED && g[0].pre);
  if (pl.split() && (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255u) != 0))
    return kErrInvalid;
  Launch<NC> L;
  uint8_t* parts = static_cast<uint8_t*>(scratch);
  L.p[1] = Problem{};
  for (int i = 0; i < count; ++i) {
    for (int c = 0; c < NC; ++c)
      if (!operand_map(&L.a[i][c], g[i].a, c, g[i].M, g[i].K) ||
          !operand_map(&L.b[i][0][c], g[i].b, c, g[i].N, g[i].K) ||
          (GATED && !operand_map(&L.b[i][1][c], g[i].b2, c, g[i].N, g[i].K)))
        return kErrUnsupported;
    if (!GATED) std::copy(L.b[i][0], L.b[i][0] + NC, L.b[i][1]);
    Problem& p = L.p[i];
    const Plan& q = pl.p[i];
    p.out = g[i].out;
    p.bias = g[i].bias;
    p.pre = g[i].pre;
    p.parts = q.splits > 1 ? reinterpret_cast<float*>(parts) : nullptr;
    parts += q.part_bytes;
    p.ldc = g[i].ldc;
    p.ldp = ((static_cast<int64_t>(g[i].N) + 7) & ~7ll) * (GATED ? 2 : 1);
    p.M = g[i].M; p.N = g[i].N; p.K = g[i].K;
    p.tiles_m = q.tiles_m; p.tiles_n = q.tiles_n; p.tiles = q.tiles;
    p.splits = q.splits; p.kb_per = q.kb_per;
    p.act = g[i].act;
    p.a_kmajor = g[i].a.kmajor;
    p.b_kmajor = g[i].b.kmajor;
    p.vec = out_on(g[i], 32) ? 32 : out_on(g[i], 16) ? 16 : 0;
    if ((reinterpret_cast<uintptr_t>(p.pre) & 31u) != 0) return kErrInvalid;
  }
  L.status = ctx->status;
  L.timeout_ns = ctx->timeout_ns;
  L.jobs0 = pl.p[0].jobs();
  L.jobs1 = pl.p[1].jobs();
  L.fill = fill_of(pl, pl.pairs, NC);
  L.sub = pl.sub;
  auto start = [&](auto kern, int bytes, SmemOptIn& opt_in) {
    cudaError_t e = opt_in.ensure(kern, bytes);
    if (e != cudaSuccess) return e;
    note_launches(1);
    return launch_after(kern, 2 * pl.pairs, kThreads, bytes, s, after, L);
  };
  static SmemOptIn opt_vec, opt_any;
  cudaError_t e;
  if constexpr (NC == 1) {
    static SmemOptIn tall_vec, tall_any;
    if (pl.sub == 2)
      e = vec ? start(bf16_gemm_kernel<1, GATED, true, 2>, Ring<1, true, 2>::kSmem, tall_vec)
              : start(bf16_gemm_kernel<1, GATED, false, 2>, Ring<1, false, 2>::kSmem, tall_any);
  }
  if (pl.sub == 1)
    e = vec ? start(bf16_gemm_kernel<NC, GATED, true, 1>, Ring<NC, true, 1>::kSmem, opt_vec)
            : start(bf16_gemm_kernel<NC, GATED, false, 1>, Ring<NC, false, 1>::kSmem, opt_any);
  if (e != cudaSuccess || (!pl.split() && !sum)) return cuda_status(e);
  Tail t{};
  for (int i = 0; i < 2; ++i) {
    t.p[i] = L.p[i];
    if (pl.p[i].splits > 1)
      t.blocks[i] = static_cast<int>(std::min<int64_t>(
          (L.p[i].M * (L.p[i].ldp / (GATED ? 8 : 4)) + 255) / 256, ctx->num_sms * 16));
  }
  int blocks = t.blocks[0] + t.blocks[1];
  if (sum) {
    t.part = sum->part;
    t.sum = sum->out;
    t.rows = sum->rows;
    t.width = sum->width;
    blocks += (sum->width + 31) / 32;
  }
  note_launches(1);
  return cuda_status(launch_after(tail_kernel<T, GATED>, blocks, 256, 0, s, true, t));
}

}  // namespace

size_t bf16_gemm_scratch_bytes(const Context* ctx, const Bf16Gemm* g, int count) {
  const Plans pl = plan_of(ctx, g, count);
  return pl.p[0].part_bytes + pl.p[1].part_bytes;
}

int bf16_gemm(Context* ctx, const Bf16Gemm* g, int count, void* scratch, const Bf16ColumnSum* sum,
              bool after, cudaStream_t s) {
  if (count < 1 || count > 2 || (sum && g[0].gated) || (count == 2 && (g[0].gated || g[1].gated || g[0].copies != g[1].copies)))
    return kErrInvalid;
  for (int i = 0; i < count; ++i)
    if (g[i].M <= 0 || g[i].N <= 0 || g[i].K <= 0) return kErrInvalid;
  if (g[0].copies == 3)
    return g[0].gated ? launch<3, true>(ctx, g, count, scratch, sum, after, s)
                      : launch<3, false>(ctx, g, count, scratch, sum, after, s);
  return g[0].gated ? launch<1, true>(ctx, g, count, scratch, sum, after, s)
                    : launch<1, false>(ctx, g, count, scratch, sum, after, s);
}

}  // namespace mx
