// Matrix product on the tensor cores with the epilogue of the operator that
// uses it: the loop shared by the cross-entropy kernels and the 8-bit output
// layer.
//
// A tile is 128 * CG rows by BN columns, made by CG = 1 or 2 CTAs.  With 2 (a
// cluster, one CTA per SM of a pair) each CTA loads its 128 rows of A and half
// of the rows of B, one tcgen05.mma.cta_group::2 reads both halves, and each
// CTA keeps its own 128 rows of the accumulator: per product step an SM reads
// 32 KB of shared memory instead of 48 KB, which is what bounds a 128 x 256
// tile of 8-bit operands (188 of the 128 bytes per clock it could read) and
// costs power with 16-bit ones.
//
// Persistent CTAs of 2 + EW warps:
//   warp 0       TMA producer, STAGES stages of 128 bytes of K (128-byte
//                swizzle);
//   warp 1       TMEM allocation; in the first CTA of a pair the MMA issuer:
//                four tcgen05.mma (32 bytes of K each) per stage into one of
//                two BN-column accumulators;
//   the others   epilogue, one accumulator row per thread, the columns split
//                over EW / 4 warps.
// The two accumulators let the epilogue of a tile run under the next tile's
// products.  An operator may take the accumulator over every KC stages of K
// (a tile's parts, added by its epilogue in fp32 registers).  An operand is
// either K-major (its rows run along K) or MN-major (its rows run along M or
// N; a stage then holds 64 rows of K of as many 64-element column groups as
// the tile needs).
//
// Every wait is bounded; on a timeout all roles leave their loops, then the
// copies and products in flight are waited for (bounded) and TMEM is released,
// as in the fused LM-head kernel; the CTAs of a pair leave together.  The
// epilogue writes NaN for the tiles it could not finish.
#pragma once

#include "fw_host.cuh"
#include "fw_rowslots.cuh"
#include "fw_tc_ptx.cuh"

namespace fwb200 {
namespace {

constexpr int kGemmBM = 128;        // accumulator rows per CTA
constexpr int kGemmRowBytes = 128;  // bytes of K per stage (K-major) = one swizzle row
constexpr uint32_t kGemmABytes = kGemmBM * kGemmRowBytes;

enum TcKind { kTcBf16, kTcF16, kTcS8 };

__host__ __device__ constexpr uint32_t gemm_idesc(TcKind kind, bool a_mn, bool b_mn, int m, int n) {
  // accumulator: fp32 (1) or s32 (2); operands: f16 0, bf16 1 / u8 0, s8 1
  const uint32_t d = kind == kTcS8 ? 2u : 1u;
  const uint32_t ab = kind == kTcF16 ? 0u : 1u;
  return (d << 4) | (ab << 7) | (ab << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// MN-major operand in the 128-byte swizzle: 64 elements of M or N by 8 of K
// per 1024-byte atom, next 8 of K 1024 bytes on, next 64 of M or N 8192 bytes
// on (64 rows of K per stage).
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <int CG, bool I8>
__device__ __forceinline__ void umma_issue(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
#define FWB_MMA(group, kind)                                                       \
  asm volatile(                                                                    \
      "{\n\t.reg .pred p;\n\t"                                                     \
      "setp.ne.b32 p, %4, 0;\n\t"                                                  \
      "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), \
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate))
  if constexpr (CG == 2 && I8)
    FWB_MMA("2", "i8");
  else if constexpr (CG == 2)
    FWB_MMA("2", "f16");
  else if constexpr (I8)
    FWB_MMA("1", "i8");
  else
    FWB_MMA("1", "f16");
#undef FWB_MMA
}

// Arrives, once the products issued so far are complete, on the barrier at
// this offset in every CTA of the group.
template <int CG>
__device__ __forceinline__ void umma_commit_group(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    umma_commit(bar);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Address, in the cluster's window, of `p`'s place in CTA `rank`.
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// Tile load into this CTA that counts on a barrier given by its address in
// the cluster's window (the pair's first CTA holds it).
template <int CG>
__device__ __forceinline__ void tma_load_group(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void mbar_arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Where a tile is and how many stages of K it has.
struct TcTile {
  int m0, n0;  // first row of M, first row of N
  int ak, bk;  // start along K, in elements, of A and of B
  int nk;      // stages of K (0: the accumulator is not written)
  int rows;    // rows of A that matter, at most 128 (operators with A_BOX < 128)
  int kind;    // which of two products (operators with TWO)
};

// Division of n < 2^31 by a divisor met again and again: a multiplication and
// a shift (Granlund and Montgomery, Division by Invariant Integers using
// Multiplication, 1994).  The multiplier is floor(2^32 (2^s - d) / d) + 1 for the first
// 2^s >= d; n < 2^31 leaves room for one more, so the quotient may be a rounded
// one (a 64-bit integer division here costs a short kernel half a microsecond).
struct FastDiv {
  uint32_t d, mul, shift;
  __device__ __forceinline__ void set(int divisor) {
    d = (uint32_t)max(divisor, 1);
    shift = d > 1 ? 32 - __clz((int)d - 1) : 0;
    mul = (uint32_t)(4294967296.0 * (double)((1u << shift) - d) / (double)d) + 1u;
  }
  __device__ __forceinline__ int div(int n) const {
    return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift);
  }
};

// Order of mt x nt tiles: blocks of `group` rows of tiles, the row fastest
// inside one, so that the tiles in flight share their operands in L2.
struct TileOrder {
  int mt, nt, group;
  FastDiv by_block, by_group, by_tail;
  __device__ __forceinline__ void set(int m_tiles, int n_tiles, int group_) {
    mt = m_tiles, nt = n_tiles, group = group_;
    by_block.set(group * nt);
    by_group.set(group);
    by_tail.set(mt % group);
  }
  __device__ __forceinline__ int count() const { return mt * nt; }
  __device__ __forceinline__ void get(int w, int* m, int* n) const {
    const int g = by_block.div(w), r = w - g * group * nt;
    const bool tail = (g + 1) * group > mt;
    *n = tail ? by_tail.div(r) : by_group.div(r);
    *m = g * group + r - *n * (tail ? (int)by_tail.d : group);
  }
};

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}

// What an epilogue warp works on: 32 rows of the accumulator from row r0 of
// the tile, and a share of its columns.
struct TcPart {
  uint32_t taddr;  // TMEM address of the warp's rows, column 0
  int row;         // first row of the warp in the tile
  int lane;
  int share;       // which share of the columns
  uint8_t* smem;   // EPI_BYTES / EW of scratch
};

// P is the operator: static members CG, KIND, A_MN, B_MN, BN, STAGES, KC (0:
// all of K at once), EW, EPI_BYTES and
//   TWO              tiles of kind 1 are another product, of A2 (A_MN2) and B2
//   A_BOX            rows per load of A: 128; fewer where tiles need not be
//                    whole, and A2 then is A in boxes of that many rows
//   AHEAD            loads of A brought into L2 before the previous kernel's
//                    results are waited for (0: none; A is not written by it,
//                    or the copy in L2 is brought up to date by the write)
//   struct Plan, plan(args, group, groups, &plan)  what the tiles of a CTA
//                    group follow from, worked out once per CTA
//   get(args, plan, i, &tile)  i-th tile of the CTA group; false: done
//   struct State     what an epilogue thread keeps over a tile's parts
//   begin(args, plan, tile, part, state)  before the tile's products are done:
//                    loads that the epilogue would wait for
//   epilogue<LOST>(args, plan, tile, part, state, k, parts, done): part k of
//                    the tile's `parts`; done() hands the accumulator back once
//                    its last column has been read.  LOST: there is no
//                    accumulator, a wait gave up; what the tile would have
//                    given is written as NaN (nothing, where the operator
//                    tells by its own status word).
template <class P>
struct GemmSmem {
  static constexpr uint32_t kBRows = P::BN / P::CG;
  static constexpr uint32_t kBBytes = kBRows * kGemmRowBytes;
  static constexpr uint32_t kStage = kGemmABytes + kBBytes;
  static constexpr uint32_t kBytes = 1024 + P::STAGES * kStage + P::EPI_BYTES + 256;
  static constexpr int kThreads = 64 + 32 * P::EW;
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

template <class P>
__global__ void __launch_bounds__(GemmSmem<P>::kThreads, 1)
    fw_tc_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                      const __grid_constant__ CUtensorMap tm_a2, const __grid_constant__ CUtensorMap tm_b2,
                      const __grid_constant__ typename P::Args a, uint64_t wait_ns) {
  constexpr int S = P::STAGES, CG = P::CG;
  constexpr uint32_t kBBytes = GemmSmem<P>::kBBytes;
  constexpr bool kI8 = P::KIND == kTcS8;
  constexpr uint32_t kTmemCols = 2 * P::BN < 32 ? 32 : 2 * P::BN;
  constexpr int kStep = kI8 ? 128 : 64;  // elements of K per stage
  extern __shared__ uint8_t gemm_smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(gemm_smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* smA = base;
  uint8_t* smB = base + S * kGemmABytes;
  uint8_t* smE = smB + S * kBBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smE + P::EPI_BYTES);
  uint64_t* full = bars;           // [S] TMA -> MMA, in the first CTA, for both
  uint64_t* empty = bars + S;      // [S] MMA -> TMA, in each CTA
  uint64_t* tfull = bars + 2 * S;  // [2] MMA -> epilogue, in each CTA
  uint64_t* tempty = tfull + 2;    // [2] epilogue -> MMA, in the first CTA, from both
  uint64_t* drain = tempty + 2;    // abort path
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cluster_rank() : 0;
  const int group = (int)blockIdx.x / CG, groups = (int)gridDim.x / CG;
  __shared__ typename P::Plan plan;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], P::EW * CG);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (threadIdx.x == 32 * 3) {
    tma_prefetch_map(&tm_a);
    tma_prefetch_map(&tm_b);
    if constexpr (P::TWO || P::A_BOX < 128) tma_prefetch_map(&tm_a2);
    if constexpr (P::TWO) tma_prefetch_map(&tm_b2);
  }
  if constexpr (P::AHEAD > 0) {
    if (threadIdx.x == 32 * 2) {
      typename P::Plan early;
      P::plan(a, group, groups, &early);
      TcTile t;
      if (P::get(a, early, 0, &t))
        for (int kb = 0; kb < min(t.nk, P::AHEAD); ++kb)
          for (int i = 0; i < t.rows; i += P::A_BOX) tma_prefetch_2d(&tm_a2, t.ak + kb * kStep, t.m0 + i);
    }
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(kTmemCols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(kTmemCols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // the pair's barriers exist
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_prior_kernel();  // every thread: what follows reads its results
  allow_dependent_launch();
  if (threadIdx.x == 0) P::plan(a, group, groups, &plan);
  __syncthreads();

  uint32_t issued = 0u, issued_par = 0u;  // stages with a copy issued, and its parity
  bool mma_any = false;
  TcTile t;

  if (warp == 0) {
    uint32_t s = 0, ph = 0;
    for (int it = 0; P::get(a, plan, it, &t); ++it) {
      const int m = t.m0 + rank * kGemmBM, n = t.n0 + rank * (P::BN / CG);
      const CUtensorMap* ma = P::TWO && t.kind ? &tm_a2 : &tm_a;
      const CUtensorMap* mb = P::TWO && t.kind ? &tm_b2 : &tm_b;
      const bool a_mn = P::TWO && t.kind ? P::A_MN2 : P::A_MN;
      const uint32_t bytes =
          P::A_BOX == 128 ? kGemmABytes : (uint32_t)((t.rows + P::A_BOX - 1) / P::A_BOX * P::A_BOX * kGemmRowBytes);
      for (int kb = 0; kb < t.nk; ++kb) {
        if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag, a.status, wait_ns)) goto done;
        if (lane == 0) {
          if (rank == 0) mbar_expect_tx(&full[s], CG * (bytes + kBBytes));
          const uint32_t bar = CG == 2 ? in_cta(&full[s], 0) : smem_u32(&full[s]);
          const int ka = t.ak + kb * kStep, kbb = t.bk + kb * kStep;
          if (a_mn) {
#pragma unroll
            for (int i = 0; i < kGemmBM / 64; ++i)
              tma_load_group<CG>(smA + s * kGemmABytes + i * 8192, ma, m + 64 * i, ka, bar);
          } else if (P::A_BOX == 128 || t.rows == 128) {
            tma_load_group<CG>(smA + s * kGemmABytes, ma, ka, m, bar);
          } else {
            for (int i = 0; i < t.rows; i += P::A_BOX)
              tma_load_group<CG>(smA + s * kGemmABytes + i * kGemmRowBytes, &tm_a2, ka, m + i, bar);
          }
          if constexpr (P::B_MN) {
#pragma unroll
            for (int i = 0; i < P::BN / CG / 64; ++i)
              tma_load_group<CG>(smB + s * kBBytes + i * 8192, mb, n + 64 * i, kbb, bar);
          } else {
            tma_load_group<CG>(smB + s * kBBytes, mb, kbb, n, bar);
          }
        }
        issued |= 1u << s;
        issued_par = (issued_par & ~(1u << s)) | (ph << s);
        __syncwarp();
        if (++s == S) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    uint32_t s = 0, ph = 0, acc = 0, aph = 0;
    if (gives_up(wait_ns, abort_flag, a.status)) goto done;
    if (rank == 0) {
      for (int it = 0; P::get(a, plan, it, &t); ++it) {
        const bool a_mn = P::TWO && t.kind ? P::A_MN2 : P::A_MN;
        const uint32_t idesc = gemm_idesc(P::KIND, a_mn, P::B_MN, kGemmBM * CG, P::BN);
        const int kc = P::KC == 0 ? max(t.nk, 1) : P::KC;
        for (int k0 = 0; k0 < max(t.nk, 1); k0 += kc) {
          if (!mbar_wait(&tempty[acc], aph ^ 1u, abort_flag, a.status, wait_ns)) goto done;
          tc_fence_after();
          const uint32_t d = tmem + acc * P::BN;
          for (int kb = k0; kb < min(k0 + kc, t.nk); ++kb) {
            if (!mbar_wait(&full[s], ph, abort_flag, a.status, wait_ns)) goto done;
            tc_fence_after();
            if (lane == 0) {
              const uint32_t sa = smem_u32(smA + s * kGemmABytes);
              const uint32_t sb = smem_u32(smB + s * kBBytes);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                // 16 rows of K (MN-major) or 32 bytes of K (K-major) further on
                const uint64_t da = a_mn ? umma_desc_mn(sa + 2048 * k) : umma_desc_sw128(sa + 32 * k);
                const uint64_t db = P::B_MN ? umma_desc_mn(sb + 2048 * k) : umma_desc_sw128(sb + 32 * k);
                umma_issue<CG, kI8>(d, da, db, idesc, (kb != k0 || k != 0) ? 1u : 0u);
              }
              umma_commit_group<CG>(&empty[s]);
            }
            mma_any = true;
            __syncwarp();
            if (++s == S) {
              s = 0;
              ph ^= 1u;
            }
          }
          if (lane == 0) umma_commit_group<CG>(&tfull[acc]);
          mma_any = true;
          __syncwarp();
          if (++acc == 2) {
            acc = 0;
            aph ^= 1u;
          }
        }
      }
    }
  } else {
    const int quad = warp & 3;  // TMEM lanes this warp may read
    uint32_t acc = 0, aph = 0;
    TcPart part;
    part.row = rank * kGemmBM + quad * 32;
    part.lane = lane;
    part.share = (warp - 2) >> 2;
    part.smem = smE + (warp - 2) * (P::EPI_BYTES / P::EW);
    int it = 0;
    for (; P::get(a, plan, it, &t); ++it) {
      const int parts = P::KC == 0 ? 1 : max((t.nk + P::KC - 1) / (P::KC == 0 ? 1 : P::KC), 1);
      typename P::State state{};
      P::begin(a, plan, t, part, state);
      for (int k = 0; k < parts; ++k) {
        if (!mbar_wait(&tfull[acc], aph, abort_flag, a.status, wait_ns)) goto lost;
        tc_fence_after();
        part.taddr = tmem + (uint32_t)((quad * 32) << 16) + acc * P::BN;
        const uint32_t te = CG == 2 ? in_cta(&tempty[acc], 0) : smem_u32(&tempty[acc]);
        P::template epilogue<false>(a, plan, t, part, state, k, parts, [te, lane] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_at(te);
        });
        if (++acc == 2) {
          acc = 0;
          aph ^= 1u;
        }
      }
    }
    goto done;
  lost:  // this tile and those behind it
    for (; P::get(a, plan, it, &t); ++it) {
      typename P::State state{};
      P::begin(a, plan, t, part, state);
      P::template epilogue<true>(a, plan, t, part, state, 0, 1, [] {});
    }
  }
done:
  // Every role has left its loop: one that had finished before another gave up
  // may still have copies or products in flight.
  __syncwarp();
  __syncthreads();
  if (*abort_flag && lane == 0) {
    if (warp == 0) {
      if (rank == 0)
        for (int st = 0; st < S; ++st)
          if (issued & (1u << st)) mbar_drain(&full[st], (issued_par >> st) & 1u);
      // the pair's other copies count on the first CTA's barriers: time for them to land
      const uint64_t t0 = global_ns();
      for (int i = 0; i < (1 << 20) && global_ns() - t0 < 1000000ull; ++i) {
      }
    } else if (warp == 1 && mma_any) {
      umma_commit_group<CG>(drain);
      mbar_drain(drain, 0u);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // nobody reads or signals the other's shared memory any more
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// The warp's 32 x 32 block of fp32 values, one row per thread, turned through
// shared memory and stored as rows: 16 bytes per lane where the rows are
// aligned (`vec`), else one element per lane.  row_ptr(i) is where column 0 of
// the block's row i goes, or NULL.
template <class RowPtr>
__device__ __forceinline__ void store_block(float* sm, const float (&v)[32], int lane, int cols, bool vec,
                                            RowPtr row_ptr) {
  constexpr int V = 4, LANES = 32 / V, ROWS = 32 / LANES;  // lanes per row, rows per step
#pragma unroll
  for (int i = 0; i < 32; ++i) sm[lane * 33 + i] = v[i];
  __syncwarp();
  if (vec) {
    const int c = (lane % LANES) * V;
#pragma unroll
    for (int i0 = 0; i0 < 32; i0 += ROWS) {
      const int i = i0 + lane / LANES;
      float* p = row_ptr(i);
      const float* x = sm + i * 33 + c;
      if (p && c < cols) *reinterpret_cast<float4*>(p + c) = make_float4(x[0], x[1], x[2], x[3]);  // cols: a multiple of V
    }
  } else {
#pragma unroll 8
    for (int i = 0; i < 32; ++i) {
      float* p = row_ptr(i);
      if (p && lane < cols) p[lane] = sm[i * 33 + lane];
    }
  }
  __syncwarp();
}

// A warp's 32 x COLS block of 16-bit values: staged one row per thread, then
// stored row by row.  Rows may start anywhere: the stores are the 16-byte
// slots of the destination, single elements only at a segment's two ends (32
// lanes of 2 bytes each would write parts of sectors, at a fifth of the rate).
template <int COLS>
constexpr int kStageWords = COLS / 2 + 1;  // 32-bit words of a row, and one against bank conflicts
template <int COLS>
constexpr uint32_t kStageBytes = 32 * kStageWords<COLS> * 4;

template <class T, int COLS>
__device__ __forceinline__ void stage_block(uint32_t* sm, const float (&v)[32], int lane, int c) {
  static_assert(sizeof(T) == 2, "16-bit types");
#pragma unroll
  for (int i = 0; i < 16; ++i)
    sm[lane * kStageWords<COLS> + c / 2 + i] = pack2<T>(v[2 * i], v[2 * i + 1]);
}

// `cols` columns of every row, a lane per slot; row_ptr(i) is where column 0
// of row i goes, or NULL.
template <class T, int COLS, class RowPtr>
__device__ __forceinline__ void store_staged(const uint32_t* sm, int lane, int cols, RowPtr row_ptr) {
  __syncwarp();
  constexpr int LANES = COLS / 8;
  const int k = lane % LANES;
#pragma unroll 4
  for (int i0 = 0; i0 < 32; i0 += 32 / LANES) {
    const int i = i0 + lane / LANES;
    unsigned short* p = reinterpret_cast<unsigned short*>(row_ptr(i));
    const uint32_t* row = sm + i * kStageWords<COLS>;
    // elements before the first slot, slots, elements behind the last
    const int head = min((int)(-(reinterpret_cast<uintptr_t>(p) >> 1) & 7u), cols);
    const int whole = (cols - head) >> 3, tail = head + whole * 8;
    if (p && k < whole) {
      const int e0 = head + k * 8;
      const uint32_t* w = row + (e0 >> 1);
      uint4 u = make_uint4(w[0], w[1], w[2], w[3]);
      if (head & 1) {
        const uint32_t last = w[4];
        u = make_uint4(__funnelshift_r(u.x, u.y, 16), __funnelshift_r(u.y, u.z, 16), __funnelshift_r(u.z, u.w, 16),
                       __funnelshift_r(u.w, last, 16));
      }
      *reinterpret_cast<uint4*>(p + e0) = u;
    }
#pragma unroll
    for (int j = k; j < 16; j += LANES) {  // 0..7: head, 8..15: tail
      const int e = j < 8 ? j : tail + j - 8;
      if (p && e < (j < 8 ? head : cols)) p[e] = (unsigned short)(row[e >> 1] >> (16 * (e & 1)));
    }
  }
  __syncwarp();
}

// ------------------------------------------------------------------- host
typedef CUresult (*TcEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline TcEncodeFn tc_encode() {
  static std::atomic<TcEncodeFn> fn{nullptr};
  TcEncodeFn f = fn.load(std::memory_order_acquire);
  if (!f) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess) {
      f = reinterpret_cast<TcEncodeFn>(p);
      fn.store(f, std::memory_order_release);
    }
  }
  return f;
}

// Row-major matrix [rows, cols] with row stride ld (elements) in tiles of
// 128 bytes x box_rows; elements outside read as zero.
inline bool tc_map(CUtensorMap* m, TcKind kind, const void* ptr, int64_t rows, int64_t cols, int64_t ld,
                   int box_rows) {
  TcEncodeFn fn = tc_encode();
  if (!fn) return false;
  const int es = kind == kTcS8 ? 1 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * es};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  const CUtensorMapDataType dt = kind == kTcS8   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : kind == kTcF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  auto encode = [&] {
    return fn(m, dt, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (encode()) return true;
  // a host thread that has not used the device yet has no context current
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess && encode();
}

// At most one CTA per SM; `max_tiles` bounds the grid where the tile count is
// known on the device only.  A programmatic dependent of the kernel before it.
template <class P>
cudaError_t launch_gemm(const CUtensorMap& ma, const CUtensorMap& mb, const typename P::Args& a, int64_t max_tiles,
                        cudaStream_t st, const CUtensorMap* ma2 = nullptr, const CUtensorMap* mb2 = nullptr) {
  static std::atomic<bool> attr_set[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kMaxDevices || !attr_set[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(fw_tc_gemm_kernel<P>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)GemmSmem<P>::kBytes);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) attr_set[dev].store(true, std::memory_order_release);
  }
  int64_t grid = max_tiles * P::CG;
  const int64_t sms = sm_count() / P::CG * P::CG;
  if (grid > sms) grid = sms;
  return launch_dependent(fw_tc_gemm_kernel<P>, grid, GemmSmem<P>::kThreads, GemmSmem<P>::kBytes, P::CG, st, ma, mb,
                          ma2 ? *ma2 : ma, mb2 ? *mb2 : mb, a, tc_wait_ns());
}

}  // namespace
}  // namespace fwb200
