// Matrix product on the tensor cores with the epilogue of the operator that
// uses it: the loop shared by the cross-entropy kernels and the 8-bit output
// layer.
//
// One CTA per SM (persistent), 6 warps, as in the fused LM-head kernel:
//   warp 0       TMA producer, kGemmStages stages of a 128 x 128-byte A tile
//                and a BN x 128-byte B tile (128-byte swizzle);
//   warp 1       TMEM allocation, MMA issuer: four tcgen05.mma (32 bytes of
//                K each) per stage into one of two BN-column accumulators;
//   warps 2..5   epilogue, one accumulator row per thread.
// The two accumulators let the epilogue of a tile run under the next tile's
// products.  An operand is either K-major (its rows run along K, 128 bytes of
// K per stage) or MN-major (its rows run along M or N; the stage then holds
// 64 rows of K of as many 64-element column groups as the tile needs).
//
// Every wait is bounded; on a timeout all roles leave their loops, the copies
// and products in flight are waited for (bounded) and TMEM is released, as in
// the fused LM-head kernel.
#pragma once

#include "fw_host.cuh"
#include "fw_tc_ptx.cuh"

namespace fwb200 {
namespace {

constexpr int kGemmBM = 128;
constexpr int kGemmRowBytes = 128;  // bytes of K per stage (K-major) = one swizzle row
constexpr int kGemmThreads = 192;
constexpr uint32_t kGemmABytes = kGemmBM * kGemmRowBytes;

enum TcKind { kTcBf16, kTcF16, kTcS8 };

__host__ __device__ constexpr uint32_t gemm_idesc(TcKind kind, bool a_mn, bool b_mn, int bn) {
  // accumulator: fp32 (1) or s32 (2); operands: f16 0, bf16 1 / u8 0, s8 1
  const uint32_t d = kind == kTcS8 ? 2u : 1u;
  const uint32_t ab = kind == kTcF16 ? 0u : 1u;
  return (d << 4) | (ab << 7) | (ab << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(kGemmBM >> 4) << 24);
}

// MN-major operand in the 128-byte swizzle: 64 elements of M or N by 8 of K
// per 1024-byte atom, next 8 of K 1024 bytes on, next 64 of M or N 8192 bytes
// on (64 rows of K per stage).
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <bool I8>
__device__ __forceinline__ void umma_issue(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  if constexpr (I8)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
  else
    umma_bf16(tmem_d, adesc, bdesc, idesc, accumulate);
}

// Where a tile is and how many stages of K it has.
struct TcTile {
  int m0, n0;  // first row of M, first row of N
  int ak, bk;  // start along K, in elements, of A and of B
  int nk;      // stages of K (0: the accumulator is not written)
};

// P is the operator: static members KIND, A_MN, B_MN, BN, STAGES, smem for its epilogue
// (EPI_BYTES), and
//   tiles(args)              number of tiles (read from device memory where
//                            it depends on data)
//   tile(args, w)            tile w
//   epilogue(args, tile, acc_addr, quad, lane, has, smem, done)
// `done()` hands the accumulator back once its last column has been read.
template <class P>
struct GemmSmem {
  static constexpr uint32_t kBBytes = P::BN * kGemmRowBytes;
  static constexpr uint32_t kStage = kGemmABytes + kBBytes;
  static constexpr uint32_t kBytes = 1024 + P::STAGES * kStage + P::EPI_BYTES + 256;
};

template <class P>
__global__ void __launch_bounds__(kGemmThreads, 1)
    fw_tc_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                      const __grid_constant__ typename P::Args a) {
  constexpr int S = P::STAGES;
  constexpr uint32_t kBBytes = GemmSmem<P>::kBBytes;
  constexpr bool kI8 = P::KIND == kTcS8;
  constexpr uint32_t kTmemCols = 2 * P::BN < 32 ? 32 : 2 * P::BN;
  constexpr uint32_t kIdesc = gemm_idesc(P::KIND, P::A_MN, P::B_MN, P::BN);
  extern __shared__ uint8_t gemm_smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(gemm_smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* smA = base;
  uint8_t* smB = base + S * kGemmABytes;
  uint8_t* smE = smB + S * kBBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smE + P::EPI_BYTES);
  uint64_t* full = bars;           // [S] TMA -> MMA
  uint64_t* empty = bars + S;      // [S] MMA -> TMA
  uint64_t* tfull = bars + 2 * S;  // [2] MMA -> epilogue
  uint64_t* tempty = tfull + 2;    // [2] epilogue -> MMA
  uint64_t* drain = tempty + 2;    // abort path
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 4 * 32);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int ntiles = P::tiles(a);
  uint32_t issued = 0u, issued_par = 0u;  // stages with a copy issued, and its parity
  bool mma_any = false;

  if (warp == 0) {
    uint32_t s = 0, ph = 0;
    for (int w = blockIdx.x; w < ntiles; w += gridDim.x) {
      const TcTile t = P::tile(a, w);
      for (int kb = 0; kb < t.nk; ++kb) {
        if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag, a.status)) goto done;
        if (lane == 0) {
          mbar_expect_tx(&full[s], kGemmABytes + kBBytes);
          constexpr int kStep = kI8 ? 128 : 64;  // elements of K per stage
          const int ka = t.ak + kb * kStep, kbb = t.bk + kb * kStep;
          if constexpr (P::A_MN) {
#pragma unroll
            for (int i = 0; i < kGemmBM / 64; ++i)
              tma_load_2d(smA + s * kGemmABytes + i * 8192, &tm_a, t.m0 + 64 * i, ka, &full[s]);
          } else {
            tma_load_2d(smA + s * kGemmABytes, &tm_a, ka, t.m0, &full[s]);
          }
          if constexpr (P::B_MN) {
#pragma unroll
            for (int i = 0; i < P::BN / 64; ++i)
              tma_load_2d(smB + s * kBBytes + i * 8192, &tm_b, t.n0 + 64 * i, kbb, &full[s]);
          } else {
            tma_load_2d(smB + s * kBBytes, &tm_b, kbb, t.n0, &full[s]);
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
    for (int w = blockIdx.x; w < ntiles; w += gridDim.x) {
      const TcTile t = P::tile(a, w);
      if (!mbar_wait(&tempty[acc], aph ^ 1u, abort_flag, a.status)) goto done;
      tc_fence_after();
      const uint32_t d = tmem + acc * P::BN;
      for (int kb = 0; kb < t.nk; ++kb) {
        if (!mbar_wait(&full[s], ph, abort_flag, a.status)) goto done;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t sa = smem_u32(smA + s * kGemmABytes);
          const uint32_t sb = smem_u32(smB + s * kBBytes);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // 16 rows of K (MN-major) or 32 bytes of K (K-major) further on
            const uint64_t da = P::A_MN ? umma_desc_mn(sa + 2048 * k) : umma_desc_sw128(sa + 32 * k);
            const uint64_t db = P::B_MN ? umma_desc_mn(sb + 2048 * k) : umma_desc_sw128(sb + 32 * k);
            umma_issue<kI8>(d, da, db, kIdesc, (kb | k) != 0 ? 1u : 0u);
          }
          umma_commit(&empty[s]);
        }
        mma_any = true;
        __syncwarp();
        if (++s == S) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (lane == 0) umma_commit(&tfull[acc]);
      mma_any = true;
      __syncwarp();
      if (++acc == 2) {
        acc = 0;
        aph ^= 1u;
      }
    }
  } else {
    const int quad = warp & 3;  // TMEM lanes this warp may read
    uint32_t acc = 0, aph = 0;
    for (int w = blockIdx.x; w < ntiles; w += gridDim.x) {
      const TcTile t = P::tile(a, w);
      if (!mbar_wait(&tfull[acc], aph, abort_flag, a.status)) goto done;
      tc_fence_after();
      const uint32_t addr = tmem + (uint32_t)((quad * 32) << 16) + acc * P::BN;
      uint64_t* te = &tempty[acc];
      P::epilogue(a, t, addr, quad, lane, smE + (warp - 2) * (P::EPI_BYTES / 4), [te] {
        tc_fence_before();
        mbar_arrive(te);
      });
      if (++acc == 2) {
        acc = 0;
        aph ^= 1u;
      }
    }
  }
done:
  __syncwarp();
  if (*abort_flag && lane == 0) {
    if (warp == 0) {
      for (int st = 0; st < S; ++st)
        if (issued & (1u << st)) mbar_drain(&full[st], (issued_par >> st) & 1u);
    } else if (warp == 1 && mma_any) {
      umma_commit(drain);
      mbar_drain(drain, 0u);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
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
  return fn(m, dt, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// At most one CTA per SM; `max_tiles` bounds the grid where the tile count is
// known on the device only.
template <class P>
cudaError_t launch_gemm(const CUtensorMap& ma, const CUtensorMap& mb, const typename P::Args& a, int64_t max_tiles,
                        cudaStream_t st) {
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
  const int64_t sms = sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(max_tiles < sms ? max_tiles : sms));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = GemmSmem<P>::kBytes;
  cfg.stream = st;
  return cudaLaunchKernelEx(&cfg, fw_tc_gemm_kernel<P>, ma, mb, a);
}

}  // namespace
}  // namespace fwb200
