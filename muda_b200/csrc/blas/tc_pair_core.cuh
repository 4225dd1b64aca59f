// tc_pair_core.cuh — persistent tcgen05 loop on CTA pairs, for products whose epilogue
// needs more than tc_gemm_core.cuh's store() hook.
//
// A cluster of two CTAs walks tiles of 256 x 256 (each CTA accumulates its 128 rows x 256
// columns in its own tensor memory) with k-blocks of 64 16-bit elements.  Each CTA loads
// its 128 rows of A and its 128 of B's 256 rows, so a k-block costs a CTA 32 KB of shared
// memory traffic where the single-CTA 128 x 256 loop moves 48 KB for the same MMA time.
//   warp 0      one thread issues the CTA's TMA loads; both CTAs' loads complete on the
//               even CTA's barrier of the stage;
//   warp 1      of the even CTA: one thread issues the pair's MMAs and commits stages and
//               accumulators back to both CTAs; of both: tensor-memory allocation;
//   warps 2-9   epilogue: warp w owns 32 rows (w % 4) and 128 columns ((w - 2) / 4).
// A problem may split the k-blocks of a tile into chunks of kChunk: each chunk starts a
// fresh accumulator (two alternate) and the epilogue adds the chunks in fp32 registers,
// which bounds the drift of the tensor core's truncating accumulation.
//
// The problem type P (a __grid_constant__ parameter) supplies
//   static constexpr bool kAMn;       // A MN-major (64 x 64 boxes), else K-major; B is K-major
//   static constexpr int kChunk;      // k-blocks per accumulator, 0: the whole tile
//   static constexpr int kStageBytes; // shared memory of an epilogue warp, a multiple of 1024
//   long long tiles_total;  int num_kb;
//   const CUtensorMap* map_a() / map_b();
//   void coords(long long t, int (&c)[3]) const;    // c[1], c[2]: tile row and column
//   int k_begin(const int (&c)[3]) const;           // first k-block of the tile
//   struct Tile;                                    // per-thread epilogue state
//   void begin(Tile&, c, int row, int half) const;  // before the accumulator is waited for
//   void chunk(Tile&, c, int row, int half, uint32_t taddr, uint8_t* stage) const;
//                                                   // reads a finished accumulator
//   void end(Tile&, c, int row, int half, uint8_t* stage) const;
// Waits are bounded as in tc_gemm_core.cuh: a wait that runs out marks its CTA aborted,
// counts the event, and every role leaves its loop; all threads of both CTAs then meet at
// the final cluster barrier, so no CTA leaves while the other may still reach its memory.
#pragma once

#include "blas/tc_gemm_core.cuh"

namespace mb200::tc {

constexpr int kPairThreads = 320;
constexpr int kPairEpiWarps = 8;
constexpr int kPairN = 256;

template <class P>
struct PairShape {
  static constexpr int A_STAGE = kBM * kRowBytes;           // this CTA's rows of A
  static constexpr int B_STAGE = (kPairN / 2) * kRowBytes;  // this CTA's rows of B
  static constexpr int STAGE = A_STAGE + B_STAGE;
  static constexpr int EPI = kPairEpiWarps * P::kStageBytes;
  static constexpr int BAR_BYTES = 256;
  static constexpr int LIMIT = 227 * 1024;
  static constexpr int FIT = (LIMIT - 1024 - BAR_BYTES - EPI) / STAGE;
  static constexpr int STAGES = FIT < 6 ? FIT : 6;
  static constexpr int SMEM = STAGES * STAGE + EPI + BAR_BYTES + 1024;
  static_assert(STAGES >= 3, "the ring needs three stages");
};

template <class P, int FMT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    tc_pair_kernel(const __grid_constant__ P p, unsigned int* timeouts) {
  using S = PairShape<P>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ std::uint8_t smem_raw[];
  std::uint8_t* base = reinterpret_cast<std::uint8_t*>(
      (reinterpret_cast<std::uintptr_t>(smem_raw) + 1023) & ~std::uintptr_t{1023});
  std::uint8_t* sa = base;
  std::uint8_t* sb = sa + STAGES * S::A_STAGE;
  std::uint8_t* se = sb + STAGES * S::B_STAGE;
  std::uint64_t* full = reinterpret_cast<std::uint64_t*>(se + S::EPI);  // used in the even CTA
  std::uint64_t* empty = full + STAGES;
  std::uint64_t* acc_full = empty + STAGES;
  std::uint64_t* acc_empty = acc_full + kAcc;                            // used in the even CTA
  std::uint64_t* mma_done = acc_empty + kAcc;
  std::uint32_t* tmem_slot = reinterpret_cast<std::uint32_t*>(mma_done + 1);
  volatile int* aborted = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const std::uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kPairEpiWarps);
    }
    mbar_init(mma_done, 1);
    *aborted = 0;
    mbar_fence_init();
    prefetch_tensormap(p.map_a());
    prefetch_tensormap(p.map_b());
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, kAcc * kPairN);
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // both CTAs' barriers are set before either signals the other
  tc_fence_after();
  const std::uint32_t tmem_base = *tmem_slot;
  const int num_kb = p.num_kb;
  const long long step = gridDim.x / 2;
  const long long first_tile = blockIdx.x / 2;
  constexpr int CK = P::kChunk;
  auto fail = [&]() {
    *aborted = 1;
    atomicAdd(timeouts, 1u);
  };

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer of this CTA's halves
      int stage = 0;
      std::uint32_t phase = 0;
      std::uint32_t issued_phase[STAGES];
      bool issued[STAGES];
      for (int s = 0; s < STAGES; ++s) issued[s] = false;
      bool ok = true;
      for (long long t = first_tile; ok && t < p.tiles_total && !*aborted; t += step) {
        int c[3];
        p.coords(t, c);
        const int k0 = p.k_begin(c);
        const int am = c[1] * 2 * kBM + static_cast<int>(rank) * kBM;
        const int bn = c[2] * kPairN + static_cast<int>(rank) * (kPairN / 2);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u)) {
            fail();
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * S::STAGE);
          const std::uint32_t bar = cluster_addr(&full[stage], 0);
          std::uint8_t* a = sa + stage * S::A_STAGE;
          const int k = (k0 + kb) * kBK;
          if constexpr (P::kAMn) {
#pragma unroll
            for (int j = 0; j < kBM / 64; ++j)
              tma_load_3d_pair(a + j * kMnBoxBytes, p.map_a(), am + 64 * j, k, 0, bar);
          } else {
            tma_load_3d_pair(a, p.map_a(), k, am, 0, bar);
          }
          tma_load_3d_pair(sb + stage * S::B_STAGE, p.map_b(), k, bn, 0, bar);
          issued[stage] = true;
          issued_phase[stage] = phase;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // Drain: the even CTA's barriers cover both CTAs' copies.
      if (rank == 0) {
        for (int s = 0; s < STAGES; ++s)
          if (issued[s] && !mbar_wait(&full[s], issued_phase[s])) fail();
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // ---------------- MMA issuer of the pair
      constexpr std::uint32_t idesc = f16_idesc(FMT, 2 * kBM, kPairN, P::kAMn, false);
      int stage = 0;
      std::uint32_t phase = 0;
      int acc = 0;
      std::uint32_t acc_phase = 0;
      bool ok = true;
      for (long long t = first_tile; ok && t < p.tiles_total && !*aborted; t += step) {
        for (int kb = 0; kb < num_kb; ++kb) {
          const bool first = CK == 0 ? kb == 0 : kb % (CK == 0 ? 1 : CK) == 0;
          const bool last = kb == num_kb - 1 || (CK != 0 && kb % (CK == 0 ? 1 : CK) == CK - 1);
          if (first) {
            if (!mbar_wait_cluster(&acc_empty[acc], acc_phase ^ 1u)) {
              fail();
              ok = false;
              break;
            }
            tc_fence_after();
          }
          if (!mbar_wait(&full[stage], phase)) {
            fail();
            ok = false;
            break;
          }
          tc_fence_after();
          const std::uint32_t d_tmem = tmem_base + static_cast<std::uint32_t>(acc * kPairN);
          const std::uint32_t a0 = smem_addr(sa + stage * S::A_STAGE);
          const std::uint32_t b0 = smem_addr(sb + stage * S::B_STAGE);
#pragma unroll
          for (int k = 0; k < kRowBytes / kStepBytes; ++k)
            mma_f16_pair(d_tmem, operand_desc<P::kAMn>(a0, k), operand_desc<false>(b0, k), idesc,
                         (first && k == 0) ? 0u : 1u);
          mma_commit_pair(&empty[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
          if (last) {
            mma_commit_pair(&acc_full[acc]);
            if (++acc == kAcc) {
              acc = 0;
              acc_phase ^= 1u;
            }
          }
        }
      }
      // Drain: all issued MMAs have completed before tensor memory is freed.
      mma_commit_pair(mma_done);
      if (!mbar_wait(mma_done, 0)) fail();
    }
  } else {
    // ---------------- epilogue: quarter = warp % 4, column half = (warp - 2) / 4
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    const int row = static_cast<int>(rank) * kBM + quarter * 32 + lane;  // in the 256-row tile
    std::uint8_t* stage = se + (warp - 2) * P::kStageBytes;
    const std::uint32_t t_lane = tmem_base + (static_cast<std::uint32_t>(quarter * 32) << 16) +
                                 static_cast<std::uint32_t>(half * (kPairN / 2));
    const std::uint32_t release0 = cluster_addr(&acc_empty[0], 0);
    const int chunks = CK == 0 ? 1 : (num_kb + (CK == 0 ? 1 : CK) - 1) / (CK == 0 ? 1 : CK);
    int acc = 0;
    std::uint32_t acc_phase = 0;
    bool ok = true;
    for (long long t = first_tile; ok && t < p.tiles_total && !*aborted; t += step) {
      int c[3];
      p.coords(t, c);
      typename P::Tile tile;
      p.begin(tile, c, row, half);
      for (int ch = 0; ch < chunks; ++ch) {
        if (!mbar_wait(&acc_full[acc], acc_phase)) {
          fail();
          ok = false;
          break;
        }
        tc_fence_after();
        __syncwarp();
        p.chunk(tile, c, row, half, t_lane + static_cast<std::uint32_t>(acc * kPairN), stage);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(release0 + acc * 8);
        if (++acc == kAcc) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) break;
      p.end(tile, c, row, half, stage);
    }
    bulk_wait_all();  // this thread's stores from shared memory, if any
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kAcc * kPairN);
  }
}

template <class P, int FMT>
cudaError_t launch_tc_pair(const P& p, int sms, unsigned int* timeouts, cudaStream_t stream) {
  using S = PairShape<P>;
  auto kern = tc_pair_kernel<P, FMT>;
  static std::atomic<unsigned long long> attr_set{0};  // per device, as launch_tc_gemm
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return cudaErrorInvalidDevice;
  const unsigned long long bit = 1ull << (dev & 63);
  if ((attr_set.load(std::memory_order_acquire) & bit) == 0) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return e;
    attr_set.fetch_or(bit, std::memory_order_release);
  }
  const long long pairs = p.tiles_total < sms / 2 ? p.tiles_total : sms / 2;
  if (pairs <= 0) return cudaSuccess;
  kern<<<static_cast<unsigned>(2 * pairs), kPairThreads, S::SMEM, stream>>>(p, timeouts);
  return cudaGetLastError();
}

}  // namespace mb200::tc
