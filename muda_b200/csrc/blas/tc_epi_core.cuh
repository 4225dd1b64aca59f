// tc_epi_core.cuh — persistent tcgen05 loop for products whose epilogue needs more than
// tc_gemm_core.cuh's store() hook: 16-bit operands, k-blocks of 64 elements.
//
// Three forms, tile_n a multiple of 32 up to 256 that is chosen at run time.  kPair: a
// cluster of two CTAs walks tiles of 256 x tile_n; each CTA accumulates its 128 rows in its
// own tensor memory and loads its 128 rows of A and half of B's rows, so a k-block of a
// 256-wide tile costs a CTA 32 KB of loads where a single CTA's 128 x 256 tile costs 48 KB
// for the same MMA time.  kTall as well: tiles of 512 x tile_n, two stacked 256-row halves
// that fill tensor memory, 24 KB per CTA and MMA time; the halves drain in turn before the
// next tile's MMAs, so it is for long K.  Otherwise single CTAs walk tiles of 128 x tile_n:
// for few rows of one operand, where streaming the other is what takes the time.
//   warp 0      issues the CTA's TMA loads (a pair's complete on the even CTA's barriers);
//   warp 1      issues the MMAs (a pair's: the even CTA) and commits stages and
//               accumulators back; allocates tensor memory;
//   warps 2-9   epilogue: warp w owns 32 rows (w % 4) and half of the columns ((w - 2) / 4).
// A problem may split the k-blocks of a tile into chunks of kChunk: each chunk starts a
// fresh accumulator (two alternate) and the epilogue adds the chunks in fp32 registers,
// which bounds the drift of the tensor core's truncating accumulation.
//
// The producer and the issuer run as whole warps with one elected lane issuing: in
// single-lane code every tcgen05 and TMA operand crosses into uniform registers, and the
// issue loop took 666 clocks a k-block (measured with and without loads) against the
// MMAs' 512; warp-uniform it takes 538.
//
// The problem type P (a __grid_constant__ parameter) supplies
//   static constexpr bool kPair, kTall;   // kTall implies kPair and kChunk 0
//   static constexpr bool kAMn;       // A MN-major (64 x 64 boxes), else K-major; B is K-major
//   static constexpr int kChunk;      // k-blocks per accumulator, 0: the whole tile
//   static constexpr int kMaxN;       // most of tile_n, 256 or less: less leaves room for stages
//   static constexpr int kStageBytes; // shared memory of an epilogue warp, a multiple of 1024
//   long long tiles_total;  int num_kb;  int tile_n;
//   const CUtensorMap* map_a() / map_b();           // K-major boxes: 64 x 128 rows of A,
//                                                   // 64 x tile_n (pair: tile_n / 2) of B
//   void coords(long long t, int (&c)[3]) const;    // c[1], c[2]: tile row and column
//   int k_begin(const int (&c)[3]) const;           // first k-block of the tile
//   bool next_early() const;                        // whether the next kernel may start once a
//                                                   // CTA's loads are out
//   struct Tile;                                    // per-thread epilogue state
//   void begin(Tile&, c, int row, int half) const;  // before the accumulator is waited for
//   void chunk(Tile&, c, int row, int half, uint32_t taddr, bool first, uint8_t* stage) const;
//                                                   // reads a finished accumulator
//   void end(Tile&, c, int row, int half, uint8_t* stage) const;
// `row` is the row in the tile, `half` the column half, taddr the half's first column.  A
// tall tile calls chunk() twice, for its upper and then its lower 256 rows.
// Waits are bounded as in tc_gemm_core.cuh: a wait that runs out marks its CTA aborted,
// counts the event, and every role leaves its loop, whole warps at a time (the warp votes on
// its clocks and on the mark: tcgen05.ld and the stores need it together); all threads (of
// both CTAs) then meet at a final barrier, so no CTA leaves while the other may still reach
// its memory.
#pragma once

#include "blas/tc_gemm_core.cuh"

namespace mb200::tc {

constexpr int kEpiThreads = 320;
constexpr int kEpiWarps = 8;
constexpr int kEpiN = 256;  // columns of an accumulator

template <class P>
struct EpiShape {
  static constexpr int kCtas = P::kPair ? 2 : 1;
  static constexpr int kHalves = P::kTall ? 2 : 1;
  static constexpr int A_HALF = kBM * kRowBytes;
  static constexpr int A_STAGE = kHalves * A_HALF;           // this CTA's rows of A
  static constexpr int B_STAGE = P::kMaxN / kCtas * kRowBytes;  // and of B
  static constexpr int STAGE = A_STAGE + B_STAGE;
  static constexpr int EPI = kEpiWarps * P::kStageBytes;
  static constexpr int BAR_BYTES = 256;
  static constexpr int LIMIT = 227 * 1024;
  static constexpr int FIT = (LIMIT - 1024 - BAR_BYTES - EPI) / STAGE;
  static constexpr int STAGES = FIT < 6 ? FIT : 6;
  static constexpr int SMEM = STAGES * STAGE + EPI + BAR_BYTES + 1024;
  static_assert(STAGES >= 3, "the ring needs three stages");
  static_assert(!P::kTall || (P::kPair && P::kChunk == 0), "a tall tile is one chunk of a pair");
};

template <class P, int FMT>
__device__ __forceinline__ void epi_body(const P& p, unsigned int* timeouts) {
  using S = EpiShape<P>;
  constexpr int STAGES = S::STAGES;
  constexpr bool kPair = P::kPair;
  constexpr int CK = P::kChunk;
  extern __shared__ std::uint8_t smem_raw[];
  std::uint8_t* base = reinterpret_cast<std::uint8_t*>(
      (reinterpret_cast<std::uintptr_t>(smem_raw) + 1023) & ~std::uintptr_t{1023});
  std::uint8_t* sa = base;
  std::uint8_t* sb = sa + STAGES * S::A_STAGE;
  std::uint8_t* se = sb + STAGES * S::B_STAGE;
  std::uint64_t* full = reinterpret_cast<std::uint64_t*>(se + S::EPI);  // pair: the even CTA's
  std::uint64_t* empty = full + STAGES;
  std::uint64_t* acc_full = empty + STAGES;
  std::uint64_t* acc_empty = acc_full + kAcc;                            // pair: the even CTA's
  std::uint64_t* mma_done = acc_empty + kAcc;
  std::uint32_t* tmem_slot = reinterpret_cast<std::uint32_t*>(mma_done + 1);
  volatile int* aborted = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const std::uint32_t rank = kPair ? cluster_rank() : 0u;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], S::kCtas * kEpiWarps);
    }
    mbar_init(mma_done, 1);
    *aborted = 0;
    mbar_fence_init();
    prefetch_tensormap(p.map_a());
    prefetch_tensormap(p.map_b());
  }
  __syncwarp();
  if (warp == 1) {
    if constexpr (kPair)
      tmem_alloc_pair(tmem_slot, kAcc * kEpiN);
    else
      tmem_alloc(tmem_slot, kAcc * kEpiN);
  }
  tc_fence_before();
  if constexpr (kPair)
    cluster_sync();  // both CTAs' barriers are set before either signals the other
  else
    __syncthreads();
  tc_fence_after();
  const std::uint32_t tmem_base = *tmem_slot;
  grid_wait_previous();
  const int num_kb = p.num_kb;
  const int tile_n = p.tile_n;
  const long long step = gridDim.x / S::kCtas;
  const long long first_tile = blockIdx.x / S::kCtas;
  auto fail = [&]() {
    *aborted = 1;
    atomicAdd(timeouts, 1u);
  };
  // a whole warp leaves or stays: its lanes could read the flag, or the clock, differently
  auto stopped = [&]() { return __any_sync(0xffffffffu, *aborted != 0) != 0; };

  if (warp == 0) {
    // ---------------- TMA producer of this CTA's rows
    const std::uint32_t full0 = kPair ? cluster_addr(full, 0) : smem_addr(full);
    const std::uint32_t tx =
        S::kCtas * S::A_STAGE + static_cast<std::uint32_t>(tile_n * kRowBytes);
    int stage = 0;
    std::uint32_t phase = 0;
    std::uint32_t issued = 0, issued_phase = 0;  // bit per stage
    bool ok = true;
    for (long long t = first_tile; ok && t < p.tiles_total && !stopped(); t += step) {
      int c[3];
      p.coords(t, c);
      int k = p.k_begin(c) * kBK;
      const int am = c[1] * S::kHalves * S::kCtas * kBM + static_cast<int>(rank) * kBM;
      const int bn = c[2] * tile_n + static_cast<int>(rank) * (tile_n / 2);
      for (int kb = 0; kb < num_kb; ++kb, k += kBK) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1u)) {
          if (lane == 0) fail();
          ok = false;
          break;
        }
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], tx);
          const std::uint32_t bar = full0 + static_cast<std::uint32_t>(stage) * 8;
#pragma unroll
          for (int u = 0; u < S::kHalves; ++u) {
            std::uint8_t* a = sa + stage * S::A_STAGE + u * S::A_HALF;
            const int m = am + u * 2 * kBM;
            if constexpr (P::kAMn) {
#pragma unroll
              for (int j = 0; j < kBM / 64; ++j)
                tma_load_3d_group<S::kCtas>(a + j * kMnBoxBytes, p.map_a(), m + 64 * j, k, 0, bar);
            } else {
              tma_load_3d_group<S::kCtas>(a, p.map_a(), k, m, 0, bar);
            }
          }
          tma_load_3d_group<S::kCtas>(sb + stage * S::B_STAGE, p.map_b(), k, bn, 0, bar);
        }
        __syncwarp();
        issued |= 1u << stage;
        issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (p.next_early()) grid_launch_next();
    // Drain: a pair's copies all complete on the even CTA's barriers.
    if (rank == 0) {
      for (int s = 0; s < STAGES; ++s)
        if ((issued >> s & 1u) != 0u && !mbar_wait_warp(&full[s], issued_phase >> s & 1u) &&
            lane == 0)
          fail();
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------- MMA issuer
      const std::uint32_t idesc = f16_idesc(FMT, S::kCtas * kBM, tile_n, P::kAMn, false);
      const std::uint64_t a_desc = operand_desc<P::kAMn>(smem_addr(sa), 0);
      const std::uint64_t b_desc = operand_desc<false>(smem_addr(sb), 0);
      constexpr std::uint64_t a_step = P::kAMn ? kMnStepBytes >> 4 : kStepBytes >> 4;
      int stage = 0;
      std::uint32_t phase = 0;
      int acc = 0;
      std::uint32_t acc_phase = 0;
      bool ok = true;
      for (long long t = first_tile; ok && t < p.tiles_total && !stopped(); t += step) {
        for (int kb = 0; kb < num_kb; ++kb) {
          const bool first = CK == 0 ? kb == 0 : kb % (CK == 0 ? 1 : CK) == 0;
          const bool last = kb == num_kb - 1 || (CK != 0 && kb % (CK == 0 ? 1 : CK) == CK - 1);
          if (!mbar_wait_warp(&full[stage], phase)) {
            if (lane == 0) fail();
            ok = false;
            break;
          }
          const std::uint64_t b0 = b_desc + static_cast<std::uint32_t>(stage * (S::B_STAGE >> 4));
#pragma unroll
          for (int u = 0; u < S::kHalves; ++u) {
            const int into = P::kTall ? u : acc;  // accumulator
            if (first && !mbar_wait_warp(&acc_empty[into], acc_phase ^ 1u)) {
              if (lane == 0) fail();
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
              const std::uint32_t d_tmem = tmem_base + static_cast<std::uint32_t>(into * kEpiN);
              const std::uint64_t a0 =
                  a_desc + static_cast<std::uint32_t>((stage * S::A_STAGE + u * S::A_HALF) >> 4);
#pragma unroll
              for (int k = 0; k < kRowBytes / kStepBytes; ++k)
                mma_f16_group<S::kCtas>(d_tmem, a0 + k * a_step, b0 + k * (kStepBytes >> 4), idesc,
                                        (first && k == 0) ? 0u : 1u);
              if (u == S::kHalves - 1) mma_commit_group<S::kCtas>(&empty[stage]);
              if (last) mma_commit_group<S::kCtas>(&acc_full[into]);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
          if (last && (P::kTall || ++acc == kAcc)) {
            acc = 0;
            acc_phase ^= 1u;
          }
        }
      }
      // Drain: all issued MMAs have completed before tensor memory is freed.
      if (elect_one()) mma_commit_group<S::kCtas>(mma_done);
      __syncwarp();
      if (!mbar_wait_warp(mma_done, 0) && lane == 0) fail();
    }
  } else {
    // ---------------- epilogue: quarter = warp % 4, column half = (warp - 2) / 4
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    const int row = static_cast<int>(rank) * kBM + quarter * 32 + lane;
    std::uint8_t* stage = se + (warp - 2) * P::kStageBytes;
    const std::uint32_t t_lane = tmem_base + (static_cast<std::uint32_t>(quarter * 32) << 16) +
                                 static_cast<std::uint32_t>(half * (tile_n / 2));
    const std::uint32_t release0 = kPair ? cluster_addr(acc_empty, 0) : smem_addr(acc_empty);
    const int chunks =
        CK == 0 ? S::kHalves : (num_kb + (CK == 0 ? 1 : CK) - 1) / (CK == 0 ? 1 : CK);
    int acc = 0;
    std::uint32_t acc_phase = 0;
    bool ok = true;
    for (long long t = first_tile; ok && t < p.tiles_total && !stopped(); t += step) {
      int c[3];
      p.coords(t, c);
      typename P::Tile tile;
      p.begin(tile, c, row, half);
      for (int ch = 0; ch < chunks; ++ch) {
        if (!mbar_wait_warp_idle(&acc_full[acc], acc_phase)) {
          if (lane == 0) fail();
          ok = false;
          break;
        }
        tc_fence_after();
        __syncwarp();
        p.chunk(tile, c, row + (P::kTall ? ch * 2 * kBM : 0), half,
                t_lane + static_cast<std::uint32_t>(acc * kEpiN), ch == 0, stage);
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
  if constexpr (kPair)
    cluster_sync();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (kPair)
      tmem_dealloc_pair(tmem_base, kAcc * kEpiN);
    else
      tmem_dealloc(tmem_base, kAcc * kEpiN);
  }
}

template <class P, int FMT>
__global__ void __launch_bounds__(kEpiThreads, 1)
    tc_epi_kernel(const __grid_constant__ P p, unsigned int* timeouts) {
  epi_body<P, FMT>(p, timeouts);
}

template <class P, int FMT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kEpiThreads, 1)
    tc_epi_pair_kernel(const __grid_constant__ P p, unsigned int* timeouts) {
  epi_body<P, FMT>(p, timeouts);
}

// Launches `kern`; with `overlap` its prologue may overlap the end of the stream's previous
// kernel (it calls grid_wait_previous() before it touches memory).  Overlap only with a
// kernel that waits for its own predecessor in turn: one's own.  tc_epi kernels do not
// let the next one start before their loads are out: its waiting CTAs cost them 2-4 %.
template <typename... K, typename... A>
cudaError_t launch_overlapped(void (*kern)(K...), dim3 grid, int threads, std::size_t smem,
                              cudaStream_t stream, bool overlap, A... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<K>(args)...);
}

template <class P, int FMT>
cudaError_t launch_tc_epi(const P& p, int sms, unsigned int* timeouts, cudaStream_t stream,
                          bool overlap) {
  using S = EpiShape<P>;
  void (*kern)(P, unsigned int*);
  if constexpr (P::kPair)
    kern = tc_epi_pair_kernel<P, FMT>;
  else
    kern = tc_epi_kernel<P, FMT>;
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
  const long long groups = std::min<long long>(p.tiles_total, sms / S::kCtas);
  if (groups <= 0) return cudaSuccess;
  return launch_overlapped(kern, dim3(static_cast<unsigned>(S::kCtas * groups)), kEpiThreads,
                           S::SMEM, stream, overlap, p, timeouts);
}

}  // namespace mb200::tc
