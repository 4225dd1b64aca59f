// vocab_loss_kernels.cu — losses over a linear head's vocabulary, and their gradients
// (sm_100a, tcgen05).  The mathematics is stated in vocab_loss.hpp.
//
// The T x V logits z = x w^T / tau never exist in memory as such.  A call runs over
// pieces of tokens; in each piece
//   1. Logits walks tiles of z.  The fp32 tile stays in tensor memory and registers; the
//      epilogue reduces each token's 128 words (a unit) to one (maximum, sum) pair, lse's
//      running maximum and sum, and picks the target words' logits.  With gradients it also
//      writes the unit's numerators 2^(z2 - the maximum's) in 16 bits;
//   2. vocab_finish_kernel joins a token's pairs into its log-sum-exp and loss, and turns
//      the numerators in place into dz = dloss / tau * (p - q).  Without dw (a frozen head)
//      bf16 numerators of more than 64 tokens share a power-of-two reference per token instead,
//      and the token's factor goes into dx's epilogue: that pass over them falls away (kCommon
//      below);
//   3. Dx and Dw multiply dx = dz w and dw = dz^T x.
// All three products run on the loop of tc_epi_core.cuh.  Scores of up to 8 tokens take
// vocab_stream_kernel instead of 1.  Exponents are in powers of two: z2 = z * log2(e), with
// log2(e) / tau folded into one multiply.  The pairs keep the maximum of x w as it is, and
// differences are taken before they are scaled: a scaled maximum, rounded, may be off by more
// than the exponentials have room for (half a unit in its last place: 1 at |z2| = 2^24), and
// that of words masked with the type's lowest value overflows.
//
// Why the numerators are kept at all: the gradient needs each logit twice, before and after
// lse is known.  Computing the product again costs 2 H flops per logit, 5 us per 10^6 logits
// at H = 4096; keeping 16 bits of it costs 6 bytes of traffic, under 1 us.  The piece bounds
// them to 2 GiB whatever T is, and whatever V is up to the 8 million words where 128 tokens,
// the least piece, reach that.
//
// What bounds a training step of 8192 x 4096 x 131072 (20.3 ms, 1301 TFLOP/s): the power
// cap.  The tensor pipe is busy 95 % of the cycles at 1.15-1.4 GHz.  Of a 1546 us score of
// 2048 x 4096 x 131072 under the cap, 100 us go with the DRAM reads and 155 us with the L2
// reads of the operands (timed without them), hence the wide tiles and the banded order.
//
// Precision: products of the 16-bit inputs accumulate in fp32; maxima, sums, target
// logits and losses are fp32.  dz is a 16-bit operand of the tensor cores and rounds once; the
// 16 bits that carry the numerators to step 2 hold 2 more significant bits than dz (OwnCode;
// fp32 numerators would double the piece's traffic).  The target words, whose p - q cancels,
// are recomputed in step 2 from their fp32 logits; what the rounding of their dz leaves is
// added where it does not average out (kSplit, Left).  dx and dw round once more at the end;
// their sums run in chains of MMAs whose truncation stays well below that (dx_chain,
// kGradientRows).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <array>
#include <climits>
#include <cstdint>
#include <mutex>
#include <type_traits>
#include <utility>

#include "blas/tc_epi_core.cuh"
#include "common/device.hpp"
#include "dnn/vocab_loss.hpp"

namespace mb200::dnn {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Tile r of a rows x cols grid, walked in bands of `band` rows, down a band's column before
// the next column: the tiles in flight share their operands' panels, and a band's rows stay
// in L2 while the columns stream past.
__device__ __forceinline__ void banded(int r, int rows, int cols, int band, int* row, int* col) {
  const int in_band = band * cols;
  const int first = (r / in_band) * band;
  const int n = min(rows - first, band);
  *row = first + (r % in_band) % n;
  *col = (r % in_band) / n;
}

__device__ unsigned int g_vocab_timeouts;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ std::uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const std::uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const std::uint32_t*>(&h);
  }
}

template <typename T>
__device__ __forceinline__ float2 unpack2(std::uint32_t v) {
  if constexpr (std::is_same_v<T, __half>)
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// kOwn's numerators (0 to 1, relative to their unit's largest) become dz's 16 bits in the
// finish.  They hold more bits than dz, or the gradients would show a third rounding beside
// dz's and their own.  They are fp32's bits, rounded and without the sign and the exponent's
// top: for bf16 7 exponent and 9 mantissa bits (10 significant bits over fp32's range below
// 1), for fp16 4 and 12 (13 bits down to 2^-14, steps of 2^-26 below).  NaN does not survive
// the code, but its unit's sum is NaN and makes the whole row NaN.  Against numerators in dz's
// own type: dw's rows of words that are no target 1.01 instead of 1.13 times the error of two
// roundings, steps 0.5-2 % slower (2048 x 2048 x 32000: 672 -> 679 us).
template <typename T>
struct OwnCode {
  static constexpr bool kHalf = std::is_same_v<T, __half>;
  static constexpr float kDown = kHalf ? 0x1p-112f : 1.0f;  // brings 1's exponent below 2^4
  static constexpr int kShift = kHalf ? 11 : 14;
};

template <typename T>
__device__ __forceinline__ std::uint32_t pack_own(float a, float b) {
  using Code = OwnCode<T>;
  const std::uint32_t lo = __float_as_uint(a * Code::kDown) + (1u << (Code::kShift - 1));
  const std::uint32_t hi = __float_as_uint(b * Code::kDown) + (1u << (Code::kShift - 1));
  // (nvcc 12.9 drops the upper half where this is written as a shift, a mask and an or)
  return __byte_perm(lo >> Code::kShift, hi >> Code::kShift, 0x5410);
}

template <typename T>
__device__ __forceinline__ float2 unpack_own(std::uint32_t v) {
  using Code = OwnCode<T>;
  return make_float2(__uint_as_float((v & 0xffffu) << Code::kShift) * (1.0f / Code::kDown),
                     __uint_as_float(v >> 16 << Code::kShift) * (1.0f / Code::kDown));
}

template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same_v<T, __half>)
    return __float2half_rn(v);
  else
    return __float2bfloat16_rn(v);
}

// Target words of the rows of a piece.  Cross entropy: top_k == 0, one label per row.
// Distillation: per row `count` entries sorted by index (vocab_targets_kernel).
struct Targets {
  const std::int64_t* labels;
  int top_k;
  const int* index;       // [row][top_k], ascending, INT_MAX behind the valid entries
  const float* q;         // [row][top_k]
  const int* count;       // valid entries; 0: row left out, -1: an index of vocab or more
  const float* neg_entropy;  // sum q log q
  const std::uint32_t* hit;  // [row][hit_units]: the first target word in each unit of words
  int hit_units;
  float* z;               // [row][max(top_k, 1)]: the target words' x w, unscaled
};

// Entry of the hit map: the word's place in its unit, its rank among the row's targets, and
// whether the row's next target is in the same unit; 0: none in this unit.
constexpr std::uint32_t kHitValid = 1u << 31, kHitMore = 1u << 30;

__device__ __forceinline__ std::uint32_t hit_entry(int word, int rank, int next_word, int unit) {
  const int u = word / unit;
  const bool more = next_word != INT_MAX && next_word / unit == u;
  return kHitValid | (more ? kHitMore : 0u) | static_cast<std::uint32_t>(rank) << 8 |
         static_cast<std::uint32_t>(word - u * unit);
}

// The entry after the one at place `at` of the row's list (its hit said there is one more).
__device__ __forceinline__ std::uint32_t next_hit(const Targets& t, std::int64_t at, int row,
                                                  int unit) {
  const std::int64_t end = (row + 1ll) * t.top_k;
  const int word = t.index[at + 1];
  const int after = at + 2 < end ? t.index[at + 2] : INT_MAX;
  return hit_entry(word, static_cast<int>(at + 1 - (end - t.top_k)), after, unit);
}

// 0: left out, -1: out-of-range target, else the number of target words.
__device__ __forceinline__ int target_count(const Targets& t, int row, int vocab) {
  if (t.top_k > 0) return t.count[row];
  const std::int64_t l = t.labels[row];
  return l < 0 ? 0 : l >= vocab ? -1 : 1;
}

// ------------------------------------------------------------------ logits kernels --
// Most words of an epilogue thread's share of a tile row, its "unit" of one
// (maximum, sum) pair.
constexpr int kUnit = 128;

// k-blocks per accumulator.  Tensor-core accumulation truncates: one chain of 256 MMAs
// (H = 4096) left lse 3.4e-6 off in the 2-norm, chunks of 32 MMAs added in fp32 registers
// 4e-7, an fp32 product's level.
// Up to 8 tokens take 8 MMAs, as their streaming kernel does, so that a width that it cannot
// read is no less exact (T 4, H 4001: 3.0e-7 and 0.8e-7, streamed at 4000 0.9e-7); with more
// tokens that would cost up to 37 % (score of 128 x 768 x 50257).
constexpr int kLogitsChunk = 8, kFewLogitsChunk = 2;

// A thread's logits of one token, and what says whether a target word is among them: the
// token's label, or its entry of the hit map.  Loaded before the
// accumulator is waited for, looked at after.
struct LogitsTile {
  float v[kUnit];
  std::int64_t hint;
};

// z = x w^T.  Pairs (more than 128 tokens): 256 tokens x 256 words.  Single CTAs: all
// tokens x tile_n words; reading w bounds these.
struct LogitsProblem {
  CUtensorMap mx;    // x: dims (features, rows), box {64, 128, 1}
  CUtensorMap mw;    // w or a slice of it: dims (features, words), box {64, tile_n or half, 1}
  CUtensorMap mnum;  // numerators: dims (ldn, rows), box {64, 32, 1} (gradients only)
  long long tiles_total;
  int num_kb, tile_n, rows, vocab, tiles_m, tiles_n;
  int word0;          // the first word of mw
  int band;           // tile rows that stay in L2 while w streams past
  int unit, units;    // words per unit (tile_n / 2), units per row
  float scale;        // log2(e) / tau
  float2* stats;      // [row][units] (maximum of x w, sum of 2^(z2 - the maximum's))
  std::int64_t ldn;
  Targets targets;

  const CUtensorMap* __device__ map_a() const { return &mx; }
  const CUtensorMap* __device__ map_b() const { return &mw; }
  __device__ void coords(long long t, int (&c)[3]) const {
    c[0] = 0;
    banded(static_cast<int>(t), tiles_m, tiles_n, band, &c[1], &c[2]);
  }
  __device__ int k_begin(const int (&)[3]) const { return 0; }
};

__device__ __forceinline__ std::int64_t target_hint(const LogitsProblem& p, int row, int n0) {
  if (row >= p.rows || n0 >= p.vocab) return p.targets.top_k == 0 ? -1 : 0;
  if (p.targets.top_k == 0) return p.targets.labels[row];
  return p.targets.hit[static_cast<std::int64_t>(row) * p.targets.hit_units + n0 / p.unit];
}

// v[j] for a j that differs by lane: halves are selected seven times over.
__device__ __forceinline__ float pick128(const float (&v)[kUnit], int j) {
  float r[kUnit / 2];
#pragma unroll
  for (int i = 0; i < kUnit / 2; ++i) r[i] = (j & (kUnit / 2)) != 0 ? v[i + kUnit / 2] : v[i];
#pragma unroll
  for (int h = kUnit / 4; h > 0; h >>= 1) {
#pragma unroll
    for (int i = 0; i < kUnit / 4; ++i)
      if (i < h) r[i] = (j & h) != 0 ? r[i + h] : r[i];
  }
  return r[0];
}

// Stores the row's target logits among the `cols` words from n0 on.
__device__ __forceinline__ void pick_targets(const LogitsProblem& p, const LogitsTile& t, int row,
                                             int n0, int cols) {
  const int tk = p.targets.top_k;
  if (tk == 0) {
    if (t.hint >= n0 && t.hint < n0 + cols)
      p.targets.z[row] = pick128(t.v, static_cast<int>(t.hint) - n0);
    return;
  }
  auto hint = static_cast<std::uint32_t>(t.hint);
  while ((hint & kHitValid) != 0) {
    const std::int64_t at = static_cast<std::int64_t>(row) * tk + (hint >> 8 & 0xFF);
    p.targets.z[at] = pick128(t.v, static_cast<int>(hint & (kUnit - 1)));
    if ((hint & kHitMore) == 0) break;
    hint = next_hit(p.targets, at, row, p.unit);
  }
}

// What a unit leaves behind besides its pair: nothing, numerators relative to its own
// maximum (kOwn), or numerators relative to 2^0 (kCommon, bf16: its exponents reach as far as
// fp32's).  Units beyond 2^+-64 keep a reference of their own until the finish has seen the
// row's maximum: the nearest whole exponent, so that moving numerators from one to another is
// exact, or the maximum itself where fp32 holds no fraction of the exponent any more.
// Loss and dx of 4096 x 2048 x 65536: 1768 us with kOwn, 1657 with kCommon.
// kSplit is kOwn whose dz becomes two 16-bit rows, rounded and what rounding left, that both
// products add up.  With few tokens the target word's one rounding is common to all of a
// token's dx (and to its row of dw) and does not average out: errors of one token to 64 were
// 1.25 to 1.45 times one rounding in the mean and up to 2.4, and are 1.00 to 1.03.  w's bytes
// set the time there: steps of 39 x 6464 x 16408 162 -> 166 us, 64 x 1111 x 32003 123 -> 126,
// loss and dx of 64 x 2048 x 65536 109 -> 119; at 128 tokens a step would take 16 % more.
enum StoreMode { kNone = 0, kOwn = 1, kCommon = 2, kSplit = 3 };
constexpr int kSplitTokens = 64;
constexpr float kCommonReach = 64.0f, kWholeReach = 0x1p22f;

// Without the second row, dx alone gets what the targets' rounding left, in fp32: one entry of
// {word, left over} per target, for tokens of up to four target words (with more the errors
// average out).  Those words of w are read again for it, where dx is written.  dx's error over
// one rounding 1.3-1.6 -> 1.00; loss and dx of 4096 x 2048 x 65536 1723 -> 1750 us, 1024 x 256 x
// 65536 133 -> 138, 1315 x 1776 x 2464 55.5 -> 62.1, a step of 8192 x 4096 x 131072 the same.
constexpr int kMostLeft = 4;
struct Left {
  int word;
  float dz;
};

// kCommon's numerators of a unit with this maximum are 2^(z2 - top * scale - whole).
struct Reference {
  float top, whole;
};

__device__ __forceinline__ Reference reference(float top, float scale) {
  const float whole = rintf(__fmul_rn(top, scale));
  if (fabsf(whole) <= kCommonReach) return {0.0f, 0.0f};
  if (fabsf(whole) <= kWholeReach) return {0.0f, whole};
  return {top, 0.0f};
}

// Adds a finished accumulator's columns of the unit (taddr: this thread's lane).
__device__ __forceinline__ void add_chunk(LogitsTile& t, int unit, std::uint32_t taddr,
                                          bool first) {
  if (first && unit == kUnit) {
    tc::tmem_load_128cols(taddr, t.v);
    return;
  }
#pragma unroll
  for (int g = 0; g < kUnit / 16; ++g) {
    if (g * 16 < unit) {
      float v[16];
      tc::tmem_load_16cols(taddr + static_cast<std::uint32_t>(g * 16), v);
#pragma unroll
      for (int j = 0; j < 16; ++j) t.v[g * 16 + j] = __fadd_rn(t.v[g * 16 + j], v[j]);
    }
  }
}

// Reduces the unit's logits to its pair and picks target words; with STORE leaves the
// numerators in `stage` as two 128-byte-swizzled boxes of 32 rows x 64 words and sends
// them to memory (the whole warp calls this).
template <typename T, int STORE>
__device__ __forceinline__ void finish_unit(const LogitsProblem& p, LogitsTile& t, int row, int n0,
                                            std::uint8_t* stage) {
  const int lane = threadIdx.x & 31;
  const int cols = min(p.unit, p.vocab - n0);
  if (cols <= 0) return;
  if (cols < kUnit) {
#pragma unroll
    for (int j = 0; j < kUnit; ++j)
      if (j >= cols) t.v[j] = -INFINITY;
  }
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < kUnit; ++j) m[j & 3] = fmaxf(m[j & 3], t.v[j]);
  float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  // a row of -inf (or NaN) has no finite maximum: 0 keeps -inf's numerators at 0
  if (top == -INFINITY) top = 0.0f;
  float shift = 1.0f;
  if constexpr (STORE == kCommon) {
    const Reference ref = reference(top, p.scale);
    shift = exp2_approx(fmaf(top - ref.top, p.scale, -ref.whole));
  }
  pick_targets(p, t, row, n0, cols);
  if constexpr (STORE != kNone) {
    // the previous unit's boxes have left the stage
    if (lane == 0) tc::bulk_wait_read_all();
  }
  __syncwarp();
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int g = 0; g < kUnit / 8; ++g) {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = exp2_approx(__fmul_rn(__fsub_rn(t.v[g * 8 + j], top), p.scale));
      s[j & 3] += e[j];
    }
    if constexpr (STORE == kCommon) {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] *= shift;
    }
    if constexpr (STORE != kNone) {
      std::uint8_t* box = stage + (g >> 3) * 4096 + lane * 128 + (((g & 7) ^ (lane & 7)) << 4);
      std::uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = STORE == kOwn ? pack_own<T>(e[2 * j], e[2 * j + 1])
                             : pack2<T>(e[2 * j], e[2 * j + 1]);
      *reinterpret_cast<uint4*>(box) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (row < p.rows) {
    const float sum = (s[0] + s[1]) + (s[2] + s[3]);  // 1 at least, or 0: all -inf
    p.stats[static_cast<std::int64_t>(row) * p.units + n0 / p.unit] =
        make_float2(sum == 0.0f ? -INFINITY : top, sum);
  }
  if constexpr (STORE != kNone) {
    tc::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && row < p.rows) {  // lane 0 has the warp's first row
      tc::tma_store_3d(&p.mnum, stage, n0, row, 0);
      if (p.unit > 64 && n0 + 64 < p.ldn)
        tc::tma_store_3d(&p.mnum, stage + 4096, n0 + 64, row, 0);
      tc::bulk_commit();
    }
  }
}

// STORE needs units of 64 or 128 words: the stage's boxes are 64 wide.
template <typename T, bool PAIR, int STORE, int CHUNK>
struct Logits : LogitsProblem {
  static constexpr bool kPair = PAIR, kTall = false;
  static constexpr bool kAMn = false;
  static constexpr int kChunk = CHUNK;
  static constexpr int kStageBytes = STORE != kNone ? 8192 : 0;
  using Tile = LogitsTile;

  __device__ __forceinline__ int token(const int (&c)[3], int row) const {
    return c[1] * (PAIR ? 2 : 1) * tc::kBM + row;
  }
  __device__ __forceinline__ int word(const int (&c)[3], int half) const {
    return word0 + c[2] * tile_n + half * unit;
  }
  __device__ __forceinline__ void begin(Tile& t, const int (&c)[3], int row, int half) const {
    t.hint = target_hint(*this, token(c, row), word(c, half));
    if (unit < kUnit) {
#pragma unroll
      for (int j = 0; j < kUnit; ++j) t.v[j] = 0.0f;
    }
  }
  __device__ __forceinline__ void chunk(Tile& t, const int (&)[3], int, int, std::uint32_t taddr,
                                        bool first, std::uint8_t*) const {
    add_chunk(t, unit, taddr, first);
  }
  __device__ __forceinline__ void end(Tile& t, const int (&c)[3], int row, int half,
                                      std::uint8_t* stage) const {
    finish_unit<T, STORE>(*this, t, token(c, row), word(c, half), stage);
  }
};

// ------------------------------------------------------------- scores of few tokens --
// Up to 8 tokens, losses only: reading w is all there is to do, so w goes from memory
// straight into mma.sync operands.  A warp takes 16 words at a time: lane (g, t) = (lane / 4,
// lane % 4) loads 16 bytes of words g and g + 8 and of token g at feature 32 step + 8 t, the
// four lanes of a word a whole 64 bytes.  The MMA's K order is free as long as both operands
// agree, so the lane's 8 features serve two k16 MMAs as they lie.  Loads run four steps (4 KB
// per warp) ahead, across words.  No tensor memory, barriers or shared-memory ring to set up:
// one token against 32000 x 1024 takes 18 us with its finish, 25 us on the tiles above, and 8
// against 131072 x 4096 178 us (6.0 TB/s) and 209.
//
// A lane keeps its own running (maximum, sum) of the words it sees; the CTA joins them once
// at the end into one pair per token.  Every eight MMAs go into an fp32 sum, which bounds the
// drift of their truncating accumulation.
constexpr int kStreamTokens = 8;
constexpr int kStreamWords = 16;    // words per warp and round
constexpr int kStreamThreads = 512;
// Steps of 32 features in flight per warp: 8 x 2048 x 32000 took 25.9 us with 4 and 27.5 with
// 8, 8 x 4096 x 131072 179.8 and 177.
constexpr int kStreamSteps = 4;

struct StreamArgs {
  const void* x;
  std::int64_t ldx;
  const void* w;
  std::int64_t ldw;
  int rows, features, vocab;
  float scale;
  float2* stats;  // [row][gridDim.x]
  Targets targets;
};

// 16 bytes that are read once, zeros without `ok`.  The predicate is inside the asm: a branch
// around the load would make its result wait for the load at once.
__device__ __forceinline__ uint4 load_once(const void* p, bool ok) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@q ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"(static_cast<int>(ok)));
  return v;
}

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], std::uint32_t a0, std::uint32_t a1,
                                            std::uint32_t a2, std::uint32_t a3, std::uint32_t b0,
                                            std::uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// (m, s) joined with (m2, s2): s counts 2^((x w - m) scale); s == 0 is an empty pair.
__device__ __forceinline__ void join_pair(float& m, float& s, float m2, float s2, float scale) {
  if (s2 == 0.0f) return;
  if (s == 0.0f) {
    m = m2;
    s = s2;
    return;
  }
  const float top = fmaxf(m, m2);
  s = s * exp2_approx((m - top) * scale) + s2 * exp2_approx((m2 - top) * scale);
  m = top;
}

template <typename T>
__global__ void __launch_bounds__(kStreamThreads, 1) vocab_stream_kernel(const StreamArgs a) {
  __shared__ float2 joined[kStreamThreads / 32][kStreamTokens];
  tc::grid_launch_next();
  tc::grid_wait_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const T* x = static_cast<const T*>(a.x) + g * a.ldx + 8 * t;
  const T* w = static_cast<const T*>(a.w);
  const int rounds_all = (a.vocab + kStreamWords - 1) / kStreamWords;
  const int groups = (a.features + 32 * kStreamSteps - 1) / (32 * kStreamSteps);
  // round r of the grid's warps, CTAs fastest so that every SM gets its share
  const int first = warp * gridDim.x + blockIdx.x;
  const int stride = gridDim.x * (kStreamThreads / 32);

  int label[2];  // cross entropy: the target words of the lane's tokens 2t and 2t + 1
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    label[j] = -1;
    if (a.targets.top_k == 0 && 2 * t + j < a.rows) {
      const std::int64_t l = a.targets.labels[2 * t + j];
      if (l >= 0 && l < a.vocab) label[j] = static_cast<int>(l);
    }
  }
  float m[2] = {0.0f, 0.0f}, s[2] = {0.0f, 0.0f};

  uint4 in[kStreamSteps][2];  // words g and g + 8 of the steps in flight
  const auto fetch = [&](int round, int group, int i) {
    const int w0 = round * kStreamWords + g;
    const int k = (group * kStreamSteps + i) * 32 + 8 * t;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      in[i][h] = load_once(w + static_cast<std::int64_t>(w0 + 8 * h) * a.ldw + k,
                           round < rounds_all && w0 + 8 * h < a.vocab && k < a.features);
  };
  if (first < rounds_all) {
#pragma unroll
    for (int i = 0; i < kStreamSteps; ++i) fetch(first, 0, i);
  }
  for (int round = first; round < rounds_all; round += stride) {
    std::uint32_t hint = 0;  // distillation: the round's entry of token `lane`'s map
    if (a.targets.top_k > 0 && lane < a.rows)
      hint = a.targets.hit[static_cast<std::int64_t>(lane) * a.targets.hit_units + round];
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int group = 0; group < groups; ++group) {
      const bool more = group + 1 < groups;
      const int next_round = more ? round : round + stride, next_group = more ? group + 1 : 0;
#pragma unroll
      for (int i = 0; i < kStreamSteps; ++i) {
        const int k = (group * kStreamSteps + i) * 32;
        uint4 b = make_uint4(0, 0, 0, 0);
        if (g < a.rows && k + 8 * t < a.features) b = __ldg(reinterpret_cast<const uint4*>(x + k));
        mma_16x8x16<T>(acc, in[i][0].x, in[i][1].x, in[i][0].y, in[i][1].y, b.x, b.y);
        mma_16x8x16<T>(acc, in[i][0].z, in[i][1].z, in[i][0].w, in[i][1].w, b.z, b.w);
        fetch(next_round, next_group, i);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        z[j] = __fadd_rn(z[j], acc[j]);
        acc[j] = 0.0f;
      }
    }
    // z[0..1]: word g, tokens 2t and 2t + 1; z[2..3]: word g + 8
    const int w0 = round * kStreamWords + g;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (w0 + (j >> 1) * 8 >= a.vocab) z[j] = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (label[j] == w0) a.targets.z[2 * t + j] = z[j];
      if (label[j] == w0 + 8) a.targets.z[2 * t + j] = z[j + 2];
      const float top = fmaxf(z[j], z[j + 2]);
      // -inf adds nothing; NaN has to (fmaxf passes over it)
      const float base = top == -INFINITY ? 0.0f : top;
      join_pair(m[j], s[j], base, exp2_approx((z[j] - base) * a.scale) +
                                      exp2_approx((z[j + 2] - base) * a.scale), a.scale);
    }
    if (a.targets.top_k > 0) {
      unsigned rows = __ballot_sync(0xffffffffu, hint != 0u);
      while (rows != 0) {  // tokens with a target among these words
        const int row = __ffs(rows) - 1;
        rows &= rows - 1;
        std::uint32_t hit = __shfl_sync(0xffffffffu, hint, row);
        for (;;) {
          const std::int64_t at =
              static_cast<std::int64_t>(row) * a.targets.top_k + (hit >> 8 & 0xFF);
          const int word = static_cast<int>(hit & (kStreamWords - 1));
          if ((word & 7) == g && row >> 1 == t) {
            const float even = word < 8 ? z[0] : z[2], odd = word < 8 ? z[1] : z[3];
            a.targets.z[at] = (row & 1) != 0 ? odd : even;
          }
          if ((hit & kHitMore) == 0) break;
          hit = next_hit(a.targets, at, row, kStreamWords);
        }
      }
      __syncwarp();
    }
  }

  // join the eight lanes of a token, then the warps
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m[j], o);
      const float s2 = __shfl_xor_sync(0xffffffffu, s[j], o);
      join_pair(m[j], s[j], m2, s2, a.scale);
    }
    if (g == 0) joined[warp][2 * t + j] = make_float2(m[j], s[j]);
  }
  __syncthreads();
  const int row = threadIdx.x;
  if (row < a.rows) {
    float2 p = joined[0][row];
    for (int i = 1; i < kStreamThreads / 32; ++i)
      join_pair(p.x, p.y, joined[i][row].x, joined[i][row].y, a.scale);
    a.stats[static_cast<std::int64_t>(row) * gridDim.x + blockIdx.x] = p;
  }
}

// ----------------------------------------------------------------- small kernels --
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp per token: the teacher's distribution over the valid entries, and the entries
// sorted by word (rank counting: top_k^2 / 32 comparisons per lane), and the hit map of the
// units that the logits come in.
constexpr int kTargetWarps = 4;

__global__ void __launch_bounds__(32 * kTargetWarps)
    vocab_targets_kernel(const std::int64_t* __restrict__ teacher_index,
                         const float* __restrict__ teacher_logits, int rows, int top_k, int vocab,
                         float inv_tau, int* index, float* __restrict__ q,
                         int* __restrict__ count, float* __restrict__ neg_entropy,
                         std::uint32_t* __restrict__ hit, int hit_units, int unit) {
  tc::grid_launch_next();
  tc::grid_wait_previous();
  __shared__ int key_all[kTargetWarps][kVocabMaxTopK];
  const int lane = threadIdx.x & 31;
  int* key = key_all[threadIdx.x >> 5];
  const int row = blockIdx.x * kTargetWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const std::int64_t r0 = static_cast<std::int64_t>(row) * top_k;
  std::uint32_t* map = hit + static_cast<std::int64_t>(row) * hit_units;
  for (int k = lane; k < hit_units; k += 32) map[k] = 0u;
  float mx = -INFINITY;
  int valid = 0, bad = 0;
  for (int k = lane; k < top_k; k += 32) {
    const std::int64_t i = teacher_index[r0 + k];
    const float t = teacher_logits[r0 + k];
    const bool ok = i >= 0 && i < vocab && t != -INFINITY;
    bad |= i >= vocab;
    key[k] = ok ? static_cast<int>(i) : INT_MAX;
    if (ok) {
      mx = fmaxf(mx, t);
      ++valid;
    }
  }
  __syncwarp();
  mx = warp_max(mx);
  valid = warp_sum(valid);
  bad = __any_sync(0xffffffffu, bad);
  // differences before they are scaled, as in finish_unit
  float total = 0.0f;
  for (int k = lane; k < top_k; k += 32)
    if (key[k] != INT_MAX) total += expf((teacher_logits[r0 + k] - mx) * inv_tau);
  total = warp_sum(total);
  const float log_total = logf(total);
  float ent = 0.0f;
  for (int k = lane; k < top_k; k += 32) {
    const int mine = key[k];
    int rank = 0;
    for (int j = 0; j < top_k; ++j) rank += key[j] < mine || (key[j] == mine && j < k);
    float qk = 0.0f;
    if (mine != INT_MAX) {
      const float d = (teacher_logits[r0 + k] - mx) * inv_tau;
      qk = expf(d) / total;
      if (qk != 0.0f) ent += qk * (d - log_total);
    }
    index[r0 + rank] = mine;
    q[r0 + rank] = qk;
  }
  __syncwarp();  // the row's sorted list and its cleared map
  for (int k = lane; k < valid; k += 32) {
    const int word = index[r0 + k];
    if (k == 0 || index[r0 + k - 1] / unit != word / unit)
      map[word / unit] =
          hit_entry(word, k, k + 1 < valid ? index[r0 + k + 1] : INT_MAX, unit);
  }
  ent = warp_sum(ent);
  if (lane == 0) {
    count[row] = bad ? -1 : valid;
    neg_entropy[row] = ent;
  }
}

// fp16 only: a power of two that brings the piece's largest |dloss / tau| (over the rows
// that are not left out) to [2^13, 2^14), so dz, at most that in magnitude, fills fp16's
// range; scale[1] undoes it after the products.
__global__ void __launch_bounds__(1024)
    vocab_grad_scale_kernel(const float* __restrict__ dloss, int rows, int vocab, Targets targets,
                            float inv_tau, float* __restrict__ scale) {
  tc::grid_launch_next();
  tc::grid_wait_previous();
  __shared__ float red[32];
  float mx = 0.0f;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float g = fabsf(dloss[i] * inv_tau);
    if (target_count(targets, i, vocab) > 0 && g < INFINITY) mx = fmaxf(mx, g);
  }
  mx = warp_max(mx);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
  __syncthreads();
  if (threadIdx.x < 32) {
    mx = warp_max(red[threadIdx.x]);
    if (threadIdx.x == 0) {
      int e = 0;
      if (mx > 0.0f) frexpf(mx, &e);  // mx in [2^(e-1), 2^e)
      e = max(-100, min(100, e));
      scale[0] = ldexpf(1.0f, 14 - e);
      scale[1] = ldexpf(1.0f, e - 14);
    }
  }
}

constexpr int kFinishThreads = 256;

__device__ __forceinline__ float block_reduce(float v, bool is_max, float* red) {
  v = is_max ? warp_max(v) : warp_sum(v);
  __syncthreads();  // red[] may still be read by the previous reduction
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int i = 1; i < kFinishThreads / 32; ++i) r = is_max ? fmaxf(r, red[i]) : r + red[i];
  return r;
}

struct TransposeArgs {
  const void* x;
  std::int64_t ldx;
  int rows, features;
  bool vec;  // 16-byte reads
  void* xt;  // null: nothing to do
  std::int64_t ldt;
};

struct FinishArgs {
  const float2* stats;  // [row][units]
  int rows, parts;      // CTAs: one per row and part of its words, then the transpose's
  int units, unit, vocab;
  Targets targets;
  float* loss;  // may be null
  float* lse;   // may be null
  const float* dloss;
  float inv_tau;
  float log2e_tau;     // log2(e) / tau
  const float* scale;  // fp16: the gradient scale, else null
  void* num;
  std::int64_t ldn, pitch;  // words of a row of num, and from a token's row to the next's
  float2* row_scale;   // dz's row is both factors times what num holds; 0 for rows left out
  Left* left;          // [row][max(top_k, 1)], null: not asked for
  TransposeArgs transpose;  // with dz: x^T for dw's product, in the same launch
};

// xt[h][row] = x[row][h], rows that are left out as zeros (their x may hold anything, and
// 0 * NaN would reach dw).  K-major x for dw's product: reading x MN-major instead would
// make both operands MN-major, the slowest form of the tensor-core loop.
// 64 x 64 tiles, 16 bytes per thread and access (reads: where x's rows allow it): 8192 x 4096
// in 29 us as a launch of its own (4.6 TB/s; 2-byte accesses took 78).
// The tile's pitch of 33 words keeps its column reads to two words of a bank.
// TWICE: every token fills two columns of x^T, for dz's two rows.
template <typename T, bool TWICE>
__device__ __forceinline__ void transpose_tile(const TransposeArgs& a, const Targets& targets,
                                               int vocab, long long block) {
  __shared__ std::uint32_t tile[64][33];
  __shared__ bool in[64];
  const T* x = static_cast<const T*>(a.x);
  T* xt = static_cast<T*>(a.xt);
  const std::int64_t ldx = a.ldx, ldt = a.ldt;
  const int rows = a.rows, features = a.features;
  const int across = (rows + 63) / 64;
  const int r0 = static_cast<int>(block % across) * 64, h0 = static_cast<int>(block / across) * 64;
  if (threadIdx.x < 64)
    in[threadIdx.x] =
        r0 + threadIdx.x < rows && target_count(targets, r0 + threadIdx.x, vocab) != 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (threadIdx.x >> 3) + 32 * i, h = (threadIdx.x & 7) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (in[r] && h0 + h < features) {
      const T* src = x + static_cast<std::int64_t>(r0 + r) * ldx + h0 + h;
      if (a.vec && h0 + h + 8 <= features) {
        v = *reinterpret_cast<const uint4*>(src);
      } else {
        alignas(16) T e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = h0 + h + j < features ? src[j] : from_float<T>(0.0f);
        v = *reinterpret_cast<const uint4*>(e);
      }
    }
    std::uint32_t* d = &tile[r][h / 2];
    d[0] = v.x;
    d[1] = v.y;
    d[2] = v.z;
    d[3] = v.w;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int h = (threadIdx.x >> 3) + 32 * i, r = (threadIdx.x & 7) * 8;
    if (h0 + h >= features || r0 + r >= rows) continue;  // x^T's rows are padded to whole lines
    constexpr int kCopies = TWICE ? 2 : 1;
    std::uint32_t o[4 * kCopies];
#pragma unroll
    for (int j = 0; j < 4 * kCopies; ++j) {
      if constexpr (TWICE)
        o[j] = __byte_perm(tile[r + j][h / 2], 0u, (h & 1) != 0 ? 0x3232 : 0x1010);
      else
        o[j] = __byte_perm(tile[r + 2 * j][h / 2], tile[r + 2 * j + 1][h / 2],
                           (h & 1) != 0 ? 0x7632 : 0x5410);
    }
    uint4* dst = reinterpret_cast<uint4*>(xt + static_cast<std::int64_t>(h0 + h) * ldt +
                                          kCopies * (r0 + r));
#pragma unroll
    for (int j = 0; j < kCopies; ++j)
      dst[j] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
  }
}

// What rounding v to r left; 0 for infinities.
__device__ __forceinline__ float rest(float v, float r) { return v == r ? 0.0f : v - r; }

// Eight numerators times f, in T; kSplit: what their rounding left, in *left.
template <typename T, int STORE>
__device__ __forceinline__ uint4 scaled(uint4 u, float f, uint4* left = nullptr) {
  std::uint32_t* w = reinterpret_cast<std::uint32_t*>(&u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float2 v = STORE == kCommon ? unpack2<T>(w[j]) : unpack_own<T>(w[j]);
    v = make_float2(f * v.x, f * v.y);
    w[j] = pack2<T>(v.x, v.y);
    if constexpr (STORE == kSplit) {
      const float2 r = unpack2<T>(w[j]);
      reinterpret_cast<std::uint32_t*>(left)[j] = pack2<T>(rest(v.x, r.x), rest(v.y, r.y));
    }
  }
  return u;
}

// A CTA per row and part of its words (each part joins the row's pairs again, a few KB from
// L2), then one per tile of the transpose.  Bound by HBM: it reads and writes the numerators once, 8192 x
// 131072 in 0.68 ms (6.3 TB/s).
template <typename T, int STORE>
__global__ void __launch_bounds__(kFinishThreads) vocab_finish_kernel(const FinishArgs a) {
  tc::grid_launch_next();
  tc::grid_wait_previous();
  constexpr bool kDz = STORE == kOwn || STORE == kSplit;
  __shared__ float red[kFinishThreads / 32];
  const long long finish = static_cast<long long>(a.rows) * a.parts;
  if constexpr (kDz) {
    if (blockIdx.x >= finish) {
      transpose_tile<T, STORE == kSplit>(a.transpose, a.targets, a.vocab, blockIdx.x - finish);
      return;
    }
  }
  const int row = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.rows));
  const int part = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.rows));
  const int n = target_count(a.targets, row, a.vocab);
  // this CTA's units, and their 8-word chunks
  const int u_per = (a.units + a.parts - 1) / a.parts;
  const int u_begin = min(a.units, u_per * part);
  const int u_end = min(a.units, u_begin + u_per);
  const int per_unit = a.unit / 8;
  const std::int64_t c_begin = static_cast<std::int64_t>(u_begin) * per_unit;
  const std::int64_t c_end = min(a.ldn / 8, static_cast<std::int64_t>(u_end) * per_unit);
  uint4* num = reinterpret_cast<uint4*>(static_cast<T*>(a.num) + row * a.pitch);
  const std::int64_t low = a.ldn / 8;  // kSplit: from dz's row to that of what rounding left
  if (n == 0) {  // left out
    if (part == 0 && threadIdx.x == 0) {
      if (a.loss != nullptr) a.loss[row] = 0.0f;
      if (a.lse != nullptr) a.lse[row] = 0.0f;
      if constexpr (STORE != kNone) a.row_scale[row] = make_float2(0.0f, 0.0f);
    }
    if constexpr (STORE != kNone) {
      if (a.left != nullptr && part == 0 && threadIdx.x < max(a.targets.top_k, 1))
        a.left[static_cast<std::int64_t>(row) * max(a.targets.top_k, 1) + threadIdx.x] = {0, 0.0f};
    }
    if constexpr (kDz) {
      for (std::int64_t c = c_begin + threadIdx.x; c < c_end; c += kFinishThreads) {
        num[c] = make_uint4(0, 0, 0, 0);
        if constexpr (STORE == kSplit) num[low + c] = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  const float2* st = a.stats + static_cast<std::int64_t>(row) * a.units;
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < a.units; i += kFinishThreads)
    if (st[i].y != 0.0f) mx = fmaxf(mx, st[i].x);
  mx = block_reduce(mx, true, red);
  float sum = 0.0f;
  for (int i = threadIdx.x; i < a.units; i += kFinishThreads)
    if (st[i].y != 0.0f) sum += st[i].y * exp2f((st[i].x - mx) * a.log2e_tau);
  sum = block_reduce(sum, false, red);
  const float log_sum = log2f(sum);

  const int tk = max(a.targets.top_k, 1);
  const std::int64_t r0 = static_cast<std::int64_t>(row) * tk;
  // a target's z2 above the maximum's: a confident word's loss is far below z2's last bit
  const auto above = [&](std::int64_t i) { return (a.targets.z[i] - mx) * a.log2e_tau; };
  if (part == 0) {
    float loss;
    if (n < 0) {
      loss = NAN;
    } else if (a.targets.top_k == 0) {
      loss = (log_sum - above(r0)) * kLn2;
    } else {
      float cross = 0.0f;
      for (int k = threadIdx.x; k < n; k += kFinishThreads)
        if (a.targets.q[r0 + k] != 0.0f)
          cross += a.targets.q[r0 + k] * ((log_sum - above(r0 + k)) * kLn2);
      loss = a.targets.neg_entropy[row] + block_reduce(cross, false, red);
    }
    if (threadIdx.x == 0) {
      if (a.loss != nullptr) a.loss[row] = loss;
      if (a.lse != nullptr) a.lse[row] = fmaf(mx, a.inv_tau, log_sum * kLn2);
    }
  }
  if constexpr (STORE != kNone) {
    float g = n < 0 ? NAN : a.dloss[row] * a.inv_tau;
    if (a.scale != nullptr) g *= a.scale[0];
    float down = 0.0f;  // kCommon: the row's reference below its maximum, in z2
    if constexpr (kDz) {
      if (part == 0 && threadIdx.x == 0)
        a.row_scale[row] = make_float2(1.0f, a.scale != nullptr ? a.scale[1] : 1.0f);
    }
    if constexpr (STORE == kCommon) {
      const Reference base = reference(mx, a.log2e_tau);
      down = fmaf(base.top - mx, a.log2e_tau, base.whole);
      if (part == 0 && threadIdx.x == 0) a.row_scale[row] = make_float2(exp2f(down - log_sum), g);
      // only units whose reference is not the row's: rare
      for (int u = u_begin + (threadIdx.x >> 5); u < u_end; u += kFinishThreads / 32) {
        const Reference ref = reference(st[u].x, a.log2e_tau);
        const float move = fmaf(ref.top - base.top, a.log2e_tau, ref.whole - base.whole);
        if (st[u].y == 0.0f || move == 0.0f) continue;
        const float f = exp2f(move);
        const std::int64_t c = static_cast<std::int64_t>(u) * per_unit + (threadIdx.x & 31);
        if ((threadIdx.x & 31) < per_unit && c < c_end) num[c] = scaled<T, STORE>(num[c], f);
      }
    } else {
      const auto factor = [&](std::int64_t c) {
        return g * exp2f(fmaf(st[c / per_unit].x - mx, a.log2e_tau, -log_sum));
      };
      const auto rescale = [&](std::int64_t c, uint4 u) {
        if constexpr (STORE == kSplit) {
          uint4 left;
          num[c] = scaled<T, STORE>(u, factor(c), &left);
          num[low + c] = left;
        } else {
          num[c] = scaled<T, STORE>(u, factor(c));
        }
      };
      std::int64_t c = c_begin + threadIdx.x;
      for (; c + 3 * kFinishThreads < c_end; c += 4 * kFinishThreads) {
        uint4 u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = num[c + j * kFinishThreads];
#pragma unroll
        for (int j = 0; j < 4; ++j) rescale(c + j * kFinishThreads, u[j]);
      }
      for (; c < c_end; c += kFinishThreads) rescale(c, num[c]);
    }
    // the targets, in the numerators' units: dz, or dz / row_scale
    const float t = STORE == kCommon ? exp2f(log_sum - down) : g;
    __syncthreads();
    const auto put = [&](int word, float v) {
      T* d = reinterpret_cast<T*>(num) + word;
      *d = from_float<T>(v);
      const float r = rest(v, static_cast<float>(*d));
      if constexpr (STORE == kSplit) d[a.ldn] = from_float<T>(r);
      return Left{word, r};
    };
    // entry k, from the part that has its word; part 0 for those without one
    const auto keep = [&](int k, Left l) {
      if (a.left != nullptr) a.left[r0 + k] = l;
    };
    if (a.targets.top_k == 0) {
      const std::int64_t l = a.targets.labels[row];
      if (threadIdx.x == 0 && n > 0 && l >= c_begin * 8 && l < c_end * 8)
        keep(0, put(static_cast<int>(l), t * expm1f((above(r0) - log_sum) * kLn2)));
      else if (threadIdx.x == 0 && n < 0 && part == 0)
        keep(0, {0, 0.0f});
    } else {
      for (int k = threadIdx.x; k < tk; k += kFinishThreads) {
        const int w = k < n ? a.targets.index[r0 + k] : -1;
        // the first entry of a run of equal words adds all
        if (k >= n || (k > 0 && a.targets.index[r0 + k - 1] == w)) {
          if (part == 0) keep(k, {0, 0.0f});
          continue;
        }
        if (w < c_begin * 8 || w >= c_end * 8) continue;
        float q = a.targets.q[r0 + k];
        for (int j = k + 1; j < n && a.targets.index[r0 + j] == w; ++j) q += a.targets.q[r0 + j];
        keep(k, put(w, t * (exp2f(above(r0 + k) - log_sum) - q)));
      }
    }
  }
}

// dst[r][c] = src[r][c] into rows of ldd elements (a multiple of 64): operands whose rows
// TMA cannot read in place, or that start off a line.  A thread moves 8 elements: the
// aligned words around them, shifted by half a word where the row is odd.  There the first
// word also holds the element before them (never src's first chunk, see below); of the fifth
// only the half that is theirs is read, the other may lie past src's end.
template <typename T>
__global__ void __launch_bounds__(256)
    vocab_pack_kernel(const T* __restrict__ src, std::int64_t lds, std::int64_t rows, int cols,
                      T* __restrict__ dst, std::int64_t ldd) {
  tc::grid_launch_next();
  tc::grid_wait_previous();
  const int per = (cols + 7) / 8;
  const std::int64_t total = rows * per;
  for (std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<std::int64_t>(gridDim.x) * 256) {
    const std::int64_t r = i / per;
    const int c = static_cast<int>(i - r * per) * 8;
    const T* s = src + r * lds + c;
    T* d = dst + r * ldd + c;
    if (c + 8 > cols || i == 0) {  // the ends of the rows, and nothing before the first element
      for (int j = 0; j < 8 && c + j < cols; ++j) d[j] = s[j];
      continue;
    }
    const auto at = reinterpret_cast<std::uintptr_t>(s);
    const std::uint32_t* w = reinterpret_cast<const std::uint32_t*>(at & ~std::uintptr_t{3});
    const unsigned shift = (at & 2) * 8;
    std::uint32_t v[5];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = w[j];
    v[4] = shift != 0 ? *reinterpret_cast<const std::uint16_t*>(s + 7) : 0u;
    *reinterpret_cast<uint4*>(d) =
        make_uint4(__funnelshift_r(v[0], v[1], shift), __funnelshift_r(v[1], v[2], shift),
                   __funnelshift_r(v[2], v[3], shift), __funnelshift_r(v[3], v[4], shift));
  }
}

// ------------------------------------------------------------------ gradient GEMMs --
// A row that is left out has factor 0 and gradient 0, whatever its numerators and w hold.
// The factors stay two: kCommon's first is down to 2^-64 / V, and its product with a small
// dloss would leave fp32's range where dx does not.
__device__ __forceinline__ float by_row(float2 factor, float v) {
  return factor.x == 0.0f ? 0.0f : factor.x * v * factor.y;
}

template <typename T>
__device__ __forceinline__ float add_left(float v, Left l, T w) {
  return l.dz == 0.0f ? v : fmaf(l.dz, static_cast<float>(w), v);
}

// dx^T = w^T dz^T: A = w^T is MN-major in w, B = dz is K-major, the faster operand forms;
// a thread's columns are tokens of one feature, so a warp's stores of one token are 32
// consecutive features.  The words (K) split across `ksplit` groups of CTAs.  Pairs (more
// than 128 tokens): 256 features x 256 tokens, or tall tiles of 512; else 128 features x
// all tokens.  SPLIT: a token has two rows of dz side by side, and so do a thread's columns.
template <typename T, bool PAIR, bool TALL, bool SPLIT>
struct Dx {
  static constexpr bool kPair = PAIR, kTall = TALL;
  static constexpr bool kAMn = true;
  static constexpr int kChunk = 0;
  static constexpr int kStageBytes = 0;
  static constexpr int kRows = (TALL ? 4 : PAIR ? 2 : 1) * tc::kBM;  // features per tile
  // With K this long nothing stays in L2 from tile to tile: 8 x 9 tiles in flight read the
  // fewest panels (measured: 8 rows 5.0 GB of DRAM reads at 8192 x 4096 x 65536, 4 rows 5.7).
  static constexpr int kBand = 8;
  struct Tile {};
  CUtensorMap ma;  // w or a slice of it: dims (features, words), box {64, 64, 1}
  CUtensorMap mb;  // dz of these words: dims (words, its rows), box {64, tile_n or half, 1}
  long long tiles_total;
  int num_kb;  // k-blocks per split
  int tile_n, rows, features, tiles_m, tiles_n;
  T* dx;
  std::int64_t lddx;
  float* partial;  // several splits or slices: [split][row][feature]
  bool add;        // to what an earlier slice left in partial
  const float2* row_scale;  // [row]
  const Left* left;         // [row][lefts], 0: none; without partial sums
  int lefts;
  const T* w;               // all words, rows of `features`

  const CUtensorMap* __device__ map_a() const { return &ma; }
  const CUtensorMap* __device__ map_b() const { return &mb; }
  __device__ void coords(long long t, int (&c)[3]) const {
    const int per = tiles_m * tiles_n;
    const int r = static_cast<int>(t % per);
    c[0] = static_cast<int>(t / per);
    banded(r, tiles_m, tiles_n, kBand, &c[1], &c[2]);
  }
  __device__ int k_begin(const int (&c)[3]) const { return c[0] * num_kb; }
  __device__ void begin(Tile&, const int (&)[3], int, int) const {}
  __device__ void end(Tile&, const int (&)[3], int, int, std::uint8_t*) const {}
  __device__ __forceinline__ void chunk(Tile&, const int (&c)[3], int row, int half,
                                        std::uint32_t taddr, bool, std::uint8_t*) const {
    const int h = c[1] * kRows + row;
    const int cols = tile_n / 2;
    constexpr int kTokens = SPLIT ? 8 : 16;  // of 16 columns
#pragma unroll 1
    for (int c0 = 0; c0 < cols; c0 += 16) {
      float v[16];
      __syncwarp();
      tc::tmem_load_16cols(taddr + static_cast<std::uint32_t>(c0), v);
      if constexpr (SPLIT) {
#pragma unroll
        for (int j = 0; j < kTokens; ++j) v[j] = v[2 * j] + v[2 * j + 1];
      }
      const int t0 = (c[2] * tile_n + half * cols + c0) / (16 / kTokens);
      if (h >= features) continue;
      for (int m = 0; m < lefts; ++m) {
        Left l[kTokens];
        T x[kTokens];
#pragma unroll
        for (int j = 0; j < kTokens; ++j)
          l[j] = left[static_cast<std::int64_t>(min(t0 + j, rows - 1)) * lefts + m];
#pragma unroll
        for (int j = 0; j < kTokens; ++j)
          x[j] = w[static_cast<std::int64_t>(l[j].word) * features + h];
#pragma unroll
        for (int j = 0; j < kTokens; ++j) v[j] = add_left(v[j], l[j], x[j]);
      }
      if (partial != nullptr) {
        float* o = partial + (static_cast<std::int64_t>(c[0]) * rows + t0) * features + h;
        if (add) {
#pragma unroll
          for (int j = 0; j < kTokens; ++j)
            if (t0 + j < rows) v[j] += o[static_cast<std::int64_t>(j) * features];
        }
#pragma unroll
        for (int j = 0; j < kTokens; ++j)
          if (t0 + j < rows) o[static_cast<std::int64_t>(j) * features] = v[j];
      } else {
        T* o = dx + static_cast<std::int64_t>(t0) * lddx + h;
#pragma unroll
        for (int j = 0; j < kTokens; ++j)
          if (t0 + j < rows) o[j * lddx] = from_float<T>(by_row(row_scale[t0 + j], v[j]));
      }
    }
  }
};

// dx = row_scale * (sum of the splits, in split order); VEC features per thread, 1 where rows
// are not whole 16-byte runs.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
    vocab_dx_reduce_kernel(const float* __restrict__ partial, int ksplit, int rows, int features,
                           T* __restrict__ dx, std::int64_t lddx, const float2* row_scale,
                           const Left* left, int lefts, const T* w) {
  tc::grid_launch_next();
  tc::grid_wait_previous();
  const std::int64_t plane = static_cast<std::int64_t>(rows) * features;
  const std::int64_t per = features / VEC;
  const std::int64_t total = rows * per;
  for (std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<std::int64_t>(gridDim.x) * 256) {
    const std::int64_t r = i / per, h = (i - r * per) * VEC;
    const float* p = partial + r * features + h;
    T* o = dx + r * lddx + h;
    const float2 f = row_scale[r];
    if constexpr (VEC == 4) {
      float4 s = __ldcs(reinterpret_cast<const float4*>(p));
#pragma unroll 4
      for (int k = 1; k < ksplit; ++k) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(p + k * plane));
        s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
      }
      for (int m = 0; m < lefts; ++m) {
        const Left l = left[r * lefts + m];
        const T* x = w + static_cast<std::int64_t>(l.word) * features + h;
        s = make_float4(add_left(s.x, l, x[0]), add_left(s.y, l, x[1]), add_left(s.z, l, x[2]),
                        add_left(s.w, l, x[3]));
      }
      *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(by_row(f, s.x), by_row(f, s.y)),
                                                pack2<T>(by_row(f, s.z), by_row(f, s.w)));
    } else {
      float s = __ldcs(p);
#pragma unroll 4
      for (int k = 1; k < ksplit; ++k) s += __ldcs(p + k * plane);
      for (int m = 0; m < lefts; ++m) {
        const Left l = left[r * lefts + m];
        s = add_left(s, l, w[static_cast<std::int64_t>(l.word) * features + h]);
      }
      *o = from_float<T>(by_row(f, s));
    }
  }
}

// dw = dz^T x on CTA pairs: A = dz^T is MN-major in dz, B = x^T (transposed copy) K-major.
// Each epilogue warp stages its words' features as 128-byte-swizzled boxes of 32 x 64 and
// sends them by TMA; rows that TMA cannot address go out of the stage in coalesced 2-byte
// stores (aligned 4-byte pairs, with a shuffle where a row starts at an odd element, were
// slower: 73 against 64 us at 777 x 1111 x 32003).  A call of several pieces adds its
// pieces in fp32 and rounds once, in the last.
template <typename T, bool TALL>
struct Dw {
  static constexpr bool kPair = true, kTall = TALL;
  static constexpr bool kAMn = true;
  static constexpr int kChunk = 0;
  static constexpr int kStageBytes = 4096;
  static constexpr int kRows = (TALL ? 4 : 2) * tc::kBM;  // words per tile
  struct Tile {};
  CUtensorMap ma;   // dz: dims (vocab, rows), box {64, 64, 1}
  CUtensorMap mb;   // x^T: dims (rows, features), box {64, tile_n / 2, 1}
  CUtensorMap mdw;  // dw: dims (features, vocab), box {64, 32, 1}, when `tma`
  long long tiles_total;
  int num_kb;
  int tile_n;  // 128 or 256 with `tma`: its boxes are 64 wide
  int vocab, features, tiles_m, tiles_n;
  int band;    // tile columns (features) that stay in L2 while dz streams past
  T* dw;
  float* sum;  // pieces: [word][sum_ld] running sum, else null
  std::int64_t sum_ld;
  bool first, last;
  bool tma;    // dw's rows are 16-byte aligned
  const float* scale;

  const CUtensorMap* __device__ map_a() const { return &ma; }
  const CUtensorMap* __device__ map_b() const { return &mb; }
  __device__ void coords(long long t, int (&c)[3]) const {
    c[0] = 0;
    banded(static_cast<int>(t), tiles_n, tiles_m, band, &c[2], &c[1]);
  }
  __device__ int k_begin(const int (&)[3]) const { return 0; }
  __device__ void begin(Tile&, const int (&)[3], int, int) const {}
  __device__ void end(Tile&, const int (&)[3], int, int, std::uint8_t*) const {}
  __device__ __forceinline__ void chunk(Tile&, const int (&c)[3], int row, int half,
                                        std::uint32_t taddr, bool, std::uint8_t* stage) const {
    const int lane = threadIdx.x & 31;
    const int w = c[1] * kRows + row;
    const int hw = c[2] * tile_n + half * (tile_n / 2);
    const float a = scale != nullptr ? scale[1] : 1.0f;
    // 64 features at a time through the stage's one box
#pragma unroll 1
    for (int b = 0; b < 2; ++b) {
      const int h0 = hw + b * 64;
      const int cols = min(min(64, tile_n / 2 - b * 64), features - h0);  // of this box
      if (cols <= 0) break;
      if (lane == 0) tc::bulk_wait_read_all();  // the previous box has left the stage
#pragma unroll 1
      for (int g = 0; g < 2; ++g) {
        if (g * 32 >= cols) break;
        float v[32];
        __syncwarp();
        tc::tmem_load_32cols(taddr + static_cast<std::uint32_t>(b * 64 + g * 32), v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= a;
        if (sum != nullptr && w < vocab) {
          float* o = sum + static_cast<std::int64_t>(w) * sum_ld + h0 + g * 32;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {  // sum's rows are whole 16-byte runs
            if (g * 32 + j >= cols) continue;
            if (!first) {
              const float4 was = *reinterpret_cast<const float4*>(o + j);
              v[j] += was.x;
              v[j + 1] += was.y;
              v[j + 2] += was.z;
              v[j + 3] += was.w;
            }
            if (!last)
              *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          std::uint8_t* box = stage + lane * 128 + (((g * 4 + k) ^ (lane & 7)) << 4);
          *reinterpret_cast<uint4*>(box) =
              make_uint4(pack2<T>(v[8 * k], v[8 * k + 1]), pack2<T>(v[8 * k + 2], v[8 * k + 3]),
                         pack2<T>(v[8 * k + 4], v[8 * k + 5]), pack2<T>(v[8 * k + 6], v[8 * k + 7]));
        }
      }
      if (!last) continue;
      if (tma) {
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && w < vocab) {  // lane 0 has the warp's first word
          tc::tma_store_3d(&mdw, stage, h0, w, 0);
          tc::bulk_commit();
        }
      } else {
        __syncwarp();
        const int rows = min(32, vocab - (w - lane));
        for (int r = 0; r < rows; ++r) {
          T* o = dw + static_cast<std::int64_t>(w - lane + r) * features + h0;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int col = i * 32 + lane;
            const T* e =
                reinterpret_cast<const T*>(stage + r * 128 + (((col >> 3) ^ (r & 7)) << 4));
            if (col < cols) o[col] = e[col & 7];
          }
        }
        __syncwarp();
      }
    }
  }
};

// ------------------------------------------------------------------------- planning --
// Bytes of a piece's numerators.  Every further piece reads and writes dw's fp32 sum: 16384 x
// 1024 x 131072 took 11.9 ms in one piece of 4 GiB or two of 2 GiB, 12.7 in four of 1 GiB.
constexpr std::size_t kNumeratorCap = std::size_t{2} << 30;
// Bytes of everything else that grows with a piece's tokens, and its tokens.  The tokens also
// bound dw's sums: within a piece the tensor cores truncate, pieces add in fp32.
constexpr std::size_t kGradientCap = std::size_t{960} << 20, kScoreCap = std::size_t{224} << 20;
constexpr int kGradientRows = 32768, kScoreRows = 16384;
constexpr int kLeastRows = 128;

// Elements of a 128-byte line: rows that start on one cost the loads of a 64-wide box one
// line each, others two.
constexpr int kLine = 64;

std::int64_t round_up(std::int64_t v, std::int64_t m) { return (v + m - 1) / m * m; }

int sms() {
  const int n = sm_count(current_device());
  return n > 0 ? n : 148;
}

// Width of the tiles of `cols` columns in `rows` tile rows on `groups` CTAs or pairs: the
// multiple of `step` whose waves end soonest.  A k-block of a 256 x n pair tile takes about
// 256 + n clocks (below 256 columns shared memory, not the MMAs, sets the pace), of a single
// CTA's tile n times what one word's line takes to arrive.
int tile_width(std::int64_t rows, int cols, int groups, int step, bool pair) {
  int best = tc::kEpiN;
  std::int64_t least = INT64_MAX;
  for (int n = tc::kEpiN; n >= step; n -= step) {
    const std::int64_t tiles = rows * ((cols + n - 1) / n);
    const std::int64_t cost = (tiles + groups - 1) / groups * (pair ? 256 + n : n);
    if (cost < least) {
      least = cost;
      best = n;
    }
  }
  return best;
}

// Words per tile of the logits; stored numerators need units (half tiles) of 64 or 128.
int logits_tile_n(int rows, int vocab, bool store) {
  const bool pair = rows > tc::kBM;
  return tile_width(pair ? (rows + 255) / 256 : 1, vocab, pair ? sms() / 2 : sms(),
                    store ? 128 : 32, pair);
}

// Columns per tile: as few tiles as 256 columns need, of even width.
int even_tile_n(int cols) {
  const int tiles = (cols + tc::kEpiN - 1) / tc::kEpiN;
  return static_cast<int>(round_up((cols + tiles - 1) / tiles, 32));
}

// dx on tall tiles: for a vocabulary that makes K long against the drain of a tile and dz too
// large for L2.  Measured (loss and dx, flat and tall): 2048 x 2048 x 16384 212-241 and 247 us,
// x 32768 479 and 492; 4096 x 4096 x 65536 3644 and 3503; the bound lies between the last two.
// Widths that leave part of a 512-row tile empty (768, 1280) go by the same rule, unmeasured.
bool dx_tall(int vocab) { return vocab >= 49152; }

// Most words that dx adds up in one chain of truncating MMAs.  Each loses up to half a unit in
// the sum's last place, all toward zero, and with one large term (the target's) early in the
// sum they add up: over 110000 words 1.3e-4 of dx, beside 3.0e-4 from fp16's two roundings and
// 2.4e-3 from bf16's.  A split of this length stays below an eighth of them.
int dx_chain(bool bf16) { return bf16 ? 262144 : 32768; }

// Splits of the words in dx's product: the count that ends soonest.  A k-block takes 512
// clocks of MMAs per 256 x 256 on a pair; a single CTA's streams w at its share of memory
// bandwidth (measured 5.5 TB/s).  Each split's partial sums are written and read once, by one
// more launch.  No split is longer than dx_chain.
int dx_splits(int rows, int features, int vocab, bool bf16) {
  const bool pair = rows > tc::kBM;
  const int bm = dx_tall(vocab) ? 512 : 256;
  const std::int64_t tiles =
      pair ? static_cast<std::int64_t>((features + bm - 1) / bm) * ((rows + 255) / 256)
           : (features + tc::kBM - 1) / tc::kBM;
  const int kb = (vocab + tc::kBK - 1) / tc::kBK;
  const int n = pair ? sms() / 2 : sms();
  const double block = pair ? bm * 2 / 1.6e9 * even_tile_n(rows) / tc::kEpiN
                            : tc::kBM * tc::kRowBytes * n / 5.5e12;
  const int least = (vocab + dx_chain(bf16) - 1) / dx_chain(bf16);
  double best = 0.0;
  int pick = least;
  for (int ks = least; ks == least || (ks <= 32 && ks * 8 <= kb); ++ks) {
    const double waves = static_cast<double>((tiles * ks + n - 1) / n);
    const double loop = waves * ((kb + ks - 1) / ks) * block;
    const double join = ks == 1 ? 0.0 : 6e-6 + 8.0 * ks * rows * features / 4.5e12;
    if (ks == least || loop + join < best) {
      best = loop + join;
      pick = ks;
    }
  }
  return pick;
}

// Tile rows (of tile_bytes each) per band: what L2 keeps, in bands of equal height.
int band_of(int tiles, std::int64_t tile_bytes, std::int64_t keep) {
  const std::int64_t most = std::max<std::int64_t>(1, keep / tile_bytes);
  const std::int64_t bands = (tiles + most - 1) / most;
  return static_cast<int>((tiles + bands - 1) / bands);
}

bool tma_rows_ok(const void* p, std::int64_t ld) { return aligned_to(p, 16) && ld % 8 == 0; }

// Bytes of a copy of some words at a time, for a w that needs one in a workspace without room
// for all of it.
constexpr std::size_t kSliceBytes = std::size_t{16} << 20;

struct Plan {
  bool stream;  // scores of few tokens (vocab_stream_kernel)
  StoreMode store;
  int unit, units;  // words per pair of the logits (stream: per round), pairs per token
  int hit_units;    // entries of a token's hit map
  int rows;    // tokens per piece (the last may have fewer)
  int pieces;
  int ksplit;
  int copies;         // rows of dz per token: 2 for kSplit
  std::int64_t ldn;   // numerators' row
  std::int64_t ldt;   // x^T's row
  std::int64_t ldp;   // row of packed copies of x and w
  bool pack_x, pack_w;
  int slice;          // words of w that are packed at a time; without pack_w all
  int lefts;          // entries per token of what the targets' rounding left
  // byte offsets into the workspace
  std::size_t stats, z, index, q, count, entropy, hit, scale, row_scale, left, xp, wp, num, xt,
      partial, sum, bytes;
  std::size_t rows_bytes;  // of them, what grows with the tokens, without the numerators
};

Plan plan_rows(const VocabLossArgs& a, int rows, bool sliced) {
  Plan p{};
  p.rows = rows;
  p.pieces = (a.tokens + rows - 1) / rows;
  p.ldn = round_up(a.vocab, kLine);
  p.ldp = round_up(a.features, kLine);
  p.pack_x = a.tokens > 1 ? !tma_rows_ok(a.x, a.ldx) : !aligned_to(a.x, 16);
  p.pack_w = !tma_rows_ok(a.w, a.features);
  // x is read once per 256 words: a copy with rows on lines pays at once (1537 x 1000 x
  // 50021: 532 -> 520 us).  A copy of w does not (520 -> 508..548 us, and 178 -> 219 at 300
  // tokens).
  if (rows > tc::kBM && a.ldx % kLine != 0) p.pack_x = true;
  const bool dx = a.gradients && a.dx != nullptr, dw = a.gradients && a.dw != nullptr;
  std::size_t at = 0;
  auto take = [&](std::size_t n) {
    const std::size_t o = at;
    at += (n + 255) / 256 * 256;
    return o;
  };
  const std::size_t R = rows, H = a.features, V = a.vocab, K = a.top_k;
  p.store = !a.gradients           ? kNone
            : rows <= kSplitTokens ? kSplit
            : dw || !a.bf16        ? kOwn
                                   : kCommon;
  p.copies = p.store == kSplit ? 2 : 1;
  p.ldt = round_up(p.copies * rows, kLine);
  p.stream = !a.gradients && a.tokens <= kStreamTokens && !p.pack_w;
  p.unit = p.stream ? kStreamWords : logits_tile_n(rows, a.vocab, a.gradients) / 2;
  p.units = p.stream ? sms() : (a.vocab + p.unit - 1) / p.unit;
  p.hit_units = (a.vocab + p.unit - 1) / p.unit;
  p.slice = a.vocab;
  if (p.pack_w && sliced) {  // whole tiles of the logits, whole k-blocks of dx
    const int whole = 4 * p.unit;
    const auto words = static_cast<int>(kSliceBytes / (p.ldp * 2)) / whole * whole;
    p.slice = std::min(a.vocab, std::max(whole, words));
  }
  p.ksplit = dx ? dx_splits(rows, a.features, p.slice, a.bf16) : 1;
  p.stats = take(R * p.units * sizeof(float2));
  p.z = take(R * std::max<std::size_t>(K, 1) * 4);
  p.index = take(R * K * 4);
  p.q = take(R * K * 4);
  p.count = take(K > 0 ? R * 4 : 0);
  p.entropy = take(K > 0 ? R * 4 : 0);
  p.hit = take(K > 0 ? R * p.hit_units * 4 : 0);
  p.scale = take(8);
  p.row_scale = take(a.gradients ? R * sizeof(float2) : 0);
  p.lefts = dx && p.store != kSplit && K <= kMostLeft ? std::max(a.top_k, 1) : 0;
  p.left = take(R * p.lefts * sizeof(Left));
  p.xp = take(p.pack_x ? R * p.ldp * 2 : 0);
  const std::size_t wp = p.pack_w ? static_cast<std::size_t>(p.slice) * p.ldp * 2 : 0;
  const std::size_t num = a.gradients ? p.copies * R * p.ldn * 2 : 0;
  const std::size_t sum = dw && p.pieces > 1 ? V * round_up(a.features, 4) * 4 : 0;
  p.wp = take(wp);
  p.num = take(num);
  p.xt = take(dw ? H * p.ldt * 2 : 0);
  p.partial = take(p.ksplit > 1 || (dx && p.slice < a.vocab) ? p.ksplit * R * H * 4 : 0);
  p.sum = take(sum);
  p.bytes = at;
  p.rows_bytes = at - num - wp - sum;
  return p;
}

// Pieces of equal size, each at most what the caps allow; in a workspace that has no room for
// dw's sum between them but for all tokens at once, one piece.  A copy of w is made in slices
// where the workspace has no room for all of it, or where `sliced` says so.
Plan plan_within(const VocabLossArgs& a, std::size_t limit, bool sliced, bool* ok) {
  const std::size_t cap = a.gradients ? kGradientCap : kScoreCap;
  // a token's pairs (and hits), and its share of x^T; the loop below sees to the rest
  const std::size_t per_row = (a.vocab + 127ull) / 128 * (a.top_k > 0 ? 12 : 8) +
                              (a.gradients ? 2ull * a.features : 0);
  std::int64_t most = a.gradients ? kGradientRows : kScoreRows;
  most = std::min(most, static_cast<std::int64_t>(cap / per_row));
  if (a.gradients)
    most = std::min(most, static_cast<std::int64_t>(kNumeratorCap / (round_up(a.vocab, kLine) * 2)));
  most = std::max<std::int64_t>(kLeastRows, most / kLeastRows * kLeastRows);
  int pieces = static_cast<int>((a.tokens + most - 1) / most);
  Plan p{};
  for (;;) {
    std::int64_t rows = (a.tokens + pieces - 1) / pieces;
    if (pieces > 1) rows = round_up(rows, kLeastRows);
    for (int s = sliced; s < 2; ++s) {
      p = plan_rows(a, static_cast<int>(std::min<std::int64_t>(rows, a.tokens)), s != 0);
      if (p.bytes <= limit && (p.rows_bytes <= cap || rows <= kLeastRows)) {
        *ok = true;
        return p;
      }
    }
    if (rows <= kLeastRows) break;
    // the next count that makes a piece smaller
    rows -= kLeastRows;
    pieces = static_cast<int>((a.tokens + rows - 1) / rows);
  }
  const Plan whole = plan_rows(a, a.tokens, true);
  *ok = whole.bytes <= limit;
  return *ok ? whole : p;
}

// Map of 16-bit elements: `inner` contiguous, `outer` rows of ld elements.
bool make_map(CUtensorMap* map, int fmt, const void* base, std::int64_t inner, std::int64_t outer,
              std::int64_t ld, int box_inner, int box_outer) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer), 1u};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld * 2),
                                 static_cast<cuuint64_t>(round_up(ld * 2, 16))};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer),
                             1u};
  return tc::encode_tiled(map, fmt, base, 3, dims, strides, box);
}

unsigned int* timeout_counter() {
  static std::mutex mu;
  static std::array<unsigned int*, 64> addr{};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return nullptr;
  std::lock_guard<std::mutex> g(mu);
  if (addr[dev] == nullptr) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_vocab_timeouts) != cudaSuccess) {
      (void)cudaGetLastError();
      return nullptr;
    }
    addr[dev] = static_cast<unsigned int*>(p);
  }
  return addr[dev];
}

template <typename T, int FMT, bool PAIR, int STORE, int CHUNK>
cudaError_t run_logits(const LogitsProblem& p, unsigned int* timeouts, cudaStream_t st,
                       bool overlap) {
  using Problem = Logits<T, PAIR, STORE, CHUNK>;
  Problem q;
  static_cast<LogitsProblem&>(q) = p;
  return tc::launch_tc_epi<Problem, FMT>(q, sms(), timeouts, st, overlap);
}

#define MB200_TRY(expr)                       \
  do {                                        \
    const cudaError_t e_ = (expr);            \
    if (e_ != cudaSuccess) return e_;         \
  } while (0)

// dx of the `words` words from word0 on (w is theirs); the slices of a call add up in partial.
template <typename T, int FMT, bool PAIR, bool TALL, bool SPLIT>
cudaError_t run_dx(const VocabLossArgs& a, const Plan& p, const T* w, std::int64_t ldw,
                   int word0, int words, const T* num, int rows, T* dx, char* ws,
                   unsigned int* to, cudaStream_t st) {
  using Problem = Dx<T, PAIR, TALL, SPLIT>;
  Problem g{};
  const int dz_rows = p.copies * rows;
  g.tile_n = even_tile_n(dz_rows);
  if (!make_map(&g.ma, FMT, w, a.features, words, ldw, 64, 64) ||
      !make_map(&g.mb, FMT, num + word0, words, dz_rows, p.ldn, 64,
                PAIR ? g.tile_n / 2 : g.tile_n))
    return cudaErrorInvalidValue;
  // splits of a whole slice; the last, shorter one has no more of them
  const auto blocks = [](int n) { return (n + tc::kBK - 1) / tc::kBK; };
  g.num_kb = (blocks(p.slice) + p.ksplit - 1) / p.ksplit;
  const int ks = (blocks(p.slice) + g.num_kb - 1) / g.num_kb;  // no split without words
  constexpr int kRows = Problem::kRows;
  g.rows = rows;
  g.features = a.features;
  g.tiles_m = (a.features + kRows - 1) / kRows;
  g.tiles_n = (dz_rows + g.tile_n - 1) / g.tile_n;
  g.tiles_total = static_cast<long long>(g.tiles_m) * g.tiles_n *
                  ((blocks(words) + g.num_kb - 1) / g.num_kb);
  g.dx = dx;
  g.lddx = a.lddx;
  const bool parts = ks > 1 || p.slice < a.vocab;
  g.partial = parts ? reinterpret_cast<float*>(ws + p.partial) : nullptr;
  g.add = word0 > 0;
  g.row_scale = reinterpret_cast<float2*>(ws + p.row_scale);
  g.left = reinterpret_cast<const Left*>(ws + p.left);
  g.lefts = parts ? 0 : p.lefts;
  g.w = static_cast<const T*>(a.w);
  MB200_TRY((tc::launch_tc_epi<Problem, FMT>(g, sms(), to, st, true)));
  if (parts && word0 + words == a.vocab) {
    const bool vec = a.features % 4 == 0 && a.lddx % 4 == 0 && aligned_to(dx, 8);
    const std::int64_t work = static_cast<std::int64_t>(rows) * a.features / (vec ? 4 : 1);
    const unsigned grid =
        static_cast<unsigned>(std::min<std::int64_t>((work + 255) / 256, sms() * 32));
    MB200_TRY(tc::launch_overlapped(
        vec ? vocab_dx_reduce_kernel<T, 4> : vocab_dx_reduce_kernel<T, 1>, dim3(grid), 256, 0, st, true,
        g.partial, ks, rows, a.features, dx, a.lddx, g.row_scale, g.left, p.lefts, g.w));
  }
  return cudaSuccess;
}

// dw on tall tiles: a tall tile drains before its successor starts (about 3000 clocks), but
// reads 3/4 of the operands.  Measured at 65536 x 4096, 2048 tokens: 684 us flat, 746 tall;
// 4096: 1367 and 1404; 8192: 3038 and 2836 (x^T no longer fits L2: 6.9 and 4.5 GB of reads);
// the bound is the middle of the last two.
constexpr int kTallTokens = 6144;

template <typename T, int FMT, bool TALL>
cudaError_t run_dw(const VocabLossArgs& a, const Plan& p, const void* num, const void* xt, int rows,
                   int piece, char* ws, const float* scale, unsigned int* to, cudaStream_t st) {
  Dw<T, TALL> g{};
  g.tma = tma_rows_ok(a.dw, a.features);
  constexpr int kRows = Dw<T, TALL>::kRows;
  g.tile_n = tile_width((a.vocab + kRows - 1) / kRows, a.features, sms() / 2, g.tma ? 128 : 32,
                        true);
  const int dz_rows = p.copies * rows;
  if (!make_map(&g.ma, FMT, num, a.vocab, dz_rows, p.ldn, 64, 64) ||
      !make_map(&g.mb, FMT, xt, dz_rows, a.features, p.ldt, tc::kBK, g.tile_n / 2) ||
      (g.tma && !make_map(&g.mdw, FMT, a.dw, a.features, a.vocab, a.features, 64, 32)))
    return cudaErrorInvalidValue;
  g.num_kb = (dz_rows + tc::kBK - 1) / tc::kBK;
  g.vocab = a.vocab;
  g.features = a.features;
  g.tiles_m = (a.vocab + kRows - 1) / kRows;
  g.tiles_n = (a.features + g.tile_n - 1) / g.tile_n;
  g.tiles_total = static_cast<long long>(g.tiles_m) * g.tiles_n;
  // measured at 8192 x 4096 x 65536: 33 MB of x^T kept 5.2 GB of DRAM reads, 67 MB 4.4
  g.band = band_of(g.tiles_n, 512ll * rows, 72ll << 20);
  g.dw = static_cast<T*>(a.dw);
  g.sum = p.pieces > 1 ? reinterpret_cast<float*>(ws + p.sum) : nullptr;
  g.sum_ld = round_up(a.features, 4);
  g.first = piece == 0;
  g.last = piece == p.pieces - 1;
  g.scale = scale;
  return tc::launch_tc_epi<Dw<T, TALL>, FMT>(g, sms(), to, st, true);
}

template <typename T, int FMT>
cudaError_t run(const VocabLossArgs& a, const Plan& p, char* ws, cudaStream_t st) {
  unsigned int* to = timeout_counter();
  if (to == nullptr) return cudaErrorInvalidDevice;
  // the call's first kernel starts when the stream reaches it, the others overlap
  bool overlap = false;
  const auto launch = [&](auto kern, long long ctas, int threads, auto... args) {
    return tc::launch_overlapped(kern, dim3(static_cast<unsigned>(ctas)), threads, 0, st,
                                 std::exchange(overlap, true), args...);
  };
  // the words from word0 on that the products below read at a time
  const T* w = static_cast<const T*>(a.w);
  const std::int64_t ldw = p.pack_w ? p.ldp : a.features;
  const auto words_from = [&](int word0) { return std::min(p.slice, a.vocab - word0); };
  const auto load_slice = [&](int word0) {
    if (!p.pack_w) return cudaSuccess;
    w = reinterpret_cast<T*>(ws + p.wp);
    return launch(vocab_pack_kernel<T>, sms() * 8, 256,
                  static_cast<const T*>(a.w) + static_cast<std::int64_t>(word0) * a.features,
                  static_cast<std::int64_t>(a.features), words_from(word0), a.features,
                  reinterpret_cast<T*>(ws + p.wp), p.ldp);
  };
  const bool sliced = p.slice < a.vocab;
  if (!sliced) MB200_TRY(load_slice(0));
  T* num = reinterpret_cast<T*>(ws + p.num);
  for (int piece = 0; piece < p.pieces; ++piece) {
    const std::int64_t t0 = static_cast<std::int64_t>(piece) * p.rows;
    const int rows = static_cast<int>(std::min<std::int64_t>(p.rows, a.tokens - t0));
    const T* x = static_cast<const T*>(a.x) + t0 * a.ldx;
    std::int64_t ldx = a.tokens > 1 ? a.ldx : p.ldp;  // one row: its stride is never used
    if (p.pack_x) {
      T* xp = reinterpret_cast<T*>(ws + p.xp);
      MB200_TRY(launch(vocab_pack_kernel<T>, sms() * 8, 256, x, ldx, rows, a.features, xp,
                       p.ldp));
      x = xp;
      ldx = p.ldp;
    }
    Targets tg{};
    tg.top_k = a.top_k;
    tg.z = reinterpret_cast<float*>(ws + p.z);
    if (a.top_k == 0) {
      tg.labels = a.labels + t0;
    } else {
      int* index = reinterpret_cast<int*>(ws + p.index);
      float* q = reinterpret_cast<float*>(ws + p.q);
      int* count = reinterpret_cast<int*>(ws + p.count);
      float* ent = reinterpret_cast<float*>(ws + p.entropy);
      auto* hit = reinterpret_cast<std::uint32_t*>(ws + p.hit);
      MB200_TRY(launch(vocab_targets_kernel, (rows + kTargetWarps - 1) / kTargetWarps,
                       32 * kTargetWarps, a.teacher_index + t0 * a.top_k,
                       a.teacher_logits + t0 * a.top_k, rows, a.top_k, a.vocab, a.inv_tau, index,
                       q, count, ent, hit, p.hit_units, p.unit));
      tg.index = index;
      tg.q = q;
      tg.count = count;
      tg.neg_entropy = ent;
      tg.hit = hit;
      tg.hit_units = p.hit_units;
    }

    float* scale = nullptr;
    if (a.gradients && !a.bf16) {
      scale = reinterpret_cast<float*>(ws + p.scale);
      MB200_TRY(launch(vocab_grad_scale_kernel, 1, 1024, a.dloss + t0, rows, a.vocab, tg,
                       a.inv_tau, scale));
    }

    FinishArgs f{};
    f.rows = rows;
    f.parts = 1;
    f.stats = reinterpret_cast<float2*>(ws + p.stats);
    f.units = p.units;
    f.unit = p.unit;
    f.vocab = a.vocab;
    f.targets = tg;
    f.loss = a.loss != nullptr ? a.loss + t0 : nullptr;
    f.lse = a.lse != nullptr ? a.lse + t0 : nullptr;
    f.inv_tau = a.inv_tau;
    f.log2e_tau = kLog2e * a.inv_tau;
    f.scale = scale;
    f.num = num;
    f.ldn = p.ldn;
    f.pitch = p.copies * p.ldn;
    if (p.stream) {
      const StreamArgs sa{x, ldx, w, ldw, rows, a.features, a.vocab, kLog2e * a.inv_tau,
                          reinterpret_cast<float2*>(ws + p.stats), tg};
      MB200_TRY(launch(vocab_stream_kernel<T>, p.units, kStreamThreads, sa));
      MB200_TRY(launch(vocab_finish_kernel<T, kNone>, rows, kFinishThreads, f));
      continue;
    }

    const bool pair = rows > tc::kBM;
    LogitsProblem lp{};
    lp.tile_n = 2 * p.unit;
    if (!make_map(&lp.mx, FMT, x, a.features, rows, ldx, tc::kBK, tc::kBM) ||
        (a.gradients && !make_map(&lp.mnum, FMT, num, p.ldn, rows, p.copies * p.ldn, 64, 32)))
      return cudaErrorInvalidValue;
    lp.num_kb = (a.features + tc::kBK - 1) / tc::kBK;
    lp.rows = rows;
    lp.vocab = a.vocab;
    lp.unit = p.unit;
    lp.units = p.units;
    lp.tiles_m = pair ? (rows + 2 * tc::kBM - 1) / (2 * tc::kBM) : 1;
    // measured at 8192 x 4096 x 65536: 16 MB of x kept 3.2 GB of DRAM reads, 33 MB 2.0, 50 MB
    // 3.3, all 67 MB 4.5 (the numerators pass through L2 too)
    lp.band = band_of(lp.tiles_m, 512ll * a.features, 36ll << 20);
    lp.scale = kLog2e * a.inv_tau;
    lp.stats = reinterpret_cast<float2*>(ws + p.stats);
    lp.ldn = p.ldn;
    lp.targets = tg;
    // enough CTAs to fill the GPU when there are few rows, each one round of 2048 words at least
    const int parts =
        std::max(1, std::min<int>(4 * sms() / rows, static_cast<int>((p.ldn + 2047) / 2048)));
    const auto logits = [&](auto store) {
      constexpr int kStore = decltype(store)::value;
      for (lp.word0 = 0; lp.word0 < a.vocab; lp.word0 += p.slice) {
        const int words = words_from(lp.word0);
        if (sliced) MB200_TRY(load_slice(lp.word0));
        if (!make_map(&lp.mw, FMT, w, a.features, words, ldw, tc::kBK,
                      pair ? lp.tile_n / 2 : lp.tile_n))
          return cudaErrorInvalidValue;
        lp.tiles_n = (words + lp.tile_n - 1) / lp.tile_n;
        lp.tiles_total = static_cast<long long>(lp.tiles_m) * lp.tiles_n;
        const auto form = pair                     ? run_logits<T, FMT, true, kStore, kLogitsChunk>
                          : rows <= kStreamTokens ? run_logits<T, FMT, false, kStore, kFewLogitsChunk>
                                                  : run_logits<T, FMT, false, kStore, kLogitsChunk>;
        MB200_TRY(form(lp, to, st, overlap));
        overlap = true;
      }
      return cudaSuccess;
    };
    if (p.store == kNone) {
      MB200_TRY(logits(std::integral_constant<int, kNone>{}));
      MB200_TRY(launch(vocab_finish_kernel<T, kNone>, rows, kFinishThreads, f));
      continue;
    }
    f.dloss = a.dloss + t0;
    f.row_scale = reinterpret_cast<float2*>(ws + p.row_scale);
    f.left = p.lefts > 0 ? reinterpret_cast<Left*>(ws + p.left) : nullptr;
    f.parts = parts;
    T* xt = reinterpret_cast<T*>(ws + p.xt);
    long long tiles = 0;
    if (a.dw != nullptr) {  // before dx, which may be x itself
      f.transpose = {x, ldx, rows, a.features, tma_rows_ok(x, ldx), xt, p.ldt};
      tiles = static_cast<long long>((rows + 63) / 64) * ((a.features + 63) / 64);
    }
    const long long finish = static_cast<long long>(rows) * parts;
    if (p.store == kOwn || p.store == kSplit) {
      MB200_TRY(logits(std::integral_constant<int, kOwn>{}));
      MB200_TRY(launch(p.store == kOwn ? vocab_finish_kernel<T, kOwn> : vocab_finish_kernel<T, kSplit>,
                       finish + tiles, kFinishThreads, f));
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      MB200_TRY(logits(std::integral_constant<int, kCommon>{}));
      MB200_TRY(launch(vocab_finish_kernel<T, kCommon>, finish, kFinishThreads, f));
    }

    if (a.dx != nullptr) {
      T* dx = static_cast<T*>(a.dx) + t0 * a.lddx;
      for (int word0 = 0; word0 < a.vocab; word0 += p.slice) {
        if (sliced) MB200_TRY(load_slice(word0));
        const auto product = [&](auto kern) {
          return kern(a, p, w, ldw, word0, words_from(word0), num, rows, dx, ws, to, st);
        };
        MB200_TRY(product(p.store == kSplit  ? run_dx<T, FMT, false, false, true>
                          : !pair            ? run_dx<T, FMT, false, false, false>
                          : dx_tall(p.slice) ? run_dx<T, FMT, true, true, false>
                                             : run_dx<T, FMT, true, false, false>));
      }
    }
    if (a.dw != nullptr) {
      if (rows >= kTallTokens)
        MB200_TRY((run_dw<T, FMT, true>(a, p, num, xt, rows, piece, ws, scale, to, st)));
      else
        MB200_TRY((run_dw<T, FMT, false>(a, p, num, xt, rows, piece, ws, scale, to, st)));
    }
  }
  return cudaSuccess;
}

}  // namespace

std::size_t vocab_loss_workspace(const VocabLossArgs& a) noexcept {
  bool ok = false;
  return plan_within(a, SIZE_MAX, false, &ok).bytes;
}

std::size_t vocab_loss_workspace_any(const VocabLossArgs& a) noexcept {
  std::size_t most = 0;
  for (const std::uintptr_t x : {256, 2}) {
    for (const std::uintptr_t w : {256, 2}) {
      VocabLossArgs b = a;
      b.x = reinterpret_cast<const void*>(x);
      b.w = reinterpret_cast<const void*>(w);
      // all of w is copied only where its rows ask for it, not its address alone
      bool ok = false;
      most = std::max(most, plan_within(b, SIZE_MAX, a.features % 8 == 0, &ok).bytes);
    }
  }
  return most;
}

std::size_t vocab_loss_min_workspace(const VocabLossArgs& a) noexcept {
  bool ok = false;
  return std::min({plan_rows(a, std::min(a.tokens, kLeastRows), true).bytes,
                   plan_rows(a, a.tokens, true).bytes,
                   plan_within(a, SIZE_MAX, true, &ok).bytes});
}

cudaError_t launch_vocab_loss(const VocabLossArgs& a, void* ws, std::size_t ws_bytes,
                              cudaStream_t stream) noexcept {
  bool ok = false;
  const Plan p = plan_within(a, ws_bytes, false, &ok);
  if (!ok) return cudaErrorInvalidValue;
  return a.bf16 ? run<__nv_bfloat16, 1>(a, p, static_cast<char*>(ws), stream)
                : run<__half, 0>(a, p, static_cast<char*>(ws), stream);
}

}  // namespace mb200::dnn
