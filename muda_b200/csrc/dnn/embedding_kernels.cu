// embedding_kernels.cu — embedding lookup and its gradient.  The mathematics is stated in
// embedding.hpp.  Both are bound by memory: the lookup reads a table row and writes a row per
// token; the gradient reads every row of dy once and writes all of dw (beta 0) or the rows of
// the words that occur (beta 1).
//
// The gradient adds each word's rows in the order of their positions, without atomics, so
// results are the same on every run.  Three launches:
//   1. embedding_sort_kernel orders the tokens by word, positions ascending within a word;
//   2. embedding_partial_kernel cuts the ordered tokens into blocks and adds up, in fp32, the
//      blocks' shares of words that occur more often than a block is long;
//   3. embedding_rows_kernel adds each word's rows, or the partial sums of a frequent one,
//      and writes its row of dw, zeros (or beta dw) for words that do not occur.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "blas/tc_epi_core.cuh"
#include "common/device.hpp"
#include "dnn/embedding.hpp"

namespace mb200::dnn {
namespace {

int sms() {
  const int n = sm_count(current_device());
  return n > 0 ? n : 148;
}

template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same_v<T, float>)
    return v;
  else if constexpr (std::is_same_v<T, __half>)
    return __float2half_rn(v);
  else
    return __float2bfloat16_rn(v);
}

// VEC elements of a row as they lie in memory: whole 16-byte words, or one element.
template <typename T, int VEC>
struct alignas(VEC == 1 ? sizeof(T) : 16) Run {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Run<T, VEC> load_run(const T* p) {
  Run<T, VEC> r;
  if constexpr (VEC == 1) {
    r.v[0] = *p;
  } else {
    constexpr int kWords = sizeof(T) * VEC / 16;
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  return r;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_run(T* p, const Run<T, VEC>& r) {
  if constexpr (VEC == 1) {
    *p = r.v[0];
  } else {
    constexpr int kWords = sizeof(T) * VEC / 16;
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      __stcs(reinterpret_cast<uint4*>(p) + i, reinterpret_cast<const uint4*>(&r)[i]);
  }
}

// ------------------------------------------------------------------------- lookup --
constexpr int kLookupThreads = 256;

template <typename TW, typename TY, int VEC, int RUNS>
__global__ void __launch_bounds__(kLookupThreads)
    embedding_kernel(const TW* __restrict__ w, const std::int64_t* __restrict__ token, TY* y,
                     std::int64_t ldy, int tokens, int features, int vocab, float alpha,
                     float beta) {
  const unsigned per = features / VEC;  // runs of a row
  const std::int64_t first = static_cast<std::int64_t>(blockIdx.x) * (kLookupThreads * RUNS);
  const std::int64_t row0 = first / per;
  const unsigned skip = static_cast<unsigned>(first - row0 * per) + threadIdx.x;
  Run<TW, VEC> in[RUNS];
  std::int64_t row[RUNS], word[RUNS];
  unsigned col[RUNS];
#pragma unroll
  for (int j = 0; j < RUNS; ++j) {
    const unsigned i = skip + j * kLookupThreads;
    const unsigned q = i / per;
    row[j] = row0 + q;
    col[j] = (i - q * per) * VEC;
    word[j] = row[j] < tokens ? token[row[j]] : -1;
  }
#pragma unroll
  for (int j = 0; j < RUNS; ++j) {
    if (word[j] >= 0 && word[j] < vocab) {
      in[j] = load_run<TW, VEC>(w + word[j] * features + col[j]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) in[j].v[e] = from_float<TW>(word[j] < 0 ? 0.0f : NAN);
    }
  }
#pragma unroll
  for (int j = 0; j < RUNS; ++j) {
    if (row[j] >= tokens) break;
    TY* o = y + row[j] * ldy + col[j];
    Run<TY, VEC> out, was;
    if (beta != 0.0f) was = load_run<TY, VEC>(o);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float v = alpha * static_cast<float>(in[j].v[e]);
      if (word[j] < 0) v = 0.0f;
      if (beta != 0.0f) v = fmaf(beta, static_cast<float>(was.v[e]), v);
      out.v[e] = from_float<TY>(v);
    }
    store_run<TY, VEC>(o, out);
  }
}

// ---------------------------------------------------------------------- the order --
// CTA c owns the words v with v % kOwners == c (frequent words are neighbours in most
// vocabularies, so ranges of words would leave one CTA most of the tokens).  Every CTA reads
// all tokens: it counts those of the owners before it, which gives the place of its own in the
// ordered list, and takes its own in position order; then it sorts them by word in passes of
// kDigit bits.  A warp goes over its own contiguous share of the list in both steps, so
// equal words keep their order, whatever the split between the warps.  No CTA waits for
// another.
constexpr int kOwners = 128, kOwnerBits = 7;
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kDigit = 5;
constexpr int kSharedList = 2048;  // entries that are sorted in shared memory
constexpr int kScanAhead = 8;      // loads in flight per lane

struct Entry {
  int word;  // v / kOwners
  int pos;
};

struct SortArgs {
  const std::int64_t* token;
  int tokens, vocab;
  int per_owner;  // words of an owner, at most
  int passes;
  Entry* list[2];  // [tokens] each: longer lists while they are sorted
  int* word;       // [tokens] out: the words in order
  int* pos;        // [tokens] out: and their positions
  int2* span;      // [owner][per_owner] out: a word's entries, {0, 0}: none
  int* total;      // out: entries
};

__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// v summed over the threads before this one; *all: over all threads.
__device__ __forceinline__ int block_exclusive(int v, int* warps, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += u;
  }
  __syncthreads();  // warps[] may still be read by the previous scan
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  int w = warps[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  *all = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return sum - v + (warp > 0 ? before : 0);
}

__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const SortArgs a) {
  __shared__ Entry near[2][kSharedList];
  __shared__ int count[1 << kDigit][kSortWarps + 1];  // a warp's counters in banks of their own
  __shared__ int warps[32];
  tc::grid_launch_next();
  tc::grid_wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int owner = blockIdx.x;
  const unsigned before_me = (1u << lane) - 1;

  int2* span = a.span + static_cast<std::int64_t>(owner) * a.per_owner;
  for (int i = threadIdx.x; i < a.per_owner; i += kSortThreads) span[i] = make_int2(0, 0);

  // the warp's share of the tokens; owner_of is -1 for tokens that enter nothing
  const int share = ((a.tokens + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
  const std::int64_t t0 = static_cast<std::int64_t>(warp) * share;
  const std::int64_t t1 = min(t0 + share, static_cast<std::int64_t>(a.tokens));
  const auto load = [&](std::int64_t t) -> int {
    if (t >= t1) return -1;
    const std::int64_t v = a.token[t];
    return v >= 0 && v < a.vocab ? static_cast<int>(v) : -1;
  };
  int mine = 0, below = 0;
  for (std::int64_t t = t0; t < t1; t += 32 * kScanAhead) {
    int v[kScanAhead];
#pragma unroll
    for (int j = 0; j < kScanAhead; ++j) v[j] = load(t + 32 * j + lane);
#pragma unroll
    for (int j = 0; j < kScanAhead; ++j) {
      const int o = v[j] & (kOwners - 1);
      mine += v[j] >= 0 && o == owner;
      below += v[j] >= 0 && o < owner;
    }
  }
  mine = warp_sum(mine);
  int base, n;
  (void)block_exclusive(below, warps, &base);
  int at = block_exclusive(lane == 0 ? mine : 0, warps, &n);
  at = __shfl_sync(0xffffffffu, at, 0);
  if (owner == kOwners - 1 && threadIdx.x == 0) *a.total = base + n;

  Entry* from = n <= kSharedList ? near[0] : a.list[0] + base;
  Entry* to = n <= kSharedList ? near[1] : a.list[1] + base;
  if (mine > 0) {
    for (std::int64_t t = t0; t < t1; t += 32 * kScanAhead) {
      int v[kScanAhead];
#pragma unroll
      for (int j = 0; j < kScanAhead; ++j) v[j] = load(t + 32 * j + lane);
#pragma unroll
      for (int j = 0; j < kScanAhead; ++j) {
        const bool me = v[j] >= 0 && (v[j] & (kOwners - 1)) == owner;
        const unsigned all = __ballot_sync(0xffffffffu, me);
        if (me)
          from[at + __popc(all & before_me)] = {v[j] >> kOwnerBits,
                                                static_cast<int>(t + 32 * j + lane)};
        at += __popc(all);
      }
    }
  }

  const int chunk = ((n + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
  const int i0 = min(n, warp * chunk), i1 = min(n, i0 + chunk);
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * kDigit;
    const auto digit = [&](int i) {
      return i < i1 ? (from[i].word >> shift) & ((1 << kDigit) - 1) : 1 << kDigit;
    };
    static_assert(kSortThreads == kSortWarps << kDigit, "one counter per thread");
    count[threadIdx.x >> 5][lane] = 0;
    __syncthreads();  // the list and the counters are there
    for (int i = i0; i < i1; i += 32) {
      const int d = digit(i + lane);
      const unsigned same = __match_any_sync(0xffffffffu, d);
      if (d < 1 << kDigit && (same & before_me) == 0) count[d][warp] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    int* c = &count[threadIdx.x >> 5][lane];  // digit by digit, warp by warp
    int all;
    const int start = block_exclusive(*c, warps, &all);
    *c = start;
    __syncthreads();
    for (int i = i0; i < i1; i += 32) {
      const int d = digit(i + lane);
      const unsigned same = __match_any_sync(0xffffffffu, d);
      if (d < 1 << kDigit) to[count[d][warp] + __popc(same & before_me)] = from[i + lane];
      __syncwarp();
      if (d < 1 << kDigit && (same & before_me) == 0) count[d][warp] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    Entry* swap = from;
    from = to;
    to = swap;
  }
  __syncthreads();  // without passes: the list is there

  for (int i = threadIdx.x; i < n; i += kSortThreads) {
    const Entry e = from[i];
    a.word[base + i] = (e.word << kOwnerBits) + owner;
    a.pos[base + i] = e.pos;
    if (i == 0 || from[i - 1].word != e.word) span[e.word].x = base + i;
    if (i == n - 1 || from[i + 1].word != e.word) span[e.word].y = base + i + 1;
  }
}

__device__ __forceinline__ int2 span_of(const int2* span, int per_owner, int word) {
  return span[static_cast<std::int64_t>(word & (kOwners - 1)) * per_owner + (word >> kOwnerBits)];
}

// ----------------------------------------------------------------------- the sums --
// A warp adds rows over a slice of the features: RUNS runs of VEC elements per lane, all loads
// of a row (and of the next) in flight at once.
struct SumArgs {
  const void* dy;
  std::int64_t ld;
  int features, vocab;
  int per_owner;
  int block;      // entries per block
  const int* word;
  const int* pos;
  const int2* span;
  const int* total;
  float* partial;  // [block][2][features]: a block's share of the word that it starts with,
                   // and of the word that it ends with
  void* dw;
  float alpha, beta;
};

template <int VEC, int RUNS>
struct Slice {
  static constexpr int kFeatures = 32 * VEC * RUNS;
  float v[RUNS][VEC];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[r][e] = 0.0f;
  }
  // Adds features h0 + lane * VEC + r * 32 * VEC of the row.
  template <typename T>
  __device__ __forceinline__ void add(const Run<T, VEC> (&in)[RUNS]) {
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[r][e] += static_cast<float>(in[r].v[e]);
  }
};

template <typename T, int VEC, int RUNS>
__device__ __forceinline__ void load_slice(Run<T, VEC> (&in)[RUNS], const T* row, int h,
                                           int features) {
#pragma unroll
  for (int r = 0; r < RUNS; ++r)
    if (h + r * 32 * VEC < features) in[r] = load_run<T, VEC>(row + h + r * 32 * VEC);
}

// Rows pos[i0..i1) of dy.
template <typename T, int VEC, int RUNS>
__device__ __forceinline__ void add_rows(Slice<VEC, RUNS>& s, const SumArgs& a, int i0, int i1,
                                         int h) {
  const T* dy = static_cast<const T*>(a.dy);
  constexpr int kAhead = 2;
  Run<T, VEC> in[kAhead][RUNS] = {};
  int i = i0;
  for (; i + kAhead <= i1; i += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      load_slice<T, VEC, RUNS>(in[k], dy + a.pos[i + k] * a.ld, h, a.features);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) s.add(in[k]);
  }
  for (; i < i1; ++i) {
    load_slice<T, VEC, RUNS>(in[0], dy + a.pos[i] * a.ld, h, a.features);
    s.add(in[0]);
  }
}

constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32;

template <typename T, int VEC, int RUNS>
__global__ void __launch_bounds__(kSumThreads) embedding_partial_kernel(const SumArgs a) {
  tc::grid_launch_next();
  tc::grid_wait_previous();
  const int lane = threadIdx.x & 31;
  const int slices = (a.features + Slice<VEC, RUNS>::kFeatures - 1) / Slice<VEC, RUNS>::kFeatures;
  const int total = *a.total;
  const std::int64_t units = static_cast<std::int64_t>((total + a.block - 1) / a.block) * slices;
  for (std::int64_t u = static_cast<std::int64_t>(blockIdx.x) * kSumWarps + (threadIdx.x >> 5);
       u < units; u += static_cast<std::int64_t>(gridDim.x) * kSumWarps) {
    const std::int64_t b = u / slices;
    const int h = static_cast<int>(u - b * slices) * Slice<VEC, RUNS>::kFeatures + lane * VEC;
    const int i0 = static_cast<int>(b * a.block), i1 = min(total, i0 + a.block);
    const int2 head = span_of(a.span, a.per_owner, a.word[i0]);
    const int2 tail = span_of(a.span, a.per_owner, a.word[i1 - 1]);
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      const int2 s = k == 0 ? head : tail;
      if (s.y - s.x <= a.block || (k == 1 && s.x <= i0)) continue;
      Slice<VEC, RUNS> sum;
      sum.clear();
      add_rows<T, VEC, RUNS>(sum, a, max(i0, s.x), min(i1, s.y), h);
      float* o = a.partial + (2 * b + k) * a.features + h;
#pragma unroll
      for (int r = 0; r < RUNS; ++r) {
        if (h + r * 32 * VEC >= a.features) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[r * 32 * VEC + e] = sum.v[r][e];
      }
    }
  }
}

// TOUCHED: only the words that occur (beta 1), found among the entries; else all words.
template <typename T, typename TW, int VEC, int RUNS, bool TOUCHED>
__global__ void __launch_bounds__(kSumThreads) embedding_rows_kernel(const SumArgs a) {
  tc::grid_launch_next();
  tc::grid_wait_previous();
  const int lane = threadIdx.x & 31;
  const int slices = (a.features + Slice<VEC, RUNS>::kFeatures - 1) / Slice<VEC, RUNS>::kFeatures;
  const std::int64_t units = static_cast<std::int64_t>(TOUCHED ? *a.total : a.vocab) * slices;
  for (std::int64_t u = static_cast<std::int64_t>(blockIdx.x) * kSumWarps + (threadIdx.x >> 5);
       u < units; u += static_cast<std::int64_t>(gridDim.x) * kSumWarps) {
    const int i = static_cast<int>(u / slices);
    const int h = static_cast<int>(u % slices) * Slice<VEC, RUNS>::kFeatures + lane * VEC;
    int word = i;
    if constexpr (TOUCHED) {
      word = a.word[i];
      if (i > 0 && a.word[i - 1] == word) continue;
    }
    const int2 s = span_of(a.span, a.per_owner, word);
    Slice<VEC, RUNS> sum;
    sum.clear();
    if (s.y - s.x <= a.block) {
      add_rows<T, VEC, RUNS>(sum, a, s.x, s.y, h);
    } else {
      for (int b = s.x / a.block; b <= (s.y - 1) / a.block; ++b) {
        const int k = b * static_cast<std::int64_t>(a.block) < s.x ? 1 : 0;
        const float* p = a.partial + (2ll * b + k) * a.features;
#pragma unroll
        for (int r = 0; r < RUNS; ++r) {
          if (h + r * 32 * VEC >= a.features) continue;
#pragma unroll
          for (int e = 0; e < VEC; ++e) sum.v[r][e] += p[h + r * 32 * VEC + e];
        }
      }
    }
    TW* o = static_cast<TW*>(a.dw) + static_cast<std::int64_t>(word) * a.features + h;
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      if (h + r * 32 * VEC >= a.features) continue;
      Run<TW, VEC> out, was;
      if (a.beta != 0.0f) was = load_run<TW, VEC>(o + r * 32 * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        // a word that does not occur has no sum for an infinite alpha to multiply
        float v = s.y > s.x ? a.alpha * sum.v[r][e] : 0.0f;
        if (a.beta != 0.0f) v = fmaf(a.beta, static_cast<float>(was.v[e]), v);
        out.v[e] = from_float<TW>(v);
      }
      store_run<TW, VEC>(o + r * 32 * VEC, out);
    }
  }
}

// ------------------------------------------------------------------------- planning --
// Entries per block: long enough that the partial sums of frequent words are few, short enough
// that one warp's share of a block or of a word is (the square root of the tokens balances the
// two, for a word that all of them are).
int block_entries(int tokens) {
  int n = 16;
  while (n < 512 && 4ll * n * n < tokens) n *= 2;
  return n;
}

struct SortPlan {
  int per_owner, passes, block;
  std::size_t list[2], word, pos, span, total, partial, bytes;
};

SortPlan plan(const EmbeddingArgs& a) {
  SortPlan p{};
  p.per_owner = (a.vocab + kOwners - 1) / kOwners;
  while ((p.per_owner - 1) >> (p.passes * kDigit) != 0) ++p.passes;
  p.block = block_entries(a.tokens);
  std::size_t at = 0;
  const auto take = [&](std::size_t n) {
    const std::size_t o = at;
    at += (n + 255) / 256 * 256;
    return o;
  };
  const std::size_t T = a.tokens, H = a.features;
  for (std::size_t& l : p.list) l = take(a.tokens > kSharedList ? T * sizeof(Entry) : 0);
  p.word = take(T * 4);
  p.pos = take(T * 4);
  p.span = take(static_cast<std::size_t>(p.per_owner) * kOwners * sizeof(int2));
  p.total = take(4);
  p.partial = take((T + p.block - 1) / p.block * 2 * H * 4);
  p.bytes = at;
  return p;
}

unsigned grid_of(std::int64_t units, int per_cta, int per_sm) {
  const std::int64_t ctas = (units + per_cta - 1) / per_cta;
  return static_cast<unsigned>(
      std::max<std::int64_t>(1, std::min<std::int64_t>(ctas, std::int64_t{sms()} * per_sm)));
}

template <typename TW, typename TY, int VEC, int RUNS>
cudaError_t lookup(const EmbeddingArgs& a, cudaStream_t st) {
  const std::int64_t runs = static_cast<std::int64_t>(a.tokens) * (a.features / VEC);
  const std::int64_t per = kLookupThreads * RUNS;
  const std::int64_t ctas = (runs + per - 1) / per;
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  return tc::launch_overlapped(embedding_kernel<TW, TY, VEC, RUNS>,
                               dim3(static_cast<unsigned>(ctas)), kLookupThreads, 0, st, false,
                               static_cast<const TW*>(a.w), a.token, static_cast<TY*>(a.row),
                               a.ld, a.tokens, a.features, a.vocab, a.alpha, a.beta);
}

// Whether every row of both operands is whole runs of VEC elements on 16-byte boundaries.
bool rows_of_runs(const EmbeddingArgs& a, int vec) {
  const int ws = a.table == EmbeddingType::kF32 ? 4 : 2, rs = a.rows == EmbeddingType::kF32 ? 4 : 2;
  return a.features % vec == 0 && aligned_to(a.w, 16) && aligned_to(a.row, 16) &&
         (a.tokens == 1 || a.ld * rs % 16 == 0) && a.features * ws % 16 == 0;
}

template <typename T, typename TW, int VEC, int RUNS>
cudaError_t gradient(const EmbeddingArgs& a, const SortPlan& p, char* ws, cudaStream_t st) {
  SumArgs s{};
  s.dy = a.row;
  s.ld = a.ld;
  s.features = a.features;
  s.vocab = a.vocab;
  s.per_owner = p.per_owner;
  s.block = p.block;
  s.word = reinterpret_cast<int*>(ws + p.word);
  s.pos = reinterpret_cast<int*>(ws + p.pos);
  s.span = reinterpret_cast<int2*>(ws + p.span);
  s.total = reinterpret_cast<int*>(ws + p.total);
  s.partial = reinterpret_cast<float*>(ws + p.partial);
  s.dw = a.w;
  s.alpha = a.alpha;
  s.beta = a.beta;
  constexpr int kSlice = Slice<VEC, RUNS>::kFeatures;
  const std::int64_t slices = (a.features + kSlice - 1) / kSlice;
  const std::int64_t blocks = (a.tokens + p.block - 1) / p.block;
  if (a.tokens > p.block) {  // else no word is long
    const cudaError_t e = tc::launch_overlapped(
        embedding_partial_kernel<T, VEC, RUNS>, dim3(grid_of(blocks * slices, kSumWarps, 8)),
        kSumThreads, 0, st, true, s);
    if (e != cudaSuccess) return e;
  }
  const bool touched = a.beta == 1.0f;
  const std::int64_t rows = touched ? a.tokens : a.vocab;
  return tc::launch_overlapped(touched ? embedding_rows_kernel<T, TW, VEC, RUNS, true>
                                       : embedding_rows_kernel<T, TW, VEC, RUNS, false>,
                               dim3(grid_of(rows * slices, kSumWarps, 8)), kSumThreads, 0, st,
                               true, s);
}

}  // namespace

cudaError_t launch_embedding(const EmbeddingArgs& a, cudaStream_t st) noexcept {
  using T = EmbeddingType;
  const bool wide = rows_of_runs(a, a.rows == T::kF32 ? 4 : 8);
  if (a.rows == T::kF32)
    return wide ? lookup<float, float, 4, 4>(a, st) : lookup<float, float, 1, 8>(a, st);
  if (a.rows == T::kF16) {
    if (a.table == T::kF32)
      return wide ? lookup<float, __half, 8, 2>(a, st) : lookup<float, __half, 1, 8>(a, st);
    return wide ? lookup<__half, __half, 8, 4>(a, st) : lookup<__half, __half, 1, 8>(a, st);
  }
  if (a.table == T::kF32)
    return wide ? lookup<float, __nv_bfloat16, 8, 2>(a, st)
                : lookup<float, __nv_bfloat16, 1, 8>(a, st);
  return wide ? lookup<__nv_bfloat16, __nv_bfloat16, 8, 4>(a, st)
              : lookup<__nv_bfloat16, __nv_bfloat16, 1, 8>(a, st);
}

std::size_t embedding_gradient_workspace(const EmbeddingArgs& a) noexcept { return plan(a).bytes; }

cudaError_t launch_embedding_gradient(const EmbeddingArgs& a, void* workspace,
                                      cudaStream_t st) noexcept {
  using T = EmbeddingType;
  const SortPlan p = plan(a);
  char* ws = static_cast<char*>(workspace);
  SortArgs s{};
  s.token = a.token;
  s.tokens = a.tokens;
  s.vocab = a.vocab;
  s.per_owner = p.per_owner;
  s.passes = p.passes;
  for (int i = 0; i < 2; ++i) s.list[i] = reinterpret_cast<Entry*>(ws + p.list[i]);
  s.word = reinterpret_cast<int*>(ws + p.word);
  s.pos = reinterpret_cast<int*>(ws + p.pos);
  s.span = reinterpret_cast<int2*>(ws + p.span);
  s.total = reinterpret_cast<int*>(ws + p.total);
  const cudaError_t e =
      tc::launch_overlapped(embedding_sort_kernel, dim3(kOwners), kSortThreads, 0, st, false, s);
  if (e != cudaSuccess) return e;
  const bool wide = rows_of_runs(a, a.rows == T::kF32 ? 4 : 8);
  if (a.rows == T::kF32)
    return wide ? gradient<float, float, 4, 4>(a, p, ws, st)
                : gradient<float, float, 1, 8>(a, p, ws, st);
  if (a.rows == T::kF16) {
    if (a.table == T::kF32)
      return wide ? gradient<__half, float, 8, 2>(a, p, ws, st)
                  : gradient<__half, float, 1, 8>(a, p, ws, st);
    return wide ? gradient<__half, __half, 8, 4>(a, p, ws, st)
                : gradient<__half, __half, 1, 8>(a, p, ws, st);
  }
  if (a.table == T::kF32)
    return wide ? gradient<__nv_bfloat16, float, 8, 2>(a, p, ws, st)
                : gradient<__nv_bfloat16, float, 1, 8>(a, p, ws, st);
  return wide ? gradient<__nv_bfloat16, __nv_bfloat16, 8, 4>(a, p, ws, st)
              : gradient<__nv_bfloat16, __nv_bfloat16, 1, 8>(a, p, ws, st);
}

}  // namespace mb200::dnn
