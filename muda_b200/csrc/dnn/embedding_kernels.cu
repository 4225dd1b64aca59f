// embedding_kernels.cu — embedding lookup and its gradient.  The mathematics is stated in
// embedding.hpp.  Both are bound by memory: the lookup reads a table row and writes a row per
// token; the gradient reads every row of dy once and writes all of dw (beta 0) or the rows of
// the words that occur (beta 1).
//
// The gradient adds each word's rows in the order of their positions, whatever runs first, so
// results are the same on every run.  Two launches, or three:
//   1. embedding_sort_kernel orders the tokens by word, positions ascending within a word (many
//      tokens after embedding_part_kernel); beside that it starts filling a large dw;
//   2. embedding_sum_kernel cuts the ordered tokens into blocks of equal length, whatever words
//      they hold, and adds each block's rows up in fp32: a word that lies within a block gets
//      its row of dw, one that crosses into another leaves a partial sum.  Beside that it
//      writes the rows of the words that do not occur.  The warp that leaves a word's last
//      partial sum adds them up, in the blocks' order (a counter says which that is).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
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
struct Run {
  static constexpr int kWords = sizeof(T) * VEC / 16;
  uint4 w[kWords];
};
template <typename T>
struct Run<T, 1> {
  T v;
};

// Loads that are left out without `ok` (then the value is -1, or any).  The predicate is inside
// the asm: a branch around a load makes its result wait for it there.
__device__ __forceinline__ std::int64_t load8(const std::int64_t* p, bool ok) {
  std::int64_t v;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "mov.b64 %0, -1;\n\t"
      "@q ld.global.u64 %0, [%1];\n\t}"
      : "=&l"(v)
      : "l"(p), "r"(static_cast<int>(ok))
      : "memory");
  return v;
}

__device__ __forceinline__ uint4 load16(const void* p, bool ok) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"(static_cast<int>(ok))
      : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ T load_one(const T* p, bool ok) {
  if constexpr (sizeof(T) == 4) {
    float v;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "@q ld.global.f32 %0, [%1];\n\t}"
        : "=&f"(v)
        : "l"(p), "r"(static_cast<int>(ok))
        : "memory");
    return v;
  } else {
    std::uint16_t v;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %2, 0;\n\t"
        "@q ld.global.u16 %0, [%1];\n\t}"
        : "=&h"(v)
        : "l"(p), "r"(static_cast<int>(ok))
        : "memory");
    return *reinterpret_cast<const T*>(&v);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ Run<T, VEC> load_run(const T* p, bool ok) {
  Run<T, VEC> r;
  if constexpr (VEC == 1) {
    r.v = load_one(p, ok);
  } else {
#pragma unroll
    for (int i = 0; i < r.kWords; ++i) r.w[i] = load16(reinterpret_cast<const uint4*>(p) + i, ok);
  }
  return r;
}

template <typename T, int VEC>
__device__ __forceinline__ Run<T, VEC> load_run(const T* p) {
  Run<T, VEC> r;
  if constexpr (VEC == 1) {
    r.v = *p;
  } else {
#pragma unroll
    for (int i = 0; i < r.kWords; ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  return r;
}

// fp32 that other SMs wrote in this launch: from L2.
template <int VEC>
__device__ __forceinline__ Run<float, VEC> load_shared_run(const float* p) {
  Run<float, VEC> r;
  if constexpr (VEC == 1) {
    r.v = __ldcg(p);
  } else {
#pragma unroll
    for (int i = 0; i < r.kWords; ++i) r.w[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i);
  }
  return r;
}

// ONCE: written past the rows that L2 should keep.
template <bool ONCE, typename T, int VEC>
__device__ __forceinline__ void store_run(T* p, const Run<T, VEC>& r) {
  if constexpr (VEC == 1) {
    *p = r.v;
  } else {
#pragma unroll
    for (int i = 0; i < r.kWords; ++i) {
      if constexpr (ONCE)
        __stcs(reinterpret_cast<uint4*>(p) + i, r.w[i]);
      else
        reinterpret_cast<uint4*>(p)[i] = r.w[i];
    }
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Run<T, VEC>& r, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = static_cast<float>(r.v);
  } else {
#pragma unroll
    for (int i = 0; i < r.kWords; ++i) {
      const std::uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (std::is_same_v<T, float>) {
          v[4 * i + j] = __uint_as_float(w[j]);
        } else if constexpr (std::is_same_v<T, __half>) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          v[8 * i + 2 * j] = f.x;
          v[8 * i + 2 * j + 1] = f.y;
        } else {  // bf16 is fp32's upper half
          v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
          v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
    }
  }
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

template <typename T, int VEC>
__device__ __forceinline__ Run<T, VEC> pack(const float (&v)[VEC]) {
  Run<T, VEC> r;
  if constexpr (VEC == 1) {
    r.v = from_float<T>(v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < r.kWords; ++i) {
      if constexpr (std::is_same_v<T, float>)
        r.w[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                            __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
      else
        r.w[i] = make_uint4(
            pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
            pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
    }
  }
  return r;
}

// ------------------------------------------------------------------------- lookup --
constexpr int kLookupThreads = 256;
constexpr int kLookupCtas = 4;  // per SM

// A thread has one column of ROWS rows that lie `stride` apart, so the loads of its tokens, of
// their words' runs and its stores are ROWS at a time; it loads the next rows' tokens while
// this row's runs arrive.
template <typename TW, typename TY, int VEC, int ROWS>
__global__ void __launch_bounds__(kLookupThreads, kLookupCtas)
    embedding_kernel(const TW* __restrict__ w, const std::int64_t* __restrict__ token, TY* y,
                     std::int64_t ldy, int tokens, int features, int vocab, int stride,
                     float alpha, float beta) {
  const int per = features / VEC;  // runs of a row
  const std::int64_t first = static_cast<std::int64_t>(blockIdx.x) * kLookupThreads + threadIdx.x;
  const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * kLookupThreads;
  int row = static_cast<int>(min(first / per, static_cast<std::int64_t>(stride)));
  int col = static_cast<int>(first % per);
  const int rows_on = static_cast<int>(step / per);
  const int cols_on = static_cast<int>(step % per);
  int word[ROWS];  // -1: padding, vocab: past the table
  const auto words = [&](int r) {
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const std::int64_t t = r + static_cast<std::int64_t>(j) * stride;
      const std::int64_t v = load8(token + t, r < stride && t < tokens);
      word[j] = v < 0 ? -1 : v >= vocab ? vocab : static_cast<int>(v);
    }
  };
  words(row);
  while (row < stride) {
    Run<TW, VEC> in[ROWS];
    int is[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      is[j] = word[j];
      in[j] = load_run<TW, VEC>(w + static_cast<std::int64_t>(is[j]) * features + col * VEC,
                                static_cast<unsigned>(is[j]) < static_cast<unsigned>(vocab));
    }
    const bool wraps = col + cols_on >= per;
    const int next = row + rows_on + (wraps ? 1 : 0);
    words(next);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const std::int64_t t = row + static_cast<std::int64_t>(j) * stride;
      if (t >= tokens) break;
      TY* o = y + t * ldy + col * VEC;
      float v[VEC];
      unpack<TW, VEC>(in[j], v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[e] *= alpha;
        if (static_cast<unsigned>(is[j]) >= static_cast<unsigned>(vocab))
          v[e] = is[j] < 0 ? 0.0f : NAN;
      }
      if (beta != 0.0f) {
        float was[VEC];
        unpack<TY, VEC>(load_run<TY, VEC>(o), was);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = fmaf(beta, was[e], v[e]);
      }
      store_run<false>(o, pack<TY, VEC>(v));
    }
    row = next;
    col += cols_on - (wraps ? per : 0);
  }
}

// ---------------------------------------------------------------------- the order --
// CTA c owns the words v with v % kOwners == c (frequent words are neighbours in most
// vocabularies, so ranges of words would leave one CTA most of the tokens).  It finds the place
// of its own tokens in the ordered list, which is how many the owners before it have, lists its
// own in position order, and sorts them by word.  Up to kParted tokens every CTA reads them all
// to that end; more are parted first, by a kernel that orders each of kParts runs of tokens by
// owner, of which every CTA then collects its own.  A warp goes over a contiguous share of the
// tokens or of the list in all steps, so equal words keep their order, whatever the split between
// the warps.  No CTA waits for another.
//
// Latency bound: 1537 tokens of 32003 words 6 us, 8192 of 128000 9 us, 32768 of 50257 5 us and
// then 12 (clusters of eight that read the tokens together: 18, and 4 more to be launched; a
// frequent word's owner has 2400 of these and sorts the longest).
constexpr int kOwners = kEmbeddingOwners, kOwnerBits = 7;
static_assert(kOwners == 1 << kOwnerBits);
constexpr int kSortThreads = kEmbeddingSortThreads, kSortWarps = kSortThreads / 32;
constexpr int kDigit = 5, kDigits = 1 << kDigit;
constexpr int kSharedList = 4096;  // entries that are sorted in shared memory
constexpr int kScan = 4;           // tokens per lane at a time
constexpr int kCompared = 128;     // entries that are sorted by comparing each with all
constexpr int kParts = 128, kParted = kEmbeddingParted;

struct Entry {
  int word;  // v / kOwners
  int pos;
};

struct SortArgs {
  const std::int64_t* token;
  int tokens, vocab;
  int passes;
  int near_list;   // min(tokens, kSharedList)
  Entry* list[2];  // [tokens] each: longer lists while they are sorted
  int share;       // tokens of a part, a multiple of 32; 0: they are not parted
  Entry* parts;    // [part][share], ordered by owner
  int* starts;     // [owner or kOwners][part]: where the owner's tokens start in the part
  int* word;       // [tokens] out: the words in order
  int* pos;        // [tokens] out: and their positions
  int2* span;      // [owner][per_owner] out: a word's entries
  int per_owner;   // words of an owner, at most
  bool all_words;  // spans of words that do not occur are {0, 0}; else they are left as they are
  int* counters;   // out: zeros
  std::int64_t num_counters;
  int* total;      // out: entries
  uint4* fill;     // to be set to zeros by the CTAs behind the owners'
  std::int64_t num_fill;
};

__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The lanes of `among` whose low BITS bits (ballots in `bits`) are c's.
template <int BITS>
__device__ __forceinline__ unsigned lanes_of(unsigned among, const unsigned (&bits)[BITS + 1],
                                             int c) {
#pragma unroll
  for (int i = 0; i < BITS; ++i) among &= (c >> i & 1) != 0 ? bits[i] : ~bits[i];
  return among;
}

// v summed over the lanes up to this one.
__device__ __forceinline__ int warp_inclusive(int v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += u;
  }
  return v;
}

// The token at t as a word, -1 if it enters nothing.
__device__ __forceinline__ int word_of(const SortArgs& a, std::int64_t token) {
  return token >= 0 && token < a.vocab ? static_cast<int>(token) : -1;
}

// CTA q orders its part of the tokens by owner.
__global__ void __launch_bounds__(kSortThreads) embedding_part_kernel(const SortArgs a) {
  __shared__ int count[kOwners][kSortWarps + 1];
  __shared__ int totals[kOwners];
  tc::grid_launch_next();
  tc::grid_wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = blockIdx.x;
  const unsigned before_me = (1u << lane) - 1;
  for (int o = warp; o < kOwners; o += kSortWarps) count[o][lane] = 0;
  __syncthreads();
  const int per_warp = (a.share + kSortThreads - 1) / kSortThreads * 32;
  const std::int64_t first = static_cast<std::int64_t>(q) * a.share;
  const std::int64_t t0 = first + warp * per_warp;
  const std::int64_t t1 =
      min(min(t0 + per_warp, first + a.share), static_cast<std::int64_t>(a.tokens));
  // the lane's token of the 32 from t on, and the lanes whose tokens have the same owner
  const auto owners = [&](std::int64_t t, int* word) {
    *word = word_of(a, load8(a.token + t + lane, t + lane < t1));
    unsigned bits[kOwnerBits + 1];
#pragma unroll
    for (int k = 0; k < kOwnerBits; ++k)
      bits[k] = __ballot_sync(0xffffffffu, (*word >> k & 1) != 0);
    return lanes_of<kOwnerBits>(__ballot_sync(0xffffffffu, *word >= 0), bits, *word);
  };
  for (std::int64_t t = t0; t < t1; t += 32) {
    int word;
    const unsigned same = owners(t, &word);
    if (word >= 0 && (same & before_me) == 0) count[word & (kOwners - 1)][warp] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  constexpr int kEach = kOwners / kSortWarps;  // owners that a warp scans
  int upto[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int x = count[warp * kEach + k][lane];
    const int sum = warp_inclusive(x);
    upto[k] = sum - x;
    if (lane == 31) totals[warp * kEach + k] = sum;
  }
  __syncthreads();
  int mine = 0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) mine += totals[lane * kEach + k];
  int start = __shfl_sync(0xffffffffu, warp_inclusive(mine) - mine, warp);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int o = warp * kEach + k;
    count[o][lane] = start + upto[k];
    if (lane == 0) a.starts[o * kParts + q] = start;
    start += totals[o];
  }
  if (threadIdx.x == kSortThreads - 1) a.starts[kOwners * kParts + q] = start;
  __syncthreads();
  Entry* part = a.parts + first;
  for (std::int64_t t = t0; t < t1; t += 32) {
    int word;
    const unsigned same = owners(t, &word);
    int* at = &count[word & (kOwners - 1)][warp];
    if (word >= 0)
      part[*at + __popc(same & before_me)] = {word >> kOwnerBits, static_cast<int>(t) + lane};
    __syncwarp();
    if (word >= 0 && (same & before_me) == 0) *at += __popc(same);
    __syncwarp();
  }
}

// Lists the owner's tokens in position order, from parts; returns how many there are and, in
// *base, how many the owners before it have.
__device__ __forceinline__ int collect(const SortArgs& a, Entry* near, int owner, int* base,
                                       Entry** list) {
  __shared__ int before[kParts + 1], from[kParts], sums[2][kParts / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int start = 0, n = 0, upto = 0;
  if (threadIdx.x < kParts) {
    start = a.starts[owner * kParts + threadIdx.x];
    n = a.starts[(owner + 1) * kParts + threadIdx.x] - start;
    upto = warp_inclusive(n);
    const int starts = warp_sum(start);
    if (lane == 31) {
      sums[0][warp] = upto;
      sums[1][warp] = starts;
    }
  }
  __syncthreads();
  int all = 0, lower = 0;
  *base = 0;
#pragma unroll
  for (int w = 0; w < kParts / 32; ++w) {
    if (w < warp) lower += sums[0][w];
    all += sums[0][w];
    *base += sums[1][w];
  }
  if (threadIdx.x < kParts) {
    before[threadIdx.x] = lower + upto - n;
    from[threadIdx.x] = threadIdx.x * a.share + start;
  }
  __syncthreads();
  *list = all <= a.near_list ? near : a.list[0] + *base;
  constexpr int kAtOnce = 4;
  for (int i0 = threadIdx.x; i0 < all; i0 += kAtOnce * kSortThreads) {
    Entry e[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = min(i0 + j * kSortThreads, all - 1);
      int q = 0;  // the last part that starts at i or before
#pragma unroll
      for (int step = kParts / 2; step > 0; step /= 2)
        if (before[q + step] <= i) q += step;
      e[j] = a.parts[from[q] + (i - before[q])];
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (i0 + j * kSortThreads < all) (*list)[i0 + j * kSortThreads] = e[j];
  }
  __syncthreads();
  return all;
}

// The same, from the tokens.
__device__ __forceinline__ int select(const SortArgs& a, Entry* near, int owner, int* base,
                                      Entry** list) {
  __shared__ int found[2][kSortWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned before_me = (1u << lane) - 1;
  const int per_warp = (a.tokens + kSortThreads - 1) / kSortThreads * 32;
  const int t0 = warp * per_warp, t1 = min(t0 + per_warp, a.tokens);
  const bool keep = per_warp <= 32 * kScan;  // in registers between the two readings
  int v[kScan];
  const auto load = [&](int t) {
    std::int64_t w[kScan];
#pragma unroll
    for (int j = 0; j < kScan; ++j) {
      const int i = t + 32 * j + lane;
      w[j] = load8(a.token + i, i < t1);
    }
#pragma unroll
    for (int j = 0; j < kScan; ++j) v[j] = word_of(a, w[j]);
  };
  const auto mine = [&](int word) {
    return __ballot_sync(0xffffffffu, word >= 0 && (word & (kOwners - 1)) == owner);
  };
  int below = 0, n = 0;
  for (int t = t0; t < t1; t += 32 * kScan) {
    load(t);
#pragma unroll
    for (int j = 0; j < kScan; ++j) {
      below += v[j] >= 0 && (v[j] & (kOwners - 1)) < owner;
      n += __popc(mine(v[j]));
    }
  }
  below = warp_sum(below);
  if (lane == 0) {
    found[0][warp] = n;
    found[1][warp] = below;
  }
  __syncthreads();
  const int upto = warp_inclusive(found[0][lane]);
  int at = __shfl_sync(0xffffffffu, upto, warp) - n;
  const int all = __shfl_sync(0xffffffffu, upto, 31);
  *base = warp_sum(found[1][lane]);
  *list = all <= a.near_list ? near : a.list[0] + *base;
  for (int t = t0; t < t1; t += 32 * kScan) {
    if (!keep) load(t);
#pragma unroll
    for (int j = 0; j < kScan; ++j) {
      const unsigned in = mine(v[j]);
      if ((in >> lane & 1u) != 0)
        (*list)[at + __popc(in & before_me)] = {v[j] >> kOwnerBits, t + 32 * j + lane};
      at += __popc(in);
    }
  }
  __syncthreads();
  return all;
}

__global__ void __launch_bounds__(kSortThreads, 2) embedding_sort_kernel(const SortArgs a) {
  extern __shared__ Entry near[];  // two lists of near_list entries
  // by digit, by warp: a warp's counters in banks of their own; two passes in turn
  __shared__ int count[2][kDigits][kSortWarps + 1];
  __shared__ int totals[2][kDigits];
  tc::grid_launch_next();
  tc::grid_wait_previous();
  if (blockIdx.x >= kOwners) {
    const std::int64_t step = static_cast<std::int64_t>(gridDim.x - kOwners) * kSortThreads;
    const std::int64_t first = static_cast<std::int64_t>(blockIdx.x - kOwners) * kSortThreads;
#pragma unroll 4
    for (std::int64_t i = first + threadIdx.x; i < a.num_fill; i += step)
      __stcs(a.fill + i, make_uint4(0, 0, 0, 0));
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, owner = blockIdx.x;
  const unsigned before_me = (1u << lane) - 1;
  count[0][warp][lane] = 0;
  int2* span = a.span + static_cast<std::int64_t>(owner) * a.per_owner;
  for (int i = threadIdx.x; a.all_words && i < a.per_owner; i += kSortThreads)
    span[i] = make_int2(0, 0);
  for (std::int64_t i = static_cast<std::int64_t>(owner) * kSortThreads + threadIdx.x;
       i < a.num_counters; i += kOwners * kSortThreads)
    a.counters[i] = 0;

  int base;
  Entry* from;
  const int n = a.share > 0 ? collect(a, near, owner, &base, &from)
                            : select(a, near, owner, &base, &from);
  Entry* to = n <= a.near_list ? near + a.near_list : a.list[1] + base;
  if (owner == kOwners - 1 && threadIdx.x == 0) *a.total = base + n;

  if (n <= kCompared) {
    if (static_cast<int>(threadIdx.x) < n) {
      const Entry e = from[threadIdx.x];
      int place = 0;
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const int w = from[i].word;
        place += w < e.word || (w == e.word && i < static_cast<int>(threadIdx.x));
      }
      to[place] = e;
    }
    from = to;
  } else {
    const int chunk = ((n + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
    const int i0 = min(n, warp * chunk), i1 = min(n, i0 + chunk);
    for (int pass = 0; pass < a.passes; ++pass) {
      const int shift = pass * kDigit;
      auto& counts = count[pass & 1];
      // entry i's digit, and the lanes whose entries have the same (five votes)
      const auto digit = [&](int i, unsigned* same) {
        const int d = i < i1 ? from[i].word >> shift & (kDigits - 1) : kDigits;
        unsigned bits[kDigit + 1];
#pragma unroll
        for (int k = 0; k < kDigit; ++k) bits[k] = __ballot_sync(0xffffffffu, (d >> k & 1) != 0);
        *same = lanes_of<kDigit>(__ballot_sync(0xffffffffu, d < kDigits), bits, d);
        return d;
      };
      static_assert(kSortWarps == kDigits, "a warp scans a digit's counters");
      for (int i = i0; i < i1; i += 32) {
        unsigned same;
        const int d = digit(i + lane, &same);
        if (d < kDigits && (same & before_me) == 0) counts[d][warp] += __popc(same);
        __syncwarp();
      }
      __syncthreads();
      const int x = counts[warp][lane];  // of digit `warp`, by warp
      const int upto = warp_inclusive(x);
      if (lane == 31) totals[pass & 1][warp] = upto;
      count[(pass + 1) & 1][warp][lane] = 0;
      __syncthreads();
      const int digits = totals[pass & 1][lane];
      const int before_digit = __shfl_sync(0xffffffffu, warp_inclusive(digits) - digits, warp);
      counts[warp][lane] = before_digit + upto - x;
      __syncthreads();
      for (int i = i0; i < i1; i += 32) {
        unsigned same;
        const int d = digit(i + lane, &same);
        if (d < kDigits) to[counts[d][warp] + __popc(same & before_me)] = from[i + lane];
        __syncwarp();
        if (d < kDigits && (same & before_me) == 0) counts[d][warp] += __popc(same);
        __syncwarp();
      }
      __syncthreads();
      Entry* swap = from;
      from = to;
      to = swap;
    }
  }
  __syncthreads();

  for (int i = threadIdx.x; i < n; i += kSortThreads) {
    const Entry e = from[i];
    a.word[base + i] = (e.word << kOwnerBits) + owner;
    a.pos[base + i] = e.pos;
    if (i == 0 || from[i - 1].word != e.word) span[e.word].x = base + i;
    if (i == n - 1 || from[i + 1].word != e.word) span[e.word].y = base + i + 1;
  }
}

// ----------------------------------------------------------------------- the sums --
struct SumArgs {
  const void* dy;
  std::int64_t ld;
  int features, vocab;
  int block;  // entries per block
  int per_owner;
  int first_row;  // of those to be filled: the rows before it are zeros already
  int fill_rows;  // rows that a warp fills at a time
  const int* word;
  const int* pos;
  const int2* span;
  const int* total;
  float* partial;  // [block][2][features]: a block's share of a word that began before it, and
                   // of one that began in it and goes on behind it
  int* counters;   // [block][3][slices]: partial sums that are there, see join()
  void* dw;
  float alpha, beta;
};

constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32;
// CTAs per SM.  Where there is work for all warps of the GPU, three with 8 rows in flight keep the
// most bytes on their way (8192 x 4096 of 128000 words: 192 us, 197 with two and 16 rows); where a
// warp has one block or none, two whose loads of 16 rows are one latency (4096 x 512 of 8000: 17
// us, 20 with three).
constexpr int kManyCtas = 3, kFewCtas = 2;

__device__ __forceinline__ int2 span_of(const SumArgs& a, int word) {
  return a.span[static_cast<std::int64_t>(word & (kOwners - 1)) * a.per_owner +
                (word >> kOwnerBits)];
}

// A slice of the features: RUNS runs of VEC elements per lane, from h on.
template <int VEC, int RUNS>
struct Slice {
  static constexpr int kFeatures = 32 * VEC * RUNS, kStep = 32 * VEC;
  float v[RUNS][VEC];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[r][e] = 0.0f;
  }
};

template <int VEC, int RUNS>
__device__ __forceinline__ void store_partial(const Slice<VEC, RUNS>& s, float* o, int h,
                                              int features) {
#pragma unroll
  for (int r = 0; r < RUNS; ++r)
    if (h + r * s.kStep < features)
      store_run<false>(o + h + r * s.kStep, pack<float, VEC>(s.v[r]));
}

// What becomes of dw: nothing of it is left, beta of it, or (fp32 device memory, beta 1) the sums
// are added to it.  kAdd's additions are done by L2, each element's one, so that no load's latency is
// waited for (the second micro-batch of 32768 x 2048: 69 us with kScale, 60).
enum Update { kWrite = 0, kScale = 1, kAdd = 2 };

// They take numbers below 2^-126 for zeros.  A sum of kLeastAdded or more does not see that: what
// dw was rounds away, and no cancellation leaves so little (both are multiples of 2^-124 then, or
// dw is the smaller by half).  Runs with a lesser sum are loaded.
constexpr float kLeastAdded = 0x1p-100f;

template <int VEC>
__device__ __forceinline__ void add_run(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p), "f"(v[0]) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4)
      asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p + i), "f"(v[i]),
                   "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3])
                   : "memory");
  }
}

// Lane `from`'s p.
template <typename T>
__device__ __forceinline__ T* shuffled(T* p, int from) {
  return reinterpret_cast<T*>(
      __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), from));
}

// The slice of a word's row of dw (o: at h), from its sum and what it was.
template <int UPDATE, typename TW, int VEC, int RUNS>
__device__ __forceinline__ void store_row(const Slice<VEC, RUNS>& s, const SumArgs& a, TW* o, int h,
                                          const Run<TW, VEC> (&was)[RUNS]) {
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    if (h + r * s.kStep >= a.features) continue;
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = a.alpha * s.v[r][e];
    if constexpr (UPDATE == kAdd) {
      bool small = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) small |= !(fabsf(v[e]) >= kLeastAdded);
      if (!small) {
        add_run<VEC>(o + r * s.kStep, v);
        continue;
      }
      float old[VEC];
      unpack<TW, VEC>(load_run<TW, VEC>(o + r * s.kStep), old);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] += old[e];
    }
    if constexpr (UPDATE == kScale) {
      float old[VEC];
      unpack<TW, VEC>(was[r], old);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = fmaf(a.beta, old[e], v[e]);
    }
    store_run<true>(o + r * s.kStep, pack<TW, VEC>(v));
  }
}

// The sums of `n` blocks from `first` on, in their order; the first is at `slot`, the others,
// which the word enters from before, at 0.
template <int VEC, int RUNS>
__device__ __forceinline__ void add_partials(Slice<VEC, RUNS>& s, const SumArgs& a, int first,
                                             int slot, int n, int step, int h) {
  constexpr int kStep = Slice<VEC, RUNS>::kStep;
#pragma unroll 8
  for (int k = 0; k < n; ++k) {
    const int b = k == 0 ? first : (first / step + k) * step;
    const float* p = a.partial + (2ll * b + (k == 0 ? slot : 0)) * a.features + h;
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      if (h + r * kStep >= a.features) continue;
      float v[VEC];
      unpack<float, VEC>(load_shared_run<VEC>(p + r * kStep), v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s.v[r][e] += v[e];
    }
  }
}

// Blocks whose partial sums of one word are joined by themselves first.
constexpr int kJoin = 32;

// Whether this warp is the last of n to come here.  What the others wrote before is visible
// then (each lane's writes are ordered before lane 0's release); no warp waits.
__device__ __forceinline__ bool last_of(int* counter, int n) {
  __syncwarp();
  int was = 0;
  if ((threadIdx.x & 31) == 0)
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(was) : "l"(counter)
                 : "memory");
  was = __shfl_sync(0xffffffffu, was, 0);
  __syncwarp();  // and what lane 0 acquired before the other lanes' reads
  return was == n - 1;
}

// Called by each warp that has left a partial sum of this word's slice, of block b.  The last
// one adds them up; where they are many, first the last of each kJoin neighbouring blocks those.
template <int UPDATE, typename TW, int VEC, int RUNS>
__device__ __forceinline__ void join(const SumArgs& a, int word, int b, int slice, int slices,
                                     int h) {
  const int2 span = span_of(a, word);
  const int b0 = span.x / a.block, b1 = (span.y - 1) / a.block;
  const auto counter = [&](int block, int which) {
    return a.counters + (3ll * block + which) * slices + slice;
  };
  Slice<VEC, RUNS> sum;
  sum.clear();
  if (b1 - b0 < kJoin) {
    if (!last_of(counter(b0, 2), b1 - b0 + 1)) return;
    add_partials(sum, a, b0, 1, b1 - b0 + 1, 1, h);
  } else {
    const int g = b / kJoin;
    const int first = max(b0, g * kJoin), n = min(b1, g * kJoin + kJoin - 1) - first + 1;
    const int slot = first == b0 ? 1 : 0;
    if (!last_of(counter(first, slot), n)) return;
    add_partials(sum, a, first, slot, n, 1, h);
    store_partial(sum, a.partial + (2ll * first + slot) * a.features, h, a.features);
    const int groups = b1 / kJoin - b0 / kJoin + 1;
    if (!last_of(counter(b0, 2), groups)) return;
    sum.clear();
    add_partials(sum, a, b0, 1, groups, kJoin, h);
  }
  TW* o = static_cast<TW*>(a.dw) + static_cast<std::int64_t>(word) * a.features + h;
  Run<TW, VEC> was[RUNS];
  if constexpr (UPDATE == kScale) {
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
      if (h + r * sum.kStep < a.features) was[r] = load_run<TW, VEC>(o + r * sum.kStep);
  }
  store_row<UPDATE, TW>(sum, a, o, h, was);
}

// s += the run, two features to an instruction.
template <typename T, int VEC>
__device__ __forceinline__ void add(float (&s)[VEC], const Run<T, VEC>& r) {
  float v[VEC];
  unpack<T, VEC>(r, v);
  if constexpr (VEC == 1) {
    s[0] += v[0];
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e += 2)
      asm("{\n\t.reg .b64 a, b;\n\t"
          "mov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
          "add.rn.f32x2 a, a, b;\n\t"
          "mov.b64 {%0, %1}, a;\n\t}"
          : "+f"(s[e]), "+f"(s[e + 1])
          : "f"(v[e]), "f"(v[e + 1]));
  }
}

// One block's entries: AHEAD rows are loaded at a time and added in order; with beta also the
// rows of dw of the words that end among them, whose latency would otherwise be a word's each.
// A warp alone takes as long for its instructions as for its loads, so there are no branches or
// predicates but for words that end: lanes behind the features read the row's first ones, and a
// last batch its last row again.
template <int UPDATE, typename T, typename TW, int VEC, int RUNS, int AHEAD>
__device__ __forceinline__ void sum_block(const SumArgs& a, int b, int slice, int slices,
                                          int total) {
  const int lane = threadIdx.x & 31;
  const int h = slice * Slice<VEC, RUNS>::kFeatures + lane * VEC;
  const int i0 = b * a.block, i1 = min(total, i0 + a.block);
  constexpr int kStep = Slice<VEC, RUNS>::kStep;
  int at[RUNS];  // the runs' features
#pragma unroll
  for (int r = 0; r < RUNS; ++r) at[r] = h + r * kStep < a.features ? h + r * kStep : 0;
  Slice<VEC, RUNS> sum;
  sum.clear();
  bool began_before = i0 > 0 && a.word[i0 - 1] == a.word[i0];
  float* partial = a.partial + 2ll * b * a.features;
  bool open = false;  // the last entry's word goes on behind the block
  int left = -1;      // the word that began before the block and ended in it
  for (int i = i0; i < i1; i += 32) {
    const int n = min(32, i1 - i);
    const int mine = i + min(lane, n - 1);
    const int my_word = a.word[mine];
    const int next = mine + 1 < total ? a.word[mine + 1] : -1;
    const T* my_row = static_cast<const T*>(a.dy) + a.pos[mine] * a.ld;
    TW* my_dw = static_cast<TW*>(a.dw) + static_cast<std::int64_t>(my_word) * a.features;
    const unsigned ends = __ballot_sync(0xffffffffu, my_word != next);
    open = (ends >> (n - 1) & 1u) == 0;
    for (int j = 0; j < n; j += AHEAD) {
      Run<T, VEC> in[AHEAD][RUNS];
      Run<TW, VEC> was[AHEAD][RUNS];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const T* row = shuffled(my_row, (j + k) & 31);
#pragma unroll
        for (int r = 0; r < RUNS; ++r) in[k][r] = load_run<T, VEC>(row + at[r]);
        if constexpr (UPDATE == kScale) {
          const TW* o = shuffled(my_dw, (j + k) & 31);
#pragma unroll
          for (int r = 0; r < RUNS; ++r)
            was[k][r] = load_run<TW, VEC>(o + at[r], (ends >> ((j + k) & 31) & 1u) != 0);
        }
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (j + k >= n) break;
#pragma unroll
        for (int r = 0; r < RUNS; ++r) add<T, VEC>(sum.v[r], in[k][r]);
        if ((ends >> (j + k) & 1u) == 0) continue;
        if (began_before) {
          store_partial(sum, partial, h, a.features);
          left = __shfl_sync(0xffffffffu, my_word, j + k);
        } else {
          store_row<UPDATE, TW>(sum, a, shuffled(my_dw, j + k) + h, h, was[k]);
        }
        began_before = false;
        sum.clear();
      }
    }
  }
  if (open) store_partial(sum, partial + (began_before ? 0 : a.features), h, a.features);
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const int w = k == 0 ? left : open ? a.word[i1 - 1] : -1;
    if (w >= 0) join<UPDATE, TW, VEC, RUNS>(a, w, b, slice, slices, h);
  }
}

// Rows of words that do not occur: zeros, or beta dw.  A warp takes rows of some KB at a time:
// more, and the last warps are alone with theirs (8192 x 4096 of 128000 words by 8 rows 206 us,
// by one 203).
constexpr int kFillBytes = 8192, kMostFillRows = 8;

template <int UPDATE, typename TW, int VEC>
__device__ __forceinline__ void fill_rows(const SumArgs& a, int first) {
  const int lane = threadIdx.x & 31;
  const int v = first + lane;
  const bool absent = lane < a.fill_rows && v < a.vocab && span_of(a, v).y == 0;
  unsigned rows = __ballot_sync(0xffffffffu, absent);
  while (rows != 0) {
    const int row = first + __ffs(rows) - 1;
    rows &= rows - 1;
    TW* o = static_cast<TW*>(a.dw) + static_cast<std::int64_t>(row) * a.features;
    if constexpr (UPDATE == kScale) {
      for (int h = lane * VEC; h < a.features; h += 32 * VEC) {
        float v[VEC];
        unpack<TW, VEC>(load_run<TW, VEC>(o + h), v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= a.beta;
        store_run<true>(o + h, pack<TW, VEC>(v));
      }
      continue;
    }
    // elements up to the first 16-byte word, whole words, and the elements behind the last
    constexpr int kWord = 16 / sizeof(TW);
    const auto past = static_cast<int>(reinterpret_cast<std::uintptr_t>(o) & 15);
    const int lead = min(a.features, (16 - past) % 16 / static_cast<int>(sizeof(TW)));
    const int whole = (a.features - lead) / kWord;
    if (lane < lead) o[lane] = from_float<TW>(0.0f);
#pragma unroll 4
    for (int i = lane; i < whole; i += 32)
      __stcs(reinterpret_cast<uint4*>(o + lead) + i, make_uint4(0, 0, 0, 0));
    const int rest = lead + whole * kWord + lane;
    if (rest < a.features) o[rest] = from_float<TW>(0.0f);
  }
}

// A warp takes a block's slice, or rows to fill, at a time: the sums first, so that their
// latency hides behind the filling, which takes all the bandwidth that is left.
template <int UPDATE, typename T, typename TW, int VEC, int RUNS, int AHEAD, int CTAS>
__global__ void __launch_bounds__(kSumThreads, CTAS) embedding_sum_kernel(const SumArgs a) {
  tc::grid_launch_next();
  tc::grid_wait_previous();
  using S = Slice<VEC, RUNS>;
  // as many rows as the registers hold, with dw's where they are loaded too
  constexpr int kAhead = UPDATE != kScale           ? AHEAD
                         : sizeof(TW) > sizeof(T) ? AHEAD * 3 / 8
                                                  : AHEAD / 2;
  const unsigned slices = (a.features + S::kFeatures - 1) / S::kFeatures;
  const int total = *a.total;
  const std::int64_t sums = static_cast<std::int64_t>((total + a.block - 1) / a.block) * slices;
  const std::int64_t fills =
      a.beta == 1.0f ? 0 : (a.vocab - a.first_row + a.fill_rows - 1) / a.fill_rows;
  const std::int64_t step = static_cast<std::int64_t>(gridDim.x) * kSumWarps;
  for (std::int64_t u = static_cast<std::int64_t>(blockIdx.x) * kSumWarps + (threadIdx.x >> 5);
       u < sums + fills; u += step) {
    if (u < sums) {
      const int b = static_cast<int>(u / slices);
      const int slice = static_cast<int>(u - b * static_cast<std::int64_t>(slices));
      sum_block<UPDATE, T, TW, VEC, RUNS, kAhead>(a, b, slice, slices, total);
    } else {
      fill_rows<UPDATE, TW, VEC>(a, a.first_row + static_cast<int>(u - sums) * a.fill_rows);
    }
  }
}

// ------------------------------------------------------------------------- planning --
std::int64_t few_warps() { return std::int64_t{sms()} * kFewCtas * kSumWarps; }

// Entries per block: 16, one batch of loads, as long as every warp that the GPU holds has one
// block's slice (256 features) and a frequent word (a twelfth of the tokens) has no more partial
// sums than a block has entries; else 32.  More only where one word could have more than 1024
// partial sums.
int block_entries(int tokens, int features) {
  const std::int64_t slices = (features + 255) / 256;
  int n = 16;
  if (tokens / n * slices > few_warps() || 25 * n * n < tokens) n = 32;
  while (tokens / n > 1024 && n >= 32) n *= 2;
  return n;
}

constexpr int kLeastSlice = 128;  // features of the narrowest slices

struct SortPlan {
  int per_owner, passes, block, share;
  std::int64_t num_counters;
  std::size_t list[2], parts, starts, word, pos, span, total, partial, counters, bytes;
};

SortPlan plan(const EmbeddingArgs& a) {
  SortPlan p{};
  while ((a.vocab - 1) >> kOwnerBits >> (p.passes * kDigit) != 0) ++p.passes;
  p.per_owner = (a.vocab + kOwners - 1) / kOwners;
  p.block = block_entries(a.tokens, a.features);
  std::size_t at = 0;
  const auto take = [&](std::size_t n) {
    const std::size_t o = at;
    at += (n + 255) / 256 * 256;
    return o;
  };
  const std::size_t T = a.tokens, H = a.features;
  for (std::size_t& l : p.list) l = take(a.tokens > kSharedList ? T * sizeof(Entry) : 0);
  p.share = a.tokens > kParted ? (a.tokens + 32 * kParts - 1) / (32 * kParts) * 32 : 0;
  p.parts = take(static_cast<std::size_t>(p.share) * kParts * sizeof(Entry));
  p.starts = take(p.share > 0 ? (kOwners + 1) * kParts * 4 : 0);
  p.word = take(T * 4);
  p.pos = take(T * 4);
  p.span = take(static_cast<std::size_t>(p.per_owner) * kOwners * sizeof(int2));
  p.total = take(4);
  const std::size_t blocks = (T + p.block - 1) / p.block;
  p.partial = take(blocks * 2 * H * 4);
  p.num_counters = blocks * 3 * ((H + kLeastSlice - 1) / kLeastSlice);
  p.counters = take(p.num_counters * 4);
  p.bytes = at;
  return p;
}

// Rows per thread of the lookup: one where the GPU has room for a thread per run.
constexpr int kLookupRows = 4;

template <typename TW, typename TY, int VEC, int ROWS = kLookupRows>
cudaError_t lookup(const EmbeddingArgs& a, cudaStream_t st) {
  const std::int64_t per = a.features / VEC;
  const bool one = a.tokens * per <= std::int64_t{sms()} * 2048;
  const int stride = one ? a.tokens : (a.tokens + ROWS - 1) / ROWS;
  const std::int64_t ctas = std::min<std::int64_t>(
      (stride * per + kLookupThreads - 1) / kLookupThreads, sms() * (one ? 8 : kLookupCtas));
  return tc::launch_overlapped(
      one ? embedding_kernel<TW, TY, VEC, 1> : embedding_kernel<TW, TY, VEC, ROWS>,
      dim3(static_cast<unsigned>(ctas)), kLookupThreads, 0, st, false,
      static_cast<const TW*>(a.w), a.token, static_cast<TY*>(a.row), a.ld, a.tokens, a.features,
      a.vocab, stride, a.alpha, a.beta);
}

// Whether every row of both operands is whole runs of VEC elements on 16-byte boundaries.
bool rows_of_runs(const EmbeddingArgs& a, int vec) {
  const int ws = a.table == EmbeddingType::kF32 ? 4 : 2, rs = a.rows == EmbeddingType::kF32 ? 4 : 2;
  return a.features % vec == 0 && aligned_to(a.w, 16) && aligned_to(a.row, 16) &&
         (a.tokens == 1 || a.ld * rs % 16 == 0) && a.features * ws % 16 == 0;
}

template <typename T, typename TW, int VEC, int RUNS, int AHEAD>
cudaError_t gradient(const EmbeddingArgs& a, const SortPlan& p, int first_row, char* ws,
                     cudaStream_t st) {
  SumArgs s{};
  s.dy = a.row;
  s.ld = a.ld;
  s.features = a.features;
  s.vocab = a.vocab;
  s.block = p.block;
  s.word = reinterpret_cast<int*>(ws + p.word);
  s.pos = reinterpret_cast<int*>(ws + p.pos);
  s.span = reinterpret_cast<int2*>(ws + p.span);
  s.total = reinterpret_cast<int*>(ws + p.total);
  s.partial = reinterpret_cast<float*>(ws + p.partial);
  s.counters = reinterpret_cast<int*>(ws + p.counters);
  s.per_owner = p.per_owner;
  s.dw = a.w;
  s.alpha = a.alpha;
  s.beta = a.beta;
  s.first_row = first_row;
  s.fill_rows = std::clamp<int>(kFillBytes / (a.features * sizeof(TW)), 1, kMostFillRows);
  constexpr int kSlice = Slice<VEC, RUNS>::kFeatures;
  const std::int64_t slices = (a.features + kSlice - 1) / kSlice;
  const std::int64_t blocks = (a.tokens + p.block - 1) / p.block;
  const std::int64_t units =
      blocks * slices +
      (a.beta == 1.0f ? 0 : (a.vocab - first_row + s.fill_rows - 1) / s.fill_rows);
  static_assert(kSlice >= kLeastSlice, "the counters are for fewer slices");
  const auto run = [&](auto ahead, auto ctas_per_sm) {
    constexpr int kAhead = decltype(ahead)::value, kCtas = decltype(ctas_per_sm)::value;
    auto kern = a.beta != 0.0f ? embedding_sum_kernel<kScale, T, TW, VEC, RUNS, kAhead, kCtas>
                               : embedding_sum_kernel<kWrite, T, TW, VEC, RUNS, kAhead, kCtas>;
    if constexpr (std::is_same_v<TW, float>) {
      if (a.beta == 1.0f && a.device_table) kern = embedding_sum_kernel<kAdd, T, TW, VEC, RUNS, kAhead, kCtas>;
    }
    const std::int64_t ctas =
        std::min<std::int64_t>((units + kSumWarps - 1) / kSumWarps, sms() * kCtas);
    return tc::launch_overlapped(kern, dim3(static_cast<unsigned>(ctas)), kSumThreads, 0, st, true,
                                 s);
  };
  if (blocks * slices <= few_warps())
    return run(std::integral_constant<int, AHEAD>{}, std::integral_constant<int, kFewCtas>{});
  return run(std::integral_constant<int, AHEAD / 2>{}, std::integral_constant<int, kManyCtas>{});
}

}  // namespace

cudaError_t launch_embedding(const EmbeddingArgs& a, cudaStream_t st) noexcept {
  using T = EmbeddingType;
  const bool wide = rows_of_runs(a, a.rows == T::kF32 ? 4 : 8);
  if (a.rows == T::kF32)
    return wide ? lookup<float, float, 4>(a, st) : lookup<float, float, 1>(a, st);
  if (a.rows == T::kF16) {
    if (a.table == T::kF32)
      return wide ? lookup<float, __half, 8, 2>(a, st) : lookup<float, __half, 1>(a, st);
    return wide ? lookup<__half, __half, 8>(a, st) : lookup<__half, __half, 1>(a, st);
  }
  if (a.table == T::kF32)
    return wide ? lookup<float, __nv_bfloat16, 8, 2>(a, st)
                : lookup<float, __nv_bfloat16, 1>(a, st);
  return wide ? lookup<__nv_bfloat16, __nv_bfloat16, 8>(a, st)
              : lookup<__nv_bfloat16, __nv_bfloat16, 1>(a, st);
}

// Lets the sort use the shared memory that its tokens take, once per device.
static bool sort_attributes() noexcept {
  static std::atomic<unsigned long long> set{0};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return false;
  if ((set.load(std::memory_order_acquire) >> dev & 1ull) != 0) return true;
  if (cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           2 * kSharedList * sizeof(Entry)) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  set.fetch_or(1ull << dev, std::memory_order_release);
  return true;
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
  s.passes = p.passes;
  for (int i = 0; i < 2; ++i) s.list[i] = reinterpret_cast<Entry*>(ws + p.list[i]);
  s.word = reinterpret_cast<int*>(ws + p.word);
  s.pos = reinterpret_cast<int*>(ws + p.pos);
  s.span = reinterpret_cast<int2*>(ws + p.span);
  s.total = reinterpret_cast<int*>(ws + p.total);
  s.per_owner = p.per_owner;
  s.all_words = a.beta != 1.0f;
  s.counters = reinterpret_cast<int*>(ws + p.counters);
  s.num_counters = p.num_counters;
  if (!sort_attributes()) return cudaErrorInvalidDevice;
  s.near_list = std::min(a.tokens, kSharedList);
  s.share = p.share;
  s.parts = reinterpret_cast<Entry*>(ws + p.parts);
  s.starts = reinterpret_cast<int*>(ws + p.starts);
  const std::size_t shared = 2 * s.near_list * sizeof(Entry);
  const EmbeddingFill fill = embedding_fill(a, sms());
  const int first_row = fill.rows;
  s.fill = static_cast<uint4*>(a.w);
  s.num_fill = fill.words;
  if (p.share > 0) {
    const cudaError_t e = tc::launch_overlapped(embedding_part_kernel, dim3(kParts), kSortThreads,
                                                0, st, false, s);
    if (e != cudaSuccess) return e;
  }
  const cudaError_t e = tc::launch_overlapped(embedding_sort_kernel, dim3(kOwners + fill.ctas),
                                              kSortThreads, shared, st, p.share > 0, s);
  if (e != cudaSuccess) return e;
  const bool wide = rows_of_runs(a, a.rows == T::kF32 ? 4 : 8);
  if (a.rows == T::kF32)
    return wide ? gradient<float, float, 4, 1, 16>(a, p, first_row, ws, st)
                : gradient<float, float, 1, 4, 8>(a, p, first_row, ws, st);
  if (a.rows == T::kF16) {
    if (a.table == T::kF32)
      return wide ? gradient<__half, float, 8, 1, 16>(a, p, first_row, ws, st)
                  : gradient<__half, float, 1, 4, 8>(a, p, first_row, ws, st);
    return wide ? gradient<__half, __half, 8, 1, 16>(a, p, first_row, ws, st)
                : gradient<__half, __half, 1, 4, 8>(a, p, first_row, ws, st);
  }
  if (a.table == T::kF32)
    return wide ? gradient<__nv_bfloat16, float, 8, 1, 16>(a, p, first_row, ws, st)
                : gradient<__nv_bfloat16, float, 1, 4, 8>(a, p, first_row, ws, st);
  return wide ? gradient<__nv_bfloat16, __nv_bfloat16, 8, 1, 16>(a, p, first_row, ws, st)
              : gradient<__nv_bfloat16, __nv_bfloat16, 1, 4, 8>(a, p, first_row, ws, st);
}

}  // namespace mb200::dnn
