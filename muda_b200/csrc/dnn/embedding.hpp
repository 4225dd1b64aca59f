// embedding.hpp — launch interface of the embedding lookup and its gradient.
//
// With a table w (vocab x features) and a token per row:
//   lookup     y[t] = alpha w[token[t]] + beta y[t]
//   gradient   dw[v] = alpha sum_{t: token[t] = v} dy[t] + beta dw[v]
// A negative token stands for a row of zeros and enters no gradient.  A token of vocab or
// more makes its row of y NaN and enters no gradient.  beta == 0: y or dw is not read.
#pragma once

#include <cuda_runtime_api.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "common/device.hpp"

namespace mb200::dnn {

enum class EmbeddingType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

struct EmbeddingArgs {
  EmbeddingType table, rows;  // equal, or an fp32 table of 16-bit rows
  int tokens, features, vocab;
  const std::int64_t* token;
  float alpha, beta;
  void* row;           // lookup: y; gradient: dy (read only)
  std::int64_t ld;     // elements from one row to the next
  void* w;             // lookup: the table (read only); gradient: dw; rows packed
  bool device_table;   // gradient: dw is device memory, neither managed nor the host's
};

cudaError_t launch_embedding(const EmbeddingArgs& a, cudaStream_t stream) noexcept;

// Needs embedding_gradient_workspace(a) bytes (256-byte aligned); only a's sizes count.
std::size_t embedding_gradient_workspace(const EmbeddingArgs& a) noexcept;
cudaError_t launch_embedding_gradient(const EmbeddingArgs& a, void* workspace,
                                      cudaStream_t stream) noexcept;

// ----------------------------------------------------------- a part of the gradient's plan --
// CTAs of the sort, their threads, and the most tokens that it does not part first.
constexpr int kEmbeddingOwners = 128, kEmbeddingSortThreads = 1024, kEmbeddingParted = 8192;
// Bytes of a large dw that the GPU fills in the meantime (beta 0), about what the sort's time
// has room for: 8192 x 4096 of 128000 words 199 -> 193 us, 32768 x 2048 of 50257 128 -> 121,
// 1537 x 1111 of 32003 20.4 -> 19.5; a dw of 8 MB 18 -> 20.
constexpr std::int64_t kFillAtOnce = 16 << 20, kFillPerToken = 2000, kFillParted = 1000;
constexpr std::int64_t kFillLeast = 32 << 20;

struct EmbeddingFill {
  int rows;            // from the first on; the sums' launch sees to the others
  std::int64_t words;  // of 16 bytes
  unsigned ctas;       // behind the sort's own
};

// The sort's CTAs come first, two to an SM: a GPU (or a part of one) of 64 SMs or fewer has room
// for no others, and leaves all rows to the sums.
inline EmbeddingFill embedding_fill(const EmbeddingArgs& a, int sms) noexcept {
  const std::int64_t row_bytes =
      static_cast<std::int64_t>(a.features) * (a.table == EmbeddingType::kF32 ? 4 : 2);
  const std::int64_t spare = 2ll * sms - kEmbeddingOwners;
  if (a.beta != 0.0f || !aligned_to(a.w, 16) || a.vocab * row_bytes < kFillLeast || spare <= 0)
    return {0, 0, 0};
  const std::int64_t bytes =
      kFillAtOnce + a.tokens * (a.tokens <= kEmbeddingParted ? kFillPerToken : kFillParted);
  // multiples of 8 rows are whole 16-byte words
  const auto rows = static_cast<int>(std::min<std::int64_t>(a.vocab, bytes / row_bytes) / 8 * 8);
  const std::int64_t words = rows * row_bytes / 16;
  return {rows, words,
          static_cast<unsigned>(std::min<std::int64_t>(
              spare, (words + kEmbeddingSortThreads - 1) / kEmbeddingSortThreads))};
}

}  // namespace mb200::dnn
