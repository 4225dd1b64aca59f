// embedding.hpp — launch interface of the embedding lookup and its gradient.
//
// With a table w (vocab x features) and a token per row:
//   lookup     y[t] = alpha w[token[t]] + beta y[t]
//   gradient   dw[v] = alpha sum_{t: token[t] = v} dy[t] + beta dw[v]
// A negative token stands for a row of zeros and enters no gradient.  A token of vocab or
// more makes its row of y NaN and enters no gradient.  beta == 0: y or dw is not read.
#pragma once

#include <cuda_runtime_api.h>

#include <cstddef>
#include <cstdint>

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

}  // namespace mb200::dnn
