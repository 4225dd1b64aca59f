// vocab_loss.hpp — launch interface of the losses over a linear head's vocabulary.
//
// With x (tokens x features) and w (vocab x features), 16-bit, and z = x w^T / tau:
//   cross entropy   loss = lse(z) - z[label]
//   distillation    q = softmax(teacher / tau) over the row's top_k entries,
//                   loss = sum_k q_k (log q_k - (z[index_k] - lse(z)))
//   gradient        dz = dloss / tau * (softmax(z) - q scattered to its indices),
//                   dx = dz w, dw = dz^T x
// Two losses are functions of the cross entropies (nll) of the tokens; their gradients are the
// cross entropy's with dloss times the derivative by each nll in dloss's place:
//   policy          r = exp(old - nll), s = min(r A, clip(r, lo, hi) A), at least dual A
//                   where A < 0 and dual > 0; d = nll - ref;
//                   loss = kl_coef (exp(d) - d - 1) - s
//   preference      of pairs of sequences (p, pairs + p): L = sum (or mean) of ref - nll over
//                   a sequence's tokens, h = beta (L_p - L_pairs+p) - margin,
//                   loss = softplus(-h) + smoothing h, max(0, 1 - h) or ((h - 1/2) / beta)^2
// A negative label (or index) leaves its row (or entry) out; a row that is left out has
// loss 0, log-sum-exp 0 and no gradient, whatever its x holds.  A label or index of
// vocab or more turns its row's loss, and the gradients that it enters, into NaN.
#pragma once

#include <cuda_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace mb200::dnn {

constexpr int kVocabMaxTopK = 256;

enum class HeadLoss : int { kTargets = 0, kPolicy = 1, kPreference = 2 };

struct PolicyLoss {
  const float* old_nll;  // [tokens], null: the tokens' own (r = 1)
  const float* ref_nll;  // [tokens], null: no divergence
  const float* advantage;
  float lo, hi;  // bounds of the clipped ratio
  float dual, kl_coef;
  float* loss;   // [tokens] each, may be null
  float* ratio;
  float* kl;
};

enum class PreferenceMode : int { kSigmoid = 0, kHinge = 1, kSquared = 2 };

struct PreferenceLoss {
  int pairs;
  const std::int64_t* offsets;  // [2 pairs + 1]
  const float* ref_nll;         // [tokens], null: 0
  PreferenceMode mode;
  bool averaged;
  double beta, margin, smoothing;
  float* loss;     // [pairs], may be null
  float* rewards;  // [2 pairs] beta L, may be null
};

struct VocabLossArgs {
  bool bf16;  // else fp16
  int tokens, features, vocab;
  const void* x;
  std::int64_t ldx;  // elements from one row of x to the next
  const void* w;     // rows of `features` elements, packed
  const std::int64_t* labels;  // cross entropy (top_k == 0)
  int top_k;                   // distillation: entries per row
  const std::int64_t* teacher_index;
  const float* teacher_logits;
  float inv_tau;
  float* loss;  // may be null; policy and preference: the tokens' nll
  float* lse;   // may be null
  HeadLoss head;  // of the cross entropies, unless kTargets
  PolicyLoss policy;
  PreferenceLoss preference;
  // gradients; dx or dw may be null (not computed)
  bool gradients;
  const float* dloss;  // [tokens], preference: [pairs]
  void* dx;
  std::int64_t lddx;
  void* dw;
};

// Workspace sizes depend on a.head and on whether a.loss is null as well.
// Device workspace that lets a call run in the pieces it prefers, one that lets it run in
// them wherever x and w start, and the least it can run in (one piece of 128 tokens at a
// time).  Only sizes, types, alignment and which gradients there are count.
std::size_t vocab_loss_workspace(const VocabLossArgs& a) noexcept;
std::size_t vocab_loss_workspace_any(const VocabLossArgs& a) noexcept;
std::size_t vocab_loss_min_workspace(const VocabLossArgs& a) noexcept;

// Runs the call in ws_bytes >= vocab_loss_min_workspace(a) bytes (256-byte aligned).
cudaError_t launch_vocab_loss(const VocabLossArgs& a, void* ws, std::size_t ws_bytes,
                              cudaStream_t stream) noexcept;

}  // namespace mb200::dnn
