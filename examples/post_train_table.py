"""Post-trains a language model's one table, its embeddings and its head alike.

The smallest model that has both ends: a token's hidden state is its scaled row of the table
(cudnnEmbeddingForward), and the next token's logits are its products with all rows.  Two
kinds of steps train it, as a post-training program runs them on the cuDNN library:

- a clipped policy step with a divergence term on sampled tokens and their advantages
  (cudnnLinearPolicyLossBackward), from the log-probabilities that cudnnLinearPolicyLossForward
  gave when they were sampled;
- a preference step on pairs of sequences (cudnnLinearPreferenceLossBackward), against the
  log-probabilities of the table that training started from.

Either leaves the head's gradient in dw and the hidden states' in dx, and
cudnnEmbeddingBackward adds dx's rows to the same dw.  Run on a CUDA device:
``python examples/post_train_table.py``.
"""

from __future__ import annotations

import argparse
import ctypes as C
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

import torch

from muda_b200 import capi


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


class TiedTable:
    """A cuDNN handle with the descriptors of a table of V words and H features (bf16)."""

    def __init__(self, vocab: int, features: int, scale: float):
        self.lib, self.scale = capi.cudnn(), scale
        self.handle, self.table, self.rows = C.c_void_p(), C.c_void_p(), C.c_void_p()
        self._ok(self.lib.cudnnCreate(C.byref(self.handle)))
        self._ok(self.lib.cudnnCreateFilterDescriptor(C.byref(self.table)))
        self._ok(self.lib.cudnnSetFilter4dDescriptor(self.table, capi.CUDNN_DATA_BFLOAT16,
                                                     capi.CUDNN_TENSOR_NCHW, vocab, features, 1, 1))
        self._ok(self.lib.cudnnCreateTensorDescriptor(C.byref(self.rows)))

    def _ok(self, status: int) -> None:
        if status != 0:
            raise RuntimeError(self.lib.cudnnGetErrorString(status).decode())

    def hidden(self, w: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        """The tokens' scaled rows."""
        self._ok(self.lib.cudnnSetStream(
            self.handle, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        x = torch.empty(len(tokens), w.shape[1], device="cuda", dtype=w.dtype)
        self._ok(self.lib.cudnnSetTensor4dDescriptorEx(
            self.rows, capi.CUDNN_DATA_BFLOAT16, *x.shape, 1, 1, x.stride(0), 1, x.stride(0),
            x.stride(0)))
        self._ok(self.lib.cudnnEmbeddingForward(
            self.handle, C.byref(C.c_float(self.scale)), self.table, _p(w), _p(tokens),
            C.byref(C.c_float(0.0)), self.rows, _p(x)))
        return x

    def nll(self, w, tokens, labels):
        """Negative log-probabilities of the labels, 0 where a label is negative."""
        x = self.hidden(w, tokens)
        nll, unused = torch.empty(len(tokens), device="cuda"), torch.zeros(len(tokens), device="cuda")
        self._ok(self.lib.cudnnLinearPolicyLossForward(
            self.handle, self.rows, _p(x), self.table, _p(w), _p(labels), None, None, _p(unused),
            1.0, 0.2, 0.2, 0.0, 0.0, None, 0, None, _p(nll), None, None))
        return nll

    def _step(self, call, head, dloss, outs, w, x, tokens):
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        self._ok(call(*head, _p(dloss), None, 0, *map(_p, outs), self.rows, _p(dx), self.table,
                      _p(dw)))
        self._ok(self.lib.cudnnEmbeddingBackward(
            self.handle, C.byref(C.c_float(self.scale)), self.rows, _p(dx), _p(tokens), None, 0,
            C.byref(C.c_float(1.0)), self.table, _p(dw)))
        return dw

    def policy_step(self, w, tokens, labels, old, ref, advantages, dloss, clip=0.2, kl=0.05):
        """(losses, ratios, gradient of sum(dloss * losses) by the table)."""
        x = self.hidden(w, tokens)
        loss, ratio = torch.empty_like(dloss), torch.empty_like(dloss)
        head = (self.handle, self.rows, _p(x), self.table, _p(w), _p(labels), _p(old), _p(ref),
                _p(advantages), 1.0, clip, clip, 0.0, kl)
        dw = self._step(self.lib.cudnnLinearPolicyLossBackward, head, dloss,
                        (loss, None, ratio, None), w, x, tokens)
        return loss, ratio, dw

    def preference_step(self, w, tokens, labels, offsets, ref, dloss, beta=0.1):
        """(losses, rewards, gradient by the table) of len(dloss) pairs of sequences."""
        x = self.hidden(w, tokens)
        loss = torch.empty_like(dloss)
        rewards = torch.empty(2 * len(dloss), device="cuda")
        head = (self.handle, self.rows, _p(x), self.table, _p(w), _p(labels), len(dloss),
                _p(offsets), _p(ref), capi.CUDNN_PREFERENCE_SIGMOID, 0, beta, 0.0, 0.0)
        dw = self._step(self.lib.cudnnLinearPreferenceLossBackward, head, dloss,
                        (loss, rewards, None), w, x, tokens)
        return loss, rewards, dw

    def close(self) -> None:
        self._ok(self.lib.cudnnDestroyTensorDescriptor(self.rows))
        self._ok(self.lib.cudnnDestroyFilterDescriptor(self.table))
        self._ok(self.lib.cudnnDestroy(self.handle))


def train(steps=20, sequences=16, length=64, features=256, vocab=5000, rate=0.1, seed=0, log=print):
    """Policy steps, then preference steps; returns the losses of both."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sequences * length
    master = torch.randn(vocab, features, device="cuda", generator=g) / features ** 0.5
    tokens = torch.randint(0, vocab, (T,), device="cuda", generator=g)
    labels = tokens.roll(-1)
    labels.view(sequences, length)[:, :length // 4] = -100  # prompts
    labels.view(sequences, length)[:, -1] = -100            # nothing follows the last token
    good = torch.randn(sequences, device="cuda", generator=g)
    advantages = (good - good.mean()).repeat_interleave(length).contiguous()
    live = (labels >= 0).sum()
    table = TiedTable(vocab, features, features ** 0.5)
    policy, preference = [], []
    try:
        start = master.bfloat16()
        ref = table.nll(start, tokens, labels)
        dloss = torch.full((T,), 1.0, device="cuda") / live
        old = ref.clone()
        for step in range(steps):
            if step % 4 == 0:  # sampled anew
                old = table.nll(master.bfloat16(), tokens, labels)
            loss, ratio, dw = table.policy_step(master.bfloat16(), tokens, labels, old, ref,
                                                advantages, dloss)
            master -= rate * dw.float()
            policy.append(float((loss * dloss).sum()))
            clipped = ((ratio - 1).abs() > 0.2)[labels >= 0].float().mean()
            if step % 5 == 0 or step == steps - 1:
                log(f"policy step {step:3d}  loss {policy[-1]:8.4f}  clipped {float(clipped):.3f}")
        # preferences that have nothing to do with the advantages
        order = torch.randperm(sequences, device="cuda", generator=g)
        rows = (order[:, None] * length + torch.arange(length, device="cuda")).reshape(-1)
        tokens, labels, ref = tokens[rows], labels[rows], ref[rows]
        offsets = torch.arange(0, T + 1, length, device="cuda")
        dpair = torch.full((sequences // 2,), 2.0 / sequences, device="cuda")
        for step in range(steps):
            loss, rewards, dw = table.preference_step(master.bfloat16(), tokens, labels, offsets,
                                                      ref, dpair)
            master -= rate * dw.float()
            preference.append(float((loss * dpair).sum()))
            won = (rewards[:sequences // 2] > rewards[sequences // 2:]).float().mean()
            if step % 5 == 0 or step == steps - 1:
                log(f"preference step {step:3d}  loss {preference[-1]:8.4f}  won {float(won):.2f}")
    finally:
        table.close()
    return policy, preference


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--vocab", type=int, default=5000)
    a = parser.parse_args()
    train(steps=a.steps, vocab=a.vocab)
