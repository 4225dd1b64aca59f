"""Trains a student's vocabulary head on labels and on a teacher's cached top logits.

One step on T tokens, as a training program runs it on the cuDNN library's vocabulary
losses:

    loss = (1 - a) * cross entropy(labels) + a * distillation(teacher's top K logits)

cudnnLinearCrossEntropyBackward and cudnnLinearDistillationBackward return each loss with
the gradients of the hidden states and of the head; the T x V logits are never stored.  At
the end the held-out tokens are scored one by one with the Forward calls, as a decoder
would.  Run on a CUDA device: ``python examples/distill_head.py``.
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


class VocabularyLosses:
    """A cuDNN handle with the descriptors of a head of V words and H features."""

    def __init__(self, vocab: int, features: int):
        self.lib = capi.cudnn()
        self.handle = C.c_void_p()
        self._ok(self.lib.cudnnCreate(C.byref(self.handle)))
        self.w_desc = C.c_void_p()
        self._ok(self.lib.cudnnCreateFilterDescriptor(C.byref(self.w_desc)))
        self._ok(self.lib.cudnnSetFilter4dDescriptor(self.w_desc, capi.CUDNN_DATA_BFLOAT16,
                                                     capi.CUDNN_TENSOR_NCHW, vocab, features, 1, 1))
        self.x_desc = C.c_void_p()
        self._ok(self.lib.cudnnCreateTensorDescriptor(C.byref(self.x_desc)))

    def _ok(self, status: int) -> None:
        if status != 0:
            raise RuntimeError(self.lib.cudnnGetErrorString(status).decode())

    def _enter(self, x: torch.Tensor) -> None:
        self._ok(self.lib.cudnnSetStream(
            self.handle, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        self._ok(self.lib.cudnnSetTensor4dDescriptorEx(
            self.x_desc, capi.CUDNN_DATA_BFLOAT16, x.shape[0], x.shape[1], 1, 1, x.stride(0), 1,
            x.stride(0), x.stride(0)))

    def _targets(self, targets, temperature):
        if isinstance(targets, tuple):
            index, logits = targets
            return (index.shape[1], C.c_void_p(index.data_ptr()), C.c_void_p(logits.data_ptr()),
                    temperature)
        return (C.c_void_p(targets.data_ptr()),)

    def forward(self, x, w, targets, temperature=1.0):
        """Losses of the tokens; targets: labels, or (teacher indices, teacher logits)."""
        self._enter(x)
        loss = torch.empty(x.shape[0], device=x.device)
        call = (self.lib.cudnnLinearDistillationForward if isinstance(targets, tuple)
                else self.lib.cudnnLinearCrossEntropyForward)
        self._ok(call(self.handle, self.x_desc, C.c_void_p(x.data_ptr()), self.w_desc,
                      C.c_void_p(w.data_ptr()), *self._targets(targets, temperature), None, 0,
                      C.c_void_p(loss.data_ptr()), None))
        return loss

    def backward(self, x, w, targets, dloss, temperature=1.0):
        """(losses, dx, dw) of sum(dloss * loss)."""
        self._enter(x)
        loss = torch.empty(x.shape[0], device=x.device)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        call = (self.lib.cudnnLinearDistillationBackward if isinstance(targets, tuple)
                else self.lib.cudnnLinearCrossEntropyBackward)
        self._ok(call(self.handle, self.x_desc, C.c_void_p(x.data_ptr()), self.w_desc,
                      C.c_void_p(w.data_ptr()), *self._targets(targets, temperature),
                      C.c_void_p(dloss.data_ptr()), None, 0, C.c_void_p(loss.data_ptr()), None,
                      self.x_desc, C.c_void_p(dx.data_ptr()), self.w_desc,
                      C.c_void_p(dw.data_ptr())))
        return loss, dx, dw

    def close(self) -> None:
        self._ok(self.lib.cudnnDestroyTensorDescriptor(self.x_desc))
        self._ok(self.lib.cudnnDestroyFilterDescriptor(self.w_desc))
        self._ok(self.lib.cudnnDestroy(self.handle))


def train(steps=30, tokens=512, features=256, vocab=5000, top_k=16, temperature=2.0, mix=0.5,
          rate=20.0, seed=0, log=print):
    """Returns the mean combined loss before and after, and the held-out losses one by one."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    teacher = (3.0 * randn(vocab, features) / features ** 0.5).bfloat16()
    master = 0.1 * randn(vocab, features) / features ** 0.5  # the student's fp32 weights
    x = randn(tokens + 8, features).bfloat16()
    cached, index = (x.float() @ teacher.float().t()).topk(top_k, dim=1)
    labels = index[:, 0].clone()
    labels[:tokens // 16] = -100  # a prompt: its tokens are not trained on
    index[:tokens // 16] = -1
    train_x, held_x = x[:tokens], x[tokens:]

    losses = VocabularyLosses(vocab, features)
    live = int((labels[:tokens] >= 0).sum())
    dloss = torch.full((tokens,), 1.0 / live, device="cuda")
    history = []
    try:
        for step in range(steps):
            w = master.bfloat16()
            ce, _, dw_ce = losses.backward(train_x, w, labels[:tokens], (1 - mix) * dloss)
            kd, _, dw_kd = losses.backward(train_x, w, (index[:tokens], cached[:tokens]),
                                           mix * dloss, temperature)
            master -= rate * (dw_ce.float() + dw_kd.float())
            history.append(float(((1 - mix) * ce + mix * kd).sum() / live))
            if step % 10 == 0 or step == steps - 1:
                log(f"step {step:3d}  loss {history[-1]:.4f}")
        w = master.bfloat16()
        one_by_one = [float(losses.forward(held_x[i:i + 1], w, labels[tokens + i:tokens + i + 1]))
                      for i in range(held_x.shape[0])]
        together = losses.forward(held_x, w, labels[tokens:])
    finally:
        losses.close()
    log("held-out log-probabilities: " + ", ".join(f"{-v:.3f}" for v in one_by_one))
    return history, one_by_one, together.tolist()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=30)
    parser.add_argument("--tokens", type=int, default=512)
    parser.add_argument("--vocab", type=int, default=5000)
    a = parser.parse_args()
    train(steps=a.steps, tokens=a.tokens, vocab=a.vocab)
