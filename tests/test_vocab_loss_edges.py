"""Vocabulary losses where memory, streams and numbers are at their limits."""

import ctypes as C
import math

import pytest

from muda_b200 import capi
from tests.helpers import Dnn
from tests.test_vocab_loss import Head, _p

OUTPUTS = ("loss", "lse", "dx", "dw")


def _captured(torch, d, stream, call):
    """A graph of one call, after a first call on the stream has loaded the kernels."""
    assert d.L.cudnnSetStream(d.h, C.c_void_p(stream.cuda_stream)) == 0
    with torch.cuda.stream(stream):
        assert call() == 0
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert call() == 0
    return graph


@pytest.mark.gpu
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("K", [0, 7])
def test_graph_beside_other_calls_of_the_handle(cuda, built, K, own):
    """Replays on one stream and larger calls of the same handle on another, in no order
    between the two: both give the bits that each gives alone."""
    small, large = Head(cuda, 200, 96, 900, K=K, seed=1), Head(cuda, 1100, 136, 9001, K=K, seed=2)
    a, b = cuda.cuda.Stream(), cuda.cuda.Stream()
    with Dnn(cuda) as d:
        ws = cuda.empty(small.workspace_size(d, 1), device="cuda", dtype=cuda.uint8) if own else None
        cuda.cuda.synchronize()
        graph = _captured(cuda, d, a, lambda: small.backward(d, ws))
        with cuda.cuda.stream(a):
            graph.replay()
        a.synchronize()
        small.check()
        assert d.L.cudnnSetStream(d.h, C.c_void_p(b.cuda_stream)) == 0
        assert large.backward(d) == 0  # the handle's workspace grows
        b.synchronize()
        large.check()
        want = [[getattr(h, n).clone() for n in OUTPUTS] for h in (small, large)]
        for h in (small, large):
            for n in OUTPUTS:
                getattr(h, n).fill_(math.nan)
        cuda.cuda.synchronize()
        for _ in range(20):
            with cuda.cuda.stream(a):
                for _ in range(4):
                    graph.replay()
            assert large.backward(d) == 0
        cuda.cuda.synchronize()
    for h, w in zip((small, large), want):
        for n, t in zip(OUTPUTS, w):
            assert cuda.equal(getattr(h, n), t), n
    # a graph holds what it needs without the handle too
    for n in OUTPUTS:
        getattr(small, n).fill_(math.nan)
    cuda.cuda.synchronize()
    with cuda.cuda.stream(a):
        graph.replay()
    cuda.cuda.synchronize()
    for n, t in zip(OUTPUTS, want[0]):
        assert cuda.equal(getattr(small, n), t), n
    del graph
    cuda.cuda.synchronize()
