"""Embedding lookup and its gradient against their definition in 64 bits.

Tolerances follow from the arithmetic, with u the largest relative error of a rounding to the
result's type (2^-8 for bf16, 2^-11 for fp16, 2^-24 for fp32) and `tiny` half a subnormal step:
  lookup    alpha w rounds to fp32, beta y is added with one more rounding, the result rounds
            to its type: 2^-24 (2 |alpha w| + |beta y|) + u |y| + tiny;
  gradient  a word of n rows takes at most n + 1 fp32 additions, in whichever shares, then
            alpha and beta as above.
"""

import ctypes as C
import math
import subprocess

import pytest

from muda_b200 import build, capi
from tests.helpers import Dnn, fptr

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -133, "fp16": 2.0 ** -25, "fp32": 2.0 ** -149}
CODE = {"bf16": capi.CUDNN_DATA_BFLOAT16, "fp16": capi.CUDNN_DATA_HALF,
        "fp32": capi.CUDNN_DATA_FLOAT}
TYPES = [("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32"), ("bf16", "fp32"), ("fp16", "fp32")]


def _dt(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


class Table:
    """Inputs, outputs and calls of one table; `rows` and `w` start as data for either call."""

    def __init__(self, torch, T, H, V, rows="bf16", table="bf16", seed=0, ld=None, offset=0,
                 out=0.0):
        self.torch, self.rt, self.wt = torch, rows, table
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        self.w = torch.randn(V, H, device="cuda", generator=g).to(_dt(torch, table))
        ld = H if ld is None else ld
        self.flat = torch.full((T * ld + offset,), 7.0, device="cuda", dtype=_dt(torch, rows))
        self.rows = self.flat[offset:].view(T, ld)[:, :H]
        self.rows.copy_(torch.randn(T, H, device="cuda", generator=g))
        self.tokens = torch.randint(0, V, (T,), device="cuda", generator=g)
        self.tokens[torch.rand(T, device="cuda", generator=g) < out] = -1

    def descriptors(self, d):
        T, H = self.rows.shape
        s = self.rows.stride(0)
        return (d.tensor(T, H, 1, 1, dtype=CODE[self.rt], strides=(s, 1, s, s)),
                d.filter(*self.w.shape, 1, 1, dtype=CODE[self.wt]))

    def forward(self, d, alpha=1.0, beta=0.0):
        rd, wd = self.descriptors(d)
        return d.L.cudnnEmbeddingForward(d.h, fptr(alpha), wd, _p(self.w), _p(self.tokens),
                                         fptr(beta), rd, _p(self.rows))

    def backward(self, d, alpha=1.0, beta=0.0, ws=None):
        rd, wd = self.descriptors(d)
        return d.L.cudnnEmbeddingBackward(d.h, fptr(alpha), rd, _p(self.rows), _p(self.tokens),
                                          _p(ws), 0 if ws is None else ws.numel(), fptr(beta), wd,
                                          _p(self.w))

    def workspace_size(self, d):
        rd, wd = self.descriptors(d)
        n = C.c_size_t()
        assert d.L.cudnnGetEmbeddingBackwardWorkspaceSize(d.h, rd, wd, C.byref(n)) == 0
        return n.value

    def check_forward(self, was, alpha=1.0, beta=0.0):
        torch = self.torch
        live = (self.tokens >= 0)[:, None]
        wy = torch.where(live, self.w.double()[self.tokens.clamp(min=0)] * alpha, 0.0)
        old = was.double() * beta if beta else torch.zeros_like(wy)
        want = wy + old
        tol = 2.0 ** -24 * (2 * wy.abs() + old.abs()) + U[self.rt] * want.abs() * 1.01 + TINY[self.rt]
        assert ((self.rows.double() - want).abs() <= tol).all()

    def check_backward(self, was, alpha=1.0, beta=0.0):
        torch = self.torch
        V, H = self.w.shape
        kept = ((self.tokens >= 0) & (self.tokens < V)).nonzero()[:, 0]
        t, dy = self.tokens[kept], self.rows[kept].double()
        zero = torch.zeros(V, H, device="cuda", dtype=torch.float64)
        total = zero.index_add(0, t, dy) * alpha
        mass = zero.index_add(0, t, dy.abs()) * abs(alpha)
        n = torch.bincount(t, minlength=V)[:, None]
        old = was.double() * beta if beta else zero
        want = total + old
        tol = (2.0 ** -24 * ((n + 2) * mass + old.abs()) * 1.01 + U[self.wt] * want.abs() * 1.01
               + TINY[self.wt])
        assert ((self.w.double() - want).abs() <= tol).all()
        if beta == 1.0:  # rows of words that do not occur keep their bits
            rest = n[:, 0] == 0
            assert torch.equal(self.w[rest], was[rest])


# (T, H, V): one of each; odd widths; words beyond the owners and their digits; long lists
SIZES = [(1, 1, 1), (1, 8, 1), (2, 64, 3), (1, 4096, 1000), (7, 17, 129), (33, 130, 40),
         (64, 1024, 127), (300, 72, 5000), (1000, 520, 128), (1025, 33, 70001), (5000, 24, 300),
         (2049, 1032, 17), (9001, 40, 4097)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,table", TYPES)
@pytest.mark.parametrize("T,H,V", SIZES)
def test_lookup(cuda, built, T, H, V, rows, table):
    e = Table(cuda, T, H, V, rows, table, seed=T + H, out=0.2)
    e.rows.fill_(math.nan)
    with Dnn(cuda) as d:
        assert e.forward(d, 3.5) == 0
        cuda.cuda.synchronize()
        e.check_forward(None, 3.5)
        was = e.rows.clone()
        assert e.forward(d, -0.75, 0.5) == 0
        cuda.cuda.synchronize()
        e.check_forward(was, -0.75, 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,table", TYPES)
@pytest.mark.parametrize("T,H,V", SIZES)
def test_gradient(cuda, built, T, H, V, rows, table):
    e = Table(cuda, T, H, V, rows, table, seed=T + H, out=0.2)
    e.w.fill_(math.nan)
    with Dnn(cuda) as d:
        assert e.backward(d, 1.5) == 0
        cuda.cuda.synchronize()
        e.check_backward(None, 1.5)
        for alpha, beta in ((2.0, 1.0), (1.0, -0.5)):
            was = e.w.clone()
            assert e.backward(d, alpha, beta) == 0
            cuda.cuda.synchronize()
            e.check_backward(was, alpha, beta)


@pytest.mark.gpu
@pytest.mark.parametrize("beta", [0.0, 1.0])
@pytest.mark.parametrize("rows,table", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("T,tokens", [
    (20000, "one word"), (20000, "two words of one owner"), (70000, "frequent words"),
    (70000, "one owner"), (9000, "one owner"), (4096, "runs"), (33000, "mostly padding"), (777, "all padding"),
])
def test_gradient_of_uneven_counts(cuda, built, T, tokens, rows, table, beta):
    """Words far more frequent than the others, and owners with most of the tokens."""
    H, V = 72, 50000
    e = Table(cuda, T, H, V, rows, table, seed=T)
    t, u = cuda.arange(T, device="cuda"), cuda.rand(T, device="cuda", generator=e.g)
    e.tokens = {
        "one word": t * 0 + 4242,
        "two words of one owner": cuda.where(u < 0.5, 130, 130 + 128 * 33),
        "frequent words": (cuda.exp(u.double() * math.log(V)) - 1).long(),
        "one owner": (u * 390).long() * 128 + 5,
        "runs": t // 16 * 3,
        "mostly padding": cuda.where(u < 0.999, -7, 49999),
        "all padding": t * 0 - 1,
    }[tokens]
    was = e.w.clone()
    with Dnn(cuda) as d:
        assert e.backward(d, 1.0, beta) == 0
        cuda.cuda.synchronize()
    e.check_backward(was, 1.0, beta)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,table", [("bf16", "bf16"), ("fp16", "fp32")])
@pytest.mark.parametrize("T,H,V,shift", [(8192, 1031, 20000, 0), (8193, 1032, 20003, 0),
                                         (300, 1032, 20003, 0), (9000, 1032, 20003, 1),
                                         (1, 4096, 6001, 0)])
def test_gradient_of_large_tables(cuda, built, T, H, V, shift, rows, table):
    """Tables that are filled while the tokens are sorted, from either end of the counts."""
    e = Table(cuda, T, H, V, rows, table, seed=T, out=0.1 if T > 1 else 0.0)
    flat = cuda.full((V * H + shift + 8,), 5.0, device="cuda", dtype=e.w.dtype)
    e.w = flat[shift:shift + V * H].view(V, H)
    with Dnn(cuda) as d:
        assert e.backward(d, 2.0) == 0
        cuda.cuda.synchronize()
        e.check_backward(None, 2.0)
        assert (flat[:shift] == 5).all() and (flat[shift + V * H:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 3000])
def test_few_tokens_of_very_many_words(cuda, built, T):
    """Accumulation into a table of three million words, after other calls in its workspace."""
    e = Table(cuda, T, 8, 3_000_000, "bf16", "fp32", seed=T)
    with Dnn(cuda) as d:
        ws = cuda.full((e.workspace_size(d),), 255, device="cuda", dtype=cuda.uint8)
        for _ in range(2):
            was = e.w.clone()
            e.tokens = cuda.randint(0, 3_000_000, (T,), device="cuda", generator=e.g)
            e.tokens[T // 2:] = e.tokens[0]
            assert e.backward(d, 1.0, 1.0, ws) == 0
            cuda.cuda.synchronize()
            e.check_backward(was, 1.0, 1.0)


@pytest.mark.gpu
def test_two_handles_at_once(cuda, built):
    """Calls of two handles on two streams: each gives the bits that it gives alone."""
    tables = [Table(cuda, 12000, 264, 900, seed=1), Table(cuda, 5000, 520, 7000, seed=2)]
    with Dnn(cuda) as a, Dnn(cuda) as b:
        want = []
        for e in tables:
            assert e.backward(a) == 0
            cuda.cuda.synchronize()
            e.check_backward(None)
            want.append(e.w.clone())
        streams = [cuda.cuda.Stream(), cuda.cuda.Stream()]
        for d, s in zip((a, b), streams):
            assert d.L.cudnnSetStream(d.h, C.c_void_p(s.cuda_stream)) == 0
        for _ in range(10):
            for e in tables:
                e.w.fill_(math.nan)
            cuda.cuda.synchronize()
            for _ in range(3):
                for d, e in zip((a, b), tables):
                    assert e.backward(d) == 0
            cuda.cuda.synchronize()
            assert all(cuda.equal(e.w, w) for e, w in zip(tables, want))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["bf16", "fp32"])
@pytest.mark.parametrize("H,ld,offset", [(128, 136, 0), (128, 131, 0), (128, 128, 1), (121, 200, 3),
                                         (8, 300, 8)])
def test_rows_in_wider_rows(cuda, built, H, ld, offset, rows):
    """Strided and unaligned rows; nothing between the rows is written."""
    e = Table(cuda, 100, H, 60, rows, rows, ld=ld, offset=offset, out=0.1)
    with Dnn(cuda) as d:
        assert e.forward(d, 2.0) == 0
        cuda.cuda.synchronize()
        e.check_forward(None, 2.0)
        mask = cuda.ones_like(e.flat, dtype=cuda.bool)
        mask[offset:].view(100, ld)[:, :H] = False
        assert (e.flat[mask] == 7).all()
        assert e.backward(d) == 0
        cuda.cuda.synchronize()
        e.check_backward(None)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [1, 8])
def test_tables_off_their_alignment(cuda, built, shift):
    e = Table(cuda, 50, 64, 99)
    flat = cuda.zeros(99 * 64 + shift, device="cuda", dtype=e.w.dtype)
    flat[shift:] = e.w.view(-1)
    e.w = flat[shift:].view(99, 64)
    with Dnn(cuda) as d:
        assert e.forward(d) == 0
        cuda.cuda.synchronize()
        e.check_forward(None)
        assert e.backward(d) == 0
        cuda.cuda.synchronize()
        e.check_backward(None)
    assert (flat[:shift] == 0).all()


@pytest.mark.gpu
def test_positions_of_a_tensor(cuda, built):
    """Rows given as the (n, h, w) positions of a channels-last tensor."""
    e = Table(cuda, 24, 40, 30)
    with Dnn(cuda) as d:
        rd = d.tensor(2, 40, 3, 4, dtype=CODE["bf16"], strides=(480, 1, 160, 40))
        wd = d.filter(30, 40, 1, 1, dtype=CODE["bf16"])
        assert d.L.cudnnEmbeddingForward(d.h, fptr(1.0), wd, _p(e.w), _p(e.tokens), fptr(0.0), rd,
                                         _p(e.rows)) == 0
        cuda.cuda.synchronize()
        e.check_forward(None)


@pytest.mark.gpu
def test_tokens_past_the_vocabulary(cuda, built):
    e = Table(cuda, 40, 64, 100)
    e.tokens[3], e.tokens[17], e.tokens[20] = 100, 1 << 40, -(1 << 62)
    with Dnn(cuda) as d:
        dy = e.rows.clone()
        assert e.forward(d) == 0
        cuda.cuda.synchronize()
        assert e.rows[3].isnan().all() and e.rows[17].isnan().all() and (e.rows[20] == 0).all()
        keep = (e.tokens >= 0) & (e.tokens < 100)
        assert cuda.equal(e.rows[keep], e.w[e.tokens[keep]])
        e.rows.copy_(dy)
        assert e.backward(d) == 0
        cuda.cuda.synchronize()
        e.check_backward(None)


@pytest.mark.gpu
def test_padding_hides_what_it_holds(cuda, built):
    """NaN and infinities in dy's rows of padding, or in words that no token asks for."""
    e = Table(cuda, 600, 72, 50, out=0.5)
    e.rows[e.tokens < 0] = math.nan
    with Dnn(cuda) as d:
        assert e.backward(d) == 0
        cuda.cuda.synchronize()
        clean = cuda.where(e.tokens[:, None] >= 0, e.rows, 0)
        e.rows = clean
        e.check_backward(None)
        f = Table(cuda, 600, 72, 50, out=0.5)
        f.tokens[f.tokens == 11] = 12
        f.w[11] = math.nan
        f.rows.fill_(math.inf)
        assert f.forward(d) == 0
        cuda.cuda.synchronize()
        assert f.rows.isfinite().all() and (f.rows[f.tokens < 0] == 0).all()


@pytest.mark.gpu
def test_infinite_and_nan_rows_reach_their_word_alone(cuda, built):
    e = Table(cuda, 500, 64, 20)
    at = (e.tokens == 3).nonzero()[:2, 0]
    e.rows[at[0], 5], e.rows[at[1], 9] = math.inf, math.nan
    with Dnn(cuda) as d:
        assert e.backward(d) == 0
        cuda.cuda.synchronize()
    assert e.w[3, 5] == math.inf and e.w[3, 9].isnan()
    e.w[3] = 0
    assert e.w.isfinite().all()


@pytest.mark.gpu
def test_two_micro_batches(cuda, built):
    """beta 1 after beta 0 adds a second batch; the sum is that of both."""
    a, b = Table(cuda, 3000, 96, 700, "bf16", "fp32", seed=1), Table(cuda, 2000, 96, 700, "bf16",
                                                                   "fp32", seed=2)
    b.w = a.w
    with Dnn(cuda) as d:
        assert a.backward(d, 0.5) == 0
        assert b.backward(d, 0.5, 1.0) == 0
        cuda.cuda.synchronize()
    both = Table(cuda, 5000, 96, 700, "bf16", "fp32")
    both.rows, both.tokens = cuda.cat([a.rows, b.rows]), cuda.cat([a.tokens, b.tokens])
    both.w = a.w
    both.check_backward(None, 0.5)


@pytest.mark.gpu
def test_gradient_against_differences(cuda, built):
    """The lookup is linear in the table: a table moved by a power of two times an integer
    direction, exact in fp32, moves sum c y by the gradient along it, up to fp32 sums."""
    e = Table(cuda, 400, 40, 90, "fp32", "fp32")
    c = cuda.randint(-8, 9, e.rows.shape, device="cuda", generator=e.g).float()
    move = cuda.randint(-4, 5, e.w.shape, device="cuda", generator=e.g).float()
    w0 = cuda.randint(-64, 65, e.w.shape, device="cuda", generator=e.g).float()
    values = []
    with Dnn(cuda) as d:
        for sign in (1, -1):
            e.w = w0 + sign * move
            assert e.forward(d, 0.5) == 0
            cuda.cuda.synchronize()
            values.append((e.rows.double() * c.double()).sum())
        e.rows, e.w = c.clone(), cuda.empty_like(w0)
        assert e.backward(d, 0.5) == 0
        cuda.cuda.synchronize()
    # every number here is a multiple of 1/2 below 2^20: no rounding anywhere
    assert (e.w.double() * move.double()).sum() == (values[0] - values[1]) / 2


@pytest.mark.gpu
def test_same_bits_on_any_stream_and_workspace(cuda, built):
    e = Table(cuda, 9000, 264, 3000, out=0.1)
    e.tokens = (e.tokens * e.tokens) // 3000
    want = None
    with Dnn(cuda) as d:
        size = e.workspace_size(d)
        ws = cuda.full((size,), 255, device="cuda", dtype=cuda.uint8)
        busy = cuda.randn(2048, 2048, device="cuda")
        cuda.cuda.synchronize()
        for given in (None, ws, None):
            stream = cuda.cuda.Stream()
            assert d.L.cudnnSetStream(d.h, C.c_void_p(stream.cuda_stream)) == 0
            for _ in range(4):
                busy = busy @ busy * 1e-3  # other work beside it
            e.w.fill_(math.nan)
            stream.wait_stream(cuda.cuda.current_stream())
            assert e.backward(d, 1.0, 0.0, given) == 0
            stream.synchronize()
            want = e.w.clone() if want is None else want
            assert cuda.equal(e.w, want)
    e.check_backward(None)


@pytest.mark.gpu
def test_captured_in_a_graph(cuda, built):
    """A captured pair of calls replays on new tokens, beside larger calls of the handle."""
    e, other, large = (Table(cuda, 300, 96, 200, seed=1, out=0.1),
                       Table(cuda, 300, 96, 200, seed=2, out=0.3),
                       Table(cuda, 20000, 96, 5000, seed=3))
    y = Table(cuda, 300, 96, 200, seed=4)
    y.tokens, y.w = e.tokens, other.w
    a, b = cuda.cuda.Stream(), cuda.cuda.Stream()
    with Dnn(cuda) as d:
        assert d.L.cudnnSetStream(d.h, C.c_void_p(a.cuda_stream)) == 0
        with cuda.cuda.stream(a):
            assert e.backward(d) == 0 and y.forward(d, 2.0) == 0
            a.synchronize()
            graph = cuda.cuda.CUDAGraph()
            with cuda.cuda.graph(graph, stream=a):
                assert e.backward(d) == 0 and y.forward(d, 2.0) == 0
        assert d.L.cudnnSetStream(d.h, C.c_void_p(b.cuda_stream)) == 0
        assert large.backward(d) == 0
        b.synchronize()
        large.check_backward(None)
        want = large.w.clone()
        e.tokens.copy_(other.tokens)
        e.rows.copy_(other.rows)
        for _ in range(10):
            e.w.fill_(math.nan)
            y.rows.fill_(math.nan)
            large.w.fill_(math.nan)
            cuda.cuda.synchronize()
            with cuda.cuda.stream(a):
                graph.replay()
            assert large.backward(d) == 0
            cuda.cuda.synchronize()
            e.check_backward(None)
            y.check_forward(None, 2.0)
            assert cuda.equal(large.w, want)
        del graph


@pytest.mark.gpu
def test_past_32_bit_offsets(cuda, built):
    """A table and rows of more than 2^31 elements: the far ends of both."""
    H, V = 4096, 530_000
    e = Table(cuda, 8, H, 64)
    e.w = cuda.zeros(V, H, device="cuda", dtype=cuda.bfloat16)
    e.w[-64:] = cuda.randn(64, H, device="cuda", generator=e.g)
    e.tokens = cuda.tensor([V - 1, 0, V - 2, V - 64, V - 1, -1, V, V - 3], device="cuda")
    with Dnn(cuda) as d:
        dy = e.rows.clone()
        assert e.forward(d) == 0
        cuda.cuda.synchronize()
        ok = cuda.tensor([0, 1, 2, 3, 4, 7], device="cuda")
        assert cuda.equal(e.rows[ok], e.w[e.tokens[ok]]) and e.rows[6].isnan().all()
        e.rows.copy_(dy)
        e.w.fill_(1.0)
        assert e.backward(d) == 0
        cuda.cuda.synchronize()
        assert (e.w[1:-64] == 0).all()
        want = (dy[0].float() + dy[4].float()).bfloat16()
        assert cuda.equal(e.w[-1], want) and cuda.equal(e.w[-2], dy[2])
        assert cuda.equal(e.w[-64], dy[3]) and cuda.equal(e.w[0], dy[1])
        # rows: the same table read into, and summed from, the last of 530000 rows
        del e.w
        f = Table(cuda, 2, H, 30)
        f.rows = cuda.zeros(V, H, device="cuda", dtype=cuda.bfloat16)
        f.tokens = cuda.full((V,), -1, device="cuda")
        f.tokens[-3:] = cuda.tensor([29, 3, 29], device="cuda")
        assert f.forward(d) == 0
        cuda.cuda.synchronize()
        assert cuda.equal(f.rows[-3:], f.w[f.tokens[-3:]]) and (f.rows[:-3] == 0).all()
        assert f.backward(d) == 0
        cuda.cuda.synchronize()
        assert cuda.equal(f.w[3], f.rows[-2]) and (f.w[4:29] == 0).all()
        assert cuda.equal(f.w[29], (f.rows[-1].float() * 2).bfloat16())


# ------------------------------------------------------------------------ refusals --
def test_refusals_before_the_device(built):
    bad, unsupported = capi.CUDNN_STATUS_BAD_PARAM, capi.CUDNN_STATUS_NOT_SUPPORTED
    bf, half, f32 = CODE["bf16"], CODE["fp16"], CODE["fp32"]
    with Dnn() as d:
        L, p = d.L, C.c_void_p(256)
        y, w = d.tensor(4, 64, 1, 1, dtype=bf), d.filter(100, 64, 1, 1, dtype=bf)
        one = fptr(1.0)

        def forward(alpha=one, w=w, wp=p, tokens=p, beta=one, y=y, yp=p, h=d.h):
            return L.cudnnEmbeddingForward(h, alpha, w, wp, tokens, beta, y, yp)

        def backward(alpha=one, w=w, wp=p, tokens=p, beta=one, y=y, yp=p, h=d.h):
            return L.cudnnEmbeddingBackward(h, alpha, y, yp, tokens, None, 0, beta, w, wp)

        for call in (forward, backward):
            for name in ("alpha", "beta", "wp", "yp", "tokens", "h", "w", "y"):
                assert call(**{name: None}) == bad, name
            assert call(w=y, y=w) == bad                                    # descriptors exchanged
            assert call(w=d.filter(100, 63, 1, 1, dtype=bf)) == bad
            assert call(w=d.filter(100, 64, 1, 3, dtype=bf)) == bad
            assert call(w=d.filter(100, 64, 1, 1, dtype=half)) == unsupported
            assert call(y=d.tensor(4, 64, 1, 1, dtype=f32)) == unsupported  # 16-bit table
            assert call(y=d.tensor(4, 64, 1, 3, dtype=bf)) == unsupported   # channels first
            assert call(y=d.tensor(4, 64, 1, 1, dtype=bf, strides=(63, 1, 1, 1))) == unsupported
            assert call(w=d.filter((1 << 30) + 1, 64, 1, 1, dtype=bf)) == unsupported
            assert call() == bad                                  # addresses no device knows
        n = C.c_size_t()
        size = L.cudnnGetEmbeddingBackwardWorkspaceSize
        assert size(d.h, y, w, None) == bad
        assert size(None, y, w, C.byref(n)) == bad
        assert size(d.h, w, y, C.byref(n)) == bad
        assert size(d.h, y, w, C.byref(n)) == 0
        stale = C.c_void_p(d.h.value)
    assert size(stale, y, w, C.byref(n)) == bad


def test_workspace_stays_bounded(built):
    """Some words of the table's size, and a fraction of the rows'."""
    with Dnn() as d:
        for T, H, V in ((1, 64, 100), (8192, 4096, 128000), (1 << 20, 1024, 50000),
                        (1 << 30, 64, 1000), (1, 8, 1 << 30)):
            n = C.c_size_t()
            assert d.L.cudnnGetEmbeddingBackwardWorkspaceSize(
                d.h, d.tensor(T, H, 1, 1, dtype=CODE["bf16"]),
                d.filter(V, H, 1, 1, dtype=CODE["bf16"]), C.byref(n)) == 0
            assert n.value <= 24 * T + 8 * (V + 128) + T * H // 2 + 8 * H + 4096


@pytest.mark.gpu
def test_refusals_of_memory(cuda, built):
    bad = capi.CUDNN_STATUS_BAD_PARAM
    e = Table(cuda, 32, 64, 100)
    with Dnn(cuda) as d:
        rd, wd = e.descriptors(d)
        L, one, zero = d.L, fptr(1.0), fptr(0.0)
        at = lambda t, by: C.c_void_p(t.data_ptr() + by)  # noqa: E731
        before = e.w.clone(), e.rows.clone()

        def both(tokens, w, rows):
            f = L.cudnnEmbeddingForward(d.h, one, wd, w, tokens, zero, rd, rows)
            b = L.cudnnEmbeddingBackward(d.h, one, rd, rows, tokens, None, 0, zero, wd, w)
            return f == bad and b == bad

        t, w, r = _p(e.tokens), _p(e.w), _p(e.rows)
        assert both(at(e.tokens, 4), w, r)
        assert both(t, at(e.w, 1), r)
        assert both(t, w, at(e.rows, 1))
        assert both(t, w, w)                                    # rows inside the table
        assert both(t, at(e.w, 1 << 34), r)
        assert both(t, _p(cuda.zeros(100, 64, dtype=e.w.dtype)), r)  # host memory
        size = e.workspace_size(d)
        ws = cuda.empty(size + 256, device="cuda", dtype=cuda.uint8)

        def given(p, n):
            return L.cudnnEmbeddingBackward(d.h, one, rd, r, t, p, n, zero, wd, w)

        assert given(_p(ws), size - 1) == bad
        assert given(at(ws, 8), size) == bad
        assert given(_p(ws), 1 << 40) == bad
        assert given(w, 100 * 64 * 2) == bad                    # over an operand
        cuda.cuda.synchronize()
        assert cuda.equal(e.w, before[0]) and cuda.equal(e.rows, before[1])
        assert given(_p(ws), size) == 0
        cuda.cuda.synchronize()
        e.check_backward(None)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["bf16", "fp32"])
@pytest.mark.parametrize("T,H", [(100, 512), (100, 37), (3, 64), (20000, 64)])
@pytest.mark.parametrize("beta", [1.0, 0.5])
def test_sums_and_tables_of_subnormals(cuda, built, rows, T, H, beta):
    """Sums of mixed sizes into a table of them: zeros, subnormals, cancellations."""
    e = Table(cuda, T, H, 64, rows=rows, table="fp32", seed=T + H)
    sizes = cuda.tensor([0.0, 2.0 ** -133, 2.0 ** -127, 2.0 ** -125, 2.0 ** -101, 2.0 ** -99, 1.0],
                        device="cuda")

    def mixed(t):
        s = sizes[cuda.randint(0, len(sizes), t.shape, device="cuda", generator=e.g)]
        sign = cuda.randint(0, 2, t.shape, device="cuda", generator=e.g) * 2 - 1
        t.copy_((s * sign).to(t.dtype))

    mixed(e.rows)
    mixed(e.w)
    e.rows[::2] = 0.0
    e.w[5] = -e.rows[e.tokens == 5].float().sum(0)
    was = e.w.clone()
    with Dnn(cuda) as d:
        assert e.backward(d, beta=beta) == 0
    cuda.cuda.synchronize()
    e.check_backward(was, beta=beta)


@pytest.mark.gpu
@pytest.mark.parametrize("beta", [0.0, 0.5, 1.0])
def test_gradient_into_pinned_memory(cuda, built, beta):
    e = Table(cuda, 300, 64, 100, rows="bf16", table="fp32")
    device = e.w
    e.w = device.cpu().pin_memory()
    with Dnn(cuda) as d:
        assert e.backward(d, beta=beta) == 0
    cuda.cuda.synchronize()
    e.w, was = e.w.cuda(), device
    e.check_backward(was, beta=beta)

PLAN = r"""
#include <cstdio>
#include <cstdlib>
#include "dnn/embedding.hpp"
int main(int, char** v) {
  using namespace mb200::dnn;
  EmbeddingArgs a{};
  a.table = std::atoi(v[1]) == 4 ? EmbeddingType::kF32 : EmbeddingType::kBF16;
  a.tokens = std::atoi(v[2]);
  a.features = std::atoi(v[3]);
  a.vocab = std::atoi(v[4]);
  a.w = reinterpret_cast<void*>(std::uintptr_t{256});
  for (int sms = 1; sms <= 160; ++sms) {
    const EmbeddingFill f = embedding_fill(a, sms);
    std::printf("%d %d %lld %u\n", sms, f.rows, static_cast<long long>(f.words), f.ctas);
  }
}
"""


def test_filling_beside_the_sort_on_any_number_of_sms(tmp_path):
    """Rows that the sort's launch fills have CTAs that fill them, behind the sort's own 128 and
    not beyond what the GPU holds beside them."""
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PLAN)
    subprocess.run([build.CXX, "-std=c++17", f"-I{build.CSRC}", f"-I{build.CUDA_HOME / 'include'}",
                    str(src), "-o", str(exe)], check=True)
    for size, T, H, V in ((2, 8192, 4096, 128000), (2, 32768, 2048, 50257), (4, 1, 512, 20000),
                          (2, 1537, 1111, 32003), (4, 10, 1 << 20, 9), (2, 5, 8, 1000)):
        out = subprocess.run([str(exe), *map(str, (size, T, H, V))], check=True,
                             capture_output=True, text=True).stdout
        plans = [tuple(map(int, line.split())) for line in out.splitlines()]
        assert len(plans) == 160
        for sms, rows, words, ctas in plans:
            assert 0 <= rows <= V and words * 16 == rows * H * size, (sms, rows, words)
            assert (ctas > 0) == (rows > 0), (sms, rows, ctas)
            assert ctas <= max(0, 2 * sms - 128) and ctas * 1024 < words + 1024, (sms, ctas)
        large = V * H * size >= 32 << 20 and 16 << 20 >= 8 * H * size
        assert (plans[147][1] > 0) == large


@pytest.mark.gpu
def test_refuses_another_devices_memory(cuda, built):
    if cuda.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    bad = capi.CUDNN_STATUS_BAD_PARAM
    e = Table(cuda, 32, 64, 100)
    with Dnn(cuda) as d:
        for name in ("rows", "w", "tokens"):
            here = getattr(e, name)
            setattr(e, name, here.to("cuda:1"))
            assert e.forward(d) == bad and e.backward(d) == bad, name
            setattr(e, name, here)
        ws = cuda.empty(e.workspace_size(d), device="cuda:1", dtype=cuda.uint8)
        assert e.backward(d, ws=ws) == bad
