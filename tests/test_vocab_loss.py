"""Vocabulary losses (linear cross entropy, distillation from a teacher's top logits)
against their definition in 64 bits.

Tolerances follow from the arithmetic, with u the unit roundoff of the 16-bit type (2^-8
for bf16's 8 significant bits, 2^-11 for fp16's 11):
  logits   fp32 accumulation of exact products: (H + 32) 2^-23 sum |x w| / tau at most;
  lse      the largest logit error of its row, plus 2^-20 (1 + |lse|) for the exponentials,
           sums and logarithm; loss: twice the logit error likewise;
  dz       two roundings of a word's numerator, 2 u |p|, one at the targets, u |p - q|,
           plus the logit errors (relative in p);
  dx, dw   the products' |dz| |w| weighted errors, plus one rounding of the result.
"""

import ctypes as C
import math

import pytest

from muda_b200 import capi
from tests.helpers import Dnn

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
TINY = {"bf16": 2.0 ** -133, "fp16": 2.0 ** -25}  # half a subnormal step


def _dt(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _code(name):
    return {"bf16": capi.CUDNN_DATA_BFLOAT16, "fp16": capi.CUDNN_DATA_HALF}[name]


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


class Head:
    """Inputs, outputs and calls of one head; outputs start as NaN."""

    def __init__(self, torch, T, H, V, dtype="bf16", K=0, tau=1.0, seed=0, spread=1.0, ldx=None,
                 offset=0, out=0.0):
        self.torch, self.dtype, self.K, self.tau = torch, dtype, K, tau
        g = torch.Generator(device="cuda").manual_seed(seed)
        dt = _dt(torch, dtype)
        self.g = g
        self.w = (torch.randn(V, H, device="cuda", generator=g) * spread / math.sqrt(H)).to(dt)
        ldx = H if ldx is None else ldx
        flat = torch.zeros(T * ldx + offset, device="cuda", dtype=dt)
        self.x = flat[offset:].view(T, ldx)[:, :H]
        self.x.copy_(torch.randn(T, H, device="cuda", generator=g))
        left = torch.rand(T, device="cuda", generator=g) < out
        self.labels = torch.randint(0, V, (T,), device="cuda", generator=g)
        self.labels[left] = -100
        self.index = self.teacher = None
        if K:
            self.index = torch.randint(0, V, (T, K), device="cuda", generator=g)  # may repeat
            self.index[torch.rand(T, K, device="cuda", generator=g) < 0.2] = -1
            self.index[left] = -1
            self.teacher = torch.randn(T, K, device="cuda", generator=g) * 3
        self.dloss = torch.randn(T, device="cuda", generator=g) / T
        nan = dict(device="cuda", dtype=torch.float32)
        self.loss, self.lse = torch.full((T,), math.nan, **nan), torch.full((T,), math.nan, **nan)
        self.dx = torch.full((T, H), math.nan, device="cuda", dtype=dt)
        self.dw = torch.full((V, H), math.nan, device="cuda", dtype=dt)

    def _head(self, d, x=None):
        T, H = self.x.shape
        xs = (self.x if x is None else x).stride(0)
        xd = d.tensor(T, H, 1, 1, dtype=_code(self.dtype), strides=(xs, 1, xs, xs))
        wd = d.filter(*self.w.shape, 1, 1, dtype=_code(self.dtype))
        args = (d.h, xd, _p(self.x), wd, _p(self.w))
        if self.K:
            return xd, wd, args + (self.K, _p(self.index), _p(self.teacher), self.tau)
        return xd, wd, args + (_p(self.labels),)

    def forward(self, d, ws=None):
        _, _, args = self._head(d)
        fn = d.L.cudnnLinearDistillationForward if self.K else d.L.cudnnLinearCrossEntropyForward
        return fn(*args, _p(ws), 0 if ws is None else ws.numel(), _p(self.loss), _p(self.lse))

    def backward(self, d, ws=None, dx=True, dw=True, loss=True):
        xd, wd, args = self._head(d)
        dxd = None
        if dx:
            s = self.dx.stride(0)
            dxd = d.tensor(*self.dx.shape, 1, 1, dtype=_code(self.dtype), strides=(s, 1, s, s))
        fn = d.L.cudnnLinearDistillationBackward if self.K else d.L.cudnnLinearCrossEntropyBackward
        return fn(*args, _p(self.dloss), _p(ws), 0 if ws is None else ws.numel(),
                  _p(self.loss) if loss else None, _p(self.lse) if loss else None,
                  dxd, _p(self.dx) if dx else None, wd if dw else None, _p(self.dw) if dw else None)

    def workspace_size(self, d, gradients):
        xd, wd, _ = self._head(d)
        n = C.c_size_t()
        if self.K:
            s = d.L.cudnnGetLinearDistillationWorkspaceSize(d.h, xd, wd, self.K, gradients, C.byref(n))
        else:
            s = d.L.cudnnGetLinearCrossEntropyWorkspaceSize(d.h, xd, wd, gradients, C.byref(n))
        assert s == 0
        return n.value

    def definition(self):
        """loss, lse, dz, dx, dw in 64 bits, the rows that are in, and the target weights."""
        torch = self.torch
        w = self.w.double()
        T, V = self.x.shape[0], w.shape[0]
        target = torch.zeros(T, V, device="cuda", dtype=torch.float64)
        entropy = torch.zeros(T, device="cuda", dtype=torch.float64)
        if self.K:
            t = torch.where(self.index >= 0, self.teacher.double() / self.tau, -math.inf)
            live = (t > -math.inf).any(dim=1)
            q = torch.softmax(t[live], dim=1)
            target[live] = target[live].scatter_add(1, self.index[live].clamp(min=0), q)
            entropy[live] = torch.special.xlogy(q, q).sum(dim=1)
        else:
            live = self.labels >= 0
            target[live, self.labels[live]] = 1.0
        x = torch.where(live[:, None], self.x.double(), 0.0)
        z = x @ w.t() / self.tau
        lse = torch.logsumexp(z, dim=1)
        cross = torch.where(target > 0, target * z, 0.0).sum(dim=1)
        loss = torch.where(live, entropy + lse - cross, 0.0)
        dloss = torch.where(live, self.dloss.double(), 0.0) / self.tau
        p = torch.exp(z - lse[:, None])
        dz = dloss[:, None] * (p - target)
        return dict(loss=loss, lse=torch.where(live, lse, 0.0), dz=dz, dx=dz @ w, dw=dz.t() @ x,
                    live=live, p=p, target=target, x=x, w=w, dloss=dloss)

    def check(self, dx=True, dw=True, loss=True, gradients=True):
        torch, u = self.torch, U[self.dtype]
        ref = self.definition()
        x, w, live = ref["x"].abs(), ref["w"].abs(), ref["live"]
        H = x.shape[1]
        zerr = (x @ w.t()).amax(dim=1) * (H + 32) * 2.0 ** -23 / self.tau
        if loss:
            tol = zerr + 2.0 ** -20 * (1 + ref["lse"].abs())
            assert ((self.lse.double() - ref["lse"]).abs() <= tol * live).all()
            tol = 2 * zerr + 2.0 ** -19 * (1 + ref["lse"].abs() + ref["loss"].abs())
            assert ((self.loss.double() - ref["loss"]).abs() <= tol * live).all()
        if not gradients:
            return ref
        # dz: two roundings of the numerators, one at the targets, and the logit errors in p
        g = ref["dloss"].abs()[:, None]
        p = ref["p"] * live[:, None]
        derr = g * p * (2 * u * (1 + u) + 2 * zerr[:, None] + 2.0 ** -18)
        derr += (ref["target"] > 0) * (u * ref["dz"].abs() + g * (2.0 ** -19 + 2 * zerr[:, None]) * 2)
        if self.dtype == "fp16":  # subnormal numerators, and subnormal dz after the scaling
            top = g.max()
            derr += live[:, None] * (g * p.amax(dim=1, keepdim=True) + top * 2.0 ** -12) * 2.0 ** -24
        tiny = TINY[self.dtype]
        T, V = p.shape
        if dx:
            a = ref["dz"].abs() @ w
            tol = derr @ w + u * ref["dx"].abs() * 1.01 + a * (V + 32) * 2.0 ** -23 + tiny
            assert ((self.dx.double() - ref["dx"]).abs() <= tol).all()
        if dw:
            a = ref["dz"].abs().t() @ x
            tol = derr.t() @ x + u * ref["dw"].abs() * 1.01 + a * (T + 32) * 2.0 ** -23 + tiny
            assert ((self.dw.double() - ref["dw"]).abs() <= tol).all()
        return ref


# (T, H, V): single tokens, words and features; tile edges; odd sizes
SIZES = [(1, 8, 1), (1, 1, 7), (2, 16, 3), (1, 64, 129), (5, 24, 130), (127, 72, 257),
         (128, 64, 128), (129, 65, 255), (200, 136, 1000), (300, 250, 513), (64, 512, 4099),
         (513, 192, 777), (1100, 40, 2100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V", SIZES)
def test_cross_entropy(cuda, built, T, H, V, dtype):
    h = Head(cuda, T, H, V, dtype, out=0.2 if T > 4 else 0.0, seed=T + H)
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        h.check(gradients=False)
        h.loss.fill_(math.nan)
        h.lse.fill_(math.nan)
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V,K,tau", [(1, 8, 1, 1, 1.0), (1, 64, 129, 3, 2.0), (3, 16, 5, 256, 1.0),
                                         (127, 72, 257, 32, 0.5), (129, 65, 255, 33, 4.0),
                                         (300, 250, 513, 7, 1.0), (64, 512, 4099, 128, 1.5),
                                         (1100, 40, 2100, 20, 2.0)])
def test_distillation(cuda, built, T, H, V, K, tau, dtype):
    h = Head(cuda, T, H, V, dtype, K=K, tau=tau, out=0.2 if T > 4 else 0.0, seed=T + K)
    if T == 1:
        h.index[0, 0] = V - 1
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        h.check(gradients=False)
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V,K", [
    (300, 600, 20000, 0),    # dx on tall tiles, two of them along the features
    (131, 1111, 17003, 5),   # rows that suit neither TMA nor lines, uneven tile widths
    (6200, 72, 700, 0),      # dw on tall tiles
    (6200, 121, 515, 3),     # the same with rows of dw that TMA cannot address
    (2500, 1032, 3001, 0),   # several bands of tiles, five tiles of features
    (777, 264, 2003, 20),
    (9, 264, 33000, 0),      # few tokens, many words
    (128, 520, 20001, 64),
])
def test_tilings(cuda, built, T, H, V, K, dtype):
    h = Head(cuda, T, H, V, dtype, K=K, tau=1.5 if K else 1.0, out=0.1, seed=T + V)
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        h.check(gradients=False)
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V", [(1, 1000, 333), (3, 136, 5000), (7, 8, 17), (8, 2056, 1601)])
@pytest.mark.parametrize("K", [0, 1, 40])
def test_few_tokens_scored(cuda, built, T, H, V, K, dtype):
    h = Head(cuda, T, H, V, dtype, K=K, tau=2.0 if K else 1.0, seed=H)
    if K:
        h.index[:, 0] = V - 1
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
    h.check(gradients=False)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 40, 300])
def test_clustered_targets(cuda, built, T):
    """Up to 256 targets of a token among neighbouring words, some of them equal."""
    h = Head(cuda, T, 64, 3000, K=256, seed=T)
    h.index = cuda.randint(1100, 1100 + 180, (T, 256), device="cuda", generator=h.g)
    h.index[1] = 2999
    h.index[2, 3:] = -1
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        h.check(gradients=False)
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    h.check()


@pytest.mark.gpu
def test_nan_word_reaches_every_row(cuda, built):
    """A NaN in one word's weights makes every live row NaN, as the formula has it."""
    for T in (4, 100, 300):
        h = Head(cuda, T, 64, 700, seed=T)
        h.labels[0] = -1
        h.w[555, 3] = math.nan
        with Dnn(cuda) as d:
            assert h.forward(d) == 0
            cuda.cuda.synchronize()
        assert h.loss[1:].isnan().all() and h.lse[1:].isnan().all()
        assert h.loss[0] == 0 and h.lse[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("K", [0, 7])
def test_captured_in_a_graph(cuda, built, K):
    """A captured step replays on new inputs at the same addresses."""
    h = Head(cuda, 200, 96, 900, K=K, seed=1)
    other = Head(cuda, 200, 96, 900, K=K, seed=2)
    stream = cuda.cuda.Stream()
    with Dnn(cuda) as d, cuda.cuda.stream(stream):
        assert d.L.cudnnSetStream(d.h, C.c_void_p(stream.cuda_stream)) == 0
        assert h.backward(d) == 0  # grows the workspace before the capture
        stream.synchronize()
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph, stream=stream):
            assert h.backward(d) == 0
        for name in ("x", "w", "dloss", "labels") + (("index", "teacher") if K else ()):
            getattr(h, name).copy_(getattr(other, name))
        for t in (h.loss, h.lse, h.dx, h.dw):
            t.fill_(math.nan)
        graph.replay()
        stream.synchronize()
        del graph
    h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K", [0, 6])
def test_rows_left_out_may_hold_anything(cuda, built, K, dtype):
    """NaN and infinite hidden states, teachers and upstream gradients of rows that are out."""
    h = Head(cuda, 150, 72, 300, dtype, K=K, out=0.3, seed=3)
    out = (h.index < 0).all(dim=1) if K else h.labels < 0
    assert 10 < int(out.sum()) < 100
    h.x[out] = math.nan
    h.x[out.nonzero()[0, 0], ::2] = math.inf
    h.dloss[out] = math.nan
    h.dloss[out.nonzero()[1, 0]] = 3e38
    if K:
        h.teacher[out] = math.nan
        h.teacher[h.index < 0] = math.inf  # entries that are out, in rows that are in
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    assert (h.loss[out] == 0).all() and (h.lse[out] == 0).all() and (h.dx[out] == 0).all()
    h.x[out] = 0
    h.dloss[out] = 0
    h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [0, 4])
def test_every_row_left_out(cuda, built, K):
    h = Head(cuda, 70, 64, 200, K=K)
    h.labels.fill_(-1)
    if K:
        h.index[::2] = -1
        h.teacher[1::2] = -math.inf  # a teacher logit of -inf leaves its entry out too
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    for t in (h.loss, h.lse, h.dx, h.dw):
        assert (t == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [0, 5])
def test_target_past_the_vocabulary_is_nan(cuda, built, K):
    h = Head(cuda, 40, 64, 200, K=K)
    bad = 200 if not K else 1 << 40
    if K:
        h.index[7, 2] = bad
        h.index[9] = bad
    else:
        h.labels[7] = bad
        h.labels[9] = 1 << 35
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    odd = cuda.tensor([7, 9], device="cuda")
    assert h.loss[odd].isnan().all() and h.dx[odd].isnan().all()
    rest = cuda.ones(40, dtype=cuda.bool, device="cuda")
    rest[odd] = False
    assert h.loss[rest].isfinite().all() and h.dx[rest].isfinite().all()
    assert h.dw.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_large_logits(cuda, built, dtype):
    """Logits of hundreds: one word takes all, the others' exponentials vanish."""
    h = Head(cuda, 130, 128, 700, dtype, spread=60.0, seed=5)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    ref = h.check()
    assert ref["lse"].max() > 150


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gradients_show_two_roundings(cuda, built, dtype):
    """dw of the words that are no token's target, against a model in 64 bits that rounds dz
    and the result once each.  The 2 further bits that carry the numerators add 1/16 to the
    variance of one rounding, 1/32 or 1.6 % of the pair's deviation; the model scatters by
    1.5 % over seeds.  A third full rounding would add 7 to 18 %."""
    h = Head(cuda, 300, 136, 1203, dtype, seed=41)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    ref = h.check()
    bits = {"bf16": 8, "fp16": 11}[dtype]
    m, e = cuda.frexp(ref["dz"])  # dz is scaled clear of fp16's subnormals, dw is not
    model = cuda.ldexp((m * 2 ** bits).round() / 2 ** bits, e).t() @ ref["x"]
    model = model.to(h.dw.dtype).double()
    rows = (ref["target"] == 0).all(dim=0)
    error = (h.dw.double() - ref["dw"])[rows].norm()
    assert error <= 1.05 * (model - ref["dw"])[rows].norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V,K", [(1, 64, 129, 0), (7, 1000, 5003, 4), (129, 65, 255, 0),
                                     (300, 250, 513, 7), (260, 600, 50001, 0),
                                     (700, 136, 3000, 30)])
def test_frozen_head(cuda, built, T, H, V, K, dtype):
    """Only the hidden states' gradient."""
    h = Head(cuda, T, H, V, dtype, K=K, tau=2.0 if K else 1.0, out=0.2 if T > 4 else 0.0, seed=T)
    with Dnn(cuda) as d:
        assert h.backward(d, dw=False) == 0
        cuda.cuda.synchronize()
    h.check(dw=False)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [0, 5])
@pytest.mark.parametrize("T", [40, 200])
@pytest.mark.parametrize("offset", [0.0, 60.0, -60.0, 400.0, -400.0])
@pytest.mark.parametrize("spread", [1.0, 60.0])
def test_frozen_head_offset_logits(cuda, built, T, K, offset, spread):
    """Logits far from zero, by a common offset, by their spread, or both; rows that are left
    out hold NaN."""
    h = Head(cuda, T, 128, 900, K=K, spread=spread, out=0.2, seed=T + K)
    h.x[:, 0] = 8.0
    h.w[:, 0] = offset / 8.0
    out = (h.index < 0).all(dim=1) if K else h.labels < 0
    h.x[out] = math.nan
    with Dnn(cuda) as d:
        assert h.backward(d, dw=False) == 0
        cuda.cuda.synchronize()
    assert (h.dx[out] == 0).all() and (h.loss[out] == 0).all()
    h.check(dw=False)


@pytest.mark.gpu
def test_infinite_words(cuda, built):
    """A word whose logit is -inf has probability 0; all of them: NaN, as the formula."""
    h = Head(cuda, 33, 64, 300)
    h.x.abs_()
    h.x.add_(0.5)
    h.w[5:290] = -math.inf
    h.labels.fill_(2)
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        z = h.x.double() @ h.w.double()[list(range(5)) + list(range(290, 300))].t()
        lse = cuda.logsumexp(z, dim=1)
        finite = h.w[list(range(5)) + list(range(290, 300))].double().abs()
        tol = (h.x.double() @ finite.t()).amax(dim=1) * 96 * 2.0 ** -22 + 2.0 ** -18 * (1 + lse.abs())
        assert ((h.lse.double() - lse).abs() <= tol).all()
        assert ((h.loss.double() - (lse - z[:, 2])).abs() <= 2 * tol).all()
        h.w.fill_(-math.inf)
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        assert h.loss.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("ldx,offset", [(136, 0), (145, 0), (136, 3), (128, 1)])
@pytest.mark.parametrize("H", [128, 121])
def test_strided_rows(cuda, built, H, ldx, offset, dtype):
    """x and dx inside wider rows, from addresses that are aligned to one element only; the
    columns between dx's rows stay as they are."""
    h = Head(cuda, 140, H, 333, dtype, ldx=ldx, offset=offset, out=0.1)
    wide = cuda.full((140 * (ldx + 5) + offset,), 7.0, device="cuda", dtype=h.dx.dtype)
    rows = wide[offset:].view(140, ldx + 5)
    h.dx = rows[:, :H]
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    h.check()
    assert (rows[:, H:] == 7).all() and (wide[:offset] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_unaligned_weights(cuda, built, dtype):
    h = Head(cuda, 40, 64, 300, dtype)
    for name in ("w", "dw"):
        flat = cuda.empty(300 * 64 + 1, device="cuda", dtype=h.w.dtype)
        t = flat[1:].view(300, 64)
        t.copy_(getattr(h, name))
        setattr(h, name, t)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    h.check()


@pytest.mark.gpu
def test_positions_of_an_nhwc_tensor(cuda, built):
    """(B, H, 1, S) with channels last is B*S tokens."""
    h = Head(cuda, 6 * 35, 64, 300)
    with Dnn(cuda) as d:
        xd = d.tensor(6, 64, 1, 35, fmt=capi.CUDNN_TENSOR_NHWC, dtype=_code("bf16"))
        wd = d.filter(300, 64, 1, 1, fmt=capi.CUDNN_TENSOR_NHWC, dtype=_code("bf16"))
        assert d.L.cudnnLinearCrossEntropyBackward(
            d.h, xd, _p(h.x), wd, _p(h.w), _p(h.labels), _p(h.dloss), None, 0, _p(h.loss),
            _p(h.lse), xd, _p(h.dx), wd, _p(h.dw)) == 0
        cuda.cuda.synchronize()
    h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K", [0, 9])
@pytest.mark.parametrize("T,H", [(1000, 72), (385, 65)])
def test_pieces(cuda, built, T, H, K, dtype):
    """Every workspace from the least up gives the gradients within the same bounds."""
    h = Head(cuda, T, H, 600, dtype, K=K, out=0.1, seed=11)
    with Dnn(cuda) as d:
        most = h.workspace_size(d, 1)
        seen = []
        for size in (most, most * 3 // 4, most // 2, most // 4):
            ws = cuda.empty(size // 256 * 256, device="cuda", dtype=cuda.uint8)
            for t in (h.loss, h.lse, h.dx, h.dw):
                t.fill_(math.nan)
            status = h.backward(d, ws)
            cuda.cuda.synchronize()
            seen.append(status)
            if status == 0:
                h.check()
            else:
                assert status == capi.CUDNN_STATUS_BAD_PARAM and h.dw.isnan().all()
        assert seen[0] == 0
        assert T < 1000 or seen[:3] == [0, 0, 0]
        assert h.backward(d, cuda.empty(4096, device="cuda", dtype=cuda.uint8)) == \
            capi.CUDNN_STATUS_BAD_PARAM
        ws = cuda.empty(h.workspace_size(d, 0), device="cuda", dtype=cuda.uint8)
        assert h.forward(d, ws) == 0
        cuda.cuda.synchronize()
        h.check(gradients=False)


@pytest.mark.gpu
def test_many_score_pieces(cuda, built):
    """More tokens than one scoring piece holds."""
    h = Head(cuda, 40001, 16, 37, out=0.1)
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
    h.check(gradients=False)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [0, 9])
def test_one_gradient_alone_and_in_place(cuda, built, K):
    h = Head(cuda, 200, 64, 400, K=K)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        dx, dw = h.dx.clone(), h.dw.clone()
        h.dx.fill_(math.nan)
        h.dw.fill_(math.nan)
        assert h.backward(d, dw=False, loss=False) == 0
        cuda.cuda.synchronize()
        h.check(dw=False, loss=False)
        assert h.dw.isnan().all()
        h.dx.fill_(math.nan)
        assert h.backward(d, dx=False, loss=False) == 0
        cuda.cuda.synchronize()
        assert cuda.equal(h.dw, dw) and h.dx.isnan().all()
        h.dw.fill_(math.nan)
        h.dx = h.x  # the gradient over its own input
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        assert cuda.equal(h.x, dx) and cuda.equal(h.dw, dw)


@pytest.mark.gpu
def test_same_bits_on_any_stream(cuda, built):
    """Two calls give the same bits, and a call on another stream waits for the handle's
    workspace to be free."""
    a, b = Head(cuda, 700, 128, 3000, seed=1), Head(cuda, 650, 128, 2900, seed=2, K=5)
    with Dnn(cuda) as d:
        assert a.backward(d) == 0
        assert b.backward(d) == 0
        cuda.cuda.synchronize()
        want = [t.clone() for h in (a, b) for t in (h.loss, h.lse, h.dx, h.dw)]
        for t in (a.loss, a.lse, a.dx, a.dw, b.loss, b.lse, b.dx, b.dw):
            t.fill_(math.nan)
        cuda.cuda.synchronize()
        streams = [cuda.cuda.Stream(), cuda.cuda.Stream()]
        for _ in range(5):
            for h, s in zip((a, b), streams):
                assert d.L.cudnnSetStream(d.h, C.c_void_p(s.cuda_stream)) == 0
                assert h.backward(d) == 0
        cuda.cuda.synchronize()
        got = [t for h in (a, b) for t in (h.loss, h.lse, h.dx, h.dw)]
        for x, y in zip(want, got):
            assert cuda.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [0, 8])
def test_gradient_against_differences(cuda, built, K):
    """Central differences of the operator's own losses.  Along x + s d the second
    difference quotient errs by s^2/6 |f'''|, and f''' is a third central moment of
    (w d)/tau under softmax, at most 0.0963 times its range cubed; each loss carries its
    fp32 error; dx one rounding and dz's."""
    tau = 1.0 if not K else 2.0
    h = Head(cuda, 64, 128, 500, K=K, tau=tau, seed=9)
    h.x.copy_((h.x.float() * 8).round() / 8)  # so that x +- s d is exact in bf16
    h.dloss.fill_(1.0)
    s = 0.125
    d_ = cuda.randint(-1, 2, h.x.shape, device="cuda", generator=h.g).float()
    x0 = h.x.clone()
    losses = []
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        for sign in (1, -1):
            h.x.copy_(x0.float() + sign * s * d_)
            assert cuda.equal(h.x.float(), x0.float() + sign * s * d_)
            assert h.forward(d) == 0
            cuda.cuda.synchronize()
            losses.append(h.loss.double().clone())
    got = (h.dx.double() * d_.double()).sum(dim=1)
    want = (losses[0] - losses[1]) / (2 * s)
    r = d_.double() @ h.w.double().t() / tau
    span = r.amax(dim=1) - r.amin(dim=1)
    zerr = ((x0.double().abs() + s) @ h.w.double().abs().t()).amax(dim=1) * 160 * 2.0 ** -23 / tau
    tol = s * s / 6 * 0.0963 * span ** 3 + (2 * zerr + 2.0 ** -19 * 24) / s
    # dx's rounding, and dz's errors along d: |dz| sums to at most 2 before r's 1 / tau
    tol += (h.dx.double().abs() * 2.0 ** -8).sum(dim=1) * 1.01
    tol += 2.1 * 2.0 ** -8 * 2 * r.abs().amax(dim=1)
    assert ((got - want).abs() <= tol).all()
    # and the bound is worth something: well below the directional derivatives themselves
    assert tol.median() < 0.5 * want.abs().max()


@pytest.mark.gpu
def test_weights_past_32_bit_offsets(cuda, built):
    """w and dw of 2.2e9 elements: words, labels and gradients at the far end."""
    T, H, V = 3, 2000, 1_100_000
    g = cuda.Generator(device="cuda").manual_seed(4)
    h = Head(cuda, T, H, 64)
    w = cuda.zeros(V, H, device="cuda", dtype=cuda.bfloat16)
    w[-4096:] = cuda.randn(4096, H, device="cuda", generator=g) / math.sqrt(H)
    h.w, h.dw = w, cuda.full_like(w, math.nan)
    h.labels = cuda.tensor([V - 1, 0, V - 2000], device="cuda")
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    # the zero words count as 1 each in the sum; the others as themselves
    x, tail = h.x.double(), w[-4096:].double()
    z = x @ tail.t()
    lse = cuda.log(cuda.exp(z).sum(dim=1) + (V - 4096))
    assert ((h.lse.double() - lse).abs() <= 2.0 ** -18 * lse).all()
    target = cuda.stack([z[0, -1], z[1, 0] * 0, z[2, -2000]])
    assert ((h.loss.double() - (lse - target)).abs() <= 2.0 ** -17 * lse).all()
    p = cuda.exp(z - lse[:, None])
    p[0, -1] -= 1
    p[2, -2000] -= 1
    dz = p * h.dloss.double()[:, None]
    want = dz.t() @ x
    mag = dz.abs().t() @ x.abs()
    assert ((h.dw[-4096:].double() - want).abs() <= mag * 4 * 2.0 ** -8).all()
    dz0 = cuda.exp(-lse) * h.dloss.double()
    mag0 = dz0.abs() @ x.abs()
    assert ((h.dw[1:1000].double() - dz0 @ x).abs() <= mag0 * 4 * 2.0 ** -8).all()
    dxm = dz.abs() @ tail.abs()
    assert ((h.dx.double() - dz @ tail).abs() <= dxm * 4 * 2.0 ** -8).all()


# ------------------------------------------------------------------------ refusals --
def _ce(d, xd, x, wd, w, labels, dloss=None, loss=256, lse=None, dxd=None, dx=None, dwd=None,
        dw=None, ws=None, size=0):
    v = lambda q: None if q is None else C.c_void_p(q)  # noqa: E731
    if dloss is None and dx is None and dw is None:
        return d.L.cudnnLinearCrossEntropyForward(d.h, xd, v(x), wd, v(w), v(labels), v(ws), size,
                                                  v(loss), v(lse))
    return d.L.cudnnLinearCrossEntropyBackward(d.h, xd, v(x), wd, v(w), v(labels), v(dloss), v(ws),
                                               size, v(loss), v(lse), dxd, v(dx), dwd, v(dw))


def test_refusals_before_the_device(built):
    bad, unsupported = capi.CUDNN_STATUS_BAD_PARAM, capi.CUDNN_STATUS_NOT_SUPPORTED
    bf = capi.CUDNN_DATA_BFLOAT16
    with Dnn() as d:
        x = d.tensor(4, 64, 1, 1, dtype=bf)
        w = d.filter(100, 64, 1, 1, dtype=bf)
        p = 256
        assert _ce(d, x, None, w, p, p) == bad
        assert _ce(d, x, p, w, None, p) == bad
        assert _ce(d, x, p, w, p, None) == bad
        assert _ce(d, x, p, w, p, p, loss=None) == bad                      # nothing to compute
        assert _ce(d, x, p, w, p, p, dloss=p) == bad                        # no gradient asked for
        assert _ce(d, x, p, w, p, p, dxd=x, dx=p) == bad                    # no dloss
        assert _ce(d, x, p, w, p, p, dloss=p, dx=p) == bad                  # no descriptor
        assert _ce(d, x, p, w, p, p, dloss=p, dw=p) == bad
        assert _ce(d, w, p, x, p, p) == bad                                 # descriptors exchanged
        assert _ce(d, x, p, d.filter(100, 63, 1, 1, dtype=bf), p, p) == bad
        assert _ce(d, x, p, d.filter(100, 64, 3, 3, dtype=bf), p, p) == bad
        assert _ce(d, x, p, d.filter(100, 64, 1, 1, dtype=capi.CUDNN_DATA_HALF), p, p) == bad
        assert _ce(d, d.tensor(4, 64, 1, 1), p, d.filter(100, 64, 1, 1), p, p) == unsupported
        # channels first over several positions, rows that overlap, uneven positions
        assert _ce(d, d.tensor(4, 64, 1, 3, dtype=bf), p, w, p, p) == unsupported
        assert _ce(d, d.tensor(4, 64, 1, 1, dtype=bf, strides=(63, 1, 1, 1)), p, w, p, p) == unsupported
        assert _ce(d, d.tensor(4, 64, 2, 3, dtype=bf, strides=(400, 1, 200, 64)), p, w, p, p) == unsupported
        big = d.filter((1 << 30) + 1, 64, 1, 1, dtype=bf)
        assert _ce(d, x, p, big, p, p) == unsupported
        assert _ce(d, x, p, w, p, p, dloss=p, dxd=d.tensor(4, 65, 1, 1, dtype=bf), dx=p) == bad
        assert _ce(d, x, p, w, p, p, dloss=p, dwd=d.filter(101, 64, 1, 1, dtype=bf), dw=p) == bad
        # addresses that the device does not know
        assert _ce(d, x, p, w, p, p) == bad

        def kd(topk=4, index=p, teacher=p, tau=1.0):
            q = C.c_void_p(p)
            v = lambda t: None if t is None else C.c_void_p(t)  # noqa: E731
            return d.L.cudnnLinearDistillationForward(d.h, x, q, w, q, topk, v(index), v(teacher), tau,
                                                      None, 0, q, q)

        for args in (dict(topk=0), dict(topk=257), dict(topk=-1), dict(index=None), dict(teacher=None),
                     dict(tau=0.0), dict(tau=-1.0), dict(tau=math.nan), dict(tau=math.inf)):
            assert kd(**args) == bad, args
        n = C.c_size_t()
        L = d.L
        assert L.cudnnGetLinearCrossEntropyWorkspaceSize(d.h, x, w, 1, None) == bad
        assert L.cudnnGetLinearCrossEntropyWorkspaceSize(None, x, w, 1, C.byref(n)) == bad
        assert L.cudnnGetLinearDistillationWorkspaceSize(d.h, x, w, 0, 1, C.byref(n)) == bad
        assert L.cudnnGetLinearDistillationWorkspaceSize(d.h, x, w, 300, 1, C.byref(n)) == bad
        stale = C.c_void_p(d.h.value)
        assert L.cudnnGetLinearCrossEntropyWorkspaceSize(d.h, x, w, 1, C.byref(n)) == 0
    assert L.cudnnGetLinearCrossEntropyWorkspaceSize(stale, x, w, 1, C.byref(n)) == bad


def test_workspace_bounds(built):
    """The reported workspace stays bounded as the tokens grow."""
    with Dnn() as d:
        w = d.filter(131072, 4096, 1, 1, dtype=capi.CUDNN_DATA_BFLOAT16)
        sizes = []
        for T in (1, 100, 1000, 8192, 30000, 1000000):
            x = d.tensor(T, 4096, 1, 1, dtype=capi.CUDNN_DATA_BFLOAT16)
            n = C.c_size_t()
            assert d.L.cudnnGetLinearCrossEntropyWorkspaceSize(d.h, x, w, 1, C.byref(n)) == 0
            sizes.append(n.value)
            assert d.L.cudnnGetLinearCrossEntropyWorkspaceSize(d.h, x, w, 0, C.byref(n)) == 0
            assert n.value < 1 << 28
    assert sizes[0] < 64 << 20
    assert sizes[-1] < (2 << 30) + 131072 * 4096 * 4 + (1 << 30)


@pytest.mark.gpu
def test_refusals_of_memory(cuda, built):
    bad = capi.CUDNN_STATUS_BAD_PARAM
    h = Head(cuda, 32, 64, 100)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        ok = h.__dict__.copy()

        def refused(**change):
            h.__dict__.update(change)
            h.loss.fill_(5.0)
            status = h.backward(d)
            cuda.cuda.synchronize()
            untouched = bool((h.loss == 5).all())
            h.__dict__.update(ok)
            return status == bad and untouched

        dt = h.x.dtype
        odd = cuda.zeros(4097, device="cuda", dtype=cuda.uint8)

        class At:  # a tensor whose address is moved
            def __init__(self, t, by):
                self.t, self.by, self.shape = t, by, t.shape

            def data_ptr(self):
                return self.t.data_ptr() + self.by

            def stride(self, i):
                return self.t.stride(i)

        assert refused(x=At(h.x, 1))
        assert refused(w=At(h.w, 1))
        assert refused(labels=At(h.labels, 4))
        assert refused(dloss=At(h.dloss, 2))
        assert refused(lse=At(h.lse, 2))
        assert refused(lse=At(odd, 0).t[1:])
        assert refused(dx=h.w[:32])                      # outputs over inputs
        assert refused(dw=h.w)
        assert refused(lse=h.dloss)
        assert refused(lse=h.loss)
        host = cuda.zeros(100, 64, dtype=dt)
        assert refused(dw=host)
        assert refused(w=At(h.w, 1 << 34))
        shifted = cuda.zeros(33, 64, device="cuda", dtype=dt)
        assert refused(x=shifted[:32], dx=shifted[1:])   # dx's rows one below x's
        wide = cuda.zeros(32, 128, device="cuda", dtype=dt)
        wide[:, :64] = h.x
        want = h.dx.clone()
        h.x, h.dx = wide[:, :64], wide[:, 64:]           # side by side is fine
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        assert cuda.equal(h.dx, want)
        h.__dict__.update(ok)
        ws = cuda.empty(1 << 20, device="cuda", dtype=cuda.uint8)
        assert h.backward(d, ws) == 0
        assert h.backward(d, ws[8:]) == bad              # a workspace off its alignment
        assert h.backward(d, h.dw.view(cuda.uint8).view(-1)) == bad
        cuda.cuda.synchronize()


@pytest.mark.gpu
def test_example_trains(cuda, built):
    """The example's head learns, and scoring tokens one at a time agrees with together."""
    from examples.distill_head import train

    history, one_by_one, together = train(steps=12, tokens=256, features=128, vocab=2000,
                                          log=lambda line: None)
    assert history[-1] < 0.7 * history[0]
    # same inputs on the same words: fp32 losses of about 8 that differ in summation order
    assert all(abs(a - b) <= 1e-4 for a, b in zip(one_by_one, together))
