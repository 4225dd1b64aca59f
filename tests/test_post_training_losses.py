"""Policy and preference losses on a linear head against their definition in 64 bits.

Tolerances follow from the arithmetic.  With e the error that tests/test_vocab_loss.py derives
for a token's cross entropy (its nll):
  ratio    exp(old - nll): relative e, plus 2^-21 (1 + |old - nll|) for the difference and exp;
  gain     |A| times the ratio's, one more rounding;
  kl       |exp(d) - 1| e to first order, e^2 exp(|d|) beyond, 2^-20 (exp(d) + |d|) for the
           function (near 0 a series: 2^-20 kl);
  slope    the derivative by nll: |A| ratio's and klCoef exp(d) times e likewise;
  L        the sum of its tokens' e and of 2^-24 |nll|, all else in 64 bits.
dx and dw: the cross entropy's own errors for dloss * slope in dloss's place, plus the slope's
error times the gradient's factors.
"""

import ctypes as C
import math

import pytest

from muda_b200 import capi
from tests.helpers import Dnn
from tests.test_vocab_loss import Head, TINY, U, _code, _p

MODES = {"sigmoid": capi.CUDNN_PREFERENCE_SIGMOID, "hinge": capi.CUDNN_PREFERENCE_HINGE,
         "squared": capi.CUDNN_PREFERENCE_SQUARED}


class LossHead(Head):
    """A head whose loss is a function of its tokens' nll; `outputs` names what it returns."""

    def __init__(self, torch, T, H, V, dtype="bf16", tau=1.0, **kw):
        super().__init__(torch, T, H, V, dtype, tau=tau, **kw)
        self.nll = torch.full((T,), math.nan, device="cuda")

    def nll64(self):
        """nll in 64 bits (0 where left out), and its kernel's error bound."""
        torch = self.torch
        live = self.labels >= 0
        x = torch.where(live[:, None], self.x.double(), 0.0)
        w = self.w.double()
        z = x @ w.t() / self.tau
        lse = torch.logsumexp(z, dim=1)
        nll = lse - z.gather(1, self.labels.clamp(min=0)[:, None])[:, 0]
        zerr = (x.abs() @ w.abs().t()).amax(dim=1) * (x.shape[1] + 32) * 2.0 ** -23 / self.tau
        e = 2 * zerr + 2.0 ** -19 * (1 + lse.abs() + nll.abs())
        return torch.where(live, nll, 0.0), torch.where(live, e, 0.0), live, zerr

    def _outs(self, names):
        return [_p(getattr(self, n)) if n in names else None for n in self.outputs]

    def forward(self, d, ws=None, outputs=None):
        xd, wd, args = self._call(d)
        fn = getattr(d.L, f"cudnnLinear{self.kind}LossForward")
        return fn(*args, _p(ws), 0 if ws is None else ws.numel(), *self._outs(outputs or self.outputs))

    def backward(self, d, ws=None, dx=True, dw=True, outputs=None):
        xd, wd, args = self._call(d)
        dxd = None
        if dx:
            s = self.dx.stride(0)
            dxd = d.tensor(*self.dx.shape, 1, 1, dtype=_code(self.dtype), strides=(s, 1, s, s))
        fn = getattr(d.L, f"cudnnLinear{self.kind}LossBackward")
        return fn(*args, _p(self.dloss), _p(ws), 0 if ws is None else ws.numel(),
                  *self._outs(self.outputs if outputs is None else outputs),
                  dxd, _p(self.dx) if dx else None, wd if dw else None, _p(self.dw) if dw else None)

    def workspace_size(self, d, gradients):
        xd, wd, _ = self._call(d)
        n = C.c_size_t()
        fn = getattr(d.L, f"cudnnGetLinear{self.kind}LossWorkspaceSize")
        assert fn(d.h, xd, wd, gradients, C.byref(n)) == 0
        return n.value

    def clear(self):
        for n in self.outputs + ("dx", "dw"):
            getattr(self, n).fill_(math.nan)

    def check(self, gradients=True, dx=True, dw=True, outputs=None):
        """Every output against its definition; returns it."""
        torch, u = self.torch, U[self.dtype]
        want, tol, dnll, derr = self.expected()
        for n in self.outputs if outputs is None else outputs:
            off = (getattr(self, n).double() - want[n]).abs()
            assert (off <= tol[n]).all(), (n, (off / tol[n].clamp(min=1e-300)).max())
        if not gradients:
            return want
        # as a cross entropy's gradients with |dnll| for dloss, and dnll's own error
        _, _, live, zerr = self.nll64()
        x, w = torch.where(live[:, None], self.x.double(), 0.0), self.w.double()
        z = x @ w.t() / self.tau
        p = torch.softmax(z, dim=1) * live[:, None]
        target = torch.zeros_like(p)
        target[live, self.labels[live]] = 1.0
        g = (dnll / self.tau)[:, None]
        dz = g * (p - target)
        a = g.abs()
        err = a * p * (2 * u * (1 + u) + 2 * zerr[:, None] + 2.0 ** -18)
        err += target * (u * dz.abs() + a * (2.0 ** -19 + 2 * zerr[:, None]) * 2)
        err += (derr / self.tau)[:, None] * (p - target).abs() * (1 + 2 * u)
        if self.dtype == "fp16":  # subnormal numerators, and subnormal dz after the scaling
            err += live[:, None] * (a * p.amax(dim=1, keepdim=True) + a.max() * 2.0 ** -12) * 2.0 ** -24
        T, V = p.shape
        if dx:
            dx64 = dz @ w
            t = err @ w.abs() + u * dx64.abs() * 1.01 + (dz.abs() @ w.abs()) * (V + 32) * 2.0 ** -23
            assert ((self.dx.double() - dx64).abs() <= t + TINY[self.dtype]).all()
        if dw:
            dw64 = dz.t() @ x
            t = err.t() @ x.abs() + u * dw64.abs() * 1.01
            t += (dz.abs().t() @ x.abs()) * (T + 32) * 2.0 ** -23
            assert ((self.dw.double() - dw64).abs() <= t + TINY[self.dtype]).all()
        return want


class Policy(LossHead):
    kind, outputs = "Policy", ("loss", "nll", "ratio", "kl")

    def __init__(self, torch, T, H, V, dtype="bf16", tau=1.0, low=0.2, high=0.28, dual=3.0,
                 coef=0.1, old=True, ref=True, **kw):
        super().__init__(torch, T, H, V, dtype, tau=tau, **kw)
        self.low, self.high, self.dual, self.coef = low, high, dual, coef
        nan = torch.full((T,), math.nan, device="cuda")
        self.ratio, self.kl = nan.clone(), nan.clone()
        self.advantages = torch.randn(T, device="cuda", generator=self.g)
        self.advantages[::7] = 0.0
        nll, e, _, _ = self.nll64()

        def near(scale):
            return torch.randn(T, device="cuda", generator=self.g).double() * scale

        self.old = self.ref = None
        if old:
            # ratios of 0.2 to 5, and none so near a bound that nll's error could cross it
            r = torch.exp(near(0.8))
            for edge in (1 - low, 1 + high, dual):
                if edge > 0:
                    gap = 4 * e + 2.0 ** -12
                    r = torch.where((r / edge - 1).abs() < gap, edge * (1 + 2 * gap), r)
            self.old = (nll + torch.log(r)).float()
        if ref:
            self.ref = (nll + near(0.5)).float()
            self.ref[::5] = nll[::5].float()  # next to no divergence

    def _call(self, d):
        xd, wd, args = self._head(d)
        return xd, wd, args + (_p(self.old), _p(self.ref), _p(self.advantages), self.tau, self.low,
                               self.high, self.dual, self.coef)

    def expected(self):
        torch = self.torch
        nll, e, live, _ = self.nll64()
        nll.requires_grad_()
        A = self.advantages.double()
        old = self.old.double() if self.old is not None else nll.detach()
        r = torch.exp(old - nll)
        gain = torch.minimum(r * A, r.clamp(1 - self.low, 1 + self.high) * A)
        if self.old is None:  # a tie: the gradient is that of r A
            gain = r * A
        if self.dual:
            gain = torch.where(A < 0, torch.maximum(gain, self.dual * A), gain)
        d = nll - self.ref.double() if self.ref is not None else torch.zeros_like(nll)
        kl = torch.expm1(d) - d
        loss = self.coef * kl - gain
        slope = torch.autograd.grad(torch.where(live, loss, 0.0).sum(), nll)[0]
        want = dict(loss=loss, nll=nll, ratio=r, kl=kl)
        want = {k: torch.where(live, v, 0.0).detach() for k, v in want.items()}
        d, r, f = d.detach(), r.detach(), 2.0 ** -20
        tr = r * (1.01 * e + f / 2 * (1 + (old - nll.detach()).abs())) if self.old is not None else 0 * r
        tkl = d.expm1().abs() * e + e * e * d.abs().exp()
        tkl += torch.where(d.abs() < 0.4, f * (kl + e * e + e * d.abs()), f * (d.exp() + d.abs())).detach()
        tkl += d.abs() * 2.0 ** -23 * (nll.detach().abs() + 1)  # nll - ref in fp32
        tkl += 2.0 ** -46 * (nll.detach().abs() + 1) ** 2
        if self.ref is None:
            tkl = 0 * tkl
        tloss = A.abs() * (tr + f * r) + self.coef * tkl + f * want["loss"].abs()
        tslope = A.abs() * (tr + f * r) + self.coef * (d.exp() * (e + f * (1 + nll.detach().abs())))
        tol = dict(loss=tloss, nll=e, ratio=tr, kl=tkl)
        up = torch.where(live, self.dloss.double(), 0.0)
        return (want, {k: torch.where(live, v, 0.0) for k, v in tol.items()},
                torch.where(live, up * slope, 0.0),
                torch.where(live, up.abs() * (tslope + 2.0 ** -22 * slope.abs()), 0.0))


class Preference(LossHead):
    kind, outputs = "Preference", ("loss", "rewards", "nll")

    def __init__(self, torch, T, H, V, pairs, dtype="bf16", mode="sigmoid", averaged=False, beta=0.3,
                 margin=0.0, smoothing=0.0, ref=True, lengths=None, first=0, **kw):
        super().__init__(torch, T, H, V, dtype, **kw)
        self.pairs, self.mode, self.averaged = pairs, mode, averaged
        self.beta, self.margin, self.smoothing = beta, margin, smoothing
        if lengths is None:
            cuts = torch.randint(0, T - first + 1, (2 * pairs,), device="cuda", generator=self.g)
            ends = first + cuts.sort().values
        else:
            ends = first + torch.tensor(lengths, device="cuda").cumsum(0)
        assert len(ends) == 2 * pairs and ends[-1] <= T
        self.offsets = torch.cat([torch.tensor([first], device="cuda"), ends])
        self.loss = torch.full((pairs,), math.nan, device="cuda")
        self.rewards = torch.full((2 * pairs,), math.nan, device="cuda")
        self.dloss = torch.randn(pairs, device="cuda", generator=self.g) / pairs
        self.ref = None
        if ref:
            noise = torch.randn(T, device="cuda", generator=self.g).double() * 0.5
            self.ref = (self.nll64()[0] + noise).float()

    def _call(self, d):
        xd, wd, args = self._head(d)
        return xd, wd, args + (self.pairs, _p(self.offsets), _p(self.ref), MODES[self.mode],
                               int(self.averaged), self.beta, self.margin, self.smoothing)

    def expected(self):
        torch, P = self.torch, self.pairs
        nll, e, live, _ = self.nll64()
        nll.requires_grad_()
        e = torch.where(live, e + 2.0 ** -24 * nll.detach().abs(), 0.0)
        at = self.offsets.tolist()
        L, terr, counted = [], [], []
        for a, b in zip(at[:-1], at[1:]):
            on = live[a:b].nonzero()[:, 0] + a
            n = max(1, len(on)) if self.averaged else 1
            gain = (self.ref[on].double() if self.ref is not None else 0.0) - nll[on]
            L.append(gain.sum() / n)
            terr.append((e[on].sum() / n).item())
            counted.append(len(on) > 0)
        loss, rewards = torch.zeros(P).double().cuda(), torch.zeros(2 * P).double().cuda()
        tl, trw, tslope = (torch.zeros_like(loss), torch.zeros_like(rewards), torch.zeros_like(loss))
        losses = []
        for p in range(P):
            if not (counted[p] and counted[P + p]):
                losses.append(nll[0] * 0)
                continue
            h = self.beta * (L[p] - L[P + p]) - self.margin
            eh = self.beta * (terr[p] + terr[P + p])
            if self.mode == "sigmoid":
                loss_p = torch.nn.functional.softplus(-h) + self.smoothing * h
                tl[p], tslope[p] = eh, eh / 4
            elif self.mode == "hinge":
                assert abs(h.item() - 1) > 2 * eh  # else the input cannot tell the side
                loss_p = torch.relu(1 - h)
                tl[p] = eh
            else:
                loss_p = ((h - 0.5) / self.beta) ** 2
                tslope[p] = 2 * eh / self.beta ** 2
                tl[p] = (2 * (h - 0.5).abs().item() + eh) * eh / self.beta ** 2
            losses.append(loss_p)
            for s in (p, P + p):
                rewards[s] = self.beta * L[s].detach()
                trw[s] = self.beta * terr[s] + 2.0 ** -23 * rewards[s].abs()
        loss = torch.stack(losses)
        dnll = torch.autograd.grad((loss * self.dloss.double()).sum(), nll)[0]
        loss = loss.detach()
        tl += 2.0 ** -23 * loss.abs()
        derr = torch.zeros_like(nll)
        for s, (a, b) in enumerate(zip(at[:-1], at[1:])):
            n = max(1, int(live[a:b].sum())) if self.averaged else 1
            derr[a:b] = self.dloss[s % P].abs().double() * tslope[s % P] * self.beta / n
        derr = derr * live + dnll.abs() * 2.0 ** -22
        return (dict(loss=loss, rewards=rewards, nll=nll.detach()),
                dict(loss=tl, rewards=trw, nll=e), dnll, derr)


# (T, H, V): single tokens and words, tile edges, odd sizes, several bands
SIZES = [(1, 8, 1), (1, 64, 129), (5, 24, 130), (8, 264, 1601), (40, 65, 1000), (64, 512, 4099),
         (127, 72, 257), (129, 65, 255), (300, 250, 513), (513, 192, 777), (1100, 40, 2100),
         (300, 600, 20000)]


def _both(cuda, h):
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        h.check(gradients=False)
        h.clear()
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    return h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V", SIZES)
def test_policy(cuda, built, T, H, V, dtype):
    want = _both(cuda, Policy(cuda, T, H, V, dtype, out=0.2 if T > 4 else 0.0, seed=T + H))
    if T >= 300 and V > 500:  # all sides of the clips occur
        r, A = want["ratio"], want["loss"]
        assert (r < 0.8).any() and (r > 1.28).any() and (r > 3).any() and A.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("change", [
    dict(dual=0.0), dict(coef=0.0), dict(coef=0.0, ref=False), dict(old=False), dict(tau=0.5),
    dict(tau=2.0), dict(low=0.0, high=0.0), dict(low=1.0, high=50.0), dict(old=False, coef=2.0),
])
def test_policy_parameters(cuda, built, change, dtype):
    h = Policy(cuda, 200, 64, 900, dtype, out=0.1, seed=3, **change)
    if h.ref is None:
        with Dnn(cuda) as d:
            assert h.backward(d, outputs=("loss", "nll", "ratio")) == 0
            cuda.cuda.synchronize()
        h.check(outputs=("loss", "nll", "ratio"))
        assert h.kl.isnan().all()  # not asked for
    else:
        _both(cuda, h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V", [(2, 8, 1), (2, 64, 129), (8, 264, 1601), (64, 65, 1000),
                                   (129, 72, 257), (300, 250, 513), (1100, 40, 2100),
                                   (300, 600, 20000)])
def test_preference(cuda, built, T, H, V, dtype):
    _both(cuda, Preference(cuda, T, H, V, max(1, T // 40), dtype, out=0.1 if T > 8 else 0.0,
                           seed=T + H, lengths=[1, 1] if T == 2 else None))


@pytest.mark.gpu
@pytest.mark.parametrize("change", [
    dict(smoothing=0.1), dict(mode="hinge", beta=0.05), dict(mode="squared"),
    dict(averaged=True, beta=2.0, margin=0.5), dict(ref=False, averaged=True, beta=1.0),
    dict(margin=-1.0, beta=1.0), dict(mode="squared", averaged=True, margin=0.25),
    dict(beta=40.0), dict(smoothing=0.5, beta=20.0),
])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_preference_parameters(cuda, built, change, dtype):
    _both(cuda, Preference(cuda, 400, 64, 700, 5, dtype, out=0.1, seed=11, **change))


@pytest.mark.gpu
@pytest.mark.parametrize("averaged", [False, True])
def test_sequences_of_any_length(cuda, built, averaged):
    """Empty sequences, one token, all prompt, one long one; rows before, between no
    sequences and behind the last."""
    lengths = [0, 1, 30, 700, 5, 2, 9, 0, 40, 3, 8, 2]  # chosen 0..5, rejected 0..5
    h = Preference(cuda, 900, 72, 300, 6, lengths=lengths, first=17, averaged=averaged, seed=5)
    start, end = h.offsets[2].item(), h.offsets[3].item()
    h.labels[start:end] = -100                       # pair 2: its chosen sequence is all prompt
    if h.ref is not None:
        h.ref[start:end] = math.nan                  # and says nothing
    want = _both(cuda, h)
    for pair in (0, 1, 2):                           # 0: no chosen token, 1: no rejected
        assert h.loss[pair] == 0 and h.rewards[pair] == 0 and h.rewards[6 + pair] == 0
    assert (want["loss"][3:] > 0).all()
    outside = cuda.ones(900, dtype=cuda.bool, device="cuda")
    outside[h.offsets[3]:h.offsets[6]] = False
    outside[h.offsets[9]:h.offsets[12]] = False
    assert (h.dx[outside] == 0).all() and (h.dx[~outside] != 0).any()
    assert (h.nll[:17] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [5, 40, 300])
def test_tokens_left_out_may_hold_anything(cuda, built, T, dtype):
    h = Policy(cuda, T, 64, 500, dtype, seed=2)
    h.labels[1], h.labels[3:5] = -1, -100
    gone = h.labels < 0
    for t in (h.x, h.old, h.ref, h.advantages, h.dloss):
        t[gone] = math.nan
    _both(cuda, h)
    for n in Policy.outputs + ("dx",):
        assert (getattr(h, n)[gone] == 0).all()
    q = Preference(cuda, T, 64, 500, 1, dtype, seed=2, lengths=[3, T - 3])
    q.labels[1], q.labels[3] = -1, -100
    gone = q.labels < 0
    q.x[gone] = math.nan
    q.ref[gone] = math.nan
    _both(cuda, q)
    assert (q.dx[gone] == 0).all() and (q.nll[gone] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["policy", "preference"])
def test_every_token_left_out(cuda, built, kind):
    h = (Policy(cuda, 140, 64, 300) if kind == "policy" else Preference(cuda, 140, 64, 300, 3))
    h.labels.fill_(-100)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    for n in h.outputs + ("dx", "dw"):
        assert (getattr(h, n) == 0).all(), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [6, 50, 200])
def test_nan_stays_with_its_token_or_pair(cuda, built, T, dtype):
    """A label past the vocabulary, or NaN in one of a token's inputs."""
    for spoil in ("label", "old", "ref", "advantages"):
        h = Policy(cuda, T, 64, 100, dtype, seed=T)
        h.advantages[2] = 0.0 if spoil == "old" else 1.0
        if spoil == "label":
            h.labels[2] = 100
        else:
            getattr(h, spoil)[2] = math.nan
        with Dnn(cuda) as d:
            assert h.backward(d) == 0
            cuda.cuda.synchronize()
        assert h.loss[2].isnan() and h.dx[2].isnan().all(), spoil
        rest = cuda.arange(T, device="cuda") != 2
        for n in Policy.outputs + ("dx",):
            assert getattr(h, n)[rest].isfinite().all(), (spoil, n)
    for spoil in ("label", "ref"):
        q = Preference(cuda, T, 64, 100, 3, dtype, lengths=[1, 1, 1, 1, 1, T - 5], seed=T)
        if spoil == "label":
            q.labels[1] = 100
        else:
            q.ref[1] = math.nan
        with Dnn(cuda) as d:
            assert q.backward(d) == 0
            cuda.cuda.synchronize()
        assert q.loss[1].isnan() and q.rewards[1].isnan() and q.dx[1].isnan().all()
        assert q.dx[4].isnan().all()  # the other sequence of its pair
        rest = [0, 2, 3, 5]
        assert q.loss[[0, 2]].isfinite().all() and q.dx[rest].isfinite().all()


@pytest.mark.gpu
def test_offsets_that_do_not_ascend(cuda, built):
    """A pair with bad offsets is NaN and has no gradient of its own; nothing else changes."""
    for bad in ([0, 10, 5, 20, 30], [0, -4, 10, 20, 30], [0, 10, 20, 30, 51], [0, 10, 20, 30, 1 << 40]):
        h = Preference(cuda, 50, 64, 100, 2, lengths=[10, 10, 10, 10])
        h.offsets = cuda.tensor(bad, device="cuda")
        with Dnn(cuda) as d:
            assert h.backward(d) == 0
            cuda.cuda.synchronize()
            gone = [any(not 0 <= bad[s] <= bad[s + 1] <= 50 for s in (p, p + 2)) for p in (0, 1)]
            for p in (0, 1):
                assert h.loss[p].isnan() == gone[p]
            assert h.dx.isfinite().all() and h.dw.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_infinite_ratios(cuda, built, dtype):
    """An old policy that knew no other word, and one that did not know this word."""
    h = Policy(cuda, 200, 64, 300, dtype, coef=0.0, dual=0.0, seed=8)
    h.old[0], h.old[1], h.old[2], h.old[3] = math.inf, math.inf, math.inf, -math.inf
    h.advantages[0], h.advantages[1], h.advantages[2], h.advantages[3] = 1.0, 0.0, -1.0, 1.0
    with Dnn(cuda) as d:
        assert h.backward(d, dw=False) == 0
        cuda.cuda.synchronize()
    assert h.ratio[:3].isinf().all() and h.ratio[3] == 0
    assert abs(h.loss[0] + 1.28) < 1e-6 and (h.dx[0] == 0).all()   # clipped: no gradient
    assert h.loss[1] == 0 and (h.dx[1] == 0).all()                 # asks for nothing
    assert h.loss[2] == math.inf                                   # unbounded without dualClip
    assert h.loss[3] == 0 and (h.dx[3] == 0).all()
    assert h.dx[4:].isfinite().all()
    h.dual = 3.0
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    assert abs(h.loss[2] - 3.0) < 1e-6 and (h.dx[2] == 0).all() and h.dw.isfinite().all()
    # references that were sure of the token, or did not know it
    h.ref[5], h.ref[6] = -math.inf, math.inf
    h.coef = 0.5
    with Dnn(cuda) as d:
        assert h.backward(d, dw=False) == 0
        cuda.cuda.synchronize()
    assert (h.kl[5:7] == math.inf).all() and (h.loss[5:7] == math.inf).all()
    rest = cuda.arange(200, device="cuda") != 5
    assert h.dx[rest].isfinite().all()  # exp(-inf) - 1 is an ordinary slope


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_infinite_references(cuda, built, dtype):
    """A reference that did not know a chosen token, and one that did not know a rejected one."""
    h = Preference(cuda, 100, 64, 300, 3, dtype, lengths=[10] * 6, seed=8)
    h.ref[3] = math.inf    # pair 0's chosen sequence
    h.ref[45] = math.inf   # pair 1's rejected one
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    assert h.loss[0] == 0 and (h.dx[:10] == 0).all() and (h.dx[30:40] == 0).all()
    assert h.loss[1] == math.inf and h.dx.isfinite().all() and h.dw.isfinite().all()
    assert h.rewards[0] == math.inf and h.rewards[4] == math.inf and h.loss[2].isfinite()


def _sure(h, cancelling, equal=1):
    """Makes each token's label its row's largest word, with `equal` - 1 other words that equal
    it: 32 above the others, which are of order 1; or, cancelling, 0.25 above them, in logits of
    order 0 that are sums of +-768.  There the tensor cores' sums may be off by 2^-14 (the last
    place kept of numbers below 2^10, in 24 bits) for each of 17 terms of 32 MMAs, 0.033."""
    torch, (T, H), V = h.torch, h.x.shape, len(h.w)
    own = torch.arange(T, device="cuda")
    half = (H - 256) // 2
    assert T <= 256 <= H and T * equal <= V and half == 128
    h.labels = own.clone()
    if cancelling:
        x = 1 + torch.rand(T, half, device="cuda", generator=h.g)
        w = torch.rand(V, half, device="cuda", generator=h.g) * 8
        h.x[:, 256:] = torch.cat([x, x], dim=1).to(h.x.dtype)
        h.w[:, 256:] = torch.cat([w, -w], dim=1).to(h.w.dtype)
    h.x[:, :256], h.w[:, :256] = 0.0, 0.0
    h.x[own, own] = 0.5 if cancelling else 8.0
    h.w[own, own] = 0.5 if cancelling else 4.0
    for k in range(1, equal):
        h.w[k * T:(k + 1) * T] = h.w[:T]
    z = h.x.double() @ h.w.double().t()
    others = z.clone()
    for k in range(equal):
        others[own, own + k * T] = -math.inf
    assert (z[own, own] - others.amax(dim=1) > (0.24 if cancelling else 20)).all()


TEMPERATURES = [1.0, 1e-3, 1e-5, 1e-7, 1e-8, 2.0 ** -30, 2.0 ** -40, 2.0 ** -64]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 0.5])
def test_infinite_references_with_smoothing(cuda, built, smoothing, dtype):
    """softplus(-h) + smoothing h of h = inf and -inf: |h| times smoothing and 1 - smoothing.  The
    slopes are smoothing and smoothing - 1, so that the gradients are a sum of nll's."""
    h = Preference(cuda, 100, 64, 300, 3, dtype, smoothing=smoothing, lengths=[10] * 6, seed=8)
    h.ref[3] = math.inf    # pair 0's chosen sequence
    h.ref[45] = math.inf   # pair 1's rejected one
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    assert h.loss[0] == (math.inf if smoothing else 0.0) and h.loss[1] == math.inf
    assert h.loss[2].isfinite() and h.dw.isfinite().all()
    nll, _, _, zerr = h.nll64()
    p = cuda.softmax(h.x.double() @ h.w.double().t(), dim=1)
    target = cuda.nn.functional.one_hot(h.labels, 300)
    u = U[dtype]
    for pair, slope in ((0, smoothing), (1, smoothing - 1)):
        g = h.dloss[pair].item() * slope * h.beta
        for s, sign in ((pair, -1), (3 + pair, 1)):
            rows = slice(10 * s, 10 * s + 10)
            dx = sign * g * (p - target)[rows] @ h.w.double()
            # a word's dz rounds three times, and half a step of fp16's least kept (2^-26) besides;
            # p is off by its logits' errors; dx rounds once
            err = abs(g) * ((p + target)[rows] * (3 * u + 2 * zerr[rows, None] + 2.0 ** -18) + 2.0 ** -26)
            t = err @ h.w.double().abs() + 1.01 * u * dx.abs() + TINY[dtype]
            assert ((h.dx[rows].double() - dx).abs() <= t).all(), (pair, s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cancelling", [False, True])
@pytest.mark.parametrize("T", [4, 40, 200])
def test_sure_labels_at_any_temperature(cuda, built, T, cancelling, dtype):
    """The label's share is 1 to the last bit below 2^-7 (a gap of 0.17 / tau above 18): its nll
    is 0, not the noise of its logit over the temperature, and so are its gradients."""
    h = Policy(cuda, T, 512, 1200, dtype, coef=0.0, old=False, ref=False)
    _sure(h, cancelling)
    h.ref = cuda.zeros(T, device="cuda")
    for h.tau in TEMPERATURES:
        for h.old in (None, cuda.zeros(T, device="cuda")):
            for dw in (None, False, True):  # scores, a frozen head, steps
                h.clear()
                with Dnn(cuda) as d:
                    assert (h.forward(d) if dw is None else h.backward(d, dw=dw)) == 0
                    cuda.cuda.synchronize()
                assert (h.nll >= 0).all(), h.tau
                if h.tau == 1.0:
                    h.check(gradients=False, outputs=("nll",))
                    continue
                assert (h.nll == 0).all() and (h.ratio == 1).all() and (h.kl == 0).all(), h.tau
                assert (h.loss == -h.advantages).all(), h.tau
                assert dw is None or (h.dx == 0).all(), h.tau
                assert not dw or (h.dw == 0).all(), h.tau


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cancelling", [False, True])
@pytest.mark.parametrize("T,equal", [(4, 2), (40, 3), (200, 5)])
def test_equal_words_at_any_temperature(cuda, built, T, equal, cancelling, dtype):
    """Words with the label's own row share with it at any temperature: nll is log(equal), of
    which log1p rounds to 2 units of its last place at most."""
    h = Policy(cuda, T, 512, 1200, dtype, coef=0.0, old=False, ref=False)
    _sure(h, cancelling, equal)
    for h.tau in TEMPERATURES[1:]:
        h.clear()
        with Dnn(cuda) as d:
            assert h.forward(d, outputs=("nll", "ratio", "loss")) == 0
            cuda.cuda.synchronize()
        assert (abs(h.nll - math.log(equal)) <= 2.0 ** -22 * math.log(equal)).all(), h.tau


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tau", TEMPERATURES[1:])
@pytest.mark.parametrize("T", [4, 40, 200])
def test_any_label_at_any_temperature(cuda, built, T, tau, dtype):
    """Labels that are not their rows' largest words: nll to its logits' errors over tau."""
    h = Policy(cuda, T, 512, 1200, dtype, tau=tau, coef=0.0, old=False, ref=False)
    with Dnn(cuda) as d:
        assert h.forward(d, outputs=("nll",)) == 0
        cuda.cuda.synchronize()
    assert (h.nll >= 0).all()
    h.check(gradients=False, outputs=("nll",))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cancelling", [False, True])
@pytest.mark.parametrize("T", [4, 40, 200])
def test_sequences_of_sure_labels(cuda, built, T, cancelling, dtype):
    h = Preference(cuda, T, 512, 1200, 2, dtype, ref=False, lengths=[T // 4] * 4)
    _sure(h, cancelling)
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
    assert (h.nll >= 0).all()
    h.check(gradients=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["policy", "preference"])
@pytest.mark.parametrize("T,H,V", [(15, 264, 88432), (100, 65, 40000), (128, 72, 50257)])
def test_few_tokens_of_several_waves(cuda, built, T, H, V, kind, dtype):
    """Up to 128 tokens of so many words that a CTA takes several tiles of them."""
    _both(cuda, Policy(cuda, T, H, V, dtype, out=0.2, seed=T) if kind == "policy" else
          Preference(cuda, T, H, V, 3, dtype, seed=T, lengths=[T // 6] * 6))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["policy", "preference"])
@pytest.mark.parametrize("T", [4, 100, 300])
def test_nan_word_reaches_every_token(cuda, built, kind, T):
    """A NaN in a word that is no token's label, beside labels that are their rows' largest words."""
    h = (Policy(cuda, T, 64, 700, seed=T) if kind == "policy" else
         Preference(cuda, T, 64, 700, 2, seed=T, lengths=[T // 4] * 4))
    h.labels.clamp_(max=500)
    h.labels[0] = -1
    h.x.copy_(h.w[h.labels.clamp(min=0)].float() * 16)
    h.w[555, 3] = math.nan
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
    assert h.nll[1:].isnan().all() and h.nll[0] == 0
    if kind == "policy":
        assert h.loss[1:].isnan().all()
    else:  # of 4 tokens the first is all of its sequence: a pair that is left out
        assert h.loss[1].isnan() and (h.loss[0] == 0 if T == 4 else h.loss[0].isnan())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,calls", [(8, 1024, 40), (100, 1024, 4), (2000, 1024, 1)])
def test_mean_error_of_nll(cuda, built, T, H, calls, dtype):
    """What the tensor cores' sums lose on average is made up for.  A chain of n MMAs is short of
    a logit by a share of about 1.45e-8 n (bf16; fp16 1.95e-8), the chains are of 32 MMAs (8 for up
    to 8 tokens).  That alone would leave nll off by this share of the likely words' logits, about
    16, above the label's: no more than half of it may be left, and four standard errors."""
    share = (8 if T <= 8 else 32) * (1.45e-8 if dtype == "bf16" else 1.95e-8)
    off, lost = [], []
    for seed in range(calls):
        h = Policy(cuda, T, H, 8000, dtype, seed=seed, old=False, ref=False, coef=0.0)
        likely = cuda.randint(0, 8000, (T,), device="cuda", generator=h.g)
        h.x.copy_(h.x.float() + 16 * h.w[likely].float())
        with Dnn(cuda) as d:
            assert h.forward(d, outputs=("nll",)) == 0
            cuda.cuda.synchronize()
        z = h.x.double() @ h.w.double().t()
        label = z.gather(1, h.labels[:, None])[:, 0]
        off.append(h.nll.double() - (cuda.logsumexp(z, dim=1) - label))
        lost.append(share * ((cuda.softmax(z, dim=1) * z).sum(dim=1) - label))
    off, lost = cuda.cat(off), cuda.cat(lost)
    noise = off.std() / math.sqrt(len(off))
    assert lost.mean() > 12 * noise  # the inputs tell
    assert off.mean().abs() <= 0.5 * lost.mean() + 4 * noise


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_preference_piece_of_four_gib(cuda, built, dtype):
    """One piece of 2^31 numerators, the most that a preference's gradients take: every output
    against its definition, computed by blocks of tokens."""
    torch, T, H, V, u = cuda, 16384, 64, 131072, U[dtype]

    class Large(Preference):
        def nll64(self):
            if not hasattr(self, "kept"):
                parts = []
                for a in range(0, T, 1024):
                    part = Policy.__new__(Policy)
                    part.torch, part.tau, part.w = torch, self.tau, self.w
                    part.x, part.labels = self.x[a:a + 1024], self.labels[a:a + 1024]
                    parts.append(LossHead.nll64(part))
                self.kept = [torch.cat(p) for p in zip(*parts)]
            return tuple(t.clone() for t in self.kept)

    h = Large(cuda, T, H, V, 7, dtype, out=0.1, seed=3)
    with Dnn(cuda) as d:
        assert h.workspace_size(d, 1) > 4 << 30  # one piece
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    h.check(gradients=False)
    _, _, dnll, derr = h.expected()
    _, _, live, zerr = h.nll64()
    w = h.w.double()
    dw64, dwerr, dwsum = (torch.zeros(V, H, device="cuda", dtype=torch.float64) for _ in range(3))
    for a in range(0, T, 1024):
        s = slice(a, a + 1024)
        on, x, e = live[s, None], h.x[s].double(), zerr[s, None]
        p = torch.softmax(x @ w.t(), dim=1) * on
        target = torch.zeros_like(p).scatter_(1, h.labels[s, None].clamp(min=0), 1.0) * on
        g = dnll[s, None]
        dz = g * (p - target)
        err = g.abs() * p * (2 * u * (1 + u) + 2 * e + 2.0 ** -18)
        err += target * (u * dz.abs() + g.abs() * (2.0 ** -19 + 2 * e) * 2)
        err += derr[s, None] * (p - target).abs() * (1 + 2 * u)
        if dtype == "fp16":
            err += on * (g.abs() * p.amax(dim=1, keepdim=True) + dnll.abs().max() * 2.0 ** -12) * 2.0 ** -24
        dx64 = dz @ w
        t = err @ w.abs() + u * dx64.abs() * 1.01 + (dz.abs() @ w.abs()) * (V + 32) * 2.0 ** -23
        assert ((h.dx[s].double() - dx64).abs() <= t + TINY[dtype]).all(), a
        dw64 += dz.t() @ x
        dwerr += err.t() @ x.abs()
        dwsum += dz.abs().t() @ x.abs()
    t = dwerr + u * dw64.abs() * 1.01 + dwsum * (T + 32) * 2.0 ** -23 + TINY[dtype]
    assert ((h.dw.double() - dw64).abs() <= t).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["policy", "preference"])
@pytest.mark.parametrize("T,H", [(1000, 72), (385, 65)])
def test_pieces(cuda, built, T, H, kind, dtype):
    """Given workspaces from the least to the preferred: every piece count gives the result."""
    V = 1500
    h = (Policy(cuda, T, H, V, dtype, out=0.1) if kind == "policy"
         else Preference(cuda, T, H, V, 7, dtype, out=0.1))
    with Dnn(cuda) as d:
        size = h.workspace_size(d, 1)
        pool = cuda.empty(size, device="cuda", dtype=cuda.uint8)
        refused = done = 0
        for share in (0.1, 0.2, 0.4, 0.6, 0.8, 1.0):
            h.clear()
            status = h.backward(d, pool[:int(size * share)])
            cuda.cuda.synchronize()
            if status == capi.CUDNN_STATUS_BAD_PARAM:
                refused += 1
                assert done == 0
                continue
            assert status == 0
            done += 1
            h.check()
            # without outputs, whose arrays the workspace then holds
            h.dx.fill_(math.nan)
            dw = h.dw.clone()
            if h.backward(d, pool[:int(size * share)], outputs=()) == 0:
                cuda.cuda.synchronize()
                h.check(outputs=())
                assert cuda.equal(h.dw, dw) or kind == "preference"
        assert done >= 2  # all tokens in one piece, and pieces of them
        size = h.workspace_size(d, 0)
        h.clear()
        assert h.forward(d, pool[:size]) == 0
        cuda.cuda.synchronize()
        h.check(gradients=False)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["policy", "preference"])
@pytest.mark.parametrize("T", [6, 60, 200])
def test_one_gradient_alone_and_in_place(cuda, built, kind, T):
    make = lambda: (Policy(cuda, T, 64, 500, seed=1) if kind == "policy"  # noqa: E731
                    else Preference(cuda, T, 64, 500, 2, seed=1, lengths=[1, 2, 1, T - 4]))
    h = make()
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        h.check()
        both = h.dx.clone(), h.dw.clone()
        h.clear()
        assert h.backward(d, dw=False) == 0
        cuda.cuda.synchronize()
        h.check(dw=False)
        h.clear()
        assert h.backward(d, dx=False) == 0
        cuda.cuda.synchronize()
        h.check(dx=False)
        assert cuda.equal(h.dw, both[1])
        h.dx = h.x  # in place
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        assert cuda.equal(h.x, both[0]) and cuda.equal(h.dw, both[1])


@pytest.mark.gpu
def test_policy_of_its_own_samples_is_a_weighted_cross_entropy(cuda, built):
    """With ratio 1 and no divergence the gradient is that of A nll: both calls are within what
    either may be off.  nll itself is the cross entropy with a more exact target."""
    h = Policy(cuda, 300, 136, 1000, coef=0.0, old=False, dual=0.0, seed=6)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        c = Head(cuda, 300, 136, 1000, seed=6)
        c.x, c.w, c.labels = h.x, h.w, h.labels
        c.dloss = h.dloss * h.advantages
        assert c.backward(d) == 0
        cuda.cuda.synchronize()
        c.check()
        h.check()
        policy = h.dx, h.dw
        h.dx, h.dw = c.dx, c.dw
        h.check()
        c.dx, c.dw = policy
        c.check()
    nll, e, _, _ = h.nll64()
    assert ((h.nll - c.loss).abs() <= 2 * e).all()
    assert (h.nll - nll).norm() <= (c.loss - nll).norm()
    assert cuda.equal(h.loss, -h.advantages) and (h.ratio == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["policy", "preference"])
def test_gradient_against_differences(cuda, built, kind):
    """Central differences of the operator's own losses along a direction of x, with the second
    difference of the loss in 64 bits as the bound of what they leave out."""
    T, H, V, s = 32, 64, 400, 2.0 ** -5
    if kind == "policy":
        h = Policy(cuda, T, H, V, seed=9, low=0.9, high=20.0, dual=0.0, coef=0.2)
    else:
        h = Preference(cuda, T, H, V, 4, seed=9, lengths=[4] * 8, beta=0.2)
    h.x.copy_((h.x.float() * 8).round() / 8)
    nll = h.nll64()[0]
    if kind == "policy":
        h.old = (nll + 0.3).float()
    h.ref = (nll + 0.2).float()
    h.dloss.fill_(1.0)
    move = cuda.randint(-1, 2, h.x.shape, device="cuda", generator=h.g).float()
    x0 = h.x.clone()

    def loss64(sign):
        h.x.copy_(x0.float() + sign * s * move)
        want, tol, _, _ = h.expected()
        return want["loss"].sum(), tol["loss"].sum()

    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        got = (h.dx.double() * move.double()).sum()
        rounding = (h.dx.double() * move.double()).abs().sum() * 2.0 ** -8
        # dz's roundings (two of p, one at the target) along w's rows
        along = (move.double() @ h.w.double().t()).abs().amax(dim=1)
        rounding += (3.1 * 2.0 ** -8 * h.expected()[2].abs() * along).sum()
        values = []
        for sign in (1, -1):
            h.x.copy_(x0.float() + sign * s * move)
            assert cuda.equal(h.x.float(), x0.float() + sign * s * move)
            assert h.forward(d) == 0
            cuda.cuda.synchronize()
            values.append(h.loss.double().sum())
    (a, ea), (b, eb) = loss64(1), loss64(-1)
    quotient64 = (a - b) / (2 * s)
    # the operator's difference quotient is the definition's
    assert abs((values[0] - values[1]) / (2 * s) - quotient64) <= (ea + eb) / (2 * s)
    # the quotient at half the step is a third of its distance to the one before off the
    # derivative, up to terms of the fifth order: the whole distance bounds it
    s /= 2
    (a, _), (b, _) = loss64(1), loss64(-1)
    half = (a - b) / (2 * s)
    assert abs(got - half) <= abs(half - quotient64) + rounding


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["policy", "preference"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_same_bits_on_any_stream(cuda, built, kind, dtype):
    h = (Policy(cuda, 700, 136, 3001, dtype) if kind == "policy"
         else Preference(cuda, 700, 136, 3001, 9, dtype))
    want = None
    with Dnn(cuda) as d:
        for _ in range(3):
            stream = cuda.cuda.Stream()
            assert d.L.cudnnSetStream(d.h, C.c_void_p(stream.cuda_stream)) == 0
            h.clear()
            stream.wait_stream(cuda.cuda.current_stream())
            assert h.backward(d) == 0
            stream.synchronize()
            got = [getattr(h, n).clone() for n in h.outputs + ("dx", "dw")]
            want = got if want is None else want
            assert all(cuda.equal(a, b) for a, b in zip(got, want))
    h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["policy", "preference"])
def test_captured_in_a_graph(cuda, built, kind, dtype):
    """A captured step replays on new inputs at the same addresses, beside other calls."""
    make = lambda s: (Policy(cuda, 200, 96, 900, dtype, seed=s) if kind == "policy"  # noqa: E731
                      else Preference(cuda, 200, 96, 900, 4, dtype, seed=s))
    h, other = make(1), make(2)
    large = Policy(cuda, 1100, 136, 5001, dtype)
    a, b = cuda.cuda.Stream(), cuda.cuda.Stream()
    with Dnn(cuda) as d:
        assert d.L.cudnnSetStream(d.h, C.c_void_p(a.cuda_stream)) == 0
        with cuda.cuda.stream(a):
            assert h.backward(d) == 0
            a.synchronize()
            graph = cuda.cuda.CUDAGraph()
            with cuda.cuda.graph(graph, stream=a):
                assert h.backward(d) == 0
        assert d.L.cudnnSetStream(d.h, C.c_void_p(b.cuda_stream)) == 0
        names = ("x", "w", "dloss", "labels", "ref") + (("old", "advantages") if kind == "policy"
                                                        else ("offsets",))
        for n in names:
            getattr(h, n).copy_(getattr(other, n))
        for _ in range(5):
            h.clear()
            large.clear()
            cuda.cuda.synchronize()
            with cuda.cuda.stream(a):
                graph.replay()
            assert large.backward(d) == 0
            cuda.cuda.synchronize()
        del graph
    h.check()
    large.check()


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind", ["policy", "preference"])
@pytest.mark.parametrize("T,H,V", [(4, 4096, 900), (6, 1031, 2000), (20, 4096, 3001),
                                   (128, 264, 5000), (100, 1031, 700)])
def test_short_scores_follow_their_inputs(cuda, built, kind, T, H, V, captured):
    """Scores in a row, each after kernels that write its inputs where the last one's were."""
    make = lambda s: (Policy(cuda, T, H, V, seed=s) if kind == "policy"  # noqa: E731
                      else Preference(cuda, T, H, V, 2, seed=s))
    h, sets = make(0), [make(s) for s in (1, 2, 3)]
    names = ("x", "w", "labels", "ref") + (("old", "advantages") if kind == "policy"
                                           else ("offsets",))
    stream = cuda.cuda.Stream()
    with Dnn(cuda) as d:
        for s in sets:
            assert s.forward(d) == 0
        cuda.cuda.synchronize()
        assert d.L.cudnnSetStream(d.h, C.c_void_p(stream.cuda_stream)) == 0
        got = [[cuda.empty_like(getattr(h, n)) for n in h.outputs] for _ in sets]

        def scores():
            for s, outs in zip(sets, got):
                for n in names:
                    getattr(h, n).copy_(getattr(s, n))
                assert h.forward(d) == 0
                for n, o in zip(h.outputs, outs):
                    o.copy_(getattr(h, n))

        with cuda.cuda.stream(stream):
            scores()
            if captured:
                stream.synchronize()
                graph = cuda.cuda.CUDAGraph()
                with cuda.cuda.graph(graph, stream=stream):
                    scores()
                for outs in got:
                    for o in outs:
                        o.fill_(math.nan)
                for _ in range(3):
                    graph.replay()
            stream.synchronize()
        if captured:
            del graph
    for s, outs in zip(sets, got):
        s.check(gradients=False)
        for n, o in zip(h.outputs, outs):
            assert cuda.equal(o, getattr(s, n)), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_pieces_captured_in_a_graph(cuda, built, dtype):
    """A preference step of several pieces, in a given workspace that held other things."""
    h = Preference(cuda, 1000, 72, 1500, 7, dtype, out=0.1, first=3)
    stream = cuda.cuda.Stream()
    with Dnn(cuda) as d:
        size = int(h.workspace_size(d, 1) * 0.6)
        ws = cuda.full((size,), 255, device="cuda", dtype=cuda.uint8)
        cuda.cuda.synchronize()
        assert d.L.cudnnSetStream(d.h, C.c_void_p(stream.cuda_stream)) == 0
        with cuda.cuda.stream(stream):
            assert h.backward(d, ws) == 0
            stream.synchronize()
            graph = cuda.cuda.CUDAGraph()
            with cuda.cuda.graph(graph, stream=stream):
                assert h.backward(d, ws) == 0
            for _ in range(3):
                h.clear()
                ws.fill_(255)
                graph.replay()
            stream.synchronize()
        del graph
    h.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_tied_table_step(cuda, built, dtype):
    """Lookup, policy loss on the same table as head, and both gradients into one dw."""
    from tests.test_embedding import Table

    T, H, V = 150, 64, 300
    e = Table(cuda, T, H, V, dtype, dtype, seed=4, out=0.1)
    h = Policy(cuda, T, H, V, dtype, seed=4)
    h.w = e.w = (e.w.float() / 8).to(e.w.dtype)
    with Dnn(cuda) as d:
        assert e.forward(d, 8.0) == 0
        h.x = e.rows
        nll = h.nll64()[0]
        noise = cuda.randn(T, device="cuda", generator=h.g)
        h.old = (nll + cuda.where(noise > 0, 0.1, -0.5)).float()
        h.ref = (nll + noise * 0.3).float()
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        e.check_forward(None, 8.0)
        h.check()
        head = h.dw.clone()
        e.rows, e.w = h.dx, h.dw
        assert e.backward(d, 8.0, 1.0) == 0
        cuda.cuda.synchronize()
        e.check_backward(head, 8.0, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["policy", "preference"])
def test_example_gradients(cuda, built, kind):
    """The example's steps against autograd in 64 bits.  Its hidden states round to bf16 once and
    count as inputs.  dz rounds three times at most, dx and dw once each and dw's sum once
    more: six roundings of the products' magnitudes, and the nll's errors (a share of 2^-10)."""
    from examples.post_train_table import TiedTable

    T, H, V, scale = 96, 64, 300, 8.0
    g = cuda.Generator(device="cuda").manual_seed(3)
    w = (cuda.randn(V, H, device="cuda", generator=g) / 8).bfloat16()
    tokens = cuda.randint(0, V, (T,), device="cuda", generator=g)
    tokens[5] = -1
    labels = cuda.randint(0, V, (T,), device="cuda", generator=g)
    labels[::6] = -100
    live = labels >= 0
    table = TiedTable(V, H, scale)
    try:
        x = table.hidden(w, tokens)
        nll = table.nll(w, tokens, labels)
        noise = cuda.randn(T, device="cuda", generator=g)
        ref = nll + noise
        if kind == "policy":
            old, A = nll + 0.1 * noise.sign(), cuda.randn(T, device="cuda", generator=g)
            dloss = cuda.rand(T, device="cuda", generator=g) / T
            loss, _, dw = table.policy_step(w, tokens, labels, old, ref, A, dloss, kl=0.1)
        else:
            offsets = cuda.tensor([0, 20, 50, 70, T], device="cuda")
            dloss = cuda.rand(2, device="cuda", generator=g)
            loss, _, dw = table.preference_step(w, tokens, labels, offsets, ref, dloss)
        cuda.cuda.synchronize()
    finally:
        table.close()
    z = x.double() @ w.double().t()
    logp = cuda.log_softmax(z, dim=1)
    n = -logp.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    n = cuda.where(live, n, 0.0).requires_grad_()
    if kind == "policy":
        r, d = cuda.exp(old.double() - n), n - ref.double()
        gain = cuda.minimum(r * A.double(), r.clamp(0.8, 1.2) * A.double())
        want = cuda.where(live, 0.1 * (cuda.expm1(d) - d) - gain, 0.0)
    else:
        gain = cuda.where(live, ref.double() - n, 0.0)
        L = cuda.stack([gain[a:b].sum() for a, b in ((0, 20), (20, 50), (50, 70), (70, T))])
        want = cuda.nn.functional.softplus(-0.1 * (L[:2] - L[2:]))
    assert ((loss - want).abs() <= 2.0 ** -12 * (1 + want.abs())).all()
    dn = cuda.autograd.grad((want * dloss.double()).sum(), n)[0]
    dz = cuda.exp(logp)
    dz[cuda.arange(T, device="cuda"), labels.clamp(min=0)] -= 1
    dz = cuda.where(live, dn, 0.0)[:, None] * dz

    def table_gradient(dz, x, w):
        at = (tokens >= 0).nonzero()[:, 0]
        return (dz.t() @ x).index_add(0, tokens[at], scale * (dz @ w)[at])

    want = table_gradient(dz, x.double(), w.double())
    mass = table_gradient(dz.abs(), x.double().abs(), w.double().abs())
    assert ((dw - want).abs() <= (6.2 * 2.0 ** -8 + 2.0 ** -10) * mass + 2.0 ** -133).all()


@pytest.mark.gpu
def test_example_runs(cuda, built):
    from examples.post_train_table import train

    policy, preference = train(steps=3, sequences=6, length=16, features=64, vocab=300,
                               log=lambda *a: None)
    assert len(policy) == len(preference) == 3
    assert all(math.isfinite(v) for v in policy + preference)


# ------------------------------------------------------------------------ refusals --
def test_refusals_before_the_device(built):
    bad, unsupported = capi.CUDNN_STATUS_BAD_PARAM, capi.CUDNN_STATUS_NOT_SUPPORTED
    bf = capi.CUDNN_DATA_BFLOAT16
    with Dnn() as d:
        L, p = d.L, C.c_void_p(256)
        x, w = d.tensor(4, 64, 1, 1, dtype=bf), d.filter(100, 64, 1, 1, dtype=bf)

        def policy(x=x, xp=p, w=w, wp=p, labels=p, old=p, ref=p, adv=p, tau=1.0, low=0.2, high=0.2,
                   dual=0.0, coef=0.1, dloss=None, outs=(p, p, p, p), dxd=None, dx=None, dwd=None,
                   dw=None):
            head = (d.h, x, xp, w, wp, labels, old, ref, adv, tau, low, high, dual, coef)
            if dloss is None and dx is None and dw is None:
                return L.cudnnLinearPolicyLossForward(*head, None, 0, *outs)
            return L.cudnnLinearPolicyLossBackward(*head, dloss, None, 0, *outs, dxd, dx, dwd, dw)

        def preference(x=x, xp=p, w=w, wp=p, labels=p, pairs=2, offsets=p, ref=p, mode=0, averaged=0,
                       beta=0.1, margin=0.0, smoothing=0.0, dloss=None, outs=(p, p, p), dxd=None,
                       dx=None, dwd=None, dw=None):
            head = (d.h, x, xp, w, wp, labels, pairs, offsets, ref, mode, averaged, beta, margin,
                    smoothing)
            if dloss is None and dx is None and dw is None:
                return L.cudnnLinearPreferenceLossForward(*head, None, 0, *outs)
            return L.cudnnLinearPreferenceLossBackward(*head, dloss, None, 0, *outs, dxd, dx, dwd, dw)

        for call, outs in ((policy, 4), (preference, 3)):
            for name in ("xp", "wp", "labels", "x", "w"):
                assert call(**{name: None}) == bad, name
            assert call(outs=(None,) * outs) == bad                # nothing to compute
            assert call(dloss=p) == bad                            # no gradient asked for
            assert call(dxd=x, dx=p) == bad                        # no dloss
            assert call(dloss=p, dx=p) == bad                      # no descriptor
            assert call(dloss=p, dw=p) == bad
            assert call(w=d.filter(100, 63, 1, 1, dtype=bf)) == bad
            assert call(x=d.tensor(4, 64, 1, 1), w=d.filter(100, 64, 1, 1)) == unsupported
            assert call(x=d.tensor(4, 64, 1, 3, dtype=bf)) == unsupported
            assert call() == bad                                   # addresses no device knows
        for change in (dict(adv=None), dict(tau=0.0), dict(tau=math.nan), dict(tau=math.inf),
                       dict(low=-0.1), dict(low=1.1), dict(low=math.nan), dict(high=-0.1),
                       dict(high=math.inf), dict(dual=0.5), dict(dual=-1.0), dict(dual=math.nan),
                       dict(coef=-0.1), dict(coef=math.inf), dict(ref=None),
                       dict(ref=None, coef=0.0)):  # kl is asked for
            assert policy(**change) == bad, change
        for change in (dict(pairs=0), dict(pairs=-1), dict(pairs=(1 << 29) + 1), dict(offsets=None),
                       dict(mode=3), dict(mode=-1), dict(beta=0.0), dict(beta=-1.0),
                       dict(beta=math.inf), dict(margin=math.nan), dict(margin=math.inf),
                       dict(smoothing=-0.1), dict(smoothing=0.6), dict(smoothing=0.1, mode=1),
                       dict(smoothing=0.1, mode=2), dict(smoothing=math.nan)):
            assert preference(**change) == bad, change
        n = C.c_size_t()
        for size in (L.cudnnGetLinearPolicyLossWorkspaceSize, L.cudnnGetLinearPreferenceLossWorkspaceSize):
            assert size(d.h, x, w, 1, None) == bad
            assert size(None, x, w, 1, C.byref(n)) == bad
            assert size(d.h, x, x, 1, C.byref(n)) == bad
            assert size(d.h, x, w, 1, C.byref(n)) == 0


def test_workspace_bounds(built):
    """What the cross entropy takes, and a few bytes per token besides; a preference's gradients
    have pieces of twice the size."""
    with Dnn() as d:
        w = d.filter(131072, 4096, 1, 1, dtype=capi.CUDNN_DATA_HALF)
        for T in (1, 100, 8192, 30000, 1000000):
            x = d.tensor(T, 4096, 1, 1, dtype=capi.CUDNN_DATA_HALF)
            for gradients in (0, 1):
                n, ce = C.c_size_t(), C.c_size_t()
                assert d.L.cudnnGetLinearCrossEntropyWorkspaceSize(d.h, x, w, gradients, C.byref(ce)) == 0
                for name in ("Policy", "Preference"):
                    fn = getattr(d.L, f"cudnnGetLinear{name}LossWorkspaceSize")
                    assert fn(d.h, x, w, gradients, C.byref(n)) == 0
                    if name == "Preference" and gradients:
                        assert n.value <= (4 << 30) + (1 << 30) + 131072 * 4096 * 4 + 8 * T
                    else:
                        assert ce.value <= n.value <= ce.value + 8 * T + 1024, (T, name, gradients)


@pytest.mark.gpu
def test_refuses_another_devices_memory(cuda, built):
    if cuda.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    bad = capi.CUDNN_STATUS_BAD_PARAM
    with Dnn(cuda) as d:
        for h, names in ((Policy(cuda, 32, 64, 100), ("labels", "old", "ref", "advantages", "dloss")),
                         (Preference(cuda, 32, 64, 100, 2), ("labels", "offsets", "ref", "dloss"))):
            for name in names + h.outputs + ("x", "w", "dx", "dw"):
                here = getattr(h, name)
                setattr(h, name, here.to("cuda:1"))
                assert h.backward(d) == bad, name
                setattr(h, name, here)
            ws = cuda.empty(h.workspace_size(d, 1), device="cuda:1", dtype=cuda.uint8)
            assert h.backward(d, ws) == bad


@pytest.mark.gpu
def test_refusals_of_memory(cuda, built):
    bad = capi.CUDNN_STATUS_BAD_PARAM
    p, q = Policy(cuda, 32, 64, 100), Preference(cuda, 32, 64, 100, 2)
    with Dnn(cuda) as d:
        for h, inputs in ((p, ("labels", "old", "ref", "advantages", "dloss")),
                          (q, ("labels", "offsets", "ref", "dloss"))):
            assert h.backward(d) == 0
            cuda.cuda.synchronize()
            want = [getattr(h, n).clone() for n in h.outputs + ("dx", "dw")]

            def refused(name, t):
                was = getattr(h, name)
                setattr(h, name, t)
                status = h.backward(d)
                setattr(h, name, was)
                return status == bad

            class Moved:
                def __init__(self, t, by):
                    self.t, self.by = t, by

                def data_ptr(self):
                    return self.t.data_ptr() + self.by

            for name in inputs + h.outputs:
                t = getattr(h, name)
                assert refused(name, Moved(t, t.element_size() // 2)), name
                assert refused(name, Moved(t, 1 << 34)), name
                assert refused(name, cuda.zeros(200)), name              # host memory
            for name in h.outputs:
                for other in inputs + h.outputs:
                    if other != name:
                        assert refused(name, getattr(h, other)), (name, other)
            cuda.cuda.synchronize()
            got = [getattr(h, n) for n in h.outputs + ("dx", "dw")]
            assert all(cuda.equal(a, b) for a, b in zip(got, want))
            ws = cuda.empty(h.workspace_size(d, 1), device="cuda", dtype=cuda.uint8)
            assert h.backward(d, ws[:1024]) == bad
            assert h.backward(d, ws[8:]) == bad
            assert h.backward(d, ws) == 0
            cuda.cuda.synchronize()
