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


def _definition(torch, h):
    """As Head.definition, of logits below their row's largest: lse less z cancels in 64 bits
    too where the logits are huge."""
    w = h.w.double()
    T, V = h.x.shape[0], w.shape[0]
    target = torch.zeros(T, V, device="cuda", dtype=torch.float64)
    entropy = torch.zeros(T, device="cuda", dtype=torch.float64)
    if h.K:
        t = torch.where(h.index >= 0, h.teacher.double() / h.tau, -math.inf)
        live = (t > -math.inf).any(dim=1)
        q = torch.softmax(t[live], dim=1)
        target[live] = target[live].scatter_add(1, h.index[live].clamp(min=0), q)
        entropy[live] = torch.special.xlogy(q, q).sum(dim=1)
    else:
        live = h.labels >= 0
        target[live, h.labels[live]] = 1.0
    x = torch.where(live[:, None], h.x.double(), 0.0)
    z = x @ w.t()
    top = z.amax(dim=1, keepdim=True)
    z = (z - top) / h.tau
    total = torch.logsumexp(z, dim=1, keepdim=True)
    cross = torch.where(target > 0, target * (total - z), 0.0).sum(dim=1)
    p = torch.exp(z - total)
    dloss = torch.where(live, h.dloss.double(), 0.0) / h.tau
    dz = dloss[:, None] * (p - target)
    return dict(loss=torch.where(live, entropy + cross, 0.0),
                lse=torch.where(live, (top / h.tau + total)[:, 0], 0.0), dz=dz, dx=dz @ w,
                dw=dz.t() @ x, live=live, p=p, target=target, x=x, w=w, dloss=dloss)


def _check(torch, h, zerr=0.0, dx=True, dw=True, gradients=True):
    """Outputs against the definition in 64 bits, for logits z / tau that err by zerr at most.

    u is the 16-bit type's unit roundoff.  With exact logits, exponentials, sums and logarithm
    err by 2^-20 relative, and a difference of two logits as the exponent by 2^-22 of itself:
    words whose differences pass 32 have no weight, so 2^-16 covers both.  dz: two roundings
    of a numerator, one at the targets, and fp32's underflow, 2^-126 (fp16: its subnormals as
    well, steps of 2^-24 of a row's largest, and 2^-36 of the largest dz once scaled); dx, dw:
    those weighted, fp32 accumulation and one rounding of the result.
    """
    ref = _definition(torch, h)
    live = ref["live"]
    err = 2.0 ** -16 + 2 * zerr
    assert ((h.lse.double() - ref["lse"]).abs() <= (2.0 ** -21 * ref["lse"].abs() + err) * live).all()
    tol = err * (1 + ref["loss"].abs())
    assert ((h.loss.double() - ref["loss"]).abs() <= tol * live).all()
    if not gradients:
        return ref
    u = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}[h.dtype]
    tiny = {"bf16": 2.0 ** -133, "fp16": 2.0 ** -25}[h.dtype]
    g = ref["dloss"].abs()[:, None]
    p = ref["p"] * live[:, None]
    derr = g * (p * (2 * u * (1 + u) + err) + 2.0 ** -126 * live[:, None])
    derr += (ref["target"] > 0) * (u * ref["dz"].abs() + g * err)
    if h.dtype == "fp16":
        derr += live[:, None] * (g * p.amax(dim=1, keepdim=True) + g.max() * 2.0 ** -12) * 2.0 ** -24
    x, w = ref["x"].abs(), ref["w"].abs()
    T, V = p.shape
    if dx:
        tol = derr @ w + 1.01 * u * ref["dx"].abs() + ref["dz"].abs() @ w * (V + 32) * 2.0 ** -23
        assert ((h.dx.double() - ref["dx"]).abs() <= tol + tiny).all()
    if dw:
        tol = derr.t() @ x + 1.01 * u * ref["dw"].abs() + ref["dz"].abs().t() @ x * (T + 32) * 2.0 ** -23
        assert ((h.dw.double() - ref["dw"]).abs() <= tol + tiny).all()
    return ref


def _exact_logits(torch, T, V, dtype, K, tau, bx, bw, step, seed):
    """A head whose logits bx bw + step m, m whole, have no rounding in fp32."""
    h = Head(torch, T, 64, V, dtype, K=K, tau=tau, seed=seed)

    def whole(*shape):
        return torch.randint(-1, 2, shape, device="cuda", generator=h.g).float()

    h.x.copy_(whole(T, 64))
    h.w.copy_(step * whole(V, 64))
    h.x[:, 0] = bx
    h.w[:, 0] = bw
    h.dloss *= T * tau  # dz of about 1
    if K:
        h.teacher *= tau  # a teacher of ordinary spread
    return h


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [4, 40, 300])
@pytest.mark.parametrize("K,tau,bx,bw,step", [  # cross entropy (K 0) has no temperature
    (5, 2.0 ** -20, 1.0, 8.0, 2.0 ** -20),     # z / tau about 2^23, words 1 apart
    (5, 2.0 ** -22, 1.0, 8.0, 2.0 ** -20),     # 2^25, 4 apart
    (5, 2.0 ** -40, 1.0, -8.0, 2.0 ** -20),    # -2^43, and words far apart
    (5, 2.0 ** -60, 1.0, 8.0, 2.0 ** -20),
    (0, 1.0, 2.0 ** 12, 2.0 ** 13, 4.0),       # logits of 2^25, 4 apart
    (5, 1.0, 2.0 ** 12, 2.0 ** 13, 4.0),
    (0, 1.0, 2.0 ** 12, -(2.0 ** 13), 4.0),
])
def test_logits_beyond_their_exponents_fraction(cuda, built, T, K, dtype, tau, bx, bw, step):
    """|z| / tau so large that fp32 holds no fraction of it: probabilities come of differences."""
    h = _exact_logits(cuda, T, 700, dtype, K, tau, bx, bw, step, seed=T + K)
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        _check(cuda, h, gradients=False)
        for t in (h.loss, h.lse):
            t.fill_(math.nan)
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        _check(cuda, h)
        h.dx.fill_(math.nan)
        assert h.backward(d, dw=False) == 0  # a frozen head
        cuda.cuda.synchronize()
    _check(cuda, h, dw=False)


def _logit_error(h, words):
    """Most error of the logits of these words, as the fp32 sums leave it."""
    a = h.x.double().abs() @ h.w[words].double().abs().t()
    return a.amax().item() * (h.x.shape[1] + 32) * 2.0 ** -23 / h.tau


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K,tau", [(0, 1.0), (5, 1.0), (5, 0.5)])
@pytest.mark.parametrize("T", [4, 40, 300])
def test_words_masked_with_the_lowest_value(cuda, built, T, K, dtype, tau):
    """Whole tiles of words at the type's lowest value through one feature of 1: no weight."""
    h = Head(cuda, T, 64, 1500, dtype, K=K, tau=tau, seed=T + K)
    h.x[:, 0] = 1.0
    h.w[:, 0] = 0.0
    masked = cuda.zeros(1500, dtype=cuda.bool, device="cuda")
    masked[200:1100] = True
    h.w[masked, 0] = cuda.finfo(h.w.dtype).min
    if K:
        h.index = cuda.where(h.index >= 0, h.index % 200, -1)
    else:
        h.labels %= 200
    zerr = _logit_error(h, ~masked)
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        _check(cuda, h, zerr, gradients=False)
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        ref = _check(cuda, h, zerr, dx=dtype == "bf16")
        assert (ref["p"][:, masked] == 0).all() and (h.dw[masked] == 0).all()
        assert h.backward(d, dw=False) == 0
        cuda.cuda.synchronize()
        _check(cuda, h, zerr, dx=dtype == "bf16", dw=False)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [0, 5])
@pytest.mark.parametrize("T", [4, 40, 300])
def test_every_word_masked_with_the_lowest_value(cuda, built, T, K):
    """Masks that leave no word: all have the same logit, and the same weight."""
    h = Head(cuda, T, 64, 700, K=K, seed=T + K)
    h.x.zero_()  # beside the lowest value, sums could lose its last bit
    h.x[:, 0] = 1.0
    h.w[:, 0] = cuda.finfo(h.w.dtype).min
    with Dnn(cuda) as d:
        assert h.forward(d) == 0
        cuda.cuda.synchronize()
        _check(cuda, h, gradients=False)
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    ref = _check(cuda, h, dx=False)
    assert ((ref["p"] - 1 / 700).abs() < 1e-12).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [40, 300])
def test_infinite_words_below_low_logits(cuda, built, T, dtype):
    """Tiles of words at -inf among words at about -400: no gradient for those rows of dw."""
    h = Head(cuda, T, 64, 900, dtype, seed=T)
    h.x[:, 0] = 1.0
    h.w[:, 0] = -400.0
    h.w[100:600, 0] = -math.inf
    h.labels %= 100
    finite = cuda.ones(900, dtype=cuda.bool, device="cuda")
    finite[100:600] = False
    with Dnn(cuda) as d:
        assert h.backward(d, dx=False) == 0
        cuda.cuda.synchronize()
    _check(cuda, h, _logit_error(h, finite), dx=False)
    assert (h.dw[100:600] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [3e-7, 1e-9])
@pytest.mark.parametrize("T", [4, 300])
def test_teacher_logits_beyond_their_exponents_fraction(cuda, built, T, tau):
    """Teacher logits 8 + 2^-20 m, 2.7e7 and more once divided, and 3.2 m or more apart."""
    h = Head(cuda, T, 64, 700, K=9, tau=tau, seed=T)
    h.w *= tau  # a student of ordinary spread
    h.dloss *= tau
    h.teacher = 8.0 + cuda.randint(-9, 9, (T, 9), device="cuda", generator=h.g) * 2.0 ** -20
    zerr = _logit_error(h, slice(None))
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    _check(cuda, h, zerr)


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [1.0, 0.5])
@pytest.mark.parametrize("T", [4, 300])
def test_teacher_entries_masked_with_the_lowest_value(cuda, built, T, tau):
    """Entries at fp32's lowest value have no weight beside others, and equal weights alone."""
    h = Head(cuda, T, 64, 700, K=9, tau=tau, seed=T)
    h.teacher[:, 3:7] = cuda.finfo(cuda.float32).min
    h.teacher[::2] = cuda.finfo(cuda.float32).min
    zerr = _logit_error(h, slice(None))
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    ref = _check(cuda, h, zerr)
    assert ref["live"].all()


def test_workspace_stays_bounded_for_any_shape(built):
    """cudnn.h's bound: 2 GiB of numerators, 1 GiB of what else grows with a piece's tokens,
    V H floats between pieces, and a copy of w whose rows are not a multiple of 16 bytes."""
    with Dnn() as d:
        for V in (2, 256, 5000, 131072, 1000003):
            for H in (8, 64, 1000, 1001, 4096, 8192):
                w = d.filter(V, H, 1, 1, dtype=capi.CUDNN_DATA_BFLOAT16)
                for T in (1, 1000, 30000, 300000, 1 << 24):
                    x = d.tensor(T, H, 1, 1, dtype=capi.CUDNN_DATA_BFLOAT16)
                    n = C.c_size_t()
                    assert d.L.cudnnGetLinearDistillationWorkspaceSize(d.h, x, w, 256, 1,
                                                                       C.byref(n)) == 0
                    copy = V * (H + 63) // 64 * 64 * 2 if H % 8 else 0
                    assert n.value <= (3 << 30) + 4 * V * (H + 3) + copy, (T, H, V)
                    assert d.L.cudnnGetLinearDistillationWorkspaceSize(d.h, x, w, 256, 0,
                                                                       C.byref(n)) == 0
                    assert n.value <= (256 << 20) + copy or V > 1000000, (T, H, V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K", [0, 3])
def test_many_tokens_few_words(cuda, built, K, dtype):
    """More tokens than one piece of a gradient takes, though their numerators would fit."""
    h = Head(cuda, 70001, 40, 60, dtype, K=K, out=0.1, seed=8)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
    h.check()


def _moved(torch, t, by):
    """t's values in memory that starts `by` elements off an aligned address."""
    flat = torch.empty(t.numel() + by, device="cuda", dtype=t.dtype)
    m = flat[by:].view(t.shape)
    m.copy_(t)
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K", [0, 5])
@pytest.mark.parametrize("T,H,V", [(1, 64, 3000), (5, 136, 700), (100, 128, 2001), (300, 72, 900),
                                   (40, 65, 700), (1, 1001, 300)])
@pytest.mark.parametrize("x_by,w_by", [(1, 0), (4, 0), (0, 1), (0, 4), (1, 1), (4, 3)])
def test_reported_workspace_suffices_at_any_address(cuda, built, T, H, V, K, dtype, x_by, w_by):
    h = Head(cuda, T, H, V, dtype, K=K, seed=T + H)
    if T == 1 and K:
        h.index[0, 0] = V - 1
    h.x, h.w, h.dw = _moved(cuda, h.x, x_by), _moved(cuda, h.w, w_by), _moved(cuda, h.dw, w_by)
    with Dnn(cuda) as d:
        ws = cuda.empty(h.workspace_size(d, 0), device="cuda", dtype=cuda.uint8)
        assert h.forward(d, ws) == 0
        cuda.cuda.synchronize()
        h.check(gradients=False)
        ws = cuda.empty(h.workspace_size(d, 1), device="cuda", dtype=cuda.uint8)
        assert h.backward(d, ws) == 0
        cuda.cuda.synchronize()
        h.check()
        h.dx.fill_(math.nan)
        assert h.backward(d, ws, dw=False) == 0
        cuda.cuda.synchronize()
        h.check(dw=False)
        h.dw.fill_(math.nan)
        assert h.backward(d, ws, dx=False) == 0
        cuda.cuda.synchronize()
        h.check(dx=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K", [0, 7])
@pytest.mark.parametrize("T,H,V", [(1, 520, 40000), (60, 520, 31001), (300, 600, 40003),
                                   (150, 72, 140001), (700, 1031, 20011)])
def test_head_copied_in_slices(cuda, built, T, H, V, K, dtype):
    """A w that TMA cannot read, in a workspace with room for 16 MiB of its copy: several
    slices, with dx's partial sums on flat, tall and single-CTA tiles."""
    h = Head(cuda, T, H, V, dtype, K=K, out=0.1 if T > 4 else 0.0, seed=T + H)
    if T == 1:
        h.index = None if not K else h.index.clamp(min=0)
    h.w = _moved(cuda, h.w, 4)
    with Dnn(cuda) as d:
        for gradients in (0, 1):
            size = h.workspace_size(d, gradients)
            if H % 8:  # the reported size has room for all of the copy
                size -= V * (H + 63) // 64 * 64 * 2 - (17 << 20)
            ws = cuda.empty(size // 256 * 256, device="cuda", dtype=cuda.uint8)
            for _ in range(2):
                for t in (h.loss, h.lse, h.dx, h.dw):
                    t.fill_(math.nan)
                assert (h.backward(d, ws) if gradients else h.forward(d, ws)) == 0
                cuda.cuda.synchronize()
            h.check(gradients=bool(gradients))
        h.dx.fill_(math.nan)
        assert h.backward(d, ws, dw=False) == 0
        cuda.cuda.synchronize()
        h.check(dw=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K", [0, 5])
@pytest.mark.parametrize("T,V", [(40, 900), (40, 20001), (300, 900), (300, 20001)])
def test_rows_left_out_beside_infinite_words(cuda, built, T, V, K, dtype):
    """Words at -inf leave no NaN in dx's rows that are left out (0 times infinity in the
    product), on any path of dx: with dw and alone, in one sum and in several."""
    h = Head(cuda, T, 64, V, dtype, K=K, out=0.3, seed=T + K)
    h.x.abs_()
    h.x += 0.5
    h.w[V // 3:V // 2] = -math.inf
    out = (h.index < 0).all(dim=1) if K else h.labels < 0
    assert out.any() and not out.all()
    with Dnn(cuda) as d:
        for dw in (True, False):
            h.dx.fill_(math.nan)
            assert h.backward(d, dw=dw) == 0
            cuda.cuda.synchronize()
            assert (h.dx[out] == 0).all()
            assert h.dx[~out].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [0, 5])
@pytest.mark.parametrize("T", [40, 300])
@pytest.mark.parametrize("offset", [40.0, -40.0])
def test_small_upstream_gradients(cuda, built, T, K, offset):
    """dloss of 1e-24 on logits of about 40: dx of 1e-24 is far inside bf16's range."""
    h = Head(cuda, T, 64, 900, K=K, out=0.1, seed=T + K)
    h.x[:, 0] = 8.0
    h.w[:, 0] = offset / 8.0
    h.dloss *= T * 1e-24
    with Dnn(cuda) as d:
        for dw in (True, False):
            h.dx.fill_(math.nan)
            assert h.backward(d, dw=dw) == 0
            cuda.cuda.synchronize()
            h.check(dw=dw)
            assert (h.dx.double().abs() > 0).double().mean() > 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("gradients", [False, True])
def test_odd_width_is_as_exact_for_few_tokens(cuda, built, gradients):
    """Log-sum-exps of 8 tokens at a width that 16-byte loads cannot read, against those at one
    that they can: root mean squares over 64 of them scatter by a tenth, so a factor of two
    is no accident."""
    def error(H):
        total = 0.0
        for seed in range(8):
            h = Head(cuda, 8, H, 2000, seed=seed)
            h.x += 14 * h.w[h.labels]  # tokens that one word explains: its logit is the sum
            with Dnn(cuda) as d:
                assert (h.backward(d) if gradients and H % 8 else h.forward(d)) == 0
                cuda.cuda.synchronize()
            total += (h.lse.double() - _definition(cuda, h)["lse"]).square().sum().item()
        return math.sqrt(total / 64)

    assert error(4001) <= 2 * error(4000)


@pytest.mark.gpu
@pytest.mark.parametrize("dw", [True, False])
def test_dx_over_a_long_vocabulary_shows_two_roundings(cuda, built, dw):
    """dx of 113000 words in fp16, against a model in 64 bits that rounds dz and the result once
    each: what the sum itself loses does not grow with its length.  Tokens and features fill
    the GPU's tiles once, so that speed alone asks for no split of the words.  The norm over
    256 x 1024 entries scatters by less than a percent; one chain of MMAs adds 9 %."""
    T, H, V, part = 9472, 1024, 113000, 256
    h = Head(cuda, T, H, V, "fp16", seed=5)
    h.x += (8 * cuda.rand(T, 1, device="cuda", generator=h.g) * h.w[h.labels].float()).half()
    h.dloss = 0.5 + cuda.rand(T, device="cuda", generator=h.g)
    with Dnn(cuda) as d:
        assert h.backward(d, dw=dw) == 0
        cuda.cuda.synchronize()
    w, got = h.w.double(), h.dx[:part].double()
    dz = cuda.softmax(h.x[:part].double() @ w.t(), dim=1)
    dz[cuda.arange(part), h.labels[:part]] -= 1
    dz *= h.dloss[:part, None].double()
    want = dz @ w
    m, e = cuda.frexp(dz)
    model = (cuda.ldexp((m * 2 ** 11).round() / 2 ** 11, e) @ w).half().double()
    assert (got - want).norm() <= 1.05 * (model - want).norm()


def _trained(torch, T, H, V, dtype, K=0, seed=0, **more):
    """A head whose words explain their tokens more or less, as after training."""
    h = Head(torch, T, H, V, dtype, K=K, seed=seed, **more)
    h.x += (12 * torch.rand(T, 1, device="cuda", generator=h.g) * h.w[h.labels].float()).to(h.x.dtype)
    if K:
        h.index[:, 0] = h.labels.clamp(min=0)
    h.dloss = 0.5 + torch.rand(T, device="cuda", generator=h.g)
    return h


def _over_one_rounding(got, exact):
    """Error of a 16-bit result over that of the exact one rounded once."""
    return ((got.double() - exact).norm() / (exact.to(got.dtype).double() - exact).norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V,K", [(1, 512, 5003, 0), (4, 512, 5003, 0), (4, 512, 5003, 16),
                                     (33, 264, 20000, 0), (64, 1000, 3001, 5), (64, 505, 3001, 0)])
def test_gradients_of_few_tokens_show_one_rounding(cuda, built, T, H, V, K, dtype):
    """A token's one large dz would pass its rounding on to all of its dx, and to a row of dw:
    few tokens carry what that rounding left as well.  The numerators' 2 further bits add 3 %
    to one rounding at most."""
    h = _trained(cuda, T, H, V, dtype, K=K, seed=T)
    with Dnn(cuda) as d:
        assert h.backward(d) == 0
        cuda.cuda.synchronize()
        ref = h.check()
        assert _over_one_rounding(h.dx, ref["dx"]) <= 1.1
        assert _over_one_rounding(h.dw, ref["dw"]) <= 1.1
        assert h.backward(d, dw=False) == 0
        cuda.cuda.synchronize()
        assert _over_one_rounding(h.dx, ref["dx"]) <= 1.1
        dw = h.dw.clone()
        assert h.backward(d, dx=False) == 0
        cuda.cuda.synchronize()
        assert cuda.equal(h.dw, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,V,K", [(100, 512, 20011, 0), (300, 520, 20011, 0), (300, 136, 1500, 3),
                                     (2000, 512, 2500, 0), (300, 513, 60001, 2)])
def test_dx_of_few_targets_shows_one_rounding(cuda, built, T, H, V, K, dtype):
    """dx of up to four target words per token gets what the rounding of their dz left, on flat,
    tall and single-CTA tiles, in one sum and in several, with dw and for a frozen head.  The
    other words' roundings average out."""
    h = _trained(cuda, T, H, V, dtype, K=K, seed=T, out=0.1)
    with Dnn(cuda) as d:
        for dw in (True, False):
            h.dx.fill_(math.nan)
            assert h.backward(d, dw=dw) == 0
            cuda.cuda.synchronize()
            ref = h.check(dw=dw)
            assert _over_one_rounding(h.dx, ref["dx"]) <= 1.1
        h.w = _moved(cuda, h.w, 1)  # w copied, in slices where there are more than 16 MiB
        ws = cuda.empty(h.workspace_size(d, 1) - (V * (H + 63) // 64 * 128 if H % 8 else 0)
                        + (17 << 20), device="cuda", dtype=cuda.uint8)
        h.dx.fill_(math.nan)
        assert h.backward(d, ws) == 0
        cuda.cuda.synchronize()
        h.check()
        assert _over_one_rounding(h.dx, ref["dx"]) <= 1.1
