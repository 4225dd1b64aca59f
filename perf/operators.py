"""The vocabulary losses on real work: the cases they are measured on, their plain torch
forms, the calls a program makes of them, and their definition in 64 bits.

Two operators share the linear head ``z = x w^T`` of a language model, T tokens of H
features against a vocabulary of V rows, and never hand out the T x V logits:

- cross entropy: ``loss = lse(z) - z[label]``; a negative label leaves its row out;
- distillation from a teacher's K best logits: ``q = softmax(teacher / tau)`` over the K
  entries, ``loss = sum q (log q - log softmax(z / tau))``; a negative index leaves its
  entry out, a row without entries is left out.

Rows that are left out have loss 0, log-sum-exp 0 and no gradient.  ``grad`` says what a
case asks for: "none" (scores), "x" (a frozen head) or "xw" (a training step).
"""

import ctypes as C
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the log-probability of one sampled token under a small head: launch latency
        dict(name="ce_score_token", op="ce", grad="none", T=1, H=1024, V=32000, K=1, tau=1.0,
             dtype="bf16", out=0.0, pad=0),
        # a few drafted tokens checked against a large head: one read of the weights
        dict(name="ce_score_draft", op="ce", grad="none", T=8, H=4096, V=131072, K=1, tau=1.0,
             dtype="bf16", out=0.0, pad=0),
        # perplexity of a prompt
        dict(name="ce_score_prompt", op="ce", grad="none", T=2048, H=4096, V=131072, K=1, tau=1.0,
             dtype="bf16", out=0.1, pad=0),
        # the head of a training step, one micro-batch of 8192 tokens
        dict(name="ce_train_large", op="ce", grad="xw", T=8192, H=4096, V=131072, K=1, tau=1.0,
             dtype="bf16", out=0.1, pad=0),
        # packed documents: odd lengths, an odd vocabulary, a third of the rows left out,
        # hidden states that are a slice of wider rows
        dict(name="ce_train_ragged", op="ce", grad="xw", T=1537, H=1000, V=50021, K=1, tau=1.0,
             dtype="bf16", out=0.35, pad=24),
        # 16-bit training with half precision
        dict(name="ce_train_half", op="ce", grad="xw", T=2048, H=2048, V=32000, K=1, tau=1.0,
             dtype="fp16", out=0.05, pad=0),
        # a frozen head (adapter training): only the hidden states' gradient
        dict(name="ce_train_frozen", op="ce", grad="x", T=4096, H=2048, V=65536, K=1, tau=1.0,
             dtype="bf16", out=0.1, pad=0),
        # divergence from the teacher on a few tokens while a student decodes
        dict(name="kd_score_few", op="kd", grad="none", T=4, H=2048, V=32000, K=16, tau=1.0,
             dtype="bf16", out=0.0, pad=0),
        # validation of a student
        dict(name="kd_score_eval", op="kd", grad="none", T=4096, H=2048, V=65536, K=64, tau=1.0,
             dtype="bf16", out=0.1, pad=0),
        # a distillation step with cached teacher logits
        dict(name="kd_train", op="kd", grad="xw", T=4096, H=4096, V=100000, K=32, tau=1.0,
             dtype="bf16", out=0.1, pad=0),
        # sizes that suit no tile and no vector load, a softened teacher
        dict(name="kd_train_odd", op="kd", grad="xw", T=777, H=1111, V=32003, K=20, tau=2.0,
             dtype="bf16", out=0.2, pad=0),
        # few tokens against a wide head, many teacher entries
        dict(name="kd_train_wide", op="kd", grad="xw", T=512, H=8192, V=128000, K=128, tau=1.5,
             dtype="bf16", out=0.1, pad=0),
    ]


_UNITS = {"none": 1, "x": 2, "xw": 3}  # products of T*H*V that a case cannot do without


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        T, V = spread(1, 8192), spread(1000, 160000)
        H = spread(256, 8192)
        if rng.random() < 0.75:
            H = max(256, H // 8 * 8)  # widths of real models; the others suit no vector load
        op = rng.choice(["ce", "kd"])
        grad = rng.choice(["none", "x", "xw", "xw"])
        if T * V <= 8192 * 131072 and _UNITS[grad] * T * H * V <= 3 * 8192 * 4096 * 131072:
            break
    return dict(op=op, grad=grad, T=T, H=H, V=V,
                K=1 if op == "ce" else spread(1, 128),
                tau=1.0 if op == "ce" else rng.choice([1.0, 1.5, 2.0, 4.0]),
                dtype=rng.choice(["bf16", "bf16", "bf16", "fp16"]),
                out=rng.choice([0.0, 0.1, 0.3]) if T >= 16 else 0.0, pad=rng.choice([0, 0, 8, 17]))


def _inputs(case, seed):
    """Inputs of a trained head: logits of about unit spread, the likely token's logit
    raised by 0 to 18 (probabilities from 1e-5 to nearly one)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, H, V, K = case["T"], case["H"], case["V"], case["K"]
    dt = DTYPES[case["dtype"]]

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    w = torch.empty(V, H, device="cuda", dtype=dt)
    for v0 in range(0, V, 16384):
        n = min(16384, V - v0)
        w[v0:v0 + n] = torch.randn(n, H, device="cuda", generator=g) * H ** -0.5
    likely = torch.randint(0, V, (T,), device="cuda", generator=g)
    x = torch.randn(T, H, device="cuda", generator=g)
    x += 18 * uniform(T, 1) * w[likely].float()
    rows = torch.zeros(T, H + case["pad"], device="cuda", dtype=dt)
    rows[:, :H] = x
    left_out = uniform(T) < case["out"]
    weight = (0.5 + uniform(T)) / T
    s = dict(case=dict(case), x=rows[:, :H], w=w, dloss=weight)
    if case["op"] == "ce":
        s["labels"] = torch.where(left_out, -100, likely)
    else:
        step = 1 + (uniform(T, 1) * (V // K - 1)).long()
        s["index"] = (likely[:, None] + step * torch.arange(K, device="cuda")) % V
        s["teacher"] = (torch.randn(T, K, device="cuda", generator=g) * 2).sort(
            dim=1, descending=True).values.contiguous() + 10
        kept = 1 + (uniform(T, 1) * K * 1.5).long()  # a third of the rows have fewer entries
        kept = torch.where(left_out[:, None], 0, kept)
        s["index"] = torch.where(torch.arange(K, device="cuda") < kept, s["index"], -1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    x, w = s["x"], s["w"]
    s["loss"] = torch.empty(x.shape[0], device="cuda")
    s["lse"] = torch.empty(x.shape[0], device="cuda")
    if case["grad"] != "none":
        s["dx"] = torch.empty(x.shape, device="cuda", dtype=x.dtype)
    if case["grad"] == "xw":
        s["dw"] = torch.empty_like(w)
    return s


# ------------------------------------------------------------------ the plain form --
def _plain(s):
    case, tau = s["case"], s["case"]["tau"]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if tau != 1.0:
        z /= tau
    top = z.amax(dim=1, keepdim=True)
    lse = top + (z - top).exp().sum(dim=1, keepdim=True).log()
    if case["op"] == "ce":
        index = s["labels"].clamp(min=0)[:, None]
        keep = s["labels"][:, None] >= 0
        loss = lse - z.gather(1, index)
        q = keep.float()
    else:
        index, entry = s["index"].clamp(min=0), s["index"] >= 0
        keep = entry.any(dim=1, keepdim=True)
        t = torch.where(entry, s["teacher"] / tau, -math.inf)
        t = t - torch.where(keep, t.amax(dim=1, keepdim=True), 0.0)
        total = t.exp().sum(dim=1, keepdim=True)
        q = torch.where(keep, t.exp() / total, 0.0)
        log_q = torch.where(entry, t - total.log(), 0.0)
        loss = (q * (log_q - (z.gather(1, index) - lse))).sum(dim=1, keepdim=True)
    out = {"loss": torch.where(keep, loss, 0.0)[:, 0], "lse": torch.where(keep, lse, 0.0)[:, 0]}
    if case["grad"] == "none":
        return out
    d = z.sub_(lse).exp_()
    d.scatter_add_(1, index, -q)
    d *= torch.where(keep, s["dloss"][:, None] / tau, 0.0)
    out["dx"] = (d @ w).to(s["x"].dtype)
    if case["grad"] == "xw":
        out["dw"] = (d.t() @ x).to(s["w"].dtype)
    return out


# ------------------------------------------------------------ the framework's calls --
_handle = None


def _cudnn():
    """The library and the program's one handle (its workspace grows with the largest call)."""
    global _handle
    from muda_b200 import capi

    lib = capi.cudnn()
    if _handle is None:
        _handle = C.c_void_p()
        assert lib.cudnnCreate(C.byref(_handle)) == 0
    return capi, lib, _handle


def _descriptors(s):
    """Descriptors of the state's tensors, made once as a program keeps them."""
    if "desc" in s:
        return s["desc"]
    capi, lib, _ = _cudnn()
    dt = {torch.bfloat16: capi.CUDNN_DATA_BFLOAT16, torch.float16: capi.CUDNN_DATA_HALF}[s["x"].dtype]

    def rows(t):
        d = C.c_void_p()
        assert lib.cudnnCreateTensorDescriptor(C.byref(d)) == 0
        assert lib.cudnnSetTensor4dDescriptorEx(d, dt, t.shape[0], t.shape[1], 1, 1, t.stride(0),
                                                1, t.stride(0), t.stride(0)) == 0
        return d

    f = C.c_void_p()
    assert lib.cudnnCreateFilterDescriptor(C.byref(f)) == 0
    assert lib.cudnnSetFilter4dDescriptor(f, dt, capi.CUDNN_TENSOR_NCHW, *s["w"].shape, 1, 1) == 0
    s["desc"] = rows(s["x"]), f, rows(s["dx"]) if "dx" in s else None
    return s["desc"]


def _calls(s):
    case = s["case"]
    _, lib, handle = _cudnn()
    xd, wd, dxd = _descriptors(s)

    def p(name):
        return C.c_void_p(s[name].data_ptr()) if name in s else None

    assert lib.cudnnSetStream(handle, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    if case["op"] == "ce":
        head = (handle, xd, p("x"), wd, p("w"), p("labels"))
        forward, backward = lib.cudnnLinearCrossEntropyForward, lib.cudnnLinearCrossEntropyBackward
    else:
        head = (handle, xd, p("x"), wd, p("w"), case["K"], p("index"), p("teacher"), case["tau"])
        forward, backward = lib.cudnnLinearDistillationForward, lib.cudnnLinearDistillationBackward
    if case["grad"] == "none":
        status = forward(*head, None, 0, p("loss"), p("lse"))
    else:
        status = backward(*head, p("dloss"), None, 0, p("loss"), p("lse"), dxd, p("dx"),
                          wd if "dw" in s else None, p("dw"))
    assert status == 0, lib.cudnnGetErrorString(status)
    return {k: s[k] for k in ("loss", "lse", "dx", "dw") if k in s}


def run(state):
    return _calls(state) if own else _plain(state)


def work(case):
    T, H, V, K = case["T"], case["H"], case["V"], case["K"]
    b = 2 * T * H + 2 * V * H + 8 * T  # x, w; loss and log-sum-exp
    b += 8 * T if case["op"] == "ce" else 12 * T * K
    if case["grad"] != "none":
        b += 4 * T + 2 * T * H
    if case["grad"] == "xw":
        b += 2 * V * H
    return {"bytes": b, "flops": 2 * _UNITS[case["grad"]] * T * H * V}


# ------------------------------------------------------------- the definition, 64 bits --
def exact(case, seed):
    """Row blocks of the definition in 64 bits: log p by row, then its derivative."""
    s = _inputs(case, seed)
    T, tau = case["T"], case["tau"]
    w = s["w"].double()
    out = {"loss": torch.zeros(T, device="cuda", dtype=torch.float64),
           "lse": torch.zeros(T, device="cuda", dtype=torch.float64)}
    if case["grad"] != "none":
        out["dx"] = torch.zeros(s["x"].shape, device="cuda", dtype=torch.float64)
    if case["grad"] == "xw":
        out["dw"] = torch.zeros_like(w)
    for r0 in range(0, T, 1024):
        r = slice(r0, min(T, r0 + 1024))
        x = s["x"][r].double()
        z = torch.mm(x, w.t()).div_(tau)
        lse = torch.logsumexp(z, dim=1)
        target = torch.zeros_like(z)  # the distribution that the loss compares with
        entropy = torch.zeros_like(lse)
        if case["op"] == "ce":
            on = (s["labels"][r] >= 0).nonzero()[:, 0]
            target[on, s["labels"][r][on]] = 1.0
        else:
            teacher = s["teacher"][r].double().div(tau)
            teacher = teacher.masked_fill(s["index"][r] < 0, -math.inf)
            on = (s["index"][r] >= 0).any(dim=1).nonzero()[:, 0]
            q = torch.softmax(teacher[on], dim=1)
            row, k = (s["index"][r][on] >= 0).nonzero(as_tuple=True)
            target.index_put_((on[row], s["index"][r][on][row, k]), q[row, k], accumulate=True)
            entropy[on] = torch.special.entr(q).sum(dim=1)
        live = torch.zeros_like(lse)
        live[on] = 1.0
        cross = live * lse - (target * z).sum(dim=1)
        out["loss"][r] = live * cross - entropy
        out["lse"][r] = live * lse
        if case["grad"] == "none":
            continue
        d = (z - lse[:, None]).exp_().mul_(live[:, None]).sub_(target)
        d *= s["dloss"][r].double()[:, None] / tau
        out["dx"][r] = torch.mm(d, w)
        if case["grad"] == "xw":
            out["dw"].addmm_(d.t(), x)
    return out
