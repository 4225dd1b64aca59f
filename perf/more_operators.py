"""Embeddings and the losses of post-training on real work: the cases they are measured on,
their plain torch forms, the calls a program makes of them, and their definition in 64 bits.

Three operators around the vocabulary of a language model, V words of H features:

- embedding: ``y[t] = scale * w[token[t]]`` and its gradient ``dw[v] = scale * sum of dy[t]
  over the tokens t that are v``; a negative token (padding) has a row of zeros and enters no
  gradient;
- policy loss on a linear head, ``nll = lse(z) - z[label]`` with ``z = x w^T / tau``:
  ``r = exp(old - nll)``, ``s = min(r A, clip(r) A)`` (for ``A < 0`` at least ``dual * A``),
  ``loss = -s + kl_coef * (exp(d) - d - 1)`` with ``d = nll - ref``;
- preference loss on the same head: ``L`` of a sequence is the sum (or mean) of
  ``ref - nll`` over its tokens, ``h = beta * (L_chosen - L_rejected) - margin``, and the loss
  ``softplus(-h) + smooth * h``, ``max(0, 1 - h)`` or ``((h - 1/2) / beta)^2``.

A negative label leaves its token out: 0 in every output, no gradient.  ``grad`` says what a
case of a loss asks for: "none" (scores), "x" (a frozen head) or "xw" (a training step).
"""

import ctypes as C
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MODES = ["sigmoid", "hinge", "squared"]


def _embed(name, grad, T, H, V, dtype, table, scale, out, pad, steps=1):
    return dict(name=name, op="embedding", grad=grad, T=T, H=H, V=V, dtype=dtype, table=table,
                scale=scale, out=out, pad=pad, steps=steps)


def _policy(name, grad, T, H, V, dtype, tau, lo, hi, dual, kl, out, pad):
    return dict(name=name, op="policy", grad=grad, T=T, H=H, V=V, dtype=dtype, tau=tau, lo=lo,
                hi=hi, dual=dual, kl=kl, out=out, pad=pad)


def _pairs(name, grad, T, H, V, dtype, pairs, mode, averaged, beta, margin, smooth, ref, out, pad):
    return dict(name=name, op="preference", grad=grad, T=T, H=H, V=V, dtype=dtype, pairs=pairs,
                mode=mode, averaged=averaged, beta=beta, margin=margin, smooth=smooth, ref=ref,
                out=out, pad=pad)


def listed():
    return [
        # the next token of a batch of 8 that decodes: launch latency
        _embed("embed_decode", "none", 8, 4096, 128000, "bf16", "bf16", 1.0, 0.0, 0),
        # the prompts of a batch, a model that scales its embeddings
        _embed("embed_prompt", "none", 16384, 4096, 128000, "bf16", "bf16", 64.0, 0.02, 0),
        # an untied table's whole gradient, one micro-batch
        _embed("embed_grad", "w", 8192, 4096, 128000, "bf16", "bf16", 64.0, 0.02, 0),
        # two micro-batches added up in a float gradient buffer
        _embed("embed_grad_accumulate", "w", 32768, 2048, 50257, "bf16", "fp32", 1.0, 0.1, 0,
               steps=2),
        # sizes that suit no vector load, gradients in wider rows, half precision
        _embed("embed_grad_odd", "w", 1537, 1111, 32003, "fp16", "fp16", 1.0, 0.3, 17),
        # log-probabilities, ratios and divergences of 8 sampled tokens while a policy decodes
        _policy("policy_score_few", "none", 8, 2048, 32000, "bf16", 1.0, 0.2, 0.2, 0.0, 0.05, 0.0,
                0),
        # a policy step, prompts left out
        _policy("policy_train", "xw", 4096, 4096, 100000, "bf16", 1.0, 0.2, 0.28, 3.0, 0.02, 0.3,
                0),
        # sampled at another temperature; odd sizes, half precision
        _policy("policy_train_odd", "xw", 1537, 1000, 50021, "fp16", 0.7, 0.2, 0.2, 0.0, 0.1, 0.35,
                24),
        # adapters below a frozen head
        _policy("policy_train_frozen", "x", 2048, 2048, 65536, "bf16", 1.0, 0.2, 0.2, 0.0, 0.0,
                0.1, 0),
        # rewards of a validation set
        _pairs("preference_score", "none", 2048, 2048, 65536, "bf16", 4, "sigmoid", False, 0.1,
               0.0, 0.0, True, 0.2, 0),
        # a preference step: 8 pairs of sequences with their prompts
        _pairs("preference_train", "xw", 6144, 2048, 65536, "bf16", 8, "sigmoid", False, 0.1, 0.0,
               0.1, True, 0.3, 0),
        # length-normalised without a reference, short ragged sequences, sizes that suit no tile
        _pairs("preference_train_odd", "xw", 777, 1111, 32003, "bf16", 13, "sigmoid", True, 2.0,
               0.5, 0.0, False, 0.2, 17),
    ]


_UNITS = {"none": 1, "x": 2, "xw": 3}  # products of T*H*V that a head's case cannot do without


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["embedding", "policy", "preference"])
    pad = rng.choice([0, 0, 8, 17])
    while True:
        V = spread(256, 160000) if op == "embedding" else spread(1000, 160000)
        H = spread(64, 8192) if op == "embedding" else spread(256, 8192)
        if rng.random() < 0.75:
            H = max(64, H // 8 * 8)  # widths of real models; the others suit no vector load
        T = spread(1, 65536) if op == "embedding" else spread(2, 6144)
        grad = rng.choice(["none", "w", "w"] if op == "embedding" else ["none", "x", "xw", "xw"])
        if op == "embedding":
            if T * H <= 32768 * 2048 and V * H <= 128000 * 4096:
                break
        elif T * V <= 4096 * 100000 and _UNITS[grad] * T * H * V <= 3 * 4096 * 4096 * 100000:
            break
    out = rng.choice([0.0, 0.1, 0.3]) if T >= 16 else 0.0
    if op == "embedding":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        table = rng.choice([dtype, dtype, "fp32"])
        steps = rng.choice([1, 2]) if grad == "w" and table == "fp32" else 1
        c = _embed("", grad, T, H, V, dtype, table, rng.choice([1.0, H ** 0.5]), out, pad, steps)
    elif op == "policy":
        c = _policy("", grad, T, H, V, rng.choice(["bf16", "bf16", "bf16", "fp16"]),
                    rng.choice([1.0, 1.0, 0.7, 1.5]), rng.choice([0.1, 0.2]),
                    rng.choice([0.2, 0.28]), rng.choice([0.0, 0.0, 3.0]),
                    rng.choice([0.0, 0.02, 0.1]), out, pad)
    else:
        mode = rng.choice(["sigmoid", "sigmoid", "hinge", "squared"])
        averaged = rng.random() < 0.3
        c = _pairs("", grad, T, H, V, rng.choice(["bf16", "bf16", "bf16", "fp16"]),
                   spread(1, max(1, min(64, T // 2))), mode, averaged,
                   rng.choice([1.0, 2.0]) if averaged else rng.choice([0.05, 0.1, 0.3]),
                   rng.choice([0.0, 0.5]), rng.choice([0.0, 0.1]) if mode == "sigmoid" else 0.0,
                   rng.random() < 0.8, out, pad)
    del c["name"]
    return c


# ------------------------------------------------------------------------- the inputs --
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(values, pad, dtype):
    """The values as a slice of rows that are `pad` elements wider."""
    T, H = values.shape
    rows = torch.zeros(T, H + pad, device="cuda", dtype=dtype)
    rows[:, :H] = values
    return rows[:, :H]


def _table(V, H, dtype, g):
    w = torch.empty(V, H, device="cuda", dtype=dtype)
    for v0 in range(0, V, 16384):
        n = min(16384, V - v0)
        w[v0:v0 + n] = torch.randn(n, H, device="cuda", generator=g) * H ** -0.5
    return w


def _embedding_inputs(case, seed):
    """Words as text has them: the k-th most frequent with a chance of about 1 / k, frequent
    ones first in the table."""
    g = _generator(seed)
    T, H, V = case["T"], case["H"], case["V"]
    s = dict(case=dict(case), tokens=[], dy=[])
    for _ in range(case["steps"]):
        u = torch.rand(T, device="cuda", generator=g, dtype=torch.float64)
        tokens = (torch.exp(u * math.log(V)) - 1).long().clamp(max=V - 1)
        padding = torch.rand(T, device="cuda", generator=g) < case["out"]
        s["tokens"].append(torch.where(padding, -1, tokens))
        if case["grad"] == "w":
            dy = torch.randn(T, H, device="cuda", generator=g) / T
            s["dy"].append(_rows(dy * 64 if case["dtype"] == "fp16" else dy, case["pad"],
                                 DTYPES[case["dtype"]]))
    if case["grad"] == "none":
        s["w"] = _table(V, H, DTYPES[case["table"]], g)
    return s


def _nll(x, w, labels, tau):
    """Negative log-probabilities as an earlier pass over the same tokens has them."""
    nll = torch.empty(x.shape[0], device="cuda")
    x = x.contiguous()
    for r0 in range(0, x.shape[0], 1024):
        r = slice(r0, r0 + 1024)
        z = torch.mm(x[r], w.t(), out_dtype=torch.float32).div_(tau)
        at = z.gather(1, labels[r].clamp(min=0)[:, None])[:, 0]
        nll[r] = torch.logsumexp(z, dim=1) - at
    return nll


def _head_inputs(case, seed):
    """A trained head: logits of about unit spread, the sampled token's logit raised by 0 to 18
    (probabilities from 1e-5 to nearly one)."""
    g = _generator(seed)
    T, H, V = case["T"], case["H"], case["V"]
    dt = DTYPES[case["dtype"]]

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    w = _table(V, H, dt, g)
    sampled = torch.randint(0, V, (T,), device="cuda", generator=g)
    x = normal(T, H)
    x += 18 * uniform(T, 1) * w[sampled].float()
    x = _rows(x, case["pad"], dt)
    s = dict(case=dict(case), x=x, w=w)
    tau = case.get("tau", 1.0)
    nll = _nll(x, w, sampled, tau)
    if case["op"] == "policy":
        s["labels"] = torch.where(uniform(T) < case["out"], -100, sampled)
        # ratios of a few updates after sampling; an eighth of the tokens has moved far
        moved = normal(T) * torch.where(uniform(T) < 0.125, 1.0, 0.1)
        # no ratio right on a clip, where fp32 logits cannot tell its side
        for edge in (1 - case["lo"], 1 + case["hi"]) + ((case["dual"],) if case["dual"] else ()):
            near = moved - math.log(edge)
            moved = torch.where(near.abs() < 0.0025, math.log(edge) + near.sign() * 0.0025 + near,
                                moved)
        s["old"] = nll + moved
        s["ref"] = nll + normal(T)  # the model that training started from is further away
        s["advantage"] = normal(T)
        s["dloss"] = (0.5 + uniform(T)) / T
    else:
        P = case["pairs"]
        # sequences of uneven lengths, a few rows of padding behind the last
        cuts = uniform(2 * P) + 0.2
        ends = (cuts.double().cumsum(0) / cuts.double().sum() * (T - T // 64)).round().long()
        s["offsets"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), ends])
        # a sequence's first tokens are its prompt, left out of the loss
        t = torch.arange(T, device="cuda")
        k = (torch.bucketize(t, ends, right=True)).clamp(max=2 * P - 1)
        start, end = s["offsets"][k], s["offsets"][k + 1]
        prompt = t - start < ((end - start) * case["out"] * uniform(2 * P)[k] * 2).long()
        s["labels"] = torch.where(prompt, -100, sampled)
        # the policy has moved from the reference, towards some sequences and away from others
        s["ref"] = nll + normal(T) * 0.5 + normal(2 * P)[k] * 0.2 if case["ref"] else None
        s["dloss"] = (0.5 + uniform(P)) / P
    return s


def _inputs(case, seed):
    return (_embedding_inputs if case["op"] == "embedding" else _head_inputs)(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    T, H, V = case["T"], case["H"], case["V"]

    def floats(*names, n=T):
        for name in names:
            s[name] = torch.empty(n, device="cuda")

    if case["op"] == "embedding":
        if case["grad"] == "none":
            s["y"] = torch.empty(T, H, device="cuda", dtype=DTYPES[case["dtype"]])
        else:
            s["dw"] = torch.empty(V, H, device="cuda", dtype=DTYPES[case["table"]])
        return s
    if case["op"] == "policy":
        floats("loss", "nll", "ratio", "kl")
    else:
        floats("nll")
        floats("loss", n=case["pairs"])
        floats("rewards", n=2 * case["pairs"])
    if case["grad"] != "none":
        s["dx"] = torch.empty(T, H, device="cuda", dtype=s["x"].dtype)
    if case["grad"] == "xw":
        s["dw"] = torch.empty_like(s["w"])
    return s


# --------------------------------------------------------------------- the plain form --
def _plain_embedding(s):
    case = s["case"]
    if case["grad"] == "none":
        tokens = s["tokens"][0]
        y = s["w"][tokens.clamp(min=0)].float() * case["scale"]
        return {"y": torch.where(tokens[:, None] >= 0, y, 0.0).to(s["y"].dtype)}
    dw = torch.zeros(s["dw"].shape, device="cuda")
    for tokens, dy in zip(s["tokens"], s["dy"]):
        kept = (tokens >= 0).nonzero()[:, 0]
        dw.index_add_(0, tokens[kept], dy[kept].float() * case["scale"])
    return {"dw": dw.to(s["dw"].dtype)}


def _plain_policy(s, nll, keep):
    """Outputs of the policy loss, and its derivative by each token's nll."""
    case, A = s["case"], s["advantage"]
    r = (s["old"] - nll).exp()
    plain, clipped = r * A, r.clamp(1 - case["lo"], 1 + case["hi"]) * A
    surrogate = torch.minimum(plain, clipped)
    moves = plain <= clipped
    if case["dual"]:
        floor = case["dual"] * A
        low = (A < 0) & (surrogate < floor)
        surrogate, moves = torch.where(low, floor, surrogate), moves & ~low
    d = (nll.double() - s["ref"].double())  # exp(d) - d - 1 of small d loses all digits in fp32
    kl = (d.exp() - d - 1).float()
    loss = case["kl"] * kl - surrogate
    g = torch.where(moves, plain, 0.0) + case["kl"] * d.expm1().float()
    out = {"loss": loss, "nll": nll, "ratio": r, "kl": kl}
    return {k: torch.where(keep, v, 0.0) for k, v in out.items()}, g * s["dloss"]


def _plain_preference(s, nll, keep):
    case, P = s["case"], s["case"]["pairs"]
    T = nll.shape[0]
    nll = torch.where(keep, nll, 0.0)
    gain = (s["ref"] if s["ref"] is not None else 0.0) - nll.double()  # long sums in 64 bits
    gain = torch.where(keep, gain, 0.0)
    zero = torch.zeros(1, device="cuda", dtype=torch.float64)
    sums, counts = torch.cat([zero, gain.cumsum(0)]), torch.cat([zero, keep.double().cumsum(0)])
    lo, hi = s["offsets"][:-1], s["offsets"][1:]
    n = counts[hi] - counts[lo]
    share = 1 / n.clamp(min=1) if case["averaged"] else torch.ones_like(n)
    L = (sums[hi] - sums[lo]) * share
    live = (n[:P] > 0) & (n[P:] > 0)
    beta, smooth = case["beta"], case["smooth"]
    h = beta * (L[:P] - L[P:]) - case["margin"]
    if case["mode"] == "sigmoid":
        loss = torch.log1p((-h.abs()).exp()) + (-h).clamp(min=0) + smooth * h
        slope = smooth - 1 / (1 + h.exp())
    elif case["mode"] == "hinge":
        loss = (1 - h).clamp(min=0)
        slope = -(h < 1).double()
    else:
        loss = ((h - 0.5) / beta) ** 2
        slope = 2 * (h - 0.5) / beta ** 2
    g = torch.where(live, slope * beta * s["dloss"], 0.0)
    g = torch.cat([-g, g]) * share
    t = torch.arange(T, device="cuda")
    k = torch.bucketize(t, hi, right=True)
    inside = (k < 2 * P) & keep
    g = torch.where(inside, g[k.clamp(max=2 * P - 1)], 0.0).float()
    out = {"loss": torch.where(live, loss, 0.0).float(),
           "rewards": torch.where(live.repeat(2), beta * L, 0.0).float(), "nll": nll}
    return out, g


def _plain(s):
    case = s["case"]
    if case["op"] == "embedding":
        return _plain_embedding(s)
    tau = case.get("tau", 1.0)
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if tau != 1.0:
        z /= tau
    top = z.amax(dim=1, keepdim=True)
    lse = top + (z - top).exp().sum(dim=1, keepdim=True).log()
    keep = s["labels"] >= 0
    index = s["labels"].clamp(min=0)[:, None]
    nll = (lse - z.gather(1, index))[:, 0]
    out, g = (_plain_policy if case["op"] == "policy" else _plain_preference)(s, nll, keep)
    if case["grad"] == "none":
        return out
    d = z.sub_(lse).exp_()
    d.scatter_add_(1, index, torch.full_like(nll, -1.0)[:, None])
    d *= torch.where(keep, g / tau, 0.0)[:, None]
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
    types = {torch.bfloat16: capi.CUDNN_DATA_BFLOAT16, torch.float16: capi.CUDNN_DATA_HALF,
             torch.float32: capi.CUDNN_DATA_FLOAT}

    def rows(t):
        d = C.c_void_p()
        assert lib.cudnnCreateTensorDescriptor(C.byref(d)) == 0
        assert lib.cudnnSetTensor4dDescriptorEx(d, types[t.dtype], *t.shape, 1, 1, t.stride(0), 1,
                                                t.stride(0), t.stride(0)) == 0
        return d

    def table(t):
        d = C.c_void_p()
        assert lib.cudnnCreateFilterDescriptor(C.byref(d)) == 0
        assert lib.cudnnSetFilter4dDescriptor(d, types[t.dtype], capi.CUDNN_TENSOR_NCHW, *t.shape,
                                              1, 1) == 0
        return d

    s["desc"] = {k: rows(s[k]) for k in ("x", "y", "dx") if k in s}
    s["desc"].update({k: table(s[k]) for k in ("w", "dw") if k in s})
    if s.get("dy"):
        s["desc"]["dy"] = rows(s["dy"][0])
    return s["desc"]


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _calls(s):
    case = s["case"]
    capi, lib, handle = _cudnn()
    d = _descriptors(s)
    assert lib.cudnnSetStream(handle, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0

    if case["op"] == "embedding":
        alpha = C.byref(C.c_float(case["scale"]))
        if case["grad"] == "none":
            status = lib.cudnnEmbeddingForward(handle, alpha, d["w"], _p(s["w"]),
                                               _p(s["tokens"][0]), C.byref(C.c_float(0.0)),
                                               d["y"], _p(s["y"]))
            assert status == 0, lib.cudnnGetErrorString(status)
            return {"y": s["y"]}
        for step, (tokens, dy) in enumerate(zip(s["tokens"], s["dy"])):
            status = lib.cudnnEmbeddingBackward(handle, alpha, d["dy"], _p(dy), _p(tokens), None, 0,
                                                C.byref(C.c_float(1.0 if step else 0.0)),
                                                d["dw"], _p(s["dw"]))
            assert status == 0, lib.cudnnGetErrorString(status)
        return {"dw": s["dw"]}

    head = (handle, d["x"], _p(s["x"]), d["w"], _p(s["w"]), _p(s["labels"]))
    if case["op"] == "policy":
        names = ("loss", "nll", "ratio", "kl")
        head += (_p(s["old"]), _p(s["ref"]), _p(s["advantage"]), case["tau"], case["lo"],
                 case["hi"], case["dual"], case["kl"])
        forward, backward = lib.cudnnLinearPolicyLossForward, lib.cudnnLinearPolicyLossBackward
    else:
        names = ("loss", "rewards", "nll")
        head += (case["pairs"], _p(s["offsets"]), _p(s["ref"]), MODES.index(case["mode"]),
                 int(case["averaged"]), case["beta"], case["margin"], case["smooth"])
        forward = lib.cudnnLinearPreferenceLossForward
        backward = lib.cudnnLinearPreferenceLossBackward
    outs = tuple(_p(s[n]) for n in names)
    if case["grad"] == "none":
        status = forward(*head, None, 0, *outs)
    else:
        status = backward(*head, _p(s["dloss"]), None, 0, *outs, d["dx"], _p(s["dx"]),
                          d.get("dw"), _p(s.get("dw")))
    assert status == 0, lib.cudnnGetErrorString(status)
    return {k: s[k] for k in names + ("dx", "dw") if k in s}


def run(state):
    return _calls(state) if own else _plain(state)


def _distinct(case):
    """Words that a batch of tokens is expected to hold."""
    T, V = case["T"] * (1 - case["out"]), case["V"]
    k = torch.arange(1, V + 1, dtype=torch.float64)
    chance = torch.log1p(1 / k) / math.log(V + 1)
    return float((1 - torch.exp(T * torch.log1p(-chance))).sum())


def work(case):
    T, H, V = case["T"], case["H"], case["V"]
    if case["op"] == "embedding":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}
        kept = T * (1 - case["out"])
        if case["grad"] == "none":
            return {"bytes": 8 * T + _distinct(case) * H * size[case["table"]]
                    + T * H * size[case["dtype"]], "flops": kept * H}
        b = case["steps"] * (8 * T + kept * H * size[case["dtype"]]) + V * H * size[case["table"]]
        b += (case["steps"] - 1) * 2 * _distinct(case) * H * size[case["table"]]
        return {"bytes": b, "flops": case["steps"] * 2 * kept * H}
    b = 2 * T * H + 2 * V * H + 8 * T + 4 * T  # x, w, labels; nll
    b += (12 + 12) * T if case["op"] == "policy" else 4 * T * case["ref"] + 36 * case["pairs"]
    if case["grad"] != "none":
        b += 2 * T * H + (4 * T if case["op"] == "policy" else 4 * case["pairs"])
    if case["grad"] == "xw":
        b += 2 * V * H
    return {"bytes": b, "flops": 2 * _UNITS[case["grad"]] * T * H * V}


# ------------------------------------------------------------- the definition, 64 bits --
def _exact_embedding(case, s):
    scale = case["scale"]
    if case["grad"] == "none":
        tokens = s["tokens"][0]
        y = torch.zeros(case["T"], case["H"], device="cuda", dtype=torch.float64)
        at = tokens >= 0
        y[at] = s["w"].index_select(0, tokens[at]).double().mul_(scale)
        return {"y": y}
    dw = torch.zeros(case["V"], case["H"], device="cuda", dtype=torch.float64)
    for tokens, dy in zip(s["tokens"], s["dy"]):
        order = torch.argsort(tokens, stable=True)
        for part in order.split(4096):
            part = part[tokens[part] >= 0]
            dw.index_put_((tokens[part],), dy[part].double(), accumulate=True)
    return {"dw": dw.mul_(scale)}


def exact(case, seed):
    """The definition in 64 bits; the losses' derivatives by nll from autograd."""
    s = _inputs(case, seed)
    if case["op"] == "embedding":
        return _exact_embedding(case, s)
    T, tau = case["T"], case.get("tau", 1.0)
    w = s["w"].double()
    live = s["labels"] >= 0
    logp = torch.zeros(T, device="cuda", dtype=torch.float64)
    blocks = [slice(r0, min(T, r0 + 1024)) for r0 in range(0, T, 1024)]
    for r in blocks:
        z = torch.mm(s["x"][r].double(), w.t()).div_(tau)
        z = torch.log_softmax(z, dim=1)
        logp[r] = z.gather(1, s["labels"][r].clamp(min=0)[:, None])[:, 0]
    logp = torch.where(live, logp, 0.0).requires_grad_()
    if case["op"] == "policy":
        A = s["advantage"].double()
        ratio = torch.exp(logp + s["old"].double())
        bounded = torch.clamp(ratio, 1 - case["lo"], 1 + case["hi"])
        objective = torch.where(ratio * A <= bounded * A, ratio * A, bounded * A)
        if case["dual"]:
            objective = torch.where(A < 0, torch.maximum(objective, case["dual"] * A), objective)
        log_r = -s["ref"].double() - logp  # log p_ref / p
        kl = torch.expm1(log_r) - log_r
        loss = case["kl"] * kl - objective
        out = {"loss": loss, "nll": -logp, "ratio": ratio, "kl": kl}
        out = {k: torch.where(live, v, 0.0) for k, v in out.items()}
    else:
        P = case["pairs"]
        ends = s["offsets"].tolist()
        totals, counted = [], []
        for a, b in zip(ends[:-1], ends[1:]):
            on = live[a:b].nonzero()[:, 0] + a
            gain = logp[on] + (s["ref"][on].double() if s["ref"] is not None else 0.0)
            totals.append(gain.mean() if case["averaged"] and len(on) else gain.sum())
            counted.append(len(on) > 0)
        loss, rewards = [], [torch.zeros_like(logp[0])] * (2 * P)
        for p in range(P):
            if not (counted[p] and counted[P + p]):
                loss.append(torch.zeros_like(logp[0]))
                continue
            h = case["beta"] * (totals[p] - totals[P + p]) - case["margin"]
            if case["mode"] == "sigmoid":
                sig = torch.nn.functional.logsigmoid
                loss.append(-(1 - case["smooth"]) * sig(h) - case["smooth"] * sig(-h))
            elif case["mode"] == "hinge":
                loss.append(torch.relu(1 - h))
            else:
                loss.append(((h - 0.5) / case["beta"]).square())
            for k in (p, P + p):
                rewards[k] = case["beta"] * totals[k]
        out = {"loss": torch.stack(loss), "rewards": torch.stack(rewards), "nll": -logp}
    g = None
    if case["grad"] != "none" and out["loss"].requires_grad:
        g = torch.autograd.grad((out["loss"] * s["dloss"].double()).sum(), logp,
                                allow_unused=True)[0]
    g = torch.zeros_like(logp) if g is None else torch.where(live, g, 0.0)
    out = {k: v.detach() for k, v in out.items()}
    if case["grad"] == "none":
        return out
    out["dx"] = torch.zeros(s["x"].shape, device="cuda", dtype=torch.float64)
    if case["grad"] == "xw":
        out["dw"] = torch.zeros_like(w)
    for r in blocks:
        x = s["x"][r].double()
        d = torch.softmax(torch.mm(x, w.t()).div_(tau), dim=1).neg_()
        d[torch.arange(d.shape[0], device="cuda"), s["labels"][r].clamp(min=0)] += 1.0
        d *= g[r, None] / tau
        out["dx"][r] = torch.mm(d, w)
        if case["grad"] == "xw":
            out["dw"].addmm_(d.t(), x)
    return out
