"""Operators of decoder blocks and of the scoring objective, as timed cases.

Each case is one pass through an operator: rotary positions of any layout
(``rope_positions``), a product with bias, activation and residual in its
epilogue and its backward (``gemm_act``, ``gemm_act_bwd``, ``act_bwd``), the
largest logits of a row (``top_logits``) and the distillation loss against a
teacher's list of them (``distill_loss``). ``own`` selects the framework's
kernels; otherwise the same formulas run in elementary torch operations, in
float32 (angles and probabilities near one in float64), rounded once.

The geometries are those of the repository's configurations (135M: hidden 576;
0.5B: 896; 3B: 2048; 7B: 3584) and, in the drawn cases, generic ones.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
SQRT_2_OVER_PI = math.sqrt(2.0 / math.pi)


def listed() -> list[dict]:
    return [
        # One decoding step of a 7B model: 8 sequences' newest tokens, at far
        # positions of a long context, query and key heads in the fused rows.
        dict(name="rope-decode-7b", kind="rope", tokens=8, heads=32, extra=4, d=128, rotary=128, pairing="half",
             dtype="bf16", scale=1.0, backward=False, start=-1),
        # The gradient of a rotation that covers half of each head and pairs
        # neighbours, sequences that are no whole tiles, float16.
        dict(name="rope-bwd-partial", kind="rope", tokens=4000, heads=16, extra=2, d=64, rotary=32,
             pairing="interleaved", dtype="f16", scale=1.0, backward=True, start=0),
        # The headline workload's prompts (8 x 2048 tokens of a 7B block), with
        # the magnitude correction of a scaled context.
        dict(name="rope-7b", kind="rope", tokens=16384, heads=32, extra=4, d=128, rotary=128, pairing="half",
             dtype="bf16", scale=1.1386, backward=False, start=30000),
        # The up product of a 135M ungated MLP for the newest tokens of a batch.
        dict(name="act-64x1536x576", kind="act", m=64, n=1536, k=576, f="gelu_tanh", bias=True, resid=False, save=False),
        # The up product of a 7B ungated MLP over the headline's tokens, saving
        # what the backward reads.
        dict(name="act-7b", kind="act", m=16384, n=18944, k=3584, f="silu", bias=True, resid=False, save=True),
        # A residual branch of one product with its activation last, 0.5B, a row
        # count of no whole tiles.
        dict(name="act-resid-0.5b", kind="act", m=4005, n=896, k=896, f="relu2", bias=True, resid=True, save=True),
        # That branch's backward, to the pre-activation and bias gradients.
        dict(name="act-last-bwd-0.5b", kind="act_last_bwd", m=4005, n=896, f="relu2", bias=True),
        # The backward of a 3B ungated MLP's hidden layer.
        dict(name="act-bwd-3b", kind="act_bwd", m=4096, n=11008, k=2048, f="gelu", bias=True),
        # The teacher's list for a 0.5B scoring batch (4 x 511 positions, full vocabulary).
        dict(name="top-64", kind="top", rows=2044, vocab=151936, top=64, dtype="bf16", temperature=1.0),
        # The likeliest tokens of a few decoding rows, float32, an odd vocabulary.
        dict(name="top-20-decode", kind="top", rows=8, vocab=50257, top=20, dtype="f32", temperature=0.7),
        # The scoring batch's loss and gradient against that list, the rest of
        # the vocabulary as one outcome.
        dict(name="distill-64", kind="distill", rows=2044, vocab=151936, top=64, dtype="bf16", temperature=1.0,
             tail=True, ragged=False, grad=True),
        # A smaller vocabulary in float32 at a higher temperature, the
        # teacher's list taken as its whole distribution.
        dict(name="distill-f32", kind="distill", rows=1022, vocab=49152, top=16, dtype="f32", temperature=2.0,
             tail=False, ragged=True, grad=True),
    ]


# ------------------------------------------------------------------- drawn --

def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


FUNCTIONS = ("relu", "relu2", "silu", "gelu", "gelu_tanh")


def draw(rng) -> dict:
    kind = rng.choice(("rope", "rope", "act", "act_last_bwd", "act_bwd", "top", "top", "distill", "distill"))
    if kind == "rope":
        d = rng.choice((64, 64, 80, 96, 128, 128, 256))
        heads, tokens = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
        tokens = max(1, min(tokens, 16384 * 32 * 128 // (heads * d)))
        rotary = d if rng.random() < 0.5 else 2 * max(1, int(d * rng.choice((0.25, 0.4, 0.5, 0.75))) // 2)
        return dict(kind=kind, tokens=tokens, heads=heads, extra=rng.choice((0, 1, 2, 8)), d=d, rotary=rotary,
                    pairing=rng.choice(("half", "interleaved")), dtype=rng.choice(("bf16", "bf16", "f16", "f32")),
                    scale=rng.choice((1.0, 1.0, round(rng.uniform(1.0, 1.5), 4))), backward=rng.random() < 0.5,
                    start=-1 if rng.random() < 0.3 else _log_int(rng, 1, 1000000))
    if kind in ("act", "act_last_bwd", "act_bwd"):
        n, k = 8 * _log_int(rng, 8, 2368), 64 * _log_int(rng, 1, 64)
        m = min(_log_int(rng, 1, 16384), max(1, int(1.1e12 / (n * k))))
        c = dict(kind=kind, m=m, n=n, f=rng.choice(FUNCTIONS), bias=rng.random() < 0.6)
        if kind == "act":
            c.update(resid=rng.random() < 0.3, save=rng.random() < 0.5)
        if kind != "act_last_bwd":
            c.update(k=k)
        return c
    vocab = _log_int(rng, 500, 200000)
    rows = min(_log_int(rng, 1, 4096), 2044 * 151936 // vocab)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    c = dict(kind=kind, rows=rows, vocab=vocab, top=min(vocab, _log_int(rng, 1, 512)), dtype=dtype,
             temperature=rng.choice((1.0, 1.0, round(rng.uniform(0.5, 4.0), 3))))
    if dtype == "f32":
        c["rows"] = max(1, rows // 2)
    if kind == "distill":
        c.update(tail=rng.random() < 0.6, ragged=rng.random() < 0.4, grad=rng.random() < 0.8)
    return c


# ------------------------------------------------------------------ inputs --

class _Source:
    """Random inputs made on the device from one seed."""

    def __init__(self, seed: int) -> None:
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device=DEV) * std

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV, dtype=torch.int32)


def _frequencies(c) -> torch.Tensor:
    """theta^(-2i/r), float64."""
    i = torch.arange(c["rotary"] // 2, dtype=torch.float64, device=DEV)
    return 1e6 ** (-2.0 * i / c["rotary"])


def _logits(src, rows, vocab):
    """Logits as a language model's head gives them: near normal, a few
    candidates of each row far above the rest."""
    z = src.normal(rows, vocab, std=2.0)
    z += torch.rand(rows, vocab, generator=src.g, device=DEV).pow_(256).mul_(12.0)
    return z


def prepare(case, seed):
    c, kind, src = case, case["kind"], _Source(seed)
    s = dict(c)
    if kind == "rope":
        T, d = c["tokens"], c["d"]
        s["x"] = src.normal(T, (c["heads"] + c["extra"]) * d).to(DTYPES[c["dtype"]])
        s["out"] = torch.zeros_like(s["x"])
        s["freq"] = _frequencies(c)
        # a batch's newest tokens, each at a position of its own, or a prompt's consecutive ones
        s["pos"] = (src.ints(0, 1 << 20, T) if c["start"] < 0 else
                    torch.arange(c["start"], c["start"] + T, device=DEV, dtype=torch.int32))
        return s
    if kind == "act":
        m, n, k = c["m"], c["n"], c["k"]
        s["x"] = src.normal(m, k).to(torch.bfloat16)
        s["w"] = src.normal(n, k, std=1.5 * k ** -0.5).to(torch.bfloat16)
        s["b"] = src.normal(n, std=0.1) if c["bias"] else None
        s["r"] = src.normal(m, n) if c["resid"] else None
        s["out"] = torch.empty(m, n, dtype=torch.float32 if c["resid"] else torch.bfloat16, device=DEV)
        s["pre"] = torch.empty(m, n, dtype=torch.bfloat16, device=DEV) if c["save"] else None
        return s
    if kind in ("act_last_bwd", "act_bwd"):
        m, n = c["m"], c["n"]
        if kind == "act_bwd":
            s["dd"] = src.normal(m, c["k"], std=0.1).to(torch.bfloat16)
            s["w"] = src.normal(c["k"], n, std=c["k"] ** -0.5).to(torch.bfloat16)
        else:
            s["dout"] = src.normal(m, n, std=0.1)
        s["pre"] = src.normal(m, n, std=1.5).to(torch.bfloat16)
        s["dpre"] = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
        s["dbias"] = torch.empty(n, dtype=torch.float32, device=DEV) if c["bias"] else None
        return s
    rows, vocab, top = c["rows"], c["vocab"], c["top"]
    z = _logits(src, rows, vocab)
    if kind == "top":
        s["z"] = z.to(DTYPES[c["dtype"]])
        s["values"] = torch.empty(rows, top, dtype=torch.float32, device=DEV)
        s["ids"] = torch.empty(rows, top, dtype=torch.int32, device=DEV)
        s["lse"] = torch.empty(rows, dtype=torch.float32, device=DEV)
        return s
    # the student is the teacher with noise, as a quantized model is
    teacher = z.clone()
    z += src.normal(rows, vocab, std=0.3)
    s["z"] = z.to(DTYPES[c["dtype"]])
    s["t"], ids = teacher.topk(top, dim=1)
    s["ids"] = ids.to(torch.int32)
    s["lse"] = torch.logsumexp(teacher.div_(c["temperature"]), 1) if c["tail"] else None
    if c["ragged"]:
        # lists of any length, down to none (a position without a teacher)
        length = src.ints(0, top + 1, rows, 1)
        s["ids"] = torch.where(torch.arange(top, device=DEV)[None] < length, s["ids"], -1)
    # the mean over rows; in float16 a scaled sum, which keeps the gradient in its normal range
    s["weight"] = 1024.0 if c["dtype"] == "f16" else 1.0 / rows
    s["row_loss"] = torch.empty(rows, dtype=torch.float32, device=DEV)
    s["loss"] = torch.empty(1, dtype=torch.float32, device=DEV)
    s["dz"] = torch.empty_like(s["z"]) if c["grad"] else None
    return s


# --------------------------------------------------------------------- run --

def run(state):
    kind = state["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


def _rope_own(s):
    from mround_amd import kernels as K

    K.rope_positions(s["x"], s["pos"], s["freq"], n_heads=s["heads"], head_dim=s["d"], pairing=s["pairing"],
                     scale=s["scale"], backward=s["backward"], out=s["out"])
    return s["out"][:, :s["heads"] * s["d"]]


def _act_own(s):
    from mround_amd import kernels as K

    K.gemm_act(s["x"], s["w"], s["out"], act=s["f"], bias=s["b"], pre=s["pre"], resid=s["r"])
    return {"out": s["out"]} if s["pre"] is None else {"out": s["out"], "pre": s["pre"]}


def _act_last_bwd_own(s):
    from mround_amd import kernels as K

    K.act_bwd(s["dout"], s["pre"], s["dpre"], act=s["f"], dbias=s["dbias"])
    return {"dpre": s["dpre"]} if s["dbias"] is None else {"dpre": s["dpre"], "dbias": s["dbias"]}


def _act_bwd_own(s):
    from mround_amd import kernels as K

    K.gemm_act_bwd(s["dd"], s["w"], s["pre"], s["dpre"], act=s["f"], dbias=s["dbias"])
    return {"dpre": s["dpre"]} if s["dbias"] is None else {"dpre": s["dpre"], "dbias": s["dbias"]}


def _top_own(s):
    from mround_amd import kernels as K

    K.top_logits(s["z"], V=s["vocab"], values=s["values"], ids=s["ids"], lse=s["lse"], temperature=s["temperature"])
    return {"values": s["values"], "ids": s["ids"], "lse": s["lse"]}


def _distill_own(s):
    from mround_amd import kernels as K

    K.distill_loss(s["z"], s["t"], s["ids"], V=s["vocab"], scale=s["weight"], row_loss=s["row_loss"],
                   lse=s["lse"], temperature=s["temperature"], loss_out=s["loss"], dlogits=s["dz"])
    out = {"loss": s["loss"], "row_loss": s["row_loss"]}
    return out if s["dz"] is None else dict(out, dlogits=s["dz"])


_OWN = {"rope": _rope_own, "act": _act_own, "act_last_bwd": _act_last_bwd_own, "act_bwd": _act_bwd_own,
        "top": _top_own, "distill": _distill_own}


# ------------------------------------------------------------- plain forms --

def _rope_plain(s):
    T, d, r = s["tokens"], s["d"], s["rotary"]
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = angle.cos().float()[:, None] * s["scale"], angle.sin().float()[:, None] * s["scale"]
    if s["backward"]:
        sin = -sin
    x = s["x"][:, :s["heads"] * d].float().view(T, s["heads"], d)
    rot = x[..., :r]
    if s["pairing"] == "half":
        a, b = rot[..., :r // 2], rot[..., r // 2:]
        new = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = rot[..., 0::2], rot[..., 1::2]
        new = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([new, x[..., r:]], -1).view(T, -1).to(s["x"].dtype)


def _f(x, name):
    if name == "relu":
        return x.clamp_min(0)
    if name == "relu2":
        return x.clamp_min(0).square()
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "gelu":
        return 0.5 * x * torch.erfc(x * -math.sqrt(0.5))
    return 0.5 * x * (1 + torch.tanh(SQRT_2_OVER_PI * (x + 0.044715 * x * x * x)))


def _df(x, name):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "relu2":
        return 2 * x.clamp_min(0)
    if name == "silu":
        g = torch.sigmoid(x)
        return g * (1 + x * (1 - g))
    if name == "gelu":
        return 0.5 * torch.erfc(x * -math.sqrt(0.5)) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    t = torch.tanh(SQRT_2_OVER_PI * (x + 0.044715 * x * x * x))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * SQRT_2_OVER_PI * (1 + 3 * 0.044715 * x * x)


def _act_plain(s):
    x = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        x = x + s["b"]
    y = _f(x, s["f"])
    if s["r"] is not None:
        y = y + s["r"]
    out = {"out": y.to(s["out"].dtype)}
    return out if s["pre"] is None else dict(out, pre=x.to(torch.bfloat16))


def _act_bwd_plain(s):
    dout = s["dout"] if s["kind"] == "act_last_bwd" else s["dd"].float() @ s["w"].float()
    d = dout * _df(s["pre"].float(), s["f"])
    out = {"dpre": d.to(torch.bfloat16)}
    return out if s["dbias"] is None else dict(out, dbias=d.sum(0))


def _top_plain(s):
    z = s["z"].float()
    # the float's bits as an integer of the same order, then the lower index first
    bits = (z + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key |= 0x7FFFFFFF - torch.arange(s["vocab"], device=DEV)
    ids = 0x7FFFFFFF - (key.topk(s["top"], dim=1).values & 0x7FFFFFFF)
    u = z / s["temperature"]
    m = u.amax(1, keepdim=True)
    lse = m[:, 0] + torch.log(torch.exp(u - m).sum(1))
    return {"values": z.gather(1, ids), "ids": ids.to(torch.int32), "lse": lse}


def _distill_plain(s):
    listed_, rows, dt = s["ids"] >= 0, s["z"].shape[0], s["z"].dtype
    ids = s["ids"].long().clamp_min(0)
    u = s["z"].float() / s["temperature"]
    m = u.amax(1, keepdim=True)
    e = torch.exp(u - m)
    on = torch.zeros_like(e, dtype=torch.bool).scatter_(1, torch.where(listed_, ids, s["ids"][:, :1].long().clamp_min(0)),
                                                        listed_[:, :1].expand_as(listed_))
    # the loss is a small difference of logarithms: sums and logarithms in float64
    rest = (e * ~on).sum(1, keepdim=True, dtype=torch.float64)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    log_total = m + torch.log(total)
    t = s["t"].double() / s["temperature"]
    if s["lse"] is None:
        t = torch.where(listed_, t, -math.inf)
        log_q = t - torch.logsumexp(t, 1, keepdim=True)
    else:
        log_q = t - s["lse"][:, None].double()
    q = torch.where(listed_, torch.exp(log_q), 0.0)
    q_sum = q.sum(1, keepdim=True)
    q_rest = (1 - q_sum).clamp_min(0) if s["lse"] is not None else torch.zeros_like(rest)
    q_rest = torch.where(rest > 0, q_rest, 0.0)
    q_total = q_sum + q_rest if s["lse"] is not None else torch.ones_like(rest)
    log_p = u.gather(1, ids) - log_total
    row = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1, keepdim=True)
    log_rest = torch.log(rest) - torch.log(total)
    row += torch.where(q_rest > 0, q_rest * (torch.log(q_rest) - log_rest), 0.0)
    any_listed = listed_.any(1, keepdim=True)
    row = torch.where(any_listed, row, 0.0)[:, 0]
    out = {"loss": (row.sum() * s["weight"]).float().view(1), "row_loss": row.float()}
    if s["dz"] is None:
        return out
    p = e / total.float()
    off = q_total - torch.where(q_rest > 0, q_rest * total / rest, 0.0)
    g = p * torch.where(on, q_total.float(), off.float())
    g.scatter_add_(1, ids, -q.float())
    g *= s["weight"] / s["temperature"]
    return dict(out, dlogits=torch.where(any_listed, g, 0.0).to(dt))


_PLAIN = {"rope": _rope_plain, "act": _act_plain, "act_last_bwd": _act_bwd_plain, "act_bwd": _act_bwd_plain,
          "top": _top_plain, "distill": _distill_plain}


# ---------------------------------------------------- definitions in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _rope_exact, "act": _act_exact, "act_last_bwd": _act_bwd_exact, "act_bwd": _act_bwd_exact,
            "top": _top_exact, "distill": _distill_exact}[case["kind"]](s)


def _rope_exact(s):
    """As a product of complex numbers."""
    T, d, r = s["tokens"], s["d"], s["rotary"]
    turn = torch.polar(torch.full_like(s["freq"], s["scale"]).expand(T, -1).contiguous(),
                       s["pos"].double().outer(s["freq"]) * (-1.0 if s["backward"] else 1.0))
    x = s["x"][:, :s["heads"] * d].double().reshape(T, s["heads"], d).clone()
    pairs = (x[..., :r].reshape(T, s["heads"], 2, r // 2).transpose(2, 3) if s["pairing"] == "half"
             else x[..., :r].reshape(T, s["heads"], r // 2, 2))
    new = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
    x[..., :r] = (new.transpose(2, 3) if s["pairing"] == "half" else new).reshape(T, s["heads"], r)
    return x.view(T, -1)


def _with_derivative(x, name):
    """f(x) and f'(x) in float64, by torch's own functions and autograd, a slice of rows at a time."""
    F = torch.nn.functional
    f = {"relu": F.relu, "relu2": lambda v: F.relu(v).square(), "silu": F.silu, "gelu": F.gelu,
         "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[name]
    ys, ds = [], []
    for v in x.split(1024):
        v = v.detach().requires_grad_()
        y = f(v)
        ds.append(torch.autograd.grad(y.sum(), v)[0])
        ys.append(y.detach())
    return torch.cat(ys), torch.cat(ds)


def _product(a, b):
    return torch.cat([part.double() @ b for part in a.split(2048)])


def _act_exact(s):
    x = _product(s["x"], s["w"].double().t())
    if s["b"] is not None:
        x += s["b"].double()
    y = _with_derivative(x, s["f"])[0]
    if s["r"] is not None:
        y += s["r"].double()
    return {"out": y} if s["pre"] is None else {"out": y, "pre": x}


def _act_bwd_exact(s):
    dout = s["dout"].double() if s["kind"] == "act_last_bwd" else _product(s["dd"], s["w"].double())
    d = dout * _with_derivative(s["pre"].double(), s["f"])[1]
    return {"dpre": d} if s["dbias"] is None else {"dpre": d, "dbias": d.sum(0)}


def _top_exact(s):
    values, ids, lse = [], [], []
    for z in s["z"].split(256):
        z = z.double()
        v, i = torch.sort(z, dim=1, descending=True, stable=True)
        values.append(v[:, :s["top"]].clone())
        ids.append(i[:, :s["top"]].to(torch.int32))
        lse.append(torch.logsumexp(z / s["temperature"], 1))
    return {"values": torch.cat(values), "ids": torch.cat(ids), "lse": torch.cat(lse)}


def _distill_exact(s):
    """The divergence between distributions over the listed outcomes (and the
    rest as one), its gradient by autograd, a slice of rows at a time."""
    losses, grads = [], []
    for r0 in range(0, s["rows"], 256):
        r = slice(r0, min(r0 + 256, s["rows"]))
        z = s["z"][r].double().requires_grad_()
        ids = s["ids"][r].long()
        there = ids >= 0
        some = there.any(1)
        log_p = torch.log_softmax(z / s["temperature"], 1)
        t = s["t"][r].double() / s["temperature"]
        listed_ = torch.zeros(z.shape[0], s["vocab"] + 1, dtype=torch.bool, device=DEV)
        listed_.scatter_(1, torch.where(there, ids, s["vocab"]), True)
        if s["lse"] is None:
            log_q = torch.log_softmax(torch.where(there, t, -1e300), 1)
        else:
            log_q = t - s["lse"][r].double()[:, None]
        q = torch.where(there, log_q.exp(), 0.0)
        picked = log_p.gather(1, ids.clamp_min(0))
        loss = (torch.special.xlogy(q, q) - q * picked).sum(1)
        if s["lse"] is not None:
            q_rest = (1 - q.sum(1)).clamp_min(0)
            has_rest = (~listed_[:, :s["vocab"]]).any(1)
            unlisted = log_p.masked_fill(listed_[:, :s["vocab"]], -1e300)
            log_rest = torch.logsumexp(unlisted, 1)
            loss = loss + torch.where(has_rest, torch.special.xlogy(q_rest, q_rest) - q_rest * log_rest, 0.0)
        loss = torch.where(some, loss, 0.0)
        if s["dz"] is not None:
            grads.append(torch.autograd.grad(loss.sum() * s["weight"], z)[0])
        losses.append(loss.detach())
    row = torch.cat(losses)
    out = {"loss": (row.sum() * s["weight"]).view(1), "row_loss": row}
    return out if s["dz"] is None else dict(out, dlogits=torch.cat(grads))


# -------------------------------------------------------------------- work --

def work(case):
    c, kind = case, case["kind"]
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if kind == "rope":
        n, e = c["tokens"] * c["heads"], size[c["dtype"]]
        return {"bytes": 2 * n * c["d"] * e + 4 * c["tokens"] + 4 * c["rotary"], "flops": 3 * n * c["rotary"]}
    if kind in ("act", "act_last_bwd", "act_bwd"):
        m, n, k = c["m"], c["n"], c.get("k", 0)
        b = 2 * (m * k + n * k) + (4 * n if c["bias"] else 0)
        if kind == "act":
            b += m * n * ((8 if c["resid"] else 2) + (2 if c["save"] else 0))
        else:
            b += m * n * (4 if k else 8)
        return {"bytes": b, "flops": 2 * m * n * k if k else 4 * m * n}
    rows, V, k, e = c["rows"], c["vocab"], c["top"], size[c["dtype"]]
    if kind == "top":
        return {"bytes": rows * (V * e + 8 * k + 4), "flops": 4 * rows * V}
    b = rows * (V * e * (2 if c["grad"] else 1) + 8 * k + 4 + (4 if c["tail"] else 0))
    return {"bytes": b, "flops": (7 if c["grad"] else 4) * rows * V}
