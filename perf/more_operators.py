"""Operators of decoder blocks with experts and with norms behind their branches, as timed cases.

Each case is one pass through an operator: the choice of each token's experts
and the order of the tokens by expert (``route_experts``, ``route_experts_bwd``),
products grouped by expert with ragged row counts (``gemm_experts``,
``gemm_experts_swiglu``, ``gemm_experts_swiglu_bwd``), rows dealt to their
experts and summed back (``spread_experts``, ``combine_experts``), and a branch's
end with the next norm (``norm_residual``, ``norm_residual_bwd``). ``own``
selects the framework's kernels; otherwise the same formulas run in elementary
torch operations, in float32, rounded once.

Hidden sizes are those of the repository's configurations (0.5B: 896; 3B: 2048;
7B: 3584), the experts' numbers and widths generic; drawn cases are generic.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
PRODUCTS = ("swiglu", "down", "swiglu_bwd", "dx", "dw")


def listed() -> list[dict]:
    return [
        # One decoding step: 8 sequences' newest tokens choose 8 of 64 experts.
        dict(name="route-decode", kind="route", tokens=8, experts=64, top=8, dtype="f32", normalize=False),
        # The headline's prompts (8 x 2048 tokens) over many small experts.
        dict(name="route-prompts", kind="route", tokens=16384, experts=128, top=8, dtype="bf16", normalize=True),
        # The router's gradient for a batch of no whole tiles.
        dict(name="route-bwd", kind="route_bwd", tokens=4005, experts=60, top=4, dtype="f32", normalize=False),
        # Those 8 tokens' gate/up products: one or two rows an expert, the time
        # is that of reading the chosen experts' weights.
        dict(name="experts-decode", kind="swiglu", tokens=8, experts=64, top=8, h=2048, inter=768, save=False),
        # The gate/up products of the prompts, keeping what the backward reads.
        dict(name="experts-prompts", kind="swiglu", tokens=16384, experts=128, top=8, h=2048, inter=768, save=True),
        # The down products of a few wide experts, 7B hidden size.
        dict(name="experts-down", kind="down", tokens=4005, experts=8, top=2, h=3584, inter=4864),
        # The backward through the down products and the SwiGLU.
        dict(name="experts-swiglu-bwd", kind="swiglu_bwd", tokens=4096, experts=60, top=4, h=2048, inter=1408),
        # The experts' weight gradients, each over its own number of rows.
        dict(name="experts-dw", kind="dw", tokens=8191, experts=16, top=4, h=2048, inter=1408),
        # The prompts' rows summed back, weighted, onto the residual stream.
        dict(name="combine-prompts", kind="combine", tokens=16384, experts=128, top=8, h=2048),
        # Its backward for two experts a token, to the rows' and the weights' gradients.
        dict(name="combine-bwd", kind="combine_bwd", tokens=4005, experts=8, top=2, h=3584, dtype="f32"),
        # The end of a 3B block's branch: norm, gate and scale onto the stream, and the next norm.
        dict(name="norm-3b", kind="norm", rows=4005, h=2048, post=True, gate="column", pre=True, act="bf16",
             stream="f32", scale=0.7),
        # Its backward at the headline's size, with the norms' and the gate's gradients, a gate for each sequence.
        dict(name="norm-bwd-7b", kind="norm_bwd", rows=16384, h=3584, post=True, gate="sequence", seq=2048, pre=True,
             act="bf16", stream="f32", scale=1.0),
    ]


# ------------------------------------------------------------------- drawn --

def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(("route", "route_bwd") + PRODUCTS + PRODUCTS[:1] + ("combine", "combine_bwd", "norm", "norm_bwd"))
    if kind in ("norm", "norm_bwd"):
        h = _log_int(rng, 64, 8192)
        if rng.random() < 0.8:
            h = 8 * (h // 8)
        rows = min(_log_int(rng, 1, 32768), 16384 * 3584 // h)
        act = rng.choice(("bf16", "bf16", "f16", "f32"))
        gate = rng.choice(("", "column", "sequence"))
        c = dict(kind=kind, rows=rows, h=h, post=rng.random() < 0.7, gate=gate, pre=rng.random() < 0.8, act=act,
                 stream=rng.choice(("f32", "f32", act)), scale=rng.choice((1.0, round(rng.uniform(0.2, 2.0), 3))))
        if gate == "sequence":
            c["seq"] = rng.choice((1, 100, 512, 2048))
        return c
    experts = _log_int(rng, 2, 256)
    top = min(experts, rng.choice((1, 2, 4, 6, 8)))
    tokens = _log_int(rng, 1, 16384)
    if kind in ("route", "route_bwd"):
        return dict(kind=kind, tokens=tokens, experts=experts, top=top, dtype=rng.choice(("f32", "bf16", "f16")),
                    normalize=rng.random() < 0.5)
    h = 64 * _log_int(rng, 4, 64)
    if kind in ("combine", "combine_bwd"):
        tokens = min(tokens, 16384 * 8 * 2048 // (top * h))
        c = dict(kind=kind, tokens=tokens, experts=experts, top=top, h=h)
        return dict(c, dtype=rng.choice(("f32", "bf16"))) if kind == "combine_bwd" else c
    inter = 64 * _log_int(rng, 2, 64)
    experts = max(2, min(experts, 128 * 2048 * 768 // (h * inter)))
    top = min(top, experts)
    tokens = max(1, min(tokens, 16384 * 8 * 2048 * 768 // (top * h * inter)))
    c = dict(kind=kind, tokens=tokens, experts=experts, top=top, h=h, inter=inter)
    return dict(c, save=rng.random() < 0.5) if kind == "swiglu" else c


# ------------------------------------------------------------------ inputs --

class _Source:
    """Random inputs made on the device from one seed."""

    def __init__(self, seed: int) -> None:
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device=DEV) * std

    def logits(self, tokens, experts):
        """A router's logits: some experts are liked better than others by all tokens."""
        return self.normal(tokens, experts) + self.normal(1, experts, std=0.7)


def _routing(s, src, c):
    """Each token's experts, and the order of its copies by expert."""
    T, E, k = c["tokens"], c["experts"], c["top"]
    ids = src.logits(T, E).topk(k, dim=1).indices
    order = ids.flatten().sort(stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(T * k, device=DEV)
    counts = torch.bincount(ids.flatten(), minlength=E)
    s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    s["slots"] = slots.view(T, k).to(torch.int32)
    s["rows"] = (order // k).to(torch.int32)
    s["counts"] = counts.tolist()  # for the plain form, whose loop over experts runs on the host
    return T * k


def prepare(case, seed):
    c, kind, src = case, case["kind"], _Source(seed)
    s = dict(c)
    empty = lambda *shape, dt=torch.float32: torch.empty(*shape, dtype=dt, device=DEV)
    zeros = lambda *shape, dt=torch.int32: torch.zeros(*shape, dtype=dt, device=DEV)
    bf = torch.bfloat16
    if kind in ("route", "route_bwd"):
        T, E, k = c["tokens"], c["experts"], c["top"]
        s["z"] = src.logits(T, E).to(DTYPES[c["dtype"]])
        if kind == "route":
            s.update(weights=empty(T, k), ids=zeros(T, k), offsets=zeros(E + 1), slots=zeros(T, k), rows=zeros(T * k))
        else:
            s["ids"] = _ordered(s["z"])[:, :k].to(torch.int32).contiguous()
            s["dw"] = src.normal(T, k)
            s["dz"] = torch.empty_like(s["z"])
        return s
    if kind in PRODUCTS:
        R, E, h, i = _routing(s, src, c), c["experts"], c["h"], c["inter"]
        if kind == "swiglu":
            s["x"] = src.normal(c["tokens"], h).to(bf)
            s["w"] = src.normal(E, 2 * i, h, std=h ** -0.5).to(bf)
            s["act"] = empty(R, i, dt=bf)
            s["gu"] = empty(R, 2 * i, dt=bf) if c["save"] else None
        elif kind == "down":
            s["a"] = src.normal(R, i, std=0.5).to(bf)
            s["w"] = src.normal(E, h, i, std=i ** -0.5).to(bf)
            s["y"] = empty(R, h, dt=bf)
        elif kind == "swiglu_bwd":
            s["dy"] = src.normal(R, h, std=0.1).to(bf)
            s["w"] = src.normal(E, h, i, std=i ** -0.5).to(bf)
            s["gu"] = src.normal(R, 2 * i).to(bf)
            s["dgu"] = empty(R, 2 * i, dt=bf)
        elif kind == "dx":
            s["dgu"] = src.normal(R, 2 * i, std=0.1).to(bf)
            s["w"] = src.normal(E, 2 * i, h, std=h ** -0.5).to(bf)
            s["dx"] = empty(R, h, dt=bf)
        else:
            s["dy"] = src.normal(R, h, std=0.1).to(bf)
            s["a"] = src.normal(R, i, std=0.5).to(bf)
            s["dweight"] = empty(E, h, i)
        return s
    if kind in ("combine", "combine_bwd"):
        R, T, k, h = _routing(s, src, c), c["tokens"], c["top"], c["h"]
        s["y"] = src.normal(R, h).to(bf)
        s["weights"] = torch.softmax(src.normal(T, k), 1)
        if kind == "combine":
            s["resid"] = src.normal(T, h, std=4.0)
            s["out"] = empty(T, h)
        else:
            s["dout"] = src.normal(T, h, std=0.1).to(DTYPES[c["dtype"]])
            s["dy"], s["dweights"] = empty(R, h, dt=bf), empty(T, k)
        return s
    T, h, act, stream = c["rows"], c["h"], DTYPES[c["act"]], DTYPES[c["stream"]]
    s["y"] = src.normal(T, h, std=0.5).to(act)
    s["wpost"] = 1 + src.normal(h, std=0.2) if c["post"] else None
    s["wpre"] = 1 + src.normal(h, std=0.2) if c["pre"] else None
    s["gate_rows"] = c["seq"] if c["gate"] == "sequence" else max(T, 1)
    s["gate"] = src.normal(-(-T // s["gate_rows"]), h, std=0.5) if c["gate"] else None
    s["eps"] = 1e-6
    # the stream's magnitudes differ from column to column, as a model's do
    wide = torch.exp(src.normal(h))
    if kind == "norm":
        s["resid"] = (src.normal(T, h) * wide).to(stream)
        s["out"] = torch.empty_like(s["resid"])
        s["x"] = torch.empty_like(s["y"]) if c["pre"] else None
        return s
    s["out"] = (src.normal(T, h) * wide).to(stream)
    s["dx"] = src.normal(T, h, std=0.1).to(act) if c["pre"] else None
    s["dout"] = src.normal(T, h, std=0.1).to(stream)
    s["dy"], s["dresid"] = torch.empty_like(s["y"]), torch.empty_like(s["out"])
    s["dwpost"] = empty(h) if c["post"] else None
    s["dwpre"] = empty(h) if c["pre"] else None
    s["dgate"] = torch.empty_like(s["gate"]) if c["gate"] else None
    return s


# --------------------------------------------------------------------- run --

def run(state):
    kind = state["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


def _there(**outputs):
    return {n: t for n, t in outputs.items() if t is not None}


def _route_own(s):
    from mround_amd import kernels as K

    K.route_experts(s["z"], weights=s["weights"], ids=s["ids"], offsets=s["offsets"], slots=s["slots"],
                    rows=s["rows"], normalize=s["normalize"])
    return {n: s[n] for n in ("weights", "ids", "offsets", "slots", "rows")}


def _route_bwd_own(s):
    from mround_amd import kernels as K

    K.route_experts_bwd(s["dw"], s["z"], s["ids"], s["dz"], normalize=s["normalize"])
    return s["dz"]


def _swiglu_own(s):
    from mround_amd import kernels as K

    K.gemm_experts_swiglu(s["x"], s["w"], s["act"], s["gu"], offsets=s["offsets"], rows=s["rows"])
    return _there(act=s["act"], gu=s["gu"])


def _down_own(s):
    from mround_amd import kernels as K

    K.gemm_experts("nt", s["a"], s["w"], s["y"], offsets=s["offsets"])
    return s["y"]


def _swiglu_bwd_own(s):
    from mround_amd import kernels as K

    K.gemm_experts_swiglu_bwd(s["dy"], s["w"], s["gu"], s["dgu"], offsets=s["offsets"])
    return s["dgu"]


def _dx_own(s):
    from mround_amd import kernels as K

    K.gemm_experts("nn", s["dgu"], s["w"], s["dx"], offsets=s["offsets"])
    return s["dx"]


def _dw_own(s):
    from mround_amd import kernels as K

    K.gemm_experts("tn", s["dy"], s["a"], s["dweight"], offsets=s["offsets"])
    return s["dweight"]


def _combine_own(s):
    from mround_amd import kernels as K

    K.combine_experts(s["y"], s["slots"], s["out"], weights=s["weights"], resid=s["resid"])
    return s["out"]


def _combine_bwd_own(s):
    from mround_amd import kernels as K

    K.spread_experts(s["dout"], s["slots"], s["dy"], weights=s["weights"], y=s["y"], dweights=s["dweights"])
    return {"dy": s["dy"], "dweights": s["dweights"]}


def _norm_own(s):
    from mround_amd import kernels as K

    K.norm_residual(s["y"], s["resid"], s["out"], eps=s["eps"], post=s["wpost"], gate=s["gate"],
                    gate_rows=s["gate_rows"], scale=s["scale"], pre=s["wpre"], normed=s["x"])
    return _there(out=s["out"], x=s["x"])


def _norm_bwd_own(s):
    from mround_amd import kernels as K

    K.norm_residual_bwd(s["dx"], s["dout"], s["y"], s["out"], s["dy"], s["dresid"], eps=s["eps"], post=s["wpost"],
                        gate=s["gate"], gate_rows=s["gate_rows"], scale=s["scale"], pre=s["wpre"],
                        dpost=s["dwpost"], dgate=s["dgate"], dpre=s["dwpre"])
    return _there(dy=s["dy"], dresid=s["dresid"], dpost=s["dwpost"], dgate=s["dgate"], dpre=s["dwpre"])


_OWN = {"route": _route_own, "route_bwd": _route_bwd_own, "swiglu": _swiglu_own, "down": _down_own,
        "swiglu_bwd": _swiglu_bwd_own, "dx": _dx_own, "dw": _dw_own, "combine": _combine_own,
        "combine_bwd": _combine_bwd_own, "norm": _norm_own, "norm_bwd": _norm_bwd_own}


# ------------------------------------------------------------- plain forms --

def _ordered(z):
    """Indices in descending order of the values, ties to the lower index: the
    float's bits as an integer of the same order, then the index."""
    bits = (z.float() + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key |= 0x7FFFFFFF - torch.arange(z.shape[1], device=DEV)
    return 0x7FFFFFFF - (key.sort(dim=1, descending=True).values & 0x7FFFFFFF)


def _probabilities(z):
    e = torch.exp(z - z.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _route_plain(s):
    E, k = s["experts"], s["top"]
    z = s["z"].float()
    ids = _ordered(z)[:, :k]
    w = _probabilities(z.gather(1, ids)) if s["normalize"] else _probabilities(z).gather(1, ids)
    flat = ids.flatten()
    order = (flat * flat.numel() + torch.arange(flat.numel(), device=DEV)).sort().indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(flat.numel(), device=DEV)
    counts = (flat[:, None] == torch.arange(E, device=DEV)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    i32 = torch.int32
    return {"weights": w, "ids": ids.to(i32), "offsets": offsets.to(i32), "slots": slots.view(ids.shape).to(i32),
            "rows": (order // k).to(i32)}


def _route_bwd_plain(s):
    z, ids, dw = s["z"].float(), s["ids"].long(), s["dw"]
    if s["normalize"]:
        w = _probabilities(z.gather(1, ids))
        return torch.zeros_like(z).scatter_(1, ids, w * (dw - (w * dw).sum(1, keepdim=True))).to(s["z"].dtype)
    p = _probabilities(z)
    dp = torch.zeros_like(p).scatter_(1, ids, dw)
    return (p * (dp - (p * dp).sum(1, keepdim=True))).to(s["z"].dtype)


def _groups(s):
    """(expert, its rows) for the experts that have any."""
    at = 0
    for e, n in enumerate(s["counts"]):
        if n:
            yield e, slice(at, at + n)
        at += n


def _halves(gu):
    """Gate and up columns, which alternate in runs of 32."""
    v = gu.unflatten(-1, (-1, 2, 32))
    return v[..., 0, :].flatten(-2), v[..., 1, :].flatten(-2)


def _interleaved(g, u):
    return torch.stack([g.unflatten(-1, (-1, 32)), u.unflatten(-1, (-1, 32))], -2).flatten(-3)


def _swiglu_plain(s):
    act, gu = torch.empty_like(s["act"]), None if s["gu"] is None else torch.empty_like(s["gu"])
    for e, r in _groups(s):
        p = s["x"][s["rows"][r].long()].float() @ s["w"][e].float().t()
        g, u = _halves(p)
        act[r] = (g * torch.sigmoid(g) * u).to(act.dtype)
        if gu is not None:
            gu[r] = p.to(gu.dtype)
    return _there(act=act, gu=gu)


def _down_plain(s):
    y = torch.empty_like(s["y"])
    for e, r in _groups(s):
        y[r] = (s["a"][r].float() @ s["w"][e].float().t()).to(y.dtype)
    return y


def _swiglu_bwd_plain(s):
    dgu = torch.empty_like(s["dgu"])
    for e, r in _groups(s):
        da = s["dy"][r].float() @ s["w"][e].float()
        g, u = _halves(s["gu"][r].float())
        q = torch.sigmoid(g)
        dgu[r] = _interleaved(da * u * q * (1 + g * (1 - q)), da * g * q).to(dgu.dtype)
    return dgu


def _dx_plain(s):
    dx = torch.empty_like(s["dx"])
    for e, r in _groups(s):
        dx[r] = (s["dgu"][r].float() @ s["w"][e].float()).to(dx.dtype)
    return dx


def _dw_plain(s):
    dw = torch.zeros_like(s["dweight"])
    for e, r in _groups(s):
        dw[e] = s["dy"][r].float().t() @ s["a"][r].float()
    return dw


def _combine_plain(s):
    out = s["resid"].clone()
    for j in range(s["top"]):
        out += s["weights"][:, j:j + 1] * s["y"][s["slots"][:, j].long()].float()
    return out


def _combine_bwd_plain(s):
    dy, dw = torch.empty_like(s["dy"]), torch.empty_like(s["dweights"])
    dout = s["dout"].float()
    for j in range(s["top"]):
        at = s["slots"][:, j].long()
        dw[:, j] = (dout * s["y"][at].float()).sum(1)
        dy[at] = (dout * s["weights"][:, j:j + 1]).to(dy.dtype)
    return {"dy": dy, "dweights": dw}


def _row_scale(x, eps):
    return torch.rsqrt((x * x).mean(1, keepdim=True) + eps)


def _gate_of_rows(s):
    return s["gate"].repeat_interleave(s["gate_rows"], 0)[:s["rows"]]


def _norm_plain(s):
    n = s["y"].float()
    if s["wpost"] is not None:
        n = n * _row_scale(n, s["eps"]) * s["wpost"]
    if s["gate"] is not None:
        n = n * _gate_of_rows(s)
    h = s["resid"].float() + s["scale"] * n
    x = None if s["wpre"] is None else (h * _row_scale(h, s["eps"]) * s["wpre"]).to(s["x"].dtype)
    return _there(out=h.to(s["out"].dtype), x=x)


def _norm_bwd_plain(s):
    def back(g, v, r):  # of v r(v), for the gradient g
        return r * (g - v * r * r * (g * v).mean(1, keepdim=True))

    dh, dpre, dgate, dpost = s["dout"].float(), None, None, None
    if s["wpre"] is not None:
        h, dx = s["out"].float(), s["dx"].float()
        r = _row_scale(h, s["eps"])
        dpre = (dx * h * r).sum(0)
        dh = dh + back(dx * s["wpre"], h, r)
    y = s["y"].float()
    b = dh * s["scale"]
    n = y
    if s["wpost"] is not None:
        r = _row_scale(y, s["eps"])
        n = y * r * s["wpost"]
    if s["gate"] is not None:
        d = b * n
        pad = s["gate"].shape[0] * s["gate_rows"] - s["rows"]
        dgate = torch.nn.functional.pad(d, (0, 0, 0, pad)).view(-1, s["gate_rows"], s["h"]).sum(1)
        b = b * _gate_of_rows(s)
    if s["wpost"] is not None:
        dpost = (b * y * r).sum(0)
        b = back(b * s["wpost"], y, r)
    return _there(dy=b.to(s["dy"].dtype), dresid=dh.to(s["dresid"].dtype), dpost=dpost, dgate=dgate, dpre=dpre)


_PLAIN = {"route": _route_plain, "route_bwd": _route_bwd_plain, "swiglu": _swiglu_plain, "down": _down_plain,
          "swiglu_bwd": _swiglu_bwd_plain, "dx": _dx_plain, "dw": _dw_plain, "combine": _combine_plain,
          "combine_bwd": _combine_bwd_plain, "norm": _norm_plain, "norm_bwd": _norm_bwd_plain}


# ---------------------------------------------------- definitions in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in PRODUCTS:
        return _products_exact(s)
    return {"route": _route_exact, "route_bwd": _route_bwd_exact, "combine": _combine_exact,
            "combine_bwd": _combine_bwd_exact, "norm": _norm_exact, "norm_bwd": _norm_bwd_exact}[kind](s)


def _chosen(z, ids, normalize):
    w = torch.softmax(z, 1).gather(1, ids)
    return w / w.sum(1, keepdim=True) if normalize else w


def _route_exact(s):
    z = s["z"].double()
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :s["top"]]
    experts, order = torch.sort(ids.flatten(), stable=True)
    offsets = torch.searchsorted(experts, torch.arange(s["experts"] + 1, device=DEV))
    slots = torch.argsort(order)
    i32 = torch.int32
    return {"weights": _chosen(z, ids, s["normalize"]), "ids": ids.to(i32), "offsets": offsets.to(i32),
            "slots": slots.view(ids.shape).to(i32), "rows": torch.div(order, s["top"], rounding_mode="floor").to(i32)}


def _route_bwd_exact(s):
    z = s["z"].double().requires_grad_()
    w = _chosen(z, s["ids"].long(), s["normalize"])
    return torch.autograd.grad(w, z, s["dw"].double())[0]


def _products_exact(s):
    """Each expert's product with the rows between its offsets, by torch's own functions."""
    kind, F = s["kind"], torch.nn.functional
    o = s["offsets"].tolist()
    parts = []
    for e in range(s["experts"]):
        r = slice(o[e], o[e + 1])
        if kind == "dw":
            parts.append((s["dy"][r].double().t() @ s["a"][r].double())[None])
            continue
        w = s["w"][e].double()
        if kind == "swiglu":
            p = F.linear(s["x"].double().index_select(0, s["rows"][r].long()), w)
            g, u = p.view(-1, s["inter"] // 32, 2, 32).unbind(2)
            parts.append((((F.silu(g) * u).reshape(-1, s["inter"])), p))
        elif kind == "swiglu_bwd":
            gu = s["gu"][r].double().requires_grad_()
            g, u = gu.view(-1, s["inter"] // 32, 2, 32).unbind(2)
            out = F.linear((F.silu(g) * u).reshape(-1, s["inter"]), w)
            parts.append(torch.autograd.grad(out, gu, s["dy"][r].double())[0])
        else:
            parts.append(F.linear(s["a"][r].double(), w) if kind == "down" else s["dgu"][r].double() @ w)
    if kind != "swiglu":
        return torch.cat(parts)
    return _there(act=torch.cat([a for a, _ in parts]), gu=torch.cat([p for _, p in parts]) if s["save"] else None)


def _combine_exact(s):
    parts = [(y[slots.long()].double() * w[..., None].double()).sum(1) + r.double()
             for y, slots, w, r in ((s["y"], a, b, c) for a, b, c in zip(s["slots"].split(2048), s["weights"].split(2048),
                                                                        s["resid"].split(2048)))]
    return torch.cat(parts)


def _combine_bwd_exact(s):
    rows, k = s["rows"].long(), s["top"]
    flat = torch.argsort(s["slots"].flatten())  # pair at each place
    dout = s["dout"].double().index_select(0, rows)
    dots = (dout * s["y"].double()).sum(1)
    return {"dy": dout * s["weights"].double().flatten()[flat, None], "dweights": dots[s["slots"].long()].view(-1, k)}


def _rms(x, w, eps):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w


def _norm_branch(s, y, wpost, gate):
    n = y if wpost is None else _rms(y, wpost, s["eps"])
    return s["scale"] * (n if gate is None else n * gate)


def _gate_rows_of(s, r):
    return torch.arange(s["rows"], device=DEV)[r] // s["gate_rows"]


def _double(t):
    return None if t is None else t.double()


def _row_slices(n):
    return [slice(a, min(a + 2048, n)) for a in range(0, n, 2048)]


def _norm_exact(s):
    outs, xs = [], []
    for r in _row_slices(s["rows"]):
        gate = None if s["gate"] is None else s["gate"].double()[_gate_rows_of(s, r)]
        h = s["resid"][r].double() + _norm_branch(s, s["y"][r].double(), _double(s["wpost"]), gate)
        outs.append(h)
        if s["wpre"] is not None:
            xs.append(_rms(h, s["wpre"].double(), s["eps"]))
    return _there(out=torch.cat(outs), x=torch.cat(xs) if xs else None)


def _norm_bwd_exact(s):
    """By autograd in two steps, a slice of rows at a time: the gradient at the
    stream, then through the branch."""
    names = ("wpost", "gate", "wpre")
    leaf = {n: _double(s[n]) for n in names}
    total = {n: None if t is None else torch.zeros_like(t) for n, t in leaf.items()}
    dys, drs = [], []
    for r in _row_slices(s["rows"]):
        w = {n: None if t is None else t.clone().requires_grad_() for n, t in leaf.items()}
        dh = s["dout"][r].double()
        if w["wpre"] is not None:
            h = s["out"][r].double().requires_grad_()
            g = torch.autograd.grad(_rms(h, w["wpre"], s["eps"]), (h, w["wpre"]), s["dx"][r].double())
            dh = dh + g[0]
            total["wpre"] += g[1]
        y = s["y"][r].double().requires_grad_()
        gate = None if w["gate"] is None else w["gate"][_gate_rows_of(s, r)]
        wanted = [n for n in ("wpost", "gate") if w[n] is not None]
        g = torch.autograd.grad(_norm_branch(s, y, w["wpost"], gate), [y] + [w[n] for n in wanted], dh)
        for n, t in zip(wanted, g[1:]):
            total[n] += t
        dys.append(g[0])
        drs.append(dh)
    return _there(dy=torch.cat(dys), dresid=torch.cat(drs), dpost=total["wpost"], dgate=total["gate"],
                  dpre=total["wpre"])


# -------------------------------------------------------------------- work --

def _used(c):
    """Experts that have a row, on average (taken as equally liked)."""
    E = c["experts"]
    return E * (1 - (1 - c["top"] / E) ** c["tokens"])


def work(case):
    c, kind = case, case["kind"]
    if kind in ("norm", "norm_bwd"):
        n, a, st = c["rows"] * c["h"], SIZE[c["act"]], SIZE[c["stream"]]
        weights = 4 * c["h"] * ((1 if c["post"] else 0) + (1 if c["pre"] else 0))
        if c["gate"]:
            weights += 4 * c["h"] * (-(-c["rows"] // c["seq"]) if c["gate"] == "sequence" else 1)
        if kind == "norm":
            return {"bytes": n * (a + 2 * st + (a if c["pre"] else 0)) + weights, "flops": 10 * n}
        reads = a + st + (a + st if c["pre"] else 0)
        if not (c["post"] or c["gate"]):
            reads -= a  # the branch's output is not needed for its own gradient
        return {"bytes": n * (reads + a + st) + 2 * weights, "flops": 22 * n}
    T, k, E = c["tokens"], c["top"], c["experts"]
    R = T * k
    if kind == "route":
        return {"bytes": T * E * SIZE[c["dtype"]] + 16 * R + 4 * E + 4, "flops": 4 * T * E}
    if kind == "route_bwd":
        z = SIZE[c["dtype"]]
        # where the weights are the chosen experts' alone, so are the logits read
        return {"bytes": T * (k if c["normalize"] else E) * z + T * E * z + 8 * R, "flops": 6 * T * E}
    h = c["h"]
    if kind == "combine":
        return {"bytes": R * (2 * h + 8) + 8 * T * h, "flops": 2 * R * h}
    if kind == "combine_bwd":
        return {"bytes": R * (4 * h + 12) + T * h * SIZE[c["dtype"]], "flops": 3 * R * h}
    i, used = c["inter"], _used(c)
    if kind == "swiglu":
        return {"bytes": 2 * (min(T, R) * h + used * 2 * i * h + R * i * (3 if c["save"] else 1)) + 4 * R + 4 * E,
                "flops": 4 * R * h * i}
    if kind == "down":
        return {"bytes": 2 * (R * i + used * h * i + R * h) + 4 * E, "flops": 2 * R * h * i}
    if kind == "swiglu_bwd":
        return {"bytes": 2 * (R * h + used * h * i + 4 * R * i) + 4 * E, "flops": 2 * R * h * i}
    if kind == "dx":
        return {"bytes": 2 * (2 * R * i + used * 2 * i * h + R * h) + 4 * E, "flops": 4 * R * h * i}
    return {"bytes": 2 * R * (h + i) + 4 * E * h * i + 4 * E, "flops": 2 * R * h * i}
