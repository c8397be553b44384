"""The end of a block's branch with the norm after it (``norm_residual``,
``norm_residual_bwd``) against float64, and what they refuse.

Bounds. With H columns: a mean square is off by H 2^-24 of itself and its inverse
root by half that and 2^-22; a product of five factors by 5 2^-24 more. The
backward's row sums are off by (H + 6) 2^-24 of the sum of their terms'
magnitudes, its column sums by that of the rows, T + 6, on top of their terms'
own error; outputs round by half a unit of their type.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from mround_amd import kernels as K
from mround_amd.exceptions import KernelError
from tests.helpers import dev
from tests.test_experts import address, normal, refused, rounding, strided, within

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
PAIRS = [(F32, F32), (BF, F32), (F16, F32), (BF, BF), (F16, F16)]  # branch, stream
EPS = 1e-6
U = 2.0 ** -24

# (rows, columns): one row and column, whole pieces and not, each number of pieces a
# thread and the rows past them, rows enough that a block goes on to another
SHAPES = [(1, 1), (1, 64), (3, 7), (5, 72), (130, 896), (67, 1001), (33, 4096), (9, 4104), (4, 8192), (7, 8200),
          (3, 16384), (2, 5003), (2, 16383), (3001, 200), (5000, 40), (2500, 1024)]


def inputs(T, H, act, stream, seed=0):
    wide = torch.exp(normal(H, seed=seed))
    y, r = normal(T, H, seed=seed + 1).to(act), (normal(T, H, seed=seed + 2) * wide).to(stream)
    post, pre = 1 + normal(H, seed=seed + 3, std=0.2), 1 + normal(H, seed=seed + 4, std=0.2)
    return y, r, post, pre


def forward64(y, resid, post, gate, scale, pre):
    """(h, its error's bound, x, its bound) in float64; gate a row for each row."""
    y, resid = y.double(), resid.double()
    H = y.shape[1]
    n = y if post is None else y * (y.square().mean(1, keepdim=True) + EPS).rsqrt() * post.double()
    n = scale * (n if gate is None else n * gate.double())
    h = resid + n
    eh = n.abs() * ((H / 2 + 4) * U + 6 * U) + U * (h.abs() + n.abs())
    if pre is None:
        return h, eh, None, None
    r = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
    x = h * r * pre.double()
    ex = eh * r * pre.double().abs() + x.abs() * ((H / 2 + 8) * U + r * (eh.square().mean(1, keepdim=True)).sqrt())
    return h, eh, x, ex


def gates(T, H, rows, seed=9):
    """(gate [G, H], of each row, gate_rows)"""
    if rows is None:
        g = normal(1, H, seed=seed)
        return g, g.expand(T, H), None
    g = normal(-(-T // rows), H, seed=seed)
    return g, g.repeat_interleave(rows, 0)[:T], rows


def run_forward(y, r, post, gate, gate_rows, scale, pre):
    T, H = y.shape
    out = strided(torch.full((T, H), 7.0, dtype=r.dtype, device=dev()), fill=7.0)
    x = None if pre is None else torch.full((T, H), 7.0, dtype=y.dtype, device=dev())
    K.norm_residual(y, r, out, eps=EPS, post=post, gate=gate, gate_rows=gate_rows, scale=scale, pre=pre, normed=x)
    return out, x


@pytest.mark.gpu
@pytest.mark.parametrize("act,stream", PAIRS)
@pytest.mark.parametrize("T,H", SHAPES)
def test_forward(T, H, act, stream):
    y, r, post, pre = inputs(T, H, act, stream)
    y, r = strided(y, 8 if H % 8 == 0 else 3), strided(r)
    whole, per_row, one = gates(T, H, None), gates(T, H, 1), gates(T, H, 3)
    for p, (g, rows, per), scale, q in ((post, whole, 0.7, pre), (None, per_row, 1.0, pre), (post, (None, None, None), -1.5, None),
                                        (None, (None, None, None), 1.0, pre), (post, one, 1.0, pre)):
        out, x = run_forward(y, r, p, g, per, scale, q)
        h, eh, want, ex = forward64(y, r, p, rows, scale, q)
        within(out, h, eh + rounding(h, stream), "out")
        assert bool((out._base[:, H:] == 7.0).all())
        if q is not None:
            within(x, want, ex + rounding(want, act), "normed")
    # over its inputs
    a, b = y.clone(), r.clone()
    K.norm_residual(a, b, b, eps=EPS, post=post, gate=one[0], gate_rows=3, pre=pre, normed=a)
    assert torch.equal(a, x) and torch.equal(b, out)


def backward64(dx, d, y, h, post, gate, scale, pre):
    """Gradients by the formulas in float64, and bounds of their errors."""
    T, H = y.shape
    zero = torch.zeros(1, 1, dtype=torch.float64, device=dev())
    y, h = y.double(), h.double()
    row = (H + 8) * U
    dh, edh = (d.double(), zero) if d is not None else (zero.expand(T, H), zero)
    dpre = edpre = None
    if pre is not None:
        g = dx.double() * pre.double()
        r = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
        back = r * (g - h * r * r * (g * h).mean(1, keepdim=True))
        mag = r * (g.abs() + h.abs() * r * r * (g * h).abs().mean(1, keepdim=True))
        dh, edh = dh + back, 2 * row * mag + U * (dh.abs() + mag)
        t = dx.double() * h * r
        dpre, edpre = t.sum(0), ((T + 8) * U + row) * t.abs().sum(0)
    e, ee = scale * dh, abs(scale) * (edh + U * dh.abs())
    ry = (y.square().mean(1, keepdim=True) + EPS).rsqrt() if post is not None else torch.ones_like(zero)
    w = post.double() if post is not None else torch.ones_like(zero)
    n = y * ry * w
    dgate = edgate = None
    b, eb = e, ee
    if gate is not None:
        t = e * n
        dgate, edgate = t, (ee + 2 * row * e.abs()) * n.abs() + (T + 8) * U * t.abs()
        b, eb = e * gate.double(), ee * gate.double().abs() + U * (e * gate.double()).abs()
    dy, edy, dpost, edpost = b, eb, None, None
    if post is not None:
        t = b * y * ry
        dpost, edpost = t.sum(0), ((eb + row * b.abs()) * (y * ry).abs() + (T + 8) * U * t.abs()).sum(0)
        c = b * w
        ec = eb * w.abs() + U * c.abs()
        dy = ry * (c - y * ry * ry * (c * y).mean(1, keepdim=True))
        edy = ry * (ec + y.abs() * ry * ry * (ec * y.abs()).mean(1, keepdim=True)) + 2 * row * ry * (
            c.abs() + y.abs() * ry * ry * (c * y).abs().mean(1, keepdim=True))
    return dict(dy=(dy, edy), dresid=(dh, edh), dpost=(dpost, edpost), dgate=(dgate, edgate), dpre=(dpre, edpre))


def by_group(t, per):
    """Sums of each ``per`` rows."""
    T = t.shape[0]
    if per is None:
        return t.sum(0, keepdim=True)
    return torch.nn.functional.pad(t, (0, 0, 0, -T % per)).view(-1, per, t.shape[1]).sum(1)


@pytest.mark.gpu
@pytest.mark.parametrize("act,stream", PAIRS)
@pytest.mark.parametrize("T,H", SHAPES)
def test_backward(T, H, act, stream):
    y, h, post, pre = inputs(T, H, act, stream, seed=20)
    y, h = strided(y, 8 if H % 8 == 0 else 3), strided(h)
    dx, d = strided(normal(T, H, seed=30).to(act)), strided(normal(T, H, seed=31).to(stream))
    none = (None, None, None)
    # (a gate for all, for each row, for several in a block, for more than a block has)
    cases = [(post, gates(T, H, None), 0.7, pre, True), (None, gates(T, H, 1), 1.0, pre, True), (post, none, -1.5, None, True),
             (None, none, 1.0, pre, False), (post, gates(T, H, 3), 1.0, pre, False), (post, gates(T, H, 700), 1.0, pre, True)]
    for p, (g, rows, per), scale, q, with_d in cases:
        f = lambda *s: torch.full(s, 7.0, device=dev())
        dy = strided(torch.full((T, H), 7.0, dtype=act, device=dev()), fill=7.0)
        dr = strided(torch.full((T, H), 7.0, dtype=stream, device=dev()), fill=7.0)
        dpost, dpre = None if p is None else f(H), None if q is None else f(H)
        dgate = None if g is None else torch.full_like(g, 7.0)
        args = dict(eps=EPS, post=p, gate=g, gate_rows=per, scale=scale, pre=q)
        K.norm_residual_bwd(None if q is None else dx, d if with_d else None, y, h, dy, dr, dpost=dpost, dgate=dgate,
                            dpre=dpre, **args)
        want = backward64(dx, d if with_d else None, y, h, p, rows, scale, q)
        for name, got, dtype in (("dy", dy, act), ("dresid", dr, stream)):
            v, tol = want[name]
            within(got, v, tol + rounding(v, dtype), name)
            assert bool((got._base[:, H:] == 7.0).all())
        for name, got in (("dpost", dpost), ("dpre", dpre)):
            if got is not None:
                within(got, want[name][0], want[name][1] + 1e-30, name)
        if g is not None:
            within(dgate, by_group(want["dgate"][0], per), by_group(want["dgate"][1], per) + 1e-30, "dgate")
        # without the weights' gradients, and over its inputs: the same values
        a, b = y.clone(), d.clone()
        K.norm_residual_bwd(None if q is None else dx, b if with_d else None, a, h, a, b, **args)
        assert torch.equal(a, dy) and torch.equal(b, dr)


# Rows enough that each block goes on to others, for each number of pieces a thread: one
# column at a time (4, 8 and 16 a thread) and eight (one, two, and those past 8192 columns).
MANY = [(2600, 1001), (1300, 5003), (1100, 16383), (2100, 2048), (2100, 4104), (1100, 8200), (1100, 16384)]


@pytest.mark.gpu
@pytest.mark.parametrize("act,stream", PAIRS)
@pytest.mark.parametrize("T,H", MANY)
def test_blocks_that_go_on_to_other_rows(T, H, act, stream):
    """Forward and backward with every weight's gradient."""
    y, r, post, pre = inputs(T, H, act, stream, seed=100)
    dx, d = normal(T, H, seed=110).to(act), normal(T, H, seed=111).to(stream)
    for g, rows, per in (gates(T, H, 1), gates(T, H, 3), gates(T, H, 700), (None, None, None)):
        out, x = run_forward(y, r, post, g, per, 0.7, pre)
        h, eh, want, ex = forward64(y, r, post, rows, 0.7, pre)
        within(out, h, eh + rounding(h, stream), "out")
        within(x, want, ex + rounding(want, act), "normed")
        f = lambda t: None if t is None else torch.full_like(t, 7.0)
        got = dict(dy=f(y), dresid=f(r), dpost=f(post), dgate=f(g), dpre=f(pre))
        K.norm_residual_bwd(dx, d, y, r, got["dy"], got["dresid"], eps=EPS, post=post, gate=g, gate_rows=per, scale=0.7,
                            pre=pre, dpost=got["dpost"], dgate=got["dgate"], dpre=got["dpre"])
        want = backward64(dx, d, y, r, post, rows, 0.7, pre)
        for name, dtype in (("dy", act), ("dresid", stream)):
            v, tol = want[name]
            within(got[name], v, tol + rounding(v, dtype), name)
        for name in ("dpost", "dpre"):
            within(got[name], want[name][0], want[name][1] + 1e-30, name)
        if g is not None:
            within(got["dgate"], by_group(want["dgate"][0], per), by_group(want["dgate"][1], per) + 1e-30, "dgate")


@pytest.mark.gpu
def test_backward_against_differences():
    """Central differences of sum(out d) + sum(normed dx) in float64 arithmetic of
    the operator's float32 results: a step of 2^-7 leaves its square (6e-5) times
    third derivatives of order 1, and 2^-21 / 2^-7 of the sums' rounding."""
    T, H = 6, 40
    y, r, post, pre = inputs(T, H, F32, F32, seed=40)
    r = normal(T, H, seed=42)
    gate, _, per = gates(T, H, 2)
    dx, d = normal(T, H, seed=43), normal(T, H, seed=44)
    args = dict(eps=EPS, gate_rows=per, scale=0.8)

    def value(y, r, post, gate, pre):
        out, x = torch.empty_like(r), torch.empty_like(y)
        K.norm_residual(y, r, out, post=post, gate=gate, pre=pre, normed=x, **args)
        return float((out.double() * d.double()).sum() + (x.double() * dx.double()).sum())

    inp = dict(y=y, r=r, post=post, gate=gate, pre=pre)
    out, x = torch.empty_like(r), torch.empty_like(y)
    K.norm_residual(y, r, out, post=post, gate=gate, pre=pre, normed=x, **args)
    g = {n: torch.empty_like(t) for n, t in inp.items()}
    K.norm_residual_bwd(dx, d, y, out, g["y"], g["r"], post=post, gate=gate, pre=pre, dpost=g["post"], dgate=g["gate"],
                        dpre=g["pre"], **args)
    step = 2.0 ** -7
    for n, t in inp.items():
        for seed in range(4):
            way = normal(*t.shape, seed=50 + seed)
            sides = [value(**dict(inp, **{n: t + s * way})) for s in (step, -step)]
            slope = (sides[0] - sides[1]) / (2 * step)
            want = float((g[n].double() * way.double()).sum())
            assert abs(slope - want) <= 0.01 * float(g[n].norm() * way.norm()), (n, slope, want)


@pytest.mark.gpu
def test_rows_of_zeros_and_rows_that_are_not_finite():
    """A row of zeros is scaled by eps alone; an infinity or a NaN stays in its row."""
    y, r, post, pre = inputs(9, 64, F32, F32, seed=60)
    clean = run_forward(y, r, post, None, None, 1.0, pre)
    y[2], r[2] = 0.0, 0.0
    y[4, 3], r[6, 5] = torch.nan, torch.inf
    out, x = run_forward(y, r, post, None, None, 1.0, pre)
    assert not out[2].any() and not x[2].any()
    assert bool(out[4].isnan().all()) and bool(x[4].isnan().all())
    assert bool(x[6, 5].isnan()) and bool(out[6, 5].isinf())
    keep = [0, 1, 3, 5, 7, 8]
    assert torch.equal(out[keep], clean[0][keep]) and torch.equal(x[keep], clean[1][keep])


@pytest.mark.gpu
def test_offsets_past_32_bits():
    T, H, n = 140000, 16384, 30
    y, r = torch.zeros(T, H, dtype=BF, device=dev()), torch.zeros(T, H, dtype=BF, device=dev())
    near = inputs(n, H, BF, BF, seed=70)
    y[T - n:], r[T - n:] = near[0], near[1]
    post, pre = near[2:]
    out, x = torch.empty_like(r), torch.empty_like(y)
    K.norm_residual(y, r, out, eps=EPS, post=post, pre=pre, normed=x)
    few = run_forward(near[0], near[1], post, None, None, 1.0, pre)
    assert torch.equal(out[T - n:], few[0]) and torch.equal(x[T - n:], few[1])
    dy, dr = torch.empty(n, H, dtype=BF, device=dev()), torch.empty(n, H, dtype=BF, device=dev())
    K.norm_residual_bwd(near[0], near[1], near[0], few[0].contiguous(), dy, dr, eps=EPS, post=post, pre=pre)
    K.norm_residual_bwd(x.copy_(y), r, y, out, y, r, eps=EPS, post=post, pre=pre)
    assert torch.equal(y[T - n:], dy) and torch.equal(r[T - n:], dr)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 700])
def test_a_gate_for_more_rows_than_there_are(T):
    y, r, post, pre = inputs(T, 72, BF, F32, seed=80)
    gate = normal(1, 72, seed=84)
    dx, d = normal(T, 72, seed=85).to(BF), normal(T, 72, seed=86)
    got = []
    for per in (None, T, 4096, 1 << 40):
        out, x = run_forward(y, r, post, gate, per, 0.5, pre)
        e = lambda *s, dt=F32: torch.empty(*s, dtype=dt, device=dev())
        g = [e(T, 72, dt=BF), e(T, 72), e(72), e(1, 72), e(72)]
        K.norm_residual_bwd(dx, d, y, out, g[0], g[1], eps=EPS, post=post, gate=gate, gate_rows=per, scale=0.5, pre=pre,
                            dpost=g[2], dgate=g[3], dpre=g[4])
        got.append([out, x] + g)
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    assert K.lib().mr_norm_residual_bwd_workspace_bytes(T, 72, 1 << 40, 1, 1, 1) == \
        K.lib().mr_norm_residual_bwd_workspace_bytes(T, 72, T, 1, 1, 1)


@pytest.mark.gpu
def test_no_rows():
    y, post = torch.empty(0, 64, device=dev()), torch.ones(64, device=dev())
    K.norm_residual(y, y, y.clone(), eps=EPS, post=post, pre=post, normed=y.clone())
    dpost, dpre = torch.full_like(post, 7.0), torch.full_like(post, 7.0)
    K.norm_residual_bwd(y, y, y, y, y.clone(), y.clone(), eps=EPS, post=post, pre=post, dpost=dpost, dpre=dpre)
    assert not dpost.any() and not dpre.any()


@pytest.mark.gpu
@pytest.mark.parametrize("G,per", [(1, None), (3, 5)])
def test_the_gate_of_no_rows_has_no_gradient(G, per):
    y, gate = torch.empty(0, 64, device=dev()), torch.ones(G, 64, device=dev())
    dgate = torch.full_like(gate, 7.0)
    K.norm_residual_bwd(None, y, y, y, y.clone(), y.clone(), eps=EPS, gate=gate, gate_rows=per, dgate=dgate)
    assert not dgate.any()


@pytest.mark.gpu
def test_no_rows_through_the_c_interface():
    """dpost and dpre are zeros; dgate, which has no rows then, is left."""
    w, got = torch.ones(64, device=dev()), [torch.full((64,), 7.0, device=dev()) for _ in range(3)]
    at = w.data_ptr()
    assert K.lib().mr_norm_residual_bwd(None, 0, 64, None, 0, 64, None, 64, None, 64, 0, 64, EPS, at, at, 5, 1.0, at, None, 64,
                                        None, 64, *(t.data_ptr() for t in got), None, 0, torch.cuda.current_stream().cuda_stream) == 0
    dpost, dgate, dpre = got
    assert not dpost.any() and not dpre.any() and bool((dgate == 7.0).all())


@pytest.mark.gpu
def test_two_blocks_in_a_graph():
    """Two branches' ends forward and back, captured once and replayed over other
    inputs between eager runs of the same chain."""
    T, H = 300, 256
    post, pre, gate = (normal(H, seed=1), normal(H, seed=2), normal(3, H, seed=3))
    args = dict(eps=EPS, post=post, gate=gate, gate_rows=100, scale=0.5, pre=pre)
    y, r, dx, d = (torch.zeros(T, H, dtype=t, device=dev()) for t in (BF, F32, BF, F32))

    def buffers():
        e = lambda dt, *s: torch.full(s, 3.0, dtype=dt, device=dev())
        return dict(h1=e(F32, T, H), x1=e(BF, T, H), h2=e(F32, T, H), x2=e(BF, T, H), dy=e(BF, T, H), dr=e(F32, T, H),
                    dy1=e(BF, T, H), dr1=e(F32, T, H), dpost=e(F32, H), dgate=e(F32, 3, H), dpre=e(F32, H))

    def step(b):
        K.norm_residual(y, r, b["h1"], normed=b["x1"], **args)
        K.norm_residual(b["x1"], b["h1"], b["h2"], normed=b["x2"], **args)
        K.norm_residual_bwd(dx, d, b["x1"], b["h2"], b["dy"], b["dr"], **args)
        K.norm_residual_bwd(b["dy"], b["dr"], y, b["h1"], b["dy1"], b["dr1"], dpost=b["dpost"], dgate=b["dgate"],
                            dpre=b["dpre"], **args)

    a, b = buffers(), buffers()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    for seed in range(3):
        for i, t in enumerate((y, r, dx, d)):
            t.copy_(normal(T, H, seed=10 * seed + i))
        step(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in a:
            assert torch.equal(a[name], b[name]), (seed, name)


# The gradients that may be asked for beside a gate, each with and without the others.
SUBSETS = [(a, b, c) for a in (0, 1) for b in (0, 1) for c in (0, 1) if a or b or c]


def blocks_of(T, H, rows):
    """(blocks of the backward, blocks that share a gate's row): about 512, of narrow
    rows 1024, each of whole groups or of one group's rows."""
    want = -(-T // (1024 if 512 < H <= 1024 else 512))
    if rows <= want:
        return -(-T // (want // rows * rows)), 1
    per = -(-rows // want)
    return -(-T // rows) * per, per


@pytest.mark.parametrize("T,H", [(1, 64), (600, 256), (1000, 256), (1000, 1024), (4005, 2048), (16384, 3584), (300000, 64)])
@pytest.mark.parametrize("rows", [1, 2, 3, 33, 100, 2048, 1 << 40])
def test_the_workspace_holds_what_the_blocks_leave(T, H, rows):
    """Of any gradients, with a gate or without one."""
    size = K.lib().mr_norm_residual_bwd_workspace_bytes
    gated, shared = blocks_of(T, H, min(rows, T))
    plain = blocks_of(T, H, T)[0]
    for dpost, dgate, dpre in SUBSETS:
        n = dpost + dpre + (dgate and shared > 1)
        assert size(T, H, rows, dpost, dgate, dpre) >= 4 * H * n * gated
        if not dgate:
            for any_rows in (0, rows):
                assert size(T, H, any_rows, dpost, 0, dpre) >= 4 * H * n * plain


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,rows", [(1000, 256, 3), (1000, 256, 100), (2049, 72, 33), (1500, 1000, 2), (700, 4104, 3), (900, 201, 5)])
def test_any_of_the_gradients_beside_a_gate(T, H, rows):
    """The same bits as of all of them, and nothing behind the workspace."""
    y, h, post, pre = inputs(T, H, BF, F32, seed=90)
    gate, _, per = gates(T, H, rows)
    dx, d = normal(T, H, seed=95).to(BF), normal(T, H, seed=96)
    args = dict(eps=EPS, post=post, gate=gate, gate_rows=per, scale=0.7, pre=pre)
    f = lambda t: torch.full_like(t, 7.0)
    want = [f(y), f(h), f(post), f(gate), f(pre)]
    K.norm_residual_bwd(dx, d, y, h, want[0], want[1], dpost=want[2], dgate=want[3], dpre=want[4], **args)
    lib = K.lib()
    for subset in SUBSETS:
        got = [f(y), f(h)] + [f(t) if on else None for t, on in zip((post, gate, pre), subset)]
        K.norm_residual_bwd(dx, d, y, h, got[0], got[1], dpost=got[2], dgate=got[3], dpre=got[4], **args)
        assert all(b is None or torch.equal(a, b) for a, b in zip(want, got)), subset
        size = lib.mr_norm_residual_bwd_workspace_bytes(T, H, rows, *subset)
        ws = torch.full((size + 4096,), 0x5a, dtype=torch.uint8, device=dev())
        ptr = lambda t: None if t is None else t.data_ptr()
        again = [None if t is None else f(t) for t in got]
        assert lib.mr_norm_residual_bwd(ptr(dx), 1, H, ptr(d), 0, H, ptr(y), H, ptr(h), H, T, H, EPS, ptr(post), ptr(gate), rows,
                                        0.7, ptr(pre), ptr(again[0]), H, ptr(again[1]), H, *map(ptr, again[2:]), ptr(ws), size,
                                        torch.cuda.current_stream().cuda_stream) == 0
        assert bool((ws[size:] == 0x5a).all()), subset
        assert all(a is None or torch.equal(a, b) for a, b in zip(again, got)), subset


# ---------------------------------------------------------------- refusals --

FORWARD = dict(y=address(0), act=1, ldy=64, r=address(1), st=0, ldr=64, T=10, H=64, eps=1e-6, post=address(2),
               gate=address(3), rows=5, scale=1.0, pre=address(4), out=address(5), ldo=64, x=address(6), ldn=64, stream=None)
BACKWARD = dict(dx=address(0), act=1, lddx=64, d=address(1), st=0, ldd=64, y=address(2), ldy=64, h=address(3), ldh=64, T=10,
                H=64, eps=1e-6, post=address(4), gate=address(5), rows=5, scale=1.0, pre=address(6), dy=address(7), lddy=64,
                dr=address(8), lddr=64, dpost=address(9), dgate=address(10), dpre=address(11), ws=address(12),
                bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(act=2, st=1), "of the branch's type"), (dict(act=5), "type"), (dict(H=16385, ldy=16385), "16384"), (dict(T=-1), "negative"),
    (dict(pre=None), "together"), (dict(x=None), "together"), (dict(rows=0), "gate"), (dict(ldy=63), "leading"),
    (dict(out=None), "null"), (dict(out=address(0)), "no memory"), (dict(out=address(1), ldo=65), "no memory"),
    (dict(x=address(1)), "no memory"), (dict(out=address(2)), "no memory"), (dict(x=address(3)), "no memory"),
    (dict(y=ctypes.c_void_p((1 << 20) + 1)), "aligned"), (dict(post=ctypes.c_void_p((1 << 20) + 2)), "aligned")])
def test_forward_refuses(change, message):
    refused("mr_norm_residual", list(dict(FORWARD, **change).values()), message)


@pytest.mark.parametrize("change,message", [
    (dict(act=2, st=1), "of the branch's type"), (dict(H=16385), "16384"), (dict(dx=None), "together"),
    (dict(dx=None, pre=None, dpre=None, d=None), "no gradient"), (dict(post=None), "not there"), (dict(gate=None), "not there"),
    (dict(dy=None), "null"), (dict(y=None), "null"), (dict(h=None), "null"), (dict(lddr=63), "leading"),
    (dict(ws=None), "workspace"), (dict(bytes=100), "workspace"), (dict(dy=address(0)), "no memory"),
    (dict(dr=address(1), lddr=65), "no memory"), (dict(dpost=address(4)), "no memory"), (dict(dgate=address(9)), "no memory"),
    (dict(ws=address(2)), "no memory"), (dict(dpre=ctypes.c_void_p((1 << 20) + 2)), "aligned"), (dict(rows=0), "gate")])
def test_backward_refuses(change, message):
    refused("mr_norm_residual_bwd", list(dict(BACKWARD, **change).values()), message)


@pytest.mark.parametrize("T,H,rows", [(1000, 256, 3), (4005, 2048, 100), (16384, 3584, 33)])
def test_a_workspace_too_small_for_the_blocks_beside_a_gate_is_refused(T, H, rows):
    """Where dgate is not asked for: the blocks are still those of the gate's groups."""
    lds = {n: H for n in ("lddx", "ldd", "ldy", "ldh", "lddy", "lddr")}
    far = {n: ctypes.c_void_p((i + 1) << 40) for i, n in enumerate(
        ("dx", "d", "y", "h", "post", "gate", "pre", "dy", "dr", "dpost", "dpre", "ws"))}
    base = dict(BACKWARD, **far, **lds, T=T, H=H, rows=rows, dgate=None)
    assert blocks_of(T, H, rows)[0] > blocks_of(T, H, T)[0]
    for change, n in ((dict(), 2), (dict(dpre=None), 1), (dict(dpost=None), 1)):
        for blocks in (blocks_of(T, H, T)[0], blocks_of(T, H, rows)[0] - 1):
            refused("mr_norm_residual_bwd", list(dict(base, **change, bytes=4 * H * n * blocks).values()), "workspace")


@pytest.mark.parametrize("fn,base", [("mr_norm_residual", FORWARD), ("mr_norm_residual_bwd", BACKWARD)])
@pytest.mark.parametrize("T", [2 ** 40 + 1, 1 << 62, 2 ** 63 - 1])
def test_rows_whose_bytes_pass_64_bits_are_refused(fn, base, T):
    refused(fn, list(dict(base, T=T).values()), "too many rows")
    assert K.lib().mr_norm_residual_bwd_workspace_bytes(T, 64, 5, 1, 1, 1) == 0


def test_bindings_refuse():
    y, r, w = torch.zeros(4, 8, dtype=BF), torch.zeros(4, 8), torch.zeros(8)
    for call in (
            lambda: K.norm_residual(y, r.half(), r.half(), eps=EPS),
            lambda: K.norm_residual(y, r, y, eps=EPS),
            lambda: K.norm_residual(y, r, r, eps=EPS, post=w.double()),
            lambda: K.norm_residual(y, r, r, eps=EPS, post=w[:4]),
            lambda: K.norm_residual(y, r, r, eps=EPS, pre=w),
            lambda: K.norm_residual(y, r, r, eps=EPS, pre=w, normed=r),
            lambda: K.norm_residual(y, r, r, eps=EPS, gate=torch.zeros(2, 8)),
            lambda: K.norm_residual(y, r, r, eps=EPS, gate=torch.zeros(2, 8), gate_rows=0),
            lambda: K.norm_residual(y, r, r, eps=EPS, gate=torch.zeros(2, 8), gate_rows=1),
            lambda: K.norm_residual(y[0], r, r, eps=EPS),
            lambda: K.norm_residual_bwd(None, r, y, r, y, r, eps=EPS, dpost=w),
            lambda: K.norm_residual_bwd(y, r, y, r, y, r, eps=EPS),
            lambda: K.norm_residual_bwd(None, r, y, r, y, r, eps=EPS, gate=torch.zeros(1, 8), dgate=torch.zeros(2, 8)),
            lambda: K.norm_residual(y, r, r, eps=EPS)):  # (host tensors)
        with pytest.raises(KernelError):
            call()


def test_the_gate_of_no_rows_is_a_matrix():
    """Also where there is no row to apply it to."""
    y, r = torch.zeros(0, 8, dtype=BF), torch.zeros(0, 8)
    for gate in (torch.tensor(1.0), torch.ones(8), torch.ones(1, 1, 8), torch.ones(1, 4)):
        with pytest.raises(KernelError, match="gate must be"):
            K.norm_residual(y, r, r, eps=EPS, gate=gate)
