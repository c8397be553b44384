"""The choice of experts, rows to their places and back (``route_experts``,
``spread_experts``, ``combine_experts`` and the backward) and the products
grouped by expert (``gemm_experts``, ``gemm_experts_swiglu``, ``_bwd``) against
float64, an expert MLP of them all, and what they refuse.

Bounds. A sum of K products of bfloat16 values (exact in float32) is off by at
most K 2^-24 of the sum of their magnitudes; silu has a slope of at most 1.1 and
its sigmoid is off by 2^-21 of itself (exponential, reciprocal and their
argument's rounding), its slope by that times 1 + |x|; outputs round by half a
unit of their type. A softmax over E is off by E 2^-24 for its sum, 2^-24 |z - m|
for the argument and 2^-21 for exponential, division and products.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from mround_amd import kernels as K
from mround_amd.exceptions import KernelError
from tests.helpers import dev

BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
TYPES = (F32, BF, torch.float16)


def rounding(y, dtype):
    return torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8) * y.abs() + torch.finfo(dtype).smallest_normal * 2.0 ** -9


def within(got, want, tol, what):
    got, same = got.double(), (got.double() == want) | (got.double().isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    if bool(bad.any()):
        err = torch.where(bad, (got - want).abs() / tol, 0.0)
        raise AssertionError(f"{what}: {int(bad.sum())} values past their bound, worst {float(err.nan_to_num(9e9).max())} of it")


def normal(*shape, seed=0, std=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).mul_(std).to(dev())


def strided(t, extra=8, fill=float("nan")):
    """The values of ``t`` in wider rows."""
    whole = torch.full((t.shape[0], t.shape[1] + extra), fill, dtype=t.dtype, device=t.device)
    whole[:, :t.shape[1]] = t
    return whole[:, :t.shape[1]]


# ------------------------------------------------------------------ choice --

def route(z, k, **kw):
    T, E = z.shape
    out = dict(weights=torch.full((T, k), -7.0, device=dev()), ids=torch.full((T, k), -7, dtype=I32, device=dev()),
               offsets=torch.full((E + 1,), -7, dtype=I32, device=dev()),
               slots=torch.full((T, k), -7, dtype=I32, device=dev()),
               rows=torch.full((T * k,), -7, dtype=I32, device=dev()))
    K.route_experts(z, **out, **kw)
    return out


def route_reference(z, k, normalize, scale):
    """In float64 on the CPU: (weights, ids, offsets, slots, rows or -7, bound of the weights)."""
    z = z.cpu().double()
    T, E = z.shape
    nan = z.isnan()
    order = torch.where(nan, 1e300, z.clamp(-1e299, 1e299))
    ids = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :k]
    there = z.gather(1, ids) != -torch.inf
    over = torch.where(z.new_zeros(T, E, dtype=torch.bool).scatter(1, ids, there), z, -torch.inf) if normalize else z
    p = torch.softmax(over, 1)
    w = torch.where(there, p.gather(1, ids) * scale, 0.0)
    far = torch.where(there, (z.gather(1, ids) - z.amax(1, keepdim=True)).abs(), 0.0)
    ids = torch.where(there, ids, -1)
    flat = ids.flatten()
    pairs = torch.nonzero(flat >= 0).flatten()
    pairs = pairs[torch.sort(flat[pairs], stable=True).indices]
    slots, rows = torch.full((T * k,), -1), torch.full((T * k,), -7)
    slots[pairs] = torch.arange(pairs.numel())
    rows[:pairs.numel()] = pairs // k
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(flat[pairs], minlength=E).cumsum(0)])
    tol = w.abs() * (E * 2.0 ** -24 + far * 2.0 ** -23 + 2.0 ** -21) + 2.0 ** -126
    return w, ids, offsets, slots.view(T, k), rows, tol


def check_route(z, k, normalize=False, scale=1.0):
    got = route(z, k, normalize=normalize, scale=scale)
    w, ids, offsets, slots, rows, tol = route_reference(z, k, normalize, scale)
    for name, want in (("ids", ids), ("offsets", offsets), ("slots", slots), ("rows", rows)):
        assert torch.equal(got[name].cpu().long(), want), name
    within(got["weights"].cpu(), w, tol, "weights")
    return got


# (tokens, experts, top): each width of a token's lanes and logits, several blocks, one, no whole one
ROUTES = [(1, 1, 1), (1, 7, 7), (3, 64, 8), (130, 60, 4), (300, 65, 6), (1000, 128, 8), (257, 200, 16), (200, 256, 17),
          (129, 257, 8), (131, 384, 32), (70, 512, 33), (66, 300, 64), (5000, 2, 1), (40000, 33, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", ROUTES)
def test_route(T, E, k):
    for n, dtype in enumerate(TYPES):
        z = (normal(T, E, seed=T + n) + normal(1, E, seed=1)).to(dtype)
        check_route(strided(z, 3) if n == 1 else z, k, normalize=n != 1, scale=(1.0, 2.5, 1.0)[n])
        check_route(z, k, normalize=n == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [False, True])
def test_route_ties_and_masks(normalize):
    z = normal(400, 40, seed=3)
    z[:50] = z[:50].round()             # ties, zeros of both signs
    z[50:100] = 0.0
    z[60:70, ::2] = -0.0
    z[100:200][normal(100, 40, seed=4) > 0] = -torch.inf  # some rows have fewer than k left
    z[150:160, 3:] = -torch.inf
    z[160:170] = -torch.inf             # nothing left
    z[200:210] = torch.finfo(F32).min   # masked by the lowest value, in part and throughout
    z[210:220, 5:] = torch.finfo(F32).min
    z[220] = torch.finfo(F32).max
    z[221, 7] = torch.inf               # no finite softmax: NaN weights, as torch's
    z[222, 9] = torch.nan
    z[223] = torch.nan
    z[224, :20] = -torch.nan
    z[225:230] = 3.0e38 * torch.sign(z[225:230])
    check_route(z, 6, normalize=normalize)
    check_route(z[160:170].clone(), 6, normalize=normalize)  # no token has an expert


@pytest.mark.gpu
def test_route_of_nothing_and_of_everything():
    got = route(torch.empty(0, 9, device=dev()), 2)
    assert not got["offsets"].any()
    z = torch.zeros(3000, 16, device=dev())
    z[:, 11] = 1.0
    got = check_route(z, 1)
    assert got["offsets"].tolist() == [0] * 12 + [3000] * 5
    weights, ids = torch.empty(3000, 1, device=dev()), torch.empty(3000, 1, dtype=I32, device=dev())
    K.route_experts(z, weights=weights, ids=ids)  # without the order
    assert torch.equal(ids, got["ids"]) and torch.equal(weights, got["weights"])


def probabilities(z, ids, normalize):
    there = ids >= 0
    chosen = torch.zeros(z.shape, dtype=torch.bool, device=z.device)
    chosen.scatter_(1, ids.clamp_min(0), there)  # (an id of -1 stands behind those that are there)
    chosen[:, 0] = ((ids == 0) & there).any(1)
    v = z.masked_fill(~chosen, -torch.inf) if normalize else z
    m = v.amax(1, keepdim=True)
    e = torch.exp(v - torch.where(m == -torch.inf, 0.0, m))
    total = e.sum(1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0), there


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("T,E,k", ROUTES)
def test_route_backward(T, E, k, normalize):
    for n, dtype in enumerate(TYPES):
        z = normal(T, E, seed=T + n).to(dtype)
        if T > 60:
            z[10:40][normal(30, E, seed=5) > 0] = -torch.inf
            z[50] = -torch.inf
        z = strided(z, 5)
        ids = route(z, k, normalize=normalize)["ids"]
        dw = normal(T, k, seed=6)
        dz = strided(torch.full((T, E), 7.0, dtype=dtype, device=dev()), 3, fill=7.0)
        K.route_experts_bwd(dw, z, ids, dz, normalize=normalize, scale=1.5)
        p, there = probabilities(z.double(), ids.long(), normalize)
        d = torch.zeros_like(p).scatter_add_(1, ids.long().clamp_min(0), torch.where(there, dw.double(), 0.0))
        dot = (p * d).sum(1, keepdim=True)
        want = 1.5 * p * (d - dot)
        far = (z.double() - z.double().amax(1, keepdim=True)).abs().nan_to_num(0.0, 0.0, 0.0).clamp_max(200.0)
        tol = 1.5 * p * (d.abs() + (p * d.abs()).sum(1, keepdim=True)) * (2 * E * 2.0 ** -24 + far * 2.0 ** -22 + 2.0 ** -19)
        within(dz, want, tol + rounding(want, dtype) + 2.0 ** -126, f"dlogits {dtype}")
        whole = dz._base
        assert bool((whole[:, E:] == 7.0).all())
        again = z.clone()
        K.route_experts_bwd(dw, again, ids, again, normalize=normalize, scale=1.5)
        assert torch.equal(again, dz)


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [False, True])
def test_route_backward_against_differences(normalize):
    """The gradient of the operator's own weights, by central differences. A step
    of 2^-6 leaves an error of its square times a third derivative (at most 1 for
    a softmax), 2^-12 / 6, and the weights' own errors 2 2^-20 / 2^-5."""
    z, dw = normal(5, 12, seed=8), normal(5, 3, seed=9)
    got = route(z, 3, normalize=normalize)
    dz = torch.empty_like(z)
    K.route_experts_bwd(dw, z, got["ids"], dz, normalize=normalize)
    step = 2.0 ** -6
    for e in range(12):
        sides = []
        for s in (step, -step):
            moved = z.clone()
            moved[:, e] += s
            w = route(moved, 12, normalize=False)  # every expert's probability, then those chosen before
            p = torch.zeros(5, 12, device=dev()).scatter_(1, w["ids"].long(), w["weights"]).gather(1, got["ids"].long())
            p = p / p.sum(1, keepdim=True) if normalize else p
            sides.append((p * dw).sum(1).double())
        slope = (sides[0] - sides[1]) / (2 * step)
        assert bool(((dz[:, e].double() - slope).abs() <= dw.abs().sum(1) * (2.0 ** -12 / 6 * 4 + 2.0 ** -14)).all())


# -------------------------------------------------------------------- rows --

def order_of(T, E, k, seed=0, drop=0.0):
    z = normal(T, E, seed=seed) + normal(1, E, seed=seed + 1)
    if drop:
        z[torch.rand(T, E, generator=torch.Generator().manual_seed(seed)).to(dev()) < drop] = -torch.inf
    return route(z, k)


# (tokens, experts, top, H): whole pieces and not, rows of few and many pieces, more entries than are in flight at once
ROWS = [(1, 4, 1, 8), (1, 4, 3, 896), (7, 9, 9, 33), (300, 16, 2, 896), (67, 64, 12, 2048), (130, 8, 4, 3583),
        (4100, 8, 2, 64), (4097, 60, 4, 200), (50, 20, 20, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,H", ROWS)
def test_combine_and_spread(T, E, k, H):
    o = order_of(T, E, k, seed=T, drop=0.4)
    R = T * k
    slots, n = o["slots"], int(o["offsets"][-1])
    at, there = slots.long().clamp_min(0), (slots >= 0)[..., None]
    w = normal(T, k, seed=2)
    for dy, do in ((BF, F32), (BF, BF), (F32, F32), (F32, BF)):
        y = normal(R, H, seed=3).to(dy)
        y[n:] = torch.nan  # (no entry lies there)
        y = strided(y)
        x = strided(normal(T, H, seed=4).to(do), 16)
        terms = torch.where(there, y[at.flatten()].view(T, k, H).double(), 0.0)
        for weights, resid in ((w, x), (w, None), (None, x)):
            out = torch.empty(T, H, dtype=do, device=dev())
            K.combine_experts(y, slots, out, weights=weights, resid=resid)
            t = terms if weights is None else terms * w.double()[..., None]
            base = 0.0 if resid is None else x.double()
            want = t.sum(1) + base
            tol = (k + 2) * 2.0 ** -24 * (t.abs().sum(1) + (0.0 if resid is None else x.double().abs()))
            within(out, want, tol + rounding(want, do), f"combine {dy} {do}")
        again = x.clone()
        K.combine_experts(y, slots, again, weights=w, resid=again)
        K.combine_experts(y, slots, out, weights=w, resid=x)
        assert torch.equal(out, again)
        # back: from x's type to y's
        for weights in (w, None):
            back = strided(torch.full((R, H), 7.0, dtype=dy, device=dev()), 8, fill=7.0)
            dw = torch.full((T, k), 7.0, device=dev())
            K.spread_experts(x, slots, back, weights=weights, y=y, dweights=dw)
            want = x.double()[:, None] * (1.0 if weights is None else w.double()[..., None])
            rows = back[at.flatten()].view(T, k, H)
            within(torch.where(there, rows, 0.0), torch.where(there, want, 0.0).expand(T, k, H),
                   rounding(want, dy) + 2.0 ** -24 * want.abs(), f"spread {do} {dy}")
            assert bool((back[n:] == 7.0).all()) and bool((back._base[:, H:] == 7.0).all())
            prod = x.double()[:, None] * terms
            within(dw, prod.sum(2), (H + 2) * 2.0 ** -24 * prod.abs().sum(2), "dweights")
            plain = torch.full((R, H), 7.0, dtype=dy, device=dev())
            K.spread_experts(x, slots, plain, weights=weights)
            assert torch.equal(plain, back)
        over = y.clone()
        K.spread_experts(x, slots, over, weights=w, y=over, dweights=dw)
        K.spread_experts(x, slots, back, weights=w)
        assert torch.equal(over[:n], back[:n])


@pytest.mark.gpu
def test_no_tokens_and_no_rows():
    none, slots = torch.empty(0, 16, device=dev()), torch.empty(0, 3, dtype=I32, device=dev())
    w = torch.empty(0, 3, device=dev())
    K.combine_experts(normal(4, 16), slots, none, weights=w, resid=none)
    rows = torch.full((4, 16), 7.0, device=dev())
    K.spread_experts(none, slots, rows, weights=w, y=rows, dweights=w)
    assert bool((rows == 7.0).all())
    x, away = normal(5, 16), torch.full((5, 3), -1, dtype=I32, device=dev())
    out, dw = torch.empty(5, 16, device=dev()), torch.full((5, 3), 7.0, device=dev())
    K.combine_experts(none, away, out, resid=x)
    assert torch.equal(out, x)
    K.spread_experts(x, away, none, y=none, dweights=dw)
    assert not dw.any()
    b, off = normal(2, 8, 64).to(BF), torch.zeros(3, dtype=I32, device=dev())
    K.gemm_experts("nt", torch.empty(0, 64, dtype=BF, device=dev()), b, torch.empty(0, 8, device=dev()), offsets=off)
    c = torch.full((2, 8, 16), 7.0, device=dev())
    K.gemm_experts("tn", torch.empty(0, 8, dtype=BF, device=dev()), torch.empty(0, 16, dtype=BF, device=dev()), c, offsets=off)
    assert not c.any()


@pytest.mark.gpu
def test_places_outside_the_rows_are_none():
    slots = torch.tensor([[0, 5, -1], [2, 4, 1 << 30]], dtype=I32, device=dev())
    y, out = normal(4, 16).to(BF), torch.empty(2, 16, device=dev())
    K.combine_experts(y, slots, out)
    assert torch.equal(out, torch.stack([y[0], y[2]]).float())
    x, rows, dw = normal(2, 16, seed=1), torch.zeros(4, 16, device=dev()), torch.empty(2, 3, device=dev())
    K.spread_experts(x, slots, rows, y=torch.ones_like(rows), dweights=dw)
    assert torch.equal(rows[[0, 2]], x) and not rows[[1, 3]].any()
    assert not dw[0, 1:].any() and not dw[1, 1:].any()


# ---------------------------------------------------------------- products --

# rows of each expert: none at all, one, whole tiles and not, each side of the choice of tiles
COUNTS = {"none": [0, 0, 0], "one": [1], "few": [0, 1, 2, 0, 3, 1, 0, 0], "odd": [63, 0, 65, 1, 130, 64, 7],
          "large": [300, 0, 513, 1], "many": [(37 * i * i) % 23 for i in range(150)], "skewed": [0, 5, 1500, 2],
          "whole": [256, 512], "long": [2100, 1, 0, 2900], "tall": [1900, 130, 0, 2300, 1701]}
WEIGHT_SIZES = [(8, 8), (72, 264), (264, 72), (520, 448), (2560, 2560)]
SWIGLU_SIZES = [(32, 64), (96, 128), (288, 192), (704, 448), (96, 2048), (2048, 1024)]
# (N, K): with the counts, every way that a product runs (test_products_take_every_way)
SIZES = [(8, 64), (72, 128), (264, 192), (520, 448), (768, 2048), (2048, 1024)]


def test_products_take_every_way():
    rows = [(len(n), sum(n)) for n in COUNTS.values() if sum(n)]
    for layout, output in (("nt", "bf16"), ("nt", "f32"), ("nn", "bf16"), ("nn", "f32")):
        plans = {K.gemm_experts_plan(layout, output, E, R, N, Kd)[:2] for E, R in rows for N, Kd in SIZES}
        assert {p[0] for p in plans} == {"few", "small", "large"} and any(s > 1 for _, s in plans), (layout, output, plans)
    for layout, output in (("nt", "swiglu"), ("nn", "swiglu_bwd")):
        wide = 2 if layout == "nt" else 1
        plans = {K.gemm_experts_plan(layout, output, E, R, wide * N, Kd)[:2] for E, R in rows for N, Kd in SWIGLU_SIZES}
        assert {p[0] for p in plans} == {"few", "small", "large"} and any(s > 1 for _, s in plans), (output, plans)
    for output in ("f32", "resid"):
        plans = {K.gemm_experts_plan("tn", output, E, M, N, R)[:2] for E, R in rows for M, N in WEIGHT_SIZES}
        assert {p[0] for p in plans} == {"small", "large"} and any(s > 1 for _, s in plans), (output, plans)


def offsets_of(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=I32, device=dev())


def experts_of(counts, extra):
    """The expert of each row, -1 for ``extra`` rows behind them all."""
    return torch.tensor([e for e, n in enumerate(counts) for _ in range(n)] + [-1] * extra, device=dev())


def product(a, w, counts):
    """(float64 products, bound of float32 sums) of rows ``a`` with ``w[e]`` [K, N]."""
    parts, tols, at = [], [], 0
    for e, n in enumerate(counts):
        r = a[at:at + n].double()
        parts.append(r @ w[e].double())
        tols.append(a.shape[1] * 2.0 ** -24 * (r.abs() @ w[e].double().abs()))
        at += n
    return torch.cat(parts), torch.cat(tols)


def stacked(E, rows, cols, seed, std, pad):
    """[E, rows, cols] with rows and experts apart by more than their sizes."""
    whole = torch.full((E, rows + pad, cols + 8 * pad), float("nan"), dtype=BF, device=dev())
    whole[:, :rows, :cols] = normal(E, rows, cols, seed=seed, std=std).to(BF)
    return whole[:, :rows, :cols]


@pytest.mark.gpu
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("N,Kd", SIZES)
def test_rows_products(counts, N, Kd):
    n, extra = COUNTS[counts], 5
    E, R = len(n), sum(COUNTS[counts])
    off = offsets_of(n)
    a = strided(torch.cat([normal(R, Kd, seed=1), torch.full((extra, Kd), torch.nan, device=dev())]).to(BF))
    for layout in ("nt", "nn"):
        b = stacked(E, N, Kd, 2, Kd ** -0.5, 1) if layout == "nt" else stacked(E, Kd, N, 2, Kd ** -0.5, 1)
        want, tol = product(a[:R], b.transpose(1, 2) if layout == "nt" else b, n)
        for dtype in (BF, F32):
            c = strided(torch.full((R + extra, N), 7.0, dtype=dtype, device=dev()), 8, fill=7.0)
            K.gemm_experts(layout, a, b, c, offsets=off)
            within(c[:R], want, tol + rounding(want, dtype), f"{layout} {dtype}")
            assert bool((c[R:] == 7.0).all()) and bool((c._base[:, N:] == 7.0).all())
            if layout == "nt":  # the same rows at an index
                order = torch.randperm(R + extra, generator=torch.Generator().manual_seed(3)).to(dev())
                x = torch.empty_like(a)
                x[order] = a
                other = torch.full((R + extra, N), 7.0, dtype=dtype, device=dev())
                K.gemm_experts("nt", x, b, other, offsets=off, rows=order.to(I32))
                assert torch.equal(other, c)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("M,N", WEIGHT_SIZES)
def test_weight_products(counts, M, N):
    n = COUNTS[counts]
    E, R = len(n), sum(COUNTS[counts])
    off = offsets_of(n)
    dy = strided(normal(R + 3, M, seed=1).to(BF))
    x = strided(normal(R + 3, N, seed=2).to(BF))
    dy[R:], x[R:] = torch.nan, torch.nan
    poisoned = max(range(E), key=lambda e: (n[e] > 0, -n[e]))  # one expert's rows say nothing to the others
    if n[poisoned]:
        dy[int(off[poisoned])], x[int(off[poisoned])] = torch.nan, torch.nan
    start = normal(E, M + 1, N + 8, seed=3)
    for accumulate in (False, True):
        whole = start.clone()
        c = whole[:, :M, :N]
        K.gemm_experts("tn", dy, x, c, offsets=off, accumulate=accumulate)
        for e in range(E):
            a, b = dy[int(off[e]):int(off[e + 1])].double(), x[int(off[e]):int(off[e + 1])].double()
            if e == poisoned and n[e]:
                assert bool(c[e].isnan().all())
                continue
            want, tol = a.t() @ b, n[e] * 2.0 ** -24 * (a.abs().t() @ b.abs())
            if accumulate:
                want, tol = want + start[e, :M, :N].double(), tol + 2.0 ** -24 * (want.abs() + start[e, :M, :N].double().abs())
            within(c[e], want, tol + rounding(want, F32), f"dW of {n[e]} rows")
        assert torch.equal(whole[:, M:], start[:, M:]) and torch.equal(whole[:, :, N:], start[:, :, N:])


@pytest.mark.gpu
def test_weight_products_of_few_rows_each():
    """Large tiles of one short k-tile or of none."""
    n, M, N = COUNTS["many"], 1024, 1032
    assert K.gemm_experts_plan("tn", "f32", len(n), M, N, sum(n))[0] == "large"
    dy, x = normal(sum(n), M, seed=1).to(BF), normal(sum(n), N, seed=2).to(BF)
    c = torch.full((len(n), M, N), 7.0, device=dev())
    K.gemm_experts("tn", dy, x, c, offsets=offsets_of(n))
    at = 0
    for e, rows in enumerate(n):
        a, b = dy[at:at + rows].double(), x[at:at + rows].double()
        within(c[e], a.t() @ b, rows * 2.0 ** -24 * (a.abs().t() @ b.abs()) + rounding(a.t() @ b, F32), f"dW of {rows} rows")
        at += rows


def halves(t):
    v = t.unflatten(-1, (-1, 2, 32))
    return v[..., 0, :].flatten(-2), v[..., 1, :].flatten(-2)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("N,Kd", SWIGLU_SIZES)
def test_swiglu_products(counts, N, Kd):
    n, extra = COUNTS[counts], 4
    E, R = len(n), sum(COUNTS[counts])
    off = offsets_of(n)
    x = torch.cat([normal(R, Kd, seed=1), torch.full((extra, Kd), torch.nan, device=dev())]).to(BF)
    w = stacked(E, 2 * N, Kd, 2, 1.5 * Kd ** -0.5, 1)
    p, tol = product(x[:R], w.transpose(1, 2), n)
    (g, u), (eg, eu) = halves(p), halves(tol)
    want = torch.nn.functional.silu(g) * u
    bound = 1.1 * u.abs() * eg + (torch.nn.functional.silu(g).abs() + 1.1 * eg) * eu + 2.0 ** -20 * (g * u).abs()
    act = strided(torch.full((R + extra, N), 7.0, dtype=BF, device=dev()), 8, fill=7.0)
    gu = torch.full((R + extra, 2 * N), 7.0, dtype=BF, device=dev())
    K.gemm_experts_swiglu(x, w, act, gu, offsets=off)
    within(act[:R], want, bound + rounding(want, BF), "act")
    within(gu[:R], p, tol + rounding(p, BF), "gu")
    assert bool((act[R:] == 7.0).all()) and bool((gu[R:] == 7.0).all()) and bool((act._base[:, N:] == 7.0).all())
    order = torch.randperm(R + extra, generator=torch.Generator().manual_seed(3)).to(dev())
    moved = torch.empty_like(x)
    moved[order] = x
    other = torch.full((R + extra, N), 7.0, dtype=BF, device=dev())
    K.gemm_experts_swiglu(moved, w, other, offsets=off, rows=order.to(I32))
    assert torch.equal(other, act)
    # backward: dact = dy wd[e], the saved gu
    dy = torch.cat([normal(R, Kd, seed=4), torch.full((extra, Kd), torch.nan, device=dev())]).to(BF)
    wd = stacked(E, Kd, N, 5, Kd ** -0.5, 1)
    da, e = product(dy[:R], wd, n)
    g, u = halves(gu[:R].double())
    s = torch.sigmoid(g)
    slope = s * (1 + g * (1 - s))
    for name, part, want, bound in (
            ("dgate", 0, da * u * slope, e * u.abs() * 1.1 + (da * u).abs() * (1 + g.abs()) ** 2 * 2.0 ** -20),
            ("dup", 1, da * g * s, e * g.abs() + (da * g).abs() * 2.0 ** -20)):
        dgu = torch.full((R + extra, 2 * N), 7.0, dtype=BF, device=dev())
        K.gemm_experts_swiglu_bwd(dy, wd, gu, dgu, offsets=off)
        within(halves(dgu[:R])[part], want, bound + rounding(want, BF), name)
        assert bool((dgu[R:] == 7.0).all())
    over = gu.clone()
    K.gemm_experts_swiglu_bwd(dy, wd, over, over, offsets=off)
    assert torch.equal(over, dgu)


@pytest.mark.gpu
@pytest.mark.parametrize("R,N,Kd", [(100, 40, 64), (3000, 264, 128), (8000, 2048, 1024)])
def test_offsets_that_descend_stay_inside(R, N, Kd):
    """Nothing but the product's own rows is written, whatever the offsets say."""
    off = torch.tensor([R, 0, R // 2, 7, R, -3, R, 1 << 30, 0, R], dtype=I32, device=dev())
    E = off.numel() - 1
    a, b = normal(R, Kd, seed=1).to(BF), normal(E, N, Kd, seed=2).to(BF)
    whole = torch.full((R + 16, N), 7.0, dtype=BF, device=dev())
    K.gemm_experts("nt", a, b, whole[8:R + 8], offsets=off)
    torch.cuda.synchronize()
    assert bool((whole[:8] == 7.0).all()) and bool((whole[R + 8:] == 7.0).all())
    dw = torch.full((E + 2, Kd, N), 7.0, device=dev())
    K.gemm_experts("tn", a, normal(R, N, seed=3).to(BF), dw[1:E + 1], offsets=off)
    torch.cuda.synchronize()
    assert bool((dw[0] == 7.0).all()) and bool((dw[E + 1] == 7.0).all())


@pytest.mark.gpu
def test_offsets_and_indices_outside_lead_nowhere():
    """Values that no routing gives count as the nearest that one could."""
    a, b = normal(100, 64, seed=1).to(BF), normal(3, 40, 64, seed=2).to(BF)
    c = torch.full((100, 40), 7.0, device=dev())
    K.gemm_experts("nt", a, b, c, offsets=torch.tensor([-9, 50, 1 << 30, 1 << 30], dtype=I32, device=dev()))
    want = torch.full((100, 40), 7.0, device=dev())
    K.gemm_experts("nt", a, b, want, offsets=torch.tensor([0, 50, 100, 100], dtype=I32, device=dev()))
    assert torch.equal(c, want) and not bool((c == 7.0).any())
    index = torch.arange(100, dtype=I32, device=dev())
    index[3], index[70] = -5, 1 << 30
    K.gemm_experts("nt", a, b, c, offsets=torch.tensor([0, 50, 100, 100], dtype=I32, device=dev()), rows=index)
    one = torch.empty(1, 40, device=dev())
    for r, source, e in ((3, 0, 0), (70, 99, 1)):
        K.gemm_experts("nt", a[source:source + 1], b[e:e + 1], one, offsets=torch.tensor([0, 1], dtype=I32, device=dev()))
        assert torch.allclose(c[r], one[0], rtol=0, atol=1e-4)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows that start past 2^31 elements are those that the same call on few rows
    gives."""
    R, H, T = 70000, 32768, 40
    y = torch.zeros(R, H, dtype=BF, device=dev())
    slots = torch.arange(R - 2 * T, R, dtype=I32, device=dev()).view(T, 2)
    y[R - 2 * T:] = normal(2 * T, H, seed=1).to(BF)
    w = normal(T, 2, seed=2)
    out, near = torch.empty(T, H, device=dev()), torch.empty(T, H, device=dev())
    K.combine_experts(y, slots, out, weights=w)
    K.combine_experts(y[R - 2 * T:], slots - (R - 2 * T), near, weights=w)
    assert torch.equal(out, near)
    back, dw, dw_near = torch.empty(2 * T, H, dtype=BF, device=dev()), torch.empty_like(w), torch.empty_like(w)
    K.spread_experts(near, slots - (R - 2 * T), back, weights=w, y=y[R - 2 * T:].clone(), dweights=dw_near)
    K.spread_experts(out, slots, y, weights=w, y=y, dweights=dw)
    assert torch.equal(y[R - 2 * T:], back) and torch.equal(dw, dw_near)
    del y, back
    R, Kd, N = 1 << 20, 2112, 40  # the second expert's rows start past 2^31 elements of a
    a = torch.zeros(R, Kd, dtype=BF, device=dev())
    a[R - 300:] = normal(300, Kd, seed=3).to(BF)
    b = normal(2, N, Kd, seed=4).to(BF)
    c = torch.empty(R, N, device=dev())
    K.gemm_experts("nt", a, b, c, offsets=torch.tensor([0, R - 200, R], dtype=I32, device=dev()))
    want, tol = product(a[R - 300:], b.transpose(1, 2), [100, 200])
    within(c[R - 300:], want, tol + rounding(want, F32), "far rows")
    dw = torch.empty(2, N, Kd, device=dev())
    g = torch.zeros(R, N, dtype=BF, device=dev())
    g[R - 300:] = normal(300, N, seed=5).to(BF)
    K.gemm_experts("tn", g, a, dw, offsets=torch.tensor([0, R - 200, R], dtype=I32, device=dev()))
    for e, r in ((0, slice(R - 300, R - 200)), (1, slice(R - 200, R))):
        want, mag = g[r].double().t() @ a[r].double(), g[r].double().abs().t() @ a[r].double().abs()
        within(dw[e], want, 300 * 2.0 ** -24 * mag + rounding(want, F32), "far rows' gradients")


# (rows, N, experts), a way of products each
FAR = {"few": (40, 72, 12), "small": (1500, 264, 3), "large": (8192, 2048, 2)}


def test_far_products_take_every_way():
    for way, (R, N, E) in FAR.items():
        assert K.gemm_experts_plan("nt", "bf16", E, R, N, 2048)[0] == way
        assert K.gemm_experts_plan("nt", "swiglu", E, R, 2 * N // 64 * 64, 2048)[0] == way


@pytest.mark.gpu
@pytest.mark.parametrize("way", FAR)
def test_rows_at_an_index_up_to_4_gib(way):
    """The same bits as of those rows side by side, to the last row that an index reaches."""
    R, N, E = FAR[way]
    rows, H, near = 2 ** 20 - 1, 2048, 500
    x = torch.zeros(rows, H, dtype=BF, device=dev())
    x[:near], x[rows - near:] = normal(near, H, seed=1).to(BF), normal(near, H, seed=2).to(BF)
    x[2 ** 19 - near:2 ** 19 + near] = normal(2 * near, H, seed=3).to(BF)  # either side of 2^31 bytes
    pick = torch.randint(0, 4 * near, (R,), generator=torch.Generator().manual_seed(4)).to(dev())
    pick[0], pick[-1] = 4 * near - 1, 0
    index = torch.cat([torch.arange(near), torch.arange(2 ** 19 - near, 2 ** 19 + near), torch.arange(rows - near, rows)]).to(dev())[pick]
    side = x[index]
    assert not bool((side.abs().amax(1) == 0).any())
    off = offsets_of([R // E] * (E - 1) + [R - R // E * (E - 1)])
    b = normal(E, N, H, seed=5, std=H ** -0.5).to(BF)
    got, want = torch.full((R, N), 7.0, dtype=BF, device=dev()), torch.full((R, N), 5.0, dtype=BF, device=dev())
    K.gemm_experts("nt", x, b, got, offsets=off, rows=index.to(I32))
    K.gemm_experts("nt", side, b, want, offsets=off)
    assert torch.equal(got, want)
    n = N // 64 * 32
    act, same = torch.full((R, n), 7.0, dtype=BF, device=dev()), torch.full((R, n), 5.0, dtype=BF, device=dev())
    K.gemm_experts_swiglu(x, b[:, :2 * n], act, offsets=off, rows=index.to(I32))
    K.gemm_experts_swiglu(side, b[:, :2 * n], same, offsets=off)
    assert torch.equal(act, same)


# -------------------------------------------------------------- an expert MLP --

class ExpertMLP:
    """out = x + sum of a token's k experts' SwiGLU MLPs, and its backward, as a
    user chains the operators: buffers once, no counts on the host."""

    def __init__(self, T, E, k, h, inter, seed=0):
        e = lambda *s, dt=BF: torch.full(s, 3.0, dtype=dt, device=dev())
        R = T * k
        self.T, self.E, self.k, self.h, self.inter = T, E, k, h, inter
        self.router = normal(E, h, seed=seed, std=2 * h ** -0.5).to(BF)
        self.wgu = normal(E, 2 * inter, h, seed=seed + 1, std=h ** -0.5).to(BF)
        self.wd = normal(E, h, inter, seed=seed + 2, std=inter ** -0.5).to(BF)
        self.logits, self.w, self.ids = e(T, E, dt=F32), e(T, k, dt=F32), e(T, k, dt=I32)
        self.off, self.slots, self.rows = e(E + 1, dt=I32), e(T, k, dt=I32), e(R, dt=I32)
        self.act, self.gu, self.y = e(R, inter), e(R, 2 * inter), e(R, h)
        self.out = e(T, h, dt=F32)
        self.dy, self.dgu, self.dxs, self.xs = e(R, h), e(R, 2 * inter), e(R, h), e(R, h)
        self.dw, self.dlogits, self.dx = e(T, k, dt=F32), e(T, E, dt=F32), e(T, h, dt=F32)
        self.dlogits16 = e(T, E)
        self.dwd, self.dwgu, self.drouter = e(E, h, inter, dt=F32), e(E, 2 * inter, h, dt=F32), e(E, h, dt=F32)

    def forward(self, x, x16):
        self.logits.copy_(x16.float() @ self.router.float().t())
        K.route_experts(self.logits, weights=self.w, ids=self.ids, offsets=self.off, slots=self.slots, rows=self.rows,
                        normalize=True)
        K.gemm_experts_swiglu(x16, self.wgu, self.act, self.gu, offsets=self.off, rows=self.rows)
        K.gemm_experts("nt", self.act, self.wd, self.y, offsets=self.off)
        if x is not None:
            K.combine_experts(self.y, self.slots, self.out, weights=self.w, resid=x)

    def backward(self, dout, x16, resid=True):
        K.spread_experts(dout, self.slots, self.dy, weights=self.w, y=self.y, dweights=self.dw)
        K.gemm_experts("tn", self.dy, self.act, self.dwd, offsets=self.off)
        K.gemm_experts_swiglu_bwd(self.dy, self.wd, self.gu, self.dgu, offsets=self.off)
        K.spread_experts(x16, self.slots, self.xs)
        K.gemm_experts("tn", self.dgu, self.xs, self.dwgu, offsets=self.off)
        K.gemm_experts("nn", self.dgu, self.wgu, self.dxs, offsets=self.off)
        K.route_experts_bwd(self.dw, self.logits, self.ids, self.dlogits, normalize=True)
        K.combine_experts(self.dxs, self.slots, self.dx, resid=dout if resid else None)
        self.dx += self.dlogits @ self.router.float()

    def outputs(self):
        return {n: getattr(self, n).clone() for n in ("out", "w", "dwd", "dwgu", "dlogits", "dx")}


def reference(m, x, x16, dout):
    """By autograd in float64, the experts that the operators chose."""
    x16d = x16.double().requires_grad_()
    wgu, wd = m.wgu.double().requires_grad_(), m.wd.double().requires_grad_()
    logits = (x16d @ m.router.double().t())
    logits.retain_grad()
    w = torch.softmax(logits.gather(1, m.ids.long()), 1)
    out = x.double()
    for e in range(m.E):
        t, j = torch.nonzero(m.ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        g, u = halves(x16d[t] @ wgu[e].t())
        out = out.index_add(0, t, w[t, j, None] * ((torch.nn.functional.silu(g) * u) @ wd[e].t()))
    out.backward(dout.double())
    return {"out": out, "w": w, "dwd": wd.grad, "dwgu": wgu.grad, "dlogits": logits.grad,
            "dx": x16d.grad + dout.double()}


# (tokens, experts, top, hidden, intermediate)
MLPS = [(1, 8, 2, 64, 64), (9, 64, 8, 128, 128), (500, 8, 2, 320, 192), (1300, 4, 3, 256, 320)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,h,inter", MLPS)
def test_expert_mlp(T, E, k, h, inter):
    """The chain against float64. Each bfloat16 rounding on a value's way (act, gu,
    y, dy, dgu, dx of the rows: at most four) is off by at most 2^-8 of its value, so by
    less than 2^-8 of the norm; what they are summed with grows none of it."""
    m = ExpertMLP(T, E, k, h, inter)
    x = normal(T, h, seed=7)
    x16, dout = x.to(BF), normal(T, h, seed=8)
    m.forward(x, x16)
    m.backward(dout, x16)
    got, want = m.outputs(), reference(m, x, x16, dout)
    for name, g in got.items():
        err = (g.double() - want[name]).norm() / want[name].norm()
        assert float(err.detach()) <= 4 * 2.0 ** -8, (name, float(err.detach()))


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,h,inter", MLPS)
def test_expert_mlp_between_norms(T, E, k, h, inter):
    """The MLP's half of a decoder block with norms before and behind the branch, a
    gate and a scale, forward and back, against float64. The roundings on a value's way
    are the MLP's four and those of x, the branch and their gradients: at most eight."""
    m = ExpertMLP(T, E, k, h, inter)
    stream, y0 = normal(T, h, seed=11), normal(T, h, seed=12).to(BF)
    pre, post, gate = (1 + normal(h, seed=s, std=0.2) for s in (13, 14, 15))
    dout = normal(T, h, seed=16)
    e = lambda dt: torch.full((T, h), 3.0, dtype=dt, device=dev())
    h1, x16, y1, out = e(F32), e(BF), e(BF), e(F32)
    K.norm_residual(y0, stream, h1, eps=1e-6, pre=pre, normed=x16)
    m.forward(None, x16)
    K.combine_experts(m.y, m.slots, y1, weights=m.w)
    K.norm_residual(y1, h1, out, eps=1e-6, post=post, gate=gate[None], scale=0.5)
    dy1, dh1, dx16, dy0, dstream = e(BF), e(F32), e(BF), e(BF), e(F32)
    dpost, dgate, dpre = (torch.empty(h, device=dev()) for _ in range(3))
    K.norm_residual_bwd(None, dout, y1, out, dy1, dh1, eps=1e-6, post=post, gate=gate[None], scale=0.5, dpost=dpost,
                        dgate=dgate[None])
    m.backward(dy1, x16, resid=False)
    dx16.copy_(m.dx)
    K.norm_residual_bwd(dx16, dh1, y0, h1, dy0, dstream, eps=1e-6, pre=pre, dpre=dpre)
    got = dict(out=out, dy0=dy0, dstream=dstream, dpost=dpost, dgate=dgate, dpre=dpre, dwd=m.dwd, dwgu=m.dwgu)

    leaf = {n: t.double().requires_grad_() for n, t in dict(y0=y0, stream=stream, pre=pre, post=post, gate=gate, wgu=m.wgu,
                                                             wd=m.wd).items()}
    rms = lambda v: v * (v.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    r1 = leaf["stream"] + leaf["y0"]
    x = rms(r1) * leaf["pre"]
    w = torch.softmax((x @ m.router.double().t()).gather(1, m.ids.long()), 1)
    branch = torch.zeros_like(r1)
    for i in range(E):
        t, j = torch.nonzero(m.ids == i, as_tuple=True)
        if t.numel():
            g, u = halves(x[t] @ leaf["wgu"][i].t())
            branch = branch.index_add(0, t, w[t, j, None] * ((torch.nn.functional.silu(g) * u) @ leaf["wd"][i].t()))
    r2 = r1 + 0.5 * leaf["gate"] * (rms(branch) * leaf["post"])
    r2.backward(dout.double())
    grad = {n: t.grad for n, t in leaf.items()}
    want = dict(out=r2.detach(), dy0=grad["y0"], dstream=grad["stream"], dpost=grad["post"], dgate=grad["gate"],
                dpre=grad["pre"], dwd=grad["wd"], dwgu=grad["wgu"])
    for name, v in got.items():
        err = (v.double() - want[name]).norm() / want[name].norm()
        assert float(err) <= 8 * 2.0 ** -8, (name, float(err))


@pytest.mark.gpu
def test_expert_mlp_in_a_graph():
    """One capture serves batches whose tokens choose other experts, between eager
    runs of the same chain."""
    T, E, k, h, inter = 200, 16, 4, 128, 128
    m, eager = ExpertMLP(T, E, k, h, inter), ExpertMLP(T, E, k, h, inter)
    x, x16, dout = torch.zeros(T, h, device=dev()), torch.zeros(T, h, dtype=BF, device=dev()), torch.zeros(T, h, device=dev())

    def step(mlp):
        mlp.forward(x, x16)
        mlp.backward(dout, x16)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(m)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(m)
    for seed in range(4):
        x.copy_(normal(T, h, seed=20 + seed))
        x16.copy_(x)
        dout.copy_(normal(T, h, seed=30 + seed))
        step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for (name, a), b in zip(m.outputs().items(), eager.outputs().values()):
            assert torch.equal(a, b), (seed, name)


@pytest.mark.gpu
def test_two_streams_at_once():
    a, b = ExpertMLP(300, 8, 2, 128, 128), ExpertMLP(2000, 32, 4, 128, 128, seed=5)
    data = [(normal(m.T, m.h, seed=i), normal(m.T, m.h, seed=i + 10)) for i, m in enumerate((a, b))]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for m, s, (x, dout) in zip((a, b), streams, data):
            with torch.cuda.stream(s):
                x16 = x.to(BF)
                m.forward(x, x16)
                m.backward(dout, x16)
                x16.record_stream(s)
    torch.cuda.synchronize()
    for m, (x, dout) in zip((a, b), data):
        got = m.outputs()
        m.forward(x, x.to(BF))
        m.backward(dout, x.to(BF))
        for name, want in m.outputs().items():
            assert torch.equal(got[name], want), name


# ---------------------------------------------------------------- refusals --

A = 1 << 20  # addresses that are never read: every call below is refused on the host


def address(i):
    return ctypes.c_void_p(A * (i + 1) * 4096)


def refused(fn, args, message):
    lib = K.lib()
    assert getattr(lib, fn)(*args) == K.MR_EINVAL
    assert message in lib.mr_last_error().decode(), lib.mr_last_error()


ROUTE = dict(z=address(0), dtype=0, ld=64, T=300, E=64, k=8, normalize=0, scale=1.0, w=address(1), ids=address(2),
             off=address(3), slots=address(4), rows=address(5), ws=address(6), ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=9), "dtype"), (dict(k=65, E=128, ld=128), "at most 64"), (dict(E=513, ld=513), "at most 512"),
    (dict(k=9, E=8, ld=8), "no more than"), (dict(k=0), "no experts"), (dict(E=0, k=1), "no experts"), (dict(T=-1), "negative"),
    (dict(ld=63), "leading dimension"), (dict(z=ctypes.c_void_p(A + 2)), "aligned"), (dict(w=ctypes.c_void_p(A + 2)), "aligned"),
    (dict(slots=None), "together"), (dict(off=None), "together"), (dict(z=None), "null"), (dict(ids=None), "null"),
    (dict(ws_bytes=8), "workspace"), (dict(ws=None), "workspace"), (dict(ids=address(0)), "overlap"),
    (dict(T=1 << 28), "too many"), (dict(rows=address(4)), "overlap")])
def test_route_refuses(change, message):
    refused("mr_route_experts", list(dict(ROUTE, **change).values()), message)


def test_route_refuses_tokens_whose_blocks_end_past_31_bits():
    """256 blocks of whole runs of 64 tokens: the last one ends at 2^31 from 2^31 - 2^14 + 1 tokens on."""
    most = 2 ** 31 - 2 ** 14
    ends = lambda T: -(-T // 256 // 64) * 64 * 256
    assert ends(most) < 2 ** 31 <= ends(most + 1)
    far = {n: ctypes.c_void_p((i + 1) << 40) for i, n in enumerate(("z", "w", "ids", "off", "slots", "rows", "ws"))}
    base = dict(ROUTE, **far, E=1, k=1, ld=1)
    for T in (most + 1, 2 ** 31 - 1, 2 ** 31):
        refused("mr_route_experts", list(dict(base, T=T).values()), "too many")
    refused("mr_route_experts", list(dict(base, T=most, ws_bytes=8).values()), "workspace")


BACK = dict(dw=address(1), z=address(0), dtype=0, ld=64, ids=address(2), T=300, E=64, k=8, normalize=0, scale=1.0,
            dz=address(3), lddz=64, stream=None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), "dtype"), (dict(lddz=60), "leading dimension"), (dict(dz=None), "null"), (dict(dz=address(2)), "overlaps"),
    (dict(dz=address(0), lddz=65), "may be the logits"), (dict(dz=ctypes.c_void_p(A + 2)), "aligned")])
def test_route_backward_refuses(change, message):
    refused("mr_route_experts_bwd", list(dict(BACK, **change).values()), message)


COMBINE = dict(y=address(0), ydt=1, ldy=64, R=100, slots=address(1), w=address(2), T=50, k=2, H=64, resid=address(3),
               ldr=64, out=address(4), odt=0, ldo=64, stream=None)
SPREAD = dict(x=address(0), xdt=0, ldx=64, slots=address(1), w=address(2), T=50, k=2, H=64, out=address(3), odt=1, ldo=64,
              R=100, y=address(4), ldy=64, dw=address(5), stream=None)


@pytest.mark.parametrize("fn,base,change,message", [
    ("mr_combine_experts", COMBINE, dict(ydt=2), "fp32 or bf16"), ("mr_combine_experts", COMBINE, dict(ldy=63), "leading"),
    ("mr_combine_experts", COMBINE, dict(out=address(0)), "overlaps"), ("mr_combine_experts", COMBINE, dict(slots=None), "null"),
    ("mr_combine_experts", COMBINE, dict(k=0), "no experts"), ("mr_combine_experts", COMBINE, dict(y=None), "null"),
    ("mr_combine_experts", COMBINE, dict(out=address(3), ldo=65), "may be resid"),
    ("mr_spread_experts", SPREAD, dict(odt=2), "fp32 or bf16"), ("mr_spread_experts", SPREAD, dict(ldx=63), "leading"),
    ("mr_spread_experts", SPREAD, dict(y=None), "together"), ("mr_spread_experts", SPREAD, dict(dw=None), "together"),
    ("mr_spread_experts", SPREAD, dict(out=address(0)), "overlap"), ("mr_spread_experts", SPREAD, dict(out=None), "null"),
    ("mr_spread_experts", SPREAD, dict(dw=ctypes.c_void_p(A + 2)), "aligned")])
def test_rows_refuse(fn, base, change, message):
    refused(fn, list(dict(base, **change).values()), message)


@pytest.mark.parametrize("fn,base,k", [("mr_route_experts", ROUTE, 8), ("mr_route_experts_bwd", BACK, 8),
                                       ("mr_combine_experts", COMBINE, 4), ("mr_spread_experts", SPREAD, 4)])
def test_products_of_sizes_that_pass_64_bits_are_refused(fn, base, k):
    refused(fn, list(dict(base, T=1 << 62, k=k).values()), "too")


def test_spread_refuses_columns_whose_steps_pass_31_bits():
    """A block goes over a row 256 columns at a time, and past its end by less than one step."""
    far = {n: ctypes.c_void_p((i + 1) << 40) for i, n in enumerate(("x", "slots", "w", "out", "y", "dw"))}
    for H in (2 ** 31 - 1, 2 ** 31 - 256):
        refused("mr_spread_experts", list(dict(SPREAD, **far, T=1, k=1, R=1, H=H, ldx=H, ldo=H, ldy=H).values()), "too large")
    H = 2 ** 31 - 257
    refused("mr_spread_experts", list(dict(SPREAD, **far, T=1, k=1, R=1, H=H, ldx=H, ldo=H, ldy=H - 1).values()), "leading")


@pytest.mark.parametrize("sizes", [(1 << 62, 8, 64, 64), (4, 1 << 62, 64, 64), (4, 8, 1 << 62, 64), (4, 8, 64, 1 << 62)])
def test_plans_of_sizes_past_32_bits_are_refused(sizes):
    out = [ctypes.byref(ctypes.c_int()), ctypes.byref(ctypes.c_int()), ctypes.byref(ctypes.c_size_t())]
    refused("mr_gemm_experts_plan", [0, 1, *sizes, *out], "too large")
    assert K.lib().mr_gemm_experts_workspace_bytes(0, 1, *sizes) == 0


GEMM = dict(layout=0, E=4, M=100, N=64, K=128, A=address(0), lda=128, index=None, a_rows=0, B=address(1), ldb=128,
            b_step=64 * 128, off=address(2), C=address(3), cdt=1, ldc=64, c_step=0, acc=0, ws=None, ws_bytes=0, stream=None)
TN = dict(GEMM, layout=2, M=64, K=100, lda=64, ldb=64, cdt=0, c_step=64 * 64)


@pytest.mark.parametrize("base,change,message", [
    (GEMM, dict(layout=3), "layout"), (GEMM, dict(E=0), "no experts"), (GEMM, dict(K=100), "multiple of 64"), (GEMM, dict(K=0), "64"),
    (GEMM, dict(N=60), "multiple of 8"), (GEMM, dict(cdt=2), "fp32 or bf16"), (GEMM, dict(A=None), "null"),
    (GEMM, dict(off=None), "null"), (GEMM, dict(lda=120), "smaller"), (GEMM, dict(ldc=56), "smaller"),
    (GEMM, dict(ldb=132), "multiples"), (GEMM, dict(b_step=64 * 128 - 8), "overlap"), (GEMM, dict(b_step=64 * 128 + 4), "multiples"),
    (GEMM, dict(C=address(0)), "overlap"), (GEMM, dict(acc=1), "added"), (GEMM, dict(lda=1 << 23), "leading dimensions above"),
    (GEMM, dict(index=address(4), a_rows=0), "4 GiB"), (GEMM, dict(index=address(4), a_rows=1 << 30), "4 GiB"),
    (GEMM, dict(index=address(4), layout=1, ldb=64), "nt"), (GEMM, dict(A=ctypes.c_void_p(A + 2)), "aligned"),
    (GEMM, dict(ws=address(0), ws_bytes=1 << 20), "overlap"), (GEMM, dict(ws=ctypes.c_void_p(A + 8), ws_bytes=64), "aligned"),
    (TN, dict(cdt=1), "fp32"), (TN, dict(M=60, lda=64), "multiples of 8"), (TN, dict(c_step=4092), "overlap"),
    (TN, dict(index=address(4), a_rows=5), "nt"), (TN, dict(lda=56), "smaller")])
def test_products_refuse(base, change, message):
    refused("mr_gemm_experts", list(dict(base, **change).values()), message)


def test_weight_products_refuse_rows_whose_tiles_end_past_31_bits():
    """An expert with every row has k-tiles of 64 up to the next multiple of 64."""
    far = {n: ctypes.c_void_p((i + 1) << 40) for i, n in enumerate(("A", "B", "off", "C"))}
    base = dict(TN, **far, M=8, N=8, lda=8, ldb=8, ldc=8, c_step=64)
    for rows in (2 ** 31 - 63, 2 ** 31 - 1):
        refused("mr_gemm_experts", list(dict(base, K=rows).values()), "too large")
    refused("mr_gemm_experts", list(dict(base, K=2 ** 31 - 64, c_step=56).values()), "overlap")


SWIGLU = dict(E=4, M=100, N=64, K=128, X=address(0), ldx=128, index=None, rows=0, W=address(1), ldw=128, step=128 * 128,
              off=address(2), act=address(3), ldact=64, gu=address(4), ldgu=128, ws=None, ws_bytes=0, stream=None)
SWIGLU_BWD = dict(E=4, M=100, N=64, K=128, dy=address(0), ldd=128, W=address(1), ldw=64, step=128 * 64, off=address(2),
                  gu=address(3), ldgu=128, dgu=address(4), lddgu=128, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("fn,base,change,message", [
    ("mr_gemm_experts_swiglu", SWIGLU, dict(N=40), "32"), ("mr_gemm_experts_swiglu", SWIGLU, dict(ldgu=64), "smaller"),
    ("mr_gemm_experts_swiglu", SWIGLU, dict(gu=address(3)), "overlap"), ("mr_gemm_experts_swiglu", SWIGLU, dict(step=8), "overlap"),
    ("mr_gemm_experts_swiglu", SWIGLU, dict(act=None), "null"),
    ("mr_gemm_experts_swiglu_bwd", SWIGLU_BWD, dict(N=40), "32"), ("mr_gemm_experts_swiglu_bwd", SWIGLU_BWD, dict(K=96), "64"),
    ("mr_gemm_experts_swiglu_bwd", SWIGLU_BWD, dict(dgu=address(0)), "overlap"),
    ("mr_gemm_experts_swiglu_bwd", SWIGLU_BWD, dict(dgu=address(3), lddgu=136), "unless dgu is gu"),
    ("mr_gemm_experts_swiglu_bwd", SWIGLU_BWD, dict(gu=None), "null"),
    ("mr_gemm_experts_swiglu_bwd", SWIGLU_BWD, dict(dgu=address(3), ws=address(3), ws_bytes=1 << 10), "workspace")])
def test_swiglu_refuses(fn, base, change, message):
    refused(fn, list(dict(base, **change).values()), message)


def test_bindings_refuse():
    """Types and shapes, before any address is asked for."""
    z, i = torch.zeros(4, 8), torch.zeros(4, 2, dtype=I32)
    w, off, rows = torch.zeros(4, 2), torch.zeros(9, dtype=I32), torch.zeros(8, dtype=I32)
    x, b = torch.zeros(8, 64, dtype=BF), torch.zeros(8, 16, 64, dtype=BF)
    for call in (
            lambda: K.route_experts(z, weights=w, ids=i.long()),
            lambda: K.route_experts(z, weights=w.double(), ids=i),
            lambda: K.route_experts(z, weights=w, ids=i, offsets=off),
            lambda: K.route_experts(z, weights=w, ids=i, offsets=off[:-1], slots=i, rows=rows),
            lambda: K.route_experts(z[0], weights=w, ids=i),
            lambda: K.route_experts_bwd(w, z, i, z.half()),
            lambda: K.gemm_experts("tt", x, b, torch.zeros(8, 16), offsets=off),
            lambda: K.gemm_experts("nt", x.float(), b, torch.zeros(8, 16), offsets=off),
            lambda: K.gemm_experts("nt", x, b[:7], torch.zeros(8, 16), offsets=off),
            lambda: K.gemm_experts("nt", x, b, torch.zeros(7, 16), offsets=off),
            lambda: K.gemm_experts("nt", x, b, torch.zeros(8, 16), offsets=off.long()),
            lambda: K.gemm_experts("tn", x, x, torch.zeros(8, 64, 64), offsets=off, rows=rows),
            lambda: K.gemm_experts_swiglu(x, b, torch.zeros(8, 16, dtype=BF), offsets=off),
            lambda: K.gemm_experts_swiglu_bwd(x, b.transpose(1, 2), x, x, offsets=off),
            lambda: K.combine_experts(x, i, torch.zeros(4, 64), resid=torch.zeros(4, 64, dtype=BF)),
            lambda: K.combine_experts(x, i.long(), torch.zeros(4, 64)),
            lambda: K.spread_experts(torch.zeros(4, 64), i, x, dweights=w),
            lambda: K.spread_experts(torch.zeros(4, 32), i, x),
            lambda: K.route_experts(z, weights=w, ids=i)):  # (host tensors)
        with pytest.raises(KernelError):
            call()
