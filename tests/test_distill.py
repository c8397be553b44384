"""A row's top logits (``top_logits``) and the distillation loss against them
(``distill_loss``), against their definitions in float64, and what they refuse.

Bounds. An exponential is off by 2 units of its argument's rounding and one of
its own; a thread adds at most V / 1024 + 8 of them in a row before the sums of
threads meet in a tree of 10 levels: a row's sum is off by (V / 1024 + 40) 2^-24
of itself (``unit``), its logarithm by as much. A probability carries besides
4 |u - max| 2^-24 of its argument. Outputs round by half a unit of their type.
"""

from __future__ import annotations

import ctypes
import math
import sys

import numpy as np
import pytest
import torch

from mround_amd import kernels as K
from mround_amd.exceptions import KernelError
from tests.helpers import dev

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def unit(V):
    return (V / 1024 + 40) * 2.0 ** -24


# ------------------------------------------------------------------ top logits --

def ordered(z, k):
    """ids of the k largest of each row, NaN first, ties to the lower index (a stable sort)."""
    key = np.where(np.isnan(z), np.inf, z)
    nan = np.isnan(z)
    return np.stack([np.lexsort((np.arange(z.shape[1]), -key[r], ~nan[r]))[:k] for r in range(z.shape[0])])


def run_top(z, V, k, temperature=1.0):
    T = z.shape[0]
    values = torch.empty(T, k, device=dev())
    ids = torch.empty(T, k, dtype=torch.int32, device=dev())
    lse = torch.empty(T, device=dev())
    K.top_logits(z, V=V, values=values, ids=ids, lse=lse, temperature=temperature)
    return values, ids, lse


def check_top(z, k, temperature=1.0):
    """``z`` on the CPU in its type; rows whose width is odd start off 16 bytes."""
    values, ids, lse = run_top(z.to(dev()), z.shape[1], k, temperature)
    z64 = z.double().numpy()
    want = ordered(z64, k)
    assert np.array_equal(ids.cpu().numpy(), want)
    assert np.array_equal(values.cpu().double().numpy(), np.take_along_axis(z64, want, 1), equal_nan=True)
    ref = torch.logsumexp(z.double() / temperature, 1)
    got = lse.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    finite = torch.isfinite(ref)
    assert torch.equal(got[~finite & ~torch.isnan(ref)], ref[~finite & ~torch.isnan(ref)])
    tol = unit(z.shape[1]) + 2.0 ** -24 * ref.abs()
    assert bool(((got - ref).abs() <= tol)[finite].all()), float(((got - ref).abs() - tol)[finite].max())


TOP_CASES = [(1, 1, 1), (3, 7, 7), (2, 8, 3), (5, 100, 100), (4, 1000, 1), (4, 2047, 300), (3, 2049, 1024),
             (2, 3000, 1000), (3, 8191, 512), (2, 20000, 1024), (3, 70001, 64), (2, 151936, 64), (2, 151936, 700),
             (1, 200001, 20)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", TOP_CASES, ids=lambda c: "x".join(map(str, c)))
def test_top_logits(case, dtype):
    T, V, k = case
    print("case top", case, dtype, file=sys.stderr, flush=True)
    z = (torch.randn(T, V, generator=torch.Generator().manual_seed(V + k)) * 3).to(DT[dtype])
    check_top(z, k, temperature=1.0)
    check_top(z, k, temperature=2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("V", [30, 2048, 9000, 60001])
@pytest.mark.parametrize("kind", ["equal", "two", "rising", "falling", "far", "infinite", "nan", "low", "zeros"])
def test_top_logits_of_odd_rows(kind, V, dtype):
    """Ties beyond any list, sorted rows, infinities, NaN, rows of the lowest values, zeros of both signs."""
    k = min(V, 257)
    print("case top odd", kind, V, dtype, file=sys.stderr, flush=True)
    g = torch.Generator().manual_seed(4)
    z = torch.randn(3, V, generator=g)
    if kind == "equal":
        z = torch.full((3, V), -1.5)
    elif kind == "two":
        z = (z > 0.3).float()
    elif kind == "rising":
        z = torch.arange(V).float().expand(3, V) / 64
    elif kind == "falling":
        z = -torch.arange(V).float().expand(3, V) / 64
    elif kind == "far":
        z = z * 1e4
    elif kind == "infinite":
        z[:, V // 3] = math.inf
        z[1] = -math.inf
        z[2, ::2] = -math.inf
    elif kind == "nan":
        z[0, V // 2] = z[0, 1] = math.nan
        z[1, -1] = -math.nan
        z[2, 0] = math.nan
        z[2, 3] = math.inf
    elif kind == "low":
        z = torch.full((3, V), torch.finfo(DT[dtype]).min)
        z[1, -1] = 0.0
        z[2, : V // 2] = -math.inf
    elif kind == "zeros":
        z = torch.zeros(3, V)
        z[:, 1::2] = -0.0
    check_top(z.to(DT[dtype]), k)


@pytest.mark.gpu
def test_top_logits_of_strided_rows_and_offsets_past_32_bits():
    """V of wider rows; the last row starts past 2^32 bytes."""
    T, ld, V = 17, 1 << 27, 1001  # 4.5 GB of bfloat16
    z = torch.full((T, ld), 50.0, dtype=torch.bfloat16, device=dev())
    part = torch.randn(T, V, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    z[:, :V] = part.to(dev())
    values, ids, lse = run_top(z, V, 9)
    want = ordered(part.double().numpy(), 9)
    assert np.array_equal(ids.cpu().numpy(), want)


# ---------------------------------------------------------------- distillation --

def reference(z, values, ids, *, scale, lse=None, temperature=1.0, upcast=torch.float64):
    """row losses, dlogits and what bounds them need, in float64 on the CPU, by the formulas of the definition."""
    z, t = z.to(upcast), values.to(upcast) / temperature
    u = z / temperature
    log_p = torch.log_softmax(u, 1)
    p = log_p.exp()
    T, V = z.shape
    loss, grad = torch.zeros(T, dtype=upcast), torch.zeros(T, V, dtype=upcast)
    size = torch.zeros(T, V, dtype=upcast)  # what of p a gradient's error scales with
    weight = torch.zeros(T, dtype=upcast)
    for r in range(T):
        on = ids[r] >= 0
        if not bool(on.any()):
            continue
        i = ids[r][on].long()
        off = torch.ones(V, dtype=torch.bool)
        off[i] = False
        q = torch.exp(t[r][on] - lse[r].to(upcast)) if lse is not None else torch.softmax(t[r][on], 0)
        q_rest, log_rest = 0.0, 0.0
        if lse is not None and bool((z[r][off] > -math.inf).any()):
            q_rest = max(0.0, float(1 - q.sum()))
            log_rest = float(torch.logsumexp(u[r][off], 0) - torch.logsumexp(u[r], 0))
        keep = q > 0
        loss[r] = (q[keep] * (torch.log(q[keep]) - log_p[r][i][keep])).sum()
        if q_rest > 0:
            loss[r] += q_rest * (math.log(q_rest) - log_rest)
        total = float(q.sum()) + q_rest
        share = torch.exp(log_p[r] - log_rest) if q_rest > 0 else torch.zeros_like(p[r])  # of the rest
        grad[r] = p[r] * total - q_rest * share
        size[r] = p[r] * total + q_rest * share
        grad[r][i] = p[r][i] * total - q
        size[r][i] = p[r][i] * total + q
        weight[r] = total
    gs = scale / temperature
    far = (u - u.amax(1, keepdim=True)).abs()
    return loss, grad * gs, size * gs, weight, torch.where(far < 1e30, far, torch.zeros_like(far))


def make(T, V, k, dtype, *, seed=0, ragged=False, noise=0.5):
    g = torch.Generator().manual_seed(seed)
    teacher = torch.randn(T, V, generator=g) * 2 + torch.rand(T, V, generator=g) ** 64 * 8
    z = (teacher + torch.randn(T, V, generator=g) * noise).to(DT[dtype])
    values, ids = teacher.topk(k, 1)
    ids = ids.int()
    if ragged:
        # entries absent anywhere, and rows without any
        ids[torch.rand(T, k, generator=g) < 0.4] = -1
        ids[::3] = -1
    return z, values, ids, teacher


def run(z, values, ids, *, scale, lse=None, temperature=1.0, grad=True, in_place=False, V=None):
    zd = z.to(dev())
    d = (zd if in_place else torch.full_like(zd, 3.0)) if grad else None
    row, loss = torch.full((z.shape[0],), 9.0, device=dev()), torch.full((1,), 9.0, device=dev())
    K.distill_loss(zd, values.to(dev()), ids.to(dev()), V=V or z.shape[1], scale=scale, row_loss=row,
                   lse=None if lse is None else lse.to(dev()), temperature=temperature, loss_out=loss, dlogits=d)
    return row, loss, d


def check(z, values, ids, *, scale, lse=None, temperature=1.0):
    V = z.shape[1]
    want, grad, size, weight, far = reference(z, values, ids, scale=scale, lse=lse, temperature=temperature)
    row, loss, d = run(z, values, ids, scale=scale, lse=lse, temperature=temperature)
    tol = 2 * weight * unit(V) + 2.0 ** -24 * want.abs() + 1e-12
    err = (row.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"loss: worst {float((err / tol).max())} of its bound"
    assert abs(float(loss) - scale * float(row.double().sum())) <= 2.0 ** -23 * scale * float(row.double().abs().sum())
    eps = torch.finfo(z.dtype).eps
    gtol = 2 * size * (unit(V) + 4 * far * 2.0 ** -24) + eps / 2 * grad.abs() + 2.0 ** -25 * (z.dtype == torch.float16) \
        + 2.0 ** -120 * scale
    gerr = (d.cpu().double() - grad).abs()
    assert bool((gerr <= gtol).all()), f"gradient: worst {float((gerr / gtol).max())} of its bound"
    # the gradient over the logits: the same bits; no gradient: within the same bound
    row2, _, d2 = run(z, values, ids, scale=scale, lse=lse, temperature=temperature, in_place=True)
    row3, _, _ = run(z, values, ids, scale=scale, lse=lse, temperature=temperature, grad=False)
    assert torch.equal(row, row2) and torch.equal(d, d2)
    assert bool(((row3.cpu().double() - want).abs() <= tol).all())


# rows, V, k: a piece, odd widths, each block size and registers a thread, rows read twice
DISTILL_CASES = [(1, 1, 1), (3, 5, 2), (4, 100, 100), (5, 1001, 17), (2, 5000, 1024), (3, 8193, 64), (3, 16385, 300),
                 (2, 40001, 33), (2, 52001, 33), (2, 75001, 12), (2, 90000, 8), (2, 106001, 40), (2, 151936, 64),
                 (2, 151935, 64), (2, 200001, 100), (1, 1 << 20, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("case", DISTILL_CASES, ids=lambda c: "x".join(map(str, c)))
def test_distill(case, tail, dtype):
    T, V, k = case
    print("case distill", case, tail, dtype, file=sys.stderr, flush=True)
    for temperature, ragged in ((1.0, False), (2.5, True)):
        z, values, ids, teacher = make(T, V, k, dtype, seed=V, ragged=ragged)
        lse = torch.logsumexp(teacher.double() / temperature, 1).float() if tail else None
        check(z, values, ids, scale=256.0 if dtype == "f16" else 0.37, lse=lse, temperature=temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_distill_with_nearly_all_mass_listed(dtype):
    """A teacher whose rest is 1e-6 and a student whose rest is 1e-7 of the whole: formed as
    differences of sums, neither would have a digit left."""
    T, V, k = 4, 5000, 16
    g = torch.Generator().manual_seed(2)
    teacher = torch.randn(T, V, generator=g) - 25
    teacher[:, :k] = torch.rand(T, k, generator=g) * 4
    z = teacher.clone()
    z[:, k:] -= 2.5
    values, ids = teacher.topk(k, 1)
    check(z.to(DT[dtype]), values, ids.int(), scale=1.0, lse=torch.logsumexp(teacher.double(), 1).float())


@pytest.mark.gpu
def test_gradient_against_differences():
    T, V, k, h = 3, 300, 12, 1e-4
    for tail in (True, False):
        z, values, ids, teacher = make(T, V, k, "f32", seed=9)
        lse = torch.logsumexp(teacher.double() / 1.7, 1).float() if tail else None
        kw = dict(scale=1.0, lse=lse, temperature=1.7)
        _, _, d = run(z, values, ids, **kw)
        cols = torch.cat([ids[0, :4].long(), torch.arange(0, V, 37)])
        for c in cols.tolist():
            up, down = z.double(), z.double()
            up, down = up.clone(), down.clone()
            up[:, c] += h
            down[:, c] -= h
            diff = (reference(up, values, ids, **kw)[0] - reference(down, values, ids, **kw)[0]) / (2 * h)
            # third derivatives are below 1: h^2 / 6; float64 rounding 2^-52 / h of losses below 20
            assert bool(((d[:, c].cpu().double() - diff).abs() <= h * h + 20 * 2.0 ** -52 / h + 4 * unit(V)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("V", [300, 100003])
def test_rows_that_leave_nothing(tail, V):
    """Empty lists, bad lists, lists of the whole vocabulary, logits of minus infinity, on and off the list."""
    T, k = 7, 6
    z, values, ids, teacher = make(T, V, k, "f32", seed=1)
    ids[0] = -1                       # no entry: zero, whatever the logits
    z[0, 5] = math.nan
    ids[1, 3] = ids[1, 0]             # listed twice: NaN
    ids[2, 2] = V                     # past the vocabulary: NaN
    z[3] = -math.inf                  # the student allows the list alone
    z[3, ids[3].long()] = 0.5
    z[4, ids[4, 0].long()] = -math.inf  # the student excludes what the teacher expects: infinite loss
    values[5, 1] = -math.inf          # the teacher excludes an entry
    z[5, ids[5, 1].long()] = -math.inf
    ids[6, 1:] = -1                   # a list of one
    lse = torch.logsumexp(teacher.double(), 1).float() if tail else None
    row, loss, d = run(z, values, ids, scale=1.0, lse=lse)
    row, d = row.cpu().double(), d.cpu().double()
    assert row[0] == 0 and bool((d[0] == 0).all())
    for r in (1, 2):
        assert math.isnan(row[r]) and bool(torch.isnan(d[r]).all())
    good = [3, 4, 5, 6]
    want, grad, size, weight, far = reference(z[good], values[good], ids[good], scale=1.0,
                                              lse=None if lse is None else lse[good])
    assert bool(torch.isinf(row[4])) and bool(torch.isinf(want[1]))
    fin = [0, 2, 3]
    err = (row[good].double() - want)[fin].abs()
    assert bool((err <= 2 * weight[fin] * unit(V) + 2.0 ** -24 * want[fin].abs() + 1e-12).all())
    gerr = (d[good] - grad).abs()
    assert bool((gerr <= 2 * size * (unit(V) + 4 * far * 2.0 ** -24) + 2.0 ** -24 * grad.abs() + 2.0 ** -120).all())
    assert bool((d[3][torch.isinf(z[3])] == 0).all())
    assert math.isnan(float(loss))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("V", [300, 100003])
def test_masks_of_the_lowest_value(V, dtype):
    """A mask of the type's lowest value takes logits out as minus infinity does, of most of the row and of all of
    it but the list, whatever stands in the row's first pieces; far rows keep their sums."""
    T, k = 4, 5
    low = torch.finfo(DT[dtype]).min
    z, values, ids, teacher = make(T, V, k, dtype, seed=8)
    z[0, V // 4:] = low
    z[1, : V - 3] = low
    z[1, V - 3:] = 0.5
    keep = torch.zeros(V, dtype=torch.bool)
    keep[ids[2].long()] = True
    z[2, ~keep] = low
    z[3] = (z[3].float() - 30000).to(z.dtype)  # far from zero, and in one binade
    lse = torch.logsumexp(teacher.double(), 1).float()
    # the list and the row's far part alone above the mask: what the formulas say of minus infinity
    as_inf = torch.where(z == low, torch.full_like(z, -math.inf), z) if dtype != "f16" else z
    for tail in (lse, None):
        want, grad, size, weight, far = reference(as_inf, values, ids, scale=64.0, lse=tail)
        row, _, d = run(z, values, ids, scale=64.0, lse=tail)
        row2, _, _ = run(z, values, ids, scale=64.0, lse=tail, grad=False)
        tol = 2 * weight * unit(V) + 2.0 ** -24 * want.abs() + 1e-12
        for r in (row, row2):
            err = (r.cpu().double() - want).abs()
            ok = (err <= tol) | (torch.isinf(want) & (r.cpu().double() == want))
            assert bool(ok.all()), (tail is None, r, want)
        gtol = 2 * size * (unit(V) + 4 * far * 2.0 ** -24) + torch.finfo(z.dtype).eps / 2 * grad.abs() \
            + 2.0 ** -25 * (dtype == "f16") + 2.0 ** -100
        assert bool(((d.cpu().double() - grad).abs() <= gtol).all())


@pytest.mark.gpu
def test_strided_rows_keep_what_lies_beside_them():
    """Columns past V are neither read nor written; rows start off 16 bytes."""
    T, V, k, ld = 5, 1003, 9, 1010
    z, values, ids, teacher = make(T, V, k, "bf16", seed=3)
    wide = torch.full((T, ld), math.nan, dtype=torch.bfloat16)
    wide[:, :V] = z
    lse = torch.logsumexp(teacher, 1)
    row, _, d = run(wide, values, ids, scale=1.0, lse=lse, V=V)
    want, _, dw = run(z, values, ids, scale=1.0, lse=lse)
    assert torch.equal(row, want) and torch.equal(d[:, :V], dw) and bool((d[:, V:] == 3.0).all())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    T, ld, V, k = 9, 1 << 27, 40001, 8  # float32: the last row starts at 4.3 GB
    z, values, ids, teacher = make(T, V, k, "f32", seed=6)
    wide = torch.zeros(T, ld, device=dev())
    wide[:, :V] = z.to(dev())
    row, loss = torch.empty(T, device=dev()), torch.empty(1, device=dev())
    K.distill_loss(wide, values.to(dev()), ids.to(dev()), V=V, scale=1.0, row_loss=row, loss_out=loss, dlogits=wide)
    want, _, d = run(z, values, ids, scale=1.0)
    assert torch.equal(row, want) and torch.equal(wide[:, :V], d) and bool((wide[-1, V:] == 0).all())


@pytest.mark.gpu
def test_teacher_as_its_own_student():
    """The list that ``top_logits`` gives, against the logits it came from: no divergence, no gradient."""
    z = (torch.randn(6, 151936, generator=torch.Generator().manual_seed(12)) * 3).to(torch.bfloat16).to(dev())
    for temperature in (1.0, 2.0):
        values, ids, lse = run_top(z, 151936, 64, temperature)
        row, loss, d = run(z, values, ids, scale=1.0, lse=lse, temperature=temperature)
        # lse rounds to float32 (2^-24 of at most 16) and both sums are within their unit
        bound = 4 * unit(151936) + 16 * 2.0 ** -24
        assert float(row.abs().max()) <= bound
        assert float(d.float().abs().max()) <= 2 * bound


@pytest.mark.gpu
def test_graph_and_side_stream():
    """Both captured together and replayed on new logits between eager work; two streams at once."""
    T, V, k = 33, 50257, 20
    z = torch.empty(T, V, dtype=torch.bfloat16, device=dev())
    values, ids, lse = torch.empty(T, k, device=dev()), torch.empty(T, k, dtype=torch.int32, device=dev()), torch.empty(T, device=dev())
    student, row, loss, d = torch.empty_like(z), torch.empty(T, device=dev()), torch.empty(1, device=dev()), torch.empty_like(z)

    def both(out):
        K.top_logits(z, V=V, values=out[0], ids=out[1], lse=out[2])
        K.distill_loss(student, out[0], out[1], V=V, scale=1.0 / T, row_loss=out[3], lse=out[2], loss_out=out[4],
                       dlogits=out[5])

    outs = (values, ids, lse, row, loss, d)
    fill = lambda s: (z.copy_(torch.randn(T, V, generator=torch.Generator().manual_seed(s)) * 2),
                      student.copy_(torch.randn(T, V, generator=torch.Generator().manual_seed(s + 1)) * 2))
    fill(0)
    both(outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(outs)
    side = torch.cuda.Stream()
    for s in (10, 20, 30):
        fill(s)
        want = tuple(torch.empty_like(o) for o in outs)
        other = tuple(torch.empty_like(o) for o in outs)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            both(other)
        both(want)
        torch.cuda.synchronize()
        for a, b, c in zip(outs, want, other):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_no_rows():
    e = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device=dev())
    loss = torch.full((1,), 5.0, device=dev())
    K.distill_loss(e(0, 10), e(0, 3), e(0, 3, dt=torch.int32), V=10, scale=1.0, row_loss=e(1), loss_out=loss)
    assert float(loss) == 0.0
    K.top_logits(e(0, 10), V=10, values=e(0, 3), ids=e(0, 3, dt=torch.int32))


# ------------------------------------------------------------------- refusals --

def test_top_logits_refusals_before_launch():
    lib, P, f = K.lib(), ctypes.c_void_p, ctypes.c_float

    def call(x=P(1 << 20), dt=1, ld=1000, T=4, V=1000, k=8, temp=1.0, values=P(1 << 24), ids=P(1 << 25), lse=P(1 << 26)):
        return lib.mr_top_logits(x, dt, ld, T, V, k, ctypes.c_double(temp), values, ids, lse, None)

    for bad, word in ((dict(x=None), b"null"), (dict(values=None), b"null"), (dict(ids=None), b"null"),
                      (dict(dt=5), b"dtype"), (dict(T=-1), b"sizes"), (dict(V=0), b"sizes"), (dict(k=0), b"k=0"),
                      (dict(k=1025, V=2000, ld=2000), b"k=1025"), (dict(k=9, V=8), b"k=9"), (dict(ld=999), b"leading"),
                      (dict(temp=0.0), b"temperature"), (dict(temp=math.nan), b"temperature"),
                      (dict(temp=math.inf), b"temperature"), (dict(T=1 << 31), b"large"), (dict(x=P((1 << 20) + 1)), b"aligned"),
                      (dict(values=P(1 << 20)), b"overlap"), (dict(ids=P(1 << 24)), b"overlap"),
                      (dict(lse=P((1 << 25) + 4)), b"overlap")):
        assert call(**bad) == -22, bad
        assert word in lib.mr_last_error(), (bad, lib.mr_last_error())


def test_distill_refusals_before_launch():
    lib, P, f = K.lib(), ctypes.c_void_p, ctypes.c_float

    def call(z=P(1 << 20), dt=0, ld=1000, T=4, V=1000, t=P(1 << 22), ids=P(1 << 23), k=8, lse=P(1 << 24), temp=1.0,
             row=P(1 << 25), loss=P(1 << 26), d=P(1 << 27), ldd=1000):
        return lib.mr_distill(z, dt, ld, T, V, t, ids, k, lse, ctypes.c_double(temp), f(1.0), row, loss, d, ldd, None)

    for bad, word in ((dict(z=None), b"null"), (dict(t=None), b"null"), (dict(ids=None), b"null"), (dict(row=None), b"null"),
                      (dict(dt=-1), b"dtype"), (dict(T=-2), b"sizes"), (dict(V=0), b"sizes"),
                      (dict(V=(1 << 20) + 1, ld=1 << 21, ldd=1 << 21), b"vocabularies"), (dict(k=0), b"k=0"),
                      (dict(k=1025), b"k=1025"), (dict(ld=999), b"leading"), (dict(ldd=999), b"leading"),
                      (dict(temp=-1.0), b"temperature"), (dict(T=1 << 31), b"rows"), (dict(z=P((1 << 20) + 2)), b"aligned"),
                      (dict(d=P((1 << 20) + 4)), b"overlaps"), (dict(d=P(1 << 20), ldd=1001), b"overlaps"),
                      (dict(row=P(1 << 22)), b"overlaps"), (dict(loss=P(1 << 25)), b"overlap"),
                      (dict(row=P((1 << 27) + 16)), b"overlap")):
        assert call(**bad) == -22, bad
        assert word in lib.mr_last_error(), (bad, lib.mr_last_error())


def test_bindings_refuse_on_the_host():
    z, v, i = torch.zeros(4, 100), torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int32)
    with pytest.raises(KernelError, match="int32"):
        K.top_logits(z, V=100, values=v, ids=i.long())
    with pytest.raises(KernelError, match="logits must be"):
        K.top_logits(z, V=101, values=v, ids=i)
    with pytest.raises(KernelError, match="ROCm device"):
        K.top_logits(z, V=100, values=v, ids=i)
    kw = dict(V=100, scale=1.0, row_loss=torch.zeros(4))
    with pytest.raises(KernelError, match="ids must be"):
        K.distill_loss(z, v, i[:, :7], **kw)
    with pytest.raises(KernelError, match="dlogits"):
        K.distill_loss(z, v, i, dlogits=z.half(), **kw)
    with pytest.raises(KernelError, match="one row loss"):
        K.distill_loss(z, v, i, lse=torch.zeros(3), **kw)
    with pytest.raises(KernelError, match="ROCm device"):
        K.distill_loss(z, v, i, **kw)


# ------------------------------------------------------- the ends of the range --

def test_temperatures_out_of_range_are_refused():
    lib, P, f = K.lib(), ctypes.c_void_p, ctypes.c_float
    for temp in (1e-4, 2e3):
        assert lib.mr_top_logits(P(1 << 20), 1, 1000, 4, 1000, 8, ctypes.c_double(temp), P(1 << 24), P(1 << 25), None, None) == -22
        assert b"temperature" in lib.mr_last_error()
        assert lib.mr_distill(P(1 << 20), 0, 1000, 4, 1000, P(1 << 22), P(1 << 23), 8, None, ctypes.c_double(temp), f(1.0), P(1 << 25), None,
                              None, 1000, None) == -22
        assert b"temperature" in lib.mr_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 40000, 200003])
@pytest.mark.parametrize("temperature", [2.0 ** -10, 2.0 ** 10])
def test_temperatures_at_the_ends(V, temperature):
    # (logits of the temperature's own size, so that rows are no one-hot)
    T, k = 3, 8
    z, values, ids, teacher = make(T, V, k, "f32", seed=12)
    z, values, teacher = z * temperature, values * temperature, teacher * temperature
    lse = torch.logsumexp(teacher.double() / temperature, 1).float()
    check(z, values, ids, scale=temperature, lse=lse, temperature=temperature)
    check_top(z, k, temperature=temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 40000, 100003, 200003])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logits_whose_exponents_are_no_floats(V, dtype):
    """A logit of 3e38: the largest of the list, its log-sum-exp the logit over the temperature; off a list no
    finite loss, as an infinity there."""
    z = torch.randn(4, V, generator=torch.Generator().manual_seed(3)).to(DT[dtype])
    z[1, V - 3] = z[2, 7] = 3e38
    z[3] = -3e38
    z[3, 5] = 0.0
    values, ids, lse = run_top(z.to(dev()), V, 8, 0.75)
    big = float(z[1, V - 3])
    assert ids[1, 0] == V - 3 and ids[2, 0] == 7 and ids[3, 0] == 5 and float(values[1, 0]) == big
    assert bool(torch.isinf(lse[1:3]).all()) and float(lse[3]) == 0.0
    lists, t = torch.arange(10, 18).repeat(4, 1).int(), torch.zeros(4, 8)
    for tail in (torch.full((4,), 2.5), None):
        for grad in (True, False):
            row, _, _ = run(z, t, lists, scale=1.0, lse=tail, temperature=0.75, grad=grad)
            assert bool(torch.isfinite(row[0])) and not bool(torch.isfinite(row[1:3]).any()), (tail, grad)


# the last row of each size of block, the first of the next, and lists that leave room for fewer pieces beside them
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", [(2, 126976, 8), (2, 126977, 9), (2, 151936, 1024), (2, 159744, 16), (2, 159745, 16),
                                  (1, 163840, 1000), (1, 163841, 5), (2, 63488, 7), (2, 63489, 7), (2, 76000, 1024),
                                  (1, 79873, 5), (1, 81920, 700), (1, 81921, 3)], ids=lambda c: "x".join(map(str, c)))
def test_rows_read_twice(case, dtype):
    test_distill(case, True, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [70001, 120001, 151936])
def test_odd_rows_that_are_read_twice(V):
    for tail in (True, False):
        test_rows_that_leave_nothing(tail, V)
    for dtype in ("bf16", "f32"):
        test_masks_of_the_lowest_value(V, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [70000, 120000, 151936])
def test_a_peak_anywhere(V, dtype):
    """A logit of 300, off the list, at places all over the row: the sum about the first pieces' maximum has no room
    for it and is formed anew."""
    T, k = 40, 8
    z, values, ids, teacher = make(T, V, k, dtype, seed=V + 1)
    for r in range(T):
        c = (r * V) // T + r
        while c in ids[r].tolist():
            c += 1
        z[r, c] = 300.0
    check(z, values, ids, scale=1.0, lse=torch.logsumexp(teacher.double(), 1).float())


# rows enough for small blocks of the loss alone, a row or two of each bound on a block's size
@pytest.mark.gpu
@pytest.mark.parametrize("case", [(1100, 20000, 16), (1030, 17001, 700), (3, 17001, 16), (2, 320000, 16), (2, 400000, 900),
                                  (2, 16384, 5), (2, 16385, 5)], ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_loss_alone_is_the_loss(case, dtype):
    T, V, k = case
    z, values, ids, teacher = make(T, V, k, dtype, seed=V, ragged=True)
    lse = torch.logsumexp(teacher.double(), 1).float()
    want, *_, weight, _ = reference(z, values, ids, scale=1.0, lse=lse)
    row, loss, _ = run(z, values, ids, scale=1.0, lse=lse, grad=False)
    tol = 2 * weight * unit(V) + 2.0 ** -24 * want.abs() + 1e-12
    assert bool(((row.cpu().double() - want).abs() <= tol).all())
    assert abs(float(loss) - float(row.double().sum())) <= 2.0 ** -23 * float(row.double().abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(2, 24576, 256), (2, 24577, 256), (2, 24000, 257), (2, 30000, 512), (2, 30000, 513),
                                  (2, 700, 512), (2, 700, 513), (2, 4096, 512)], ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_top_logits_by_each_block(case, dtype):
    test_top_logits(case, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.7, 1.354, 2.3])
def test_temperatures_that_are_no_floats(temperature):
    """The temperature is a double: in float32 2^-25 of a logit would be missing between the list and its log-sum-exp,
    3e-7 of every probability at logits of 10."""
    T, V, k = 8, 4363, 78
    z, values, ids, teacher = make(T, V, k, "bf16", seed=31, noise=0.1)
    check(z, values, ids, scale=1.0, lse=torch.logsumexp(teacher.double() / temperature, 1).float(), temperature=temperature)
    check_top(z, k, temperature=temperature)


# ------------------------------------------------------------ masks and far logits --

@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 16385, 40001, 100003, 151936])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("temperature", [0.75, 1.0, 1.5, 2.0, 2.034, 2.158, 2.5, 3.679, 4.0, 300.0])
def test_masks_at_any_temperature(temperature, dtype, V):
    """Every unlisted logit at a mask's value, one that is exact in powers of two over the temperature among them:
    no such outcome, with the gradient as without it, and no gradient on what is masked. In the other rows a few
    logits lie off the list and off the mask, first and last in the row."""
    T, k = 6, 5
    z, values, ids, teacher = make(T, V, k, dtype, seed=18)
    ids = torch.argsort(torch.rand(T, V - 40, generator=torch.Generator().manual_seed(V)), 1)[:, :k].int() + 20
    values = teacher.gather(1, ids.long())
    listed = torch.zeros(T, V, dtype=torch.bool).scatter_(1, ids.long(), True)
    lows = torch.tensor([torch.finfo(DT[dtype]).min, -2.0 ** 125, -2.0 ** 126]).to(z.dtype).repeat(2)[:, None]
    free = listed.clone()
    free[3, :3] = free[4, V - 3:] = free[5, V // 2] = True
    z = torch.where(free, z, lows.expand(T, V))
    as_inf = torch.where(free, z, torch.full_like(z, -math.inf))
    lse = torch.logsumexp(teacher.double() / temperature, 1).float()
    for tail in (lse, None):
        want, grad, size, weight, far = reference(as_inf, values, ids, scale=64.0, lse=tail, temperature=temperature)
        row, _, d = run(z, values, ids, scale=64.0, lse=tail, temperature=temperature)
        alone, _, _ = run(z, values, ids, scale=64.0, lse=tail, temperature=temperature, grad=False)
        tol = 2 * weight * unit(V) + 2.0 ** -24 * want.abs() + 1e-12
        for r in (row, alone):
            assert bool(((r.cpu().double() - want).abs() <= tol).all()), (tail is None, r, want)
        gtol = 2 * size * (unit(V) + 4 * far * 2.0 ** -24) + torch.finfo(z.dtype).eps / 2 * grad.abs() + 2.0 ** -100
        assert bool(((d.cpu().double() - grad).abs() <= gtol).all())
        assert bool((d.cpu()[~free] == 0).all())


def far_reference(z, values, ids, *, scale, lse, temperature):
    """``reference`` for rows whose unlisted logits lie far from the listed: the rest's shares as a softmax of its own
    (as a difference of log-probabilities of 1e10 they would keep no digit in float64 either), and of each exponent
    the distance from the largest of its kind, where that leaves anything."""
    want, _, _, weight, _ = reference(z, values, ids, scale=scale, lse=lse, temperature=temperature)
    u, t = z.double() / temperature, values.double() / temperature
    listed = torch.zeros(z.shape, dtype=torch.bool).scatter_(1, ids.long(), True)
    q = torch.exp(t - lse.double()[:, None]) if lse is not None else torch.softmax(t, 1)
    q_rest = (1 - q.sum(1, keepdim=True)).clamp_min(0) if lse is not None else torch.zeros(z.shape[0], 1).double()
    p = torch.log_softmax(u, 1).exp() * (q.sum(1, keepdim=True) + q_rest)
    target = (q_rest * torch.softmax(u.masked_fill(listed, -math.inf), 1)).scatter(1, ids.long(), q)
    away = torch.where(listed, u - u.amax(1, keepdim=True), u - u.masked_fill(listed, -math.inf).amax(1, keepdim=True)).abs()
    away = torch.where(away < 200, away, torch.zeros_like(away))
    gs = scale / temperature
    return want, (p - target) * gs, (p + target) * gs, weight, away, u.abs().amax(1)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 7, 300, 16385, 40001, 100003, 151936, 200003])
@pytest.mark.parametrize("size,dtype", [(s, t) for t in ("bf16", "f32") for s in (-3e7, -1e9, -1e10, -7e11, -1e20, -1e33, 1e10, 1e20)]
                         + [(-3e4, "f16"), (3e4, "f16")])
def test_unlisted_logits_far_from_zero(size, dtype, V):
    """Unlisted logits where a float's step is many powers of two: equal, steps of the type apart, or one far above
    the rest; the first half of a row holds the largest or none of it.

    The loss carries 2^-47 of |z / T| for each of its two logarithms (log2(e) / T is two floats), the gradient the
    errors of exponents a few steps from their largest."""
    T, k = 5, min(3, V - 2)
    for temperature in (2.0 ** -10, 0.7, 1.0, 2.0, 100.0):
        g = torch.Generator().manual_seed(V)
        z, _, _, teacher = make(T, V, k, dtype, seed=28)
        ids = torch.argsort(torch.rand(T, V, generator=g), 1)[:, :k].int()
        values = teacher.gather(1, ids.long())
        listed = torch.zeros(T, V, dtype=torch.bool).scatter_(1, ids.long(), True)
        step = 2.0 ** (math.floor(math.log2(abs(size))) - {"bf16": 7, "f16": 10, "f32": 23}[dtype])
        far = torch.full((T, V), size, dtype=torch.float64)
        far[1] -= step * torch.randint(0, 4, (V,), generator=g)
        far[2, : V // 2] *= 2 if size < 0 else 0.5
        far[3, V // 2:] *= 2 if size < 0 else 0.5
        if size > 0:
            far[4] = 0.0
        far[4, :-1] -= 64 * step * (torch.arange(V - 1) % 3)
        far[4, -1] = size
        z = torch.where(listed, z.double(), far).to(z.dtype)
        # a rest of a fifth and more
        lse = (torch.logsumexp(values.double() / temperature, 1) + 0.25).float()
        for tail in (lse, None):
            kw = dict(scale=0.37, lse=tail, temperature=temperature)
            want, grad, size_, weight, away, u_max = far_reference(z, values, ids, **kw)
            row, _, d = run(z, values, ids, **kw)
            row2, _, d2 = run(z, values, ids, in_place=True, **kw)
            alone, _, _ = run(z, values, ids, grad=False, **kw)
            tol = 2 * weight * unit(V) + 2.0 ** -24 * want.abs() + 2.0 ** -46 * weight * u_max + 1e-12
            for r in (row, alone):
                err = (r.cpu().double() - want).abs()
                assert bool((err <= tol).all()), (temperature, tail is None, r, want)
            assert torch.equal(row, row2) and torch.equal(d, d2)
            gtol = 2 * size_ * (unit(V) + 4 * away * 2.0 ** -24) + torch.finfo(z.dtype).eps / 2 * grad.abs() \
                + 2.0 ** -25 * (dtype == "f16") + 2.0 ** -120
            err = (d.cpu().double() - grad).abs()
            assert bool((err <= gtol).all()), (temperature, tail is None, float((err / gtol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [30, 2048, 9000, 60001])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("size", [-3e7, -1e9, 2.0 ** 31, -7e11, -2.0 ** 102, -2.0 ** 110, -2.0 ** 122, 1e20, 1e30])
def test_top_logits_far_from_zero(size, dtype, V):
    """Log-sum-exps of logits where a float's step is many powers of two, masks of other code's making among them:
    equal, steps of the type apart, halves of a row far from one another."""
    T, k = 4, min(V, 257)
    g = torch.Generator().manual_seed(V)
    step = 2.0 ** (math.floor(math.log2(abs(size))) - (7 if dtype == "bf16" else 23))
    z = torch.full((T, V), size, dtype=torch.float64)
    z[1] -= step * torch.randint(0, 4, (V,), generator=g)
    z[2, : V // 2] *= 2 if size < 0 else 0.5
    z[3, :-1] -= 64 * step * (torch.arange(V - 1) % 3)
    z = z.to(DT[dtype])
    for temperature in (2.0 ** -10, 0.7, 1.0, 2.0, 3.1, 100.0):
        ref = torch.logsumexp(z.double() / temperature, 1)
        over = ref.abs() >= 2.0 ** 128  # (as a float32 an infinity)
        if bool(over.any()):
            _, ids, lse = run_top(z[over].to(dev()), V, k, temperature)
            assert np.array_equal(ids.cpu().numpy(), ordered(z[over].double().numpy(), k))
            assert torch.equal(lse.cpu(), ref[over].float())
        if not bool(over.all()):
            check_top(z[~over], k, temperature)


def test_rows_past_a_launch_are_refused_before_it():
    """A block a row: blocks times threads is a 32-bit number. Every size of block, at the first row too many."""
    lib, P, f = K.lib(), ctypes.c_void_p, ctypes.c_float
    far = lambda n: P(n << 50)

    for V, k, threads in ((8, 2, 256), (24576, 256, 256), (24577, 3, 512), (300, 257, 512), (2000, 513, 1024)):
        T = (1 << 32) // threads
        assert lib.mr_top_logits(far(1), 1, V, T, V, k, ctypes.c_double(1.0), far(2), far(3), far(4), None) == -22
        assert b"too large" in lib.mr_last_error() and str(T - 1).encode() in lib.mr_last_error()
    # (elements, gradient, threads): short rows, held ones, rows read twice, the loss alone
    for V, grad, threads in ((2, True, 1024), (300, True, 256), (300, False, 256), (9000, True, 512), (16000, True, 512),
                             (80000, True, 512), (82000, True, 1024), (20000, False, 256), (200000, False, 512),
                             (1000000, False, 1024)):
        T = (1 << 32) // threads
        assert lib.mr_distill(far(1), 0, V, T, V, far(2), far(3), 2, far(4), ctypes.c_double(1.0), f(1.0), far(5), far(6),
                              far(7) if grad else None, V, None) == -22, (V, grad)
        assert b"too many rows" in lib.mr_last_error() and str(T - 1).encode() in lib.mr_last_error(), (V, grad)


def test_no_rows_have_no_addresses():
    """Tensors without elements have none: with nothing to write, nothing is refused."""
    lib, f = K.lib(), ctypes.c_float
    assert lib.mr_distill(None, 0, 10, 0, 10, None, None, 3, None, ctypes.c_double(1.0), f(1.0), None, None, None, 0, None) == 0
    assert lib.mr_top_logits(None, 0, 10, 0, 10, 3, ctypes.c_double(1.0), None, None, None, None) == 0
    assert lib.mr_rope_positions(None, 0, 64, 0, 1, 64, None, None, 64, 0, f(1.0), 0, None, 64, None) == 0


@pytest.mark.gpu
def test_a_loss_of_no_rows():
    e = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device=dev())
    loss = torch.full((1,), 5.0, device=dev())
    K.distill_loss(e(0, 10), e(0, 3), e(0, 3, dt=torch.int32), V=10, scale=1.0, row_loss=e(0), lse=e(0), loss_out=loss,
                   dlogits=e(0, 10))
    assert float(loss) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 9000, 40001, 151936, 200003])
@pytest.mark.parametrize("mask,dtype", [(m, t) for t in ("bf16", "f32") for m in (-1e6, -1e9, -1e10, -3e10, -1e12, -1e20, -1e30, -1e36)]
                         + [(-1e4, "f16"), (-65504.0, "f16")])
def test_masks_that_are_numbers(mask, dtype, V):
    """A large negative number in the place of minus infinity, at either end of a row, in most of its pieces and in
    nearly all: sums that began among the masks go on with what follows, and a NaN among them stays."""
    T, k = 6, 8
    z, values, ids, teacher = make(T, V, k, dtype, seed=V + 5)
    listed = torch.zeros(T, V, dtype=torch.bool).scatter_(1, ids.long(), True)
    out = torch.zeros(T, V, dtype=torch.bool)
    out[0, : V // 2] = out[1, V // 2:] = True
    out[2] = torch.rand(V, generator=torch.Generator().manual_seed(3)) < 0.9
    out[3, : V - 9] = out[4, 9:] = True
    z = torch.where(out, torch.full_like(z, mask), z)
    for temperature in (0.7, 1.0, 2.0, 3.1):
        check_top(z, k, temperature)
        lse = torch.logsumexp(teacher.double() / temperature, 1).float()
        zl = torch.where(listed, teacher.to(z.dtype), z)  # (no listed logit masked: a loss of 1e30 would hide the rest)
        for tail in (lse, None):
            check(zl, values, ids, scale=256.0 if dtype == "f16" else 0.37, lse=tail, temperature=temperature)
    with_nan = z.clone()
    with_nan[0, 1] = with_nan[1, V - 2] = with_nan[3, 2] = math.nan
    values_, ids_, lse_ = run_top(with_nan.to(dev()), V, k)
    assert torch.isnan(lse_.cpu()).tolist() == [True, True, False, True, False, False]
    assert ids_[0, 0] == 1 and ids_[1, 0] == V - 2 and ids_[3, 0] == 2
    zl = torch.where(listed, teacher.to(z.dtype), with_nan)
    for grad in (True, False):
        row, _, _ = run(zl, values, ids, scale=1.0, grad=grad)
        assert torch.equal(torch.isnan(row.cpu()), torch.isnan(zl).any(1))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 9000, 60001, 151936, 200003])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("temperature", [0.75, 1.1, 1.25, 1.5, 2.5, 3.0])
@pytest.mark.parametrize("gap", [20, 50, 80])
def test_a_peak_far_above_the_rest(gap, temperature, dtype, V):
    """One logit above all else by 20 to 80 temperatures, at places that the sum's correction samples and does not;
    in the loss it lies off the list."""
    T, k = 16, 4
    g = torch.Generator().manual_seed(V)
    z = (torch.randn(T, V, generator=g) - gap * temperature)
    for r in range(T):
        z[r, (r * (V - 17)) // T + r] = 0.0
    z = z.to(DT[dtype])
    check_top(z, k, temperature)
    teacher = torch.randn(T, V, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(T)]).int()
    ids = torch.where(ids == z.argmax(1, keepdim=True), (ids + 1) % V, ids)
    values = teacher.gather(1, ids.long())
    lse = torch.logsumexp(teacher.double() / temperature, 1).float()
    check(z, values, ids, scale=1.0, lse=lse, temperature=temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [5, 300, 9000, 40001, 151936, 200003])
@pytest.mark.parametrize("low,dtype", [(m, t) for t in ("bf16", "f32") for m in (0.0, -2.0 ** 125, -1e30, -1e12, 3e12)]
                         + [(-65504.0, "f16")])
def test_rows_that_a_mask_takes_whole(low, dtype, V):
    """Every logit at one value, the type's lowest (0 here) and other masks: the student's distribution is uniform over
    the list where the value counts as minus infinity off it, else over the vocabulary, whatever the value."""
    T, k = 3, 4
    low = low or torch.finfo(DT[dtype]).min
    g = torch.Generator().manual_seed(V)
    teacher = torch.randn(T, V, generator=g)
    ids = torch.argsort(torch.rand(T, V, generator=g), 1)[:, :k].int()
    values = teacher.gather(1, ids.long())
    z = torch.full((T, V), low).to(DT[dtype])
    as_zero = torch.zeros(T, V, dtype=torch.float64)  # (a shift of a row changes nothing)
    if float(z[0, 0]) <= -1e37:
        as_zero.fill_(-math.inf).scatter_(1, ids.long(), 0.0)
    for temperature in (0.7, 1.0, 2.034):
        lse = torch.logsumexp(teacher.double() / temperature, 1).float()
        for tail in (lse, None):
            kw = dict(scale=0.37, lse=tail, temperature=temperature)
            want, grad, size, weight, _ = reference(as_zero, values, ids, **kw)
            row, _, d = run(z, values, ids, **kw)
            alone, _, _ = run(z, values, ids, grad=False, **kw)
            tol = 2 * weight * unit(V) + 2.0 ** -24 * want.abs() + 1e-12
            for r in (row, alone):
                assert bool(((r.cpu().double() - want).abs() <= tol).all()), (temperature, tail is None, r, want)
            gtol = 2 * size * unit(V) + torch.finfo(z.dtype).eps / 2 * grad.abs() + 2.0 ** -25 * (dtype == "f16") + 2.0 ** -120
            assert bool(((d.cpu().double() - grad).abs() <= gtol).all()), (temperature, tail is None)
