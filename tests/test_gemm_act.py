"""Products with an activation in their epilogue and their backward
(``gemm_act``, ``gemm_act_bwd``, ``act_bwd``) against float64, and what they
refuse.

Bounds. A sum of K products of bfloat16 values (exact in float32) is off by at
most K 2^-24 of the sum of their magnitudes; an activation passes an error on by
at most its slope near the value (1.13 for the gelus, 1.1 for silu, 1 for relu,
2 |x| for its square) and adds 1e-6 of 1 + |x| of its own (the tail's fit 1.5e-7,
its float32 evaluation 4.5e-7, reciprocal and exponential 2^-22 together);
outputs round by half a unit of their type.
"""

from __future__ import annotations

import ctypes
import math
import sys

import pytest
import torch

from mround_amd import kernels as K
from mround_amd.exceptions import KernelError
from tests.helpers import dev

ACTS = ("relu", "relu2", "silu", "gelu", "gelu_tanh")
BF = torch.bfloat16


def f(x, act):
    F = torch.nn.functional
    # (by erfc and the sigmoid: torch's own, by 1 + erf and 1 + tanh, have no digit left for negative x)
    return {"relu": F.relu, "relu2": lambda v: F.relu(v).square(), "silu": F.silu,
            "gelu": lambda v: 0.5 * v * torch.erfc(v * -(0.5 ** 0.5)),
            "gelu_tanh": lambda v: v * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3))}[act](x)


def slope(x, act):
    x = x.clone().requires_grad_()
    return torch.autograd.grad(f(x, act).sum(), x)[0]


def steep(x, act):
    return 2 * x.abs() if act == "relu2" else torch.full_like(x, 1.13)


def rounding(y, dtype):
    return torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8) * y.abs()


def within(got, want, tol, what):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max())} of its bound"


def strided(rows, cols, extra, dtype, fill=7.0):
    """A view of ``cols`` columns in wider rows, and the whole."""
    whole = torch.full((rows, cols + extra), fill, dtype=dtype, device=dev())
    return whole[:, :cols], whole


# (M, N, K): plans of every kind (test_shapes_take_every_plan), rows of no whole
# tiles, one row, columns of a part of a tile, k-split partials
SHAPES = [(1, 8, 64), (3, 72, 128), (33, 1000, 576), (1000, 896, 896), (257, 264, 6144), (1001, 520, 6400),
          (700, 9728, 128), (2053, 2560, 2048), (9001, 1544, 576), (16383, 4608, 1024)]


def test_shapes_take_every_plan():
    plans = {K.gemm_plan("nt", o, M, N, Kd)[:2] for M, N, Kd in SHAPES for o in ("bf16", "resid")}
    assert {p[0] for p in plans} >= {"small", "deep", "wide", "large", "large_quarters"}
    assert any(split > 1 for _, split in plans)


def product(a, b):
    """(float64 a b, bound of a float32 sum of its terms) on the GPU."""
    return a.double() @ b.double(), a.shape[1] * 2.0 ** -24 * (a.double().abs() @ b.double().abs())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward(shape, act):
    M, N, Kd = shape
    print("case gemm_act", shape, act, file=sys.stderr, flush=True)
    g = torch.Generator(device=dev()).manual_seed(3)
    x = torch.randn(M, Kd, generator=g, device=dev()).to(BF)
    w = (torch.randn(N, Kd, generator=g, device=dev()) * 2 / Kd ** 0.5).to(BF)
    bias = torch.randn(N, generator=g, device=dev())
    resid = torch.randn(M, N, generator=g, device=dev())
    acc, err = product(x, w.t())
    for with_bias in (False, True):
        pre = acc + bias.double() if with_bias else acc
        e = err + 2.0 ** -24 * pre.abs()
        y = f(pre, act)
        ytol = e * (steep(pre, act) + 2 * e) + 1e-6 * (y.abs() + (pre < 0)) + 1e-7
        b = bias if with_bias else None
        out, whole = strided(M, N, 16, BF)
        saved, saved_whole = strided(M, N, 8, BF)
        K.gemm_act(x, w, out, act=act, bias=b, pre=saved)
        within(out, y, ytol + rounding(y, BF) + 2.0 ** -130, "bf16 output")
        within(saved, pre, e + rounding(pre, BF), "pre-activation")
        assert bool((whole[:, N:] == 7).all()) and bool((saved_whole[:, N:] == 7).all())
        plain = torch.empty(M, N, dtype=BF, device=dev())
        K.gemm_act(x, w, plain, act=act, bias=b)
        assert torch.equal(plain, out)
        out32 = torch.empty(M, N, device=dev())
        K.gemm_act(x, w, out32, act=act, bias=b)
        within(out32, y, ytol + rounding(y, torch.float32), "fp32 output")
        # over the residual, with the saved copy
        r = resid.clone()
        saved2 = torch.empty(M, N, dtype=BF, device=dev())
        K.gemm_act(x, w, r, act=act, bias=b, resid=r, pre=saved2)
        within(r, y + resid.double(), ytol + 2.0 ** -23 * (y.abs() + resid.double().abs()), "residual output")
        within(saved2, pre, e + rounding(pre, BF), "pre-activation beside a residual")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_backward_through_the_next_product(shape, act):
    M, N, Kd = shape
    print("case gemm_act_bwd", shape, act, file=sys.stderr, flush=True)
    g = torch.Generator(device=dev()).manual_seed(5)
    dd = torch.randn(M, Kd, generator=g, device=dev()).to(BF)
    wd = (torch.randn(Kd, N, generator=g, device=dev()) / Kd ** 0.5).to(BF)
    pre = (torch.randn(M, N, generator=g, device=dev()) * 2).to(BF)
    pre[0, :4] = torch.tensor([0.0, -0.0, 40.0, -40.0])
    acc, err = product(dd, wd)
    s = slope(pre.double(), act)
    want = acc * s
    tol = err * (s.abs() + 1e-6) + acc.abs() * 2e-6 * (1 + pre.double().abs())
    dpre, whole = strided(M, N, 8, BF)
    dbias = torch.empty(N, device=dev())
    K.gemm_act_bwd(dd, wd, pre, dpre, act=act, dbias=dbias)
    within(dpre, want, tol + rounding(want, BF) + 2.0 ** -130, "dpre")
    assert bool((whole[:, N:] == 7).all())
    # sums of 32 rows, then of every sixteenth of those sums, then of 16
    depth = 32 + -(-M // 512) + 16
    within(dbias, want.sum(0), tol.sum(0) + depth * 2.0 ** -24 * (want.abs() + tol).sum(0), "dbias")
    # without dbias, and over the pre-activation itself: the same bits
    again = torch.empty(M, N, dtype=BF, device=dev())
    K.gemm_act_bwd(dd, wd, pre, again, act=act)
    assert torch.equal(again, dpre)
    K.gemm_act_bwd(dd, wd, pre, pre, act=act)
    assert torch.equal(pre, dpre)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(1, 8), (31, 520), (32, 512), (1001, 1032), (4005, 896)], ids=lambda s: "x".join(map(str, s)))
def test_backward_from_the_output(shape, act, dtype):
    M, N = shape
    print("case act_bwd", shape, act, dtype, file=sys.stderr, flush=True)
    g = torch.Generator(device=dev()).manual_seed(6)
    dout = torch.randn(M, N, generator=g, device=dev()).to(dtype)
    pre = (torch.randn(M, N, generator=g, device=dev()) * 2).to(BF)
    s = slope(pre.double(), act)
    want = dout.double() * s
    tol = dout.double().abs() * (2e-6 * (1 + pre.double().abs()))
    dpre, whole = strided(M, N, 8, BF)
    dbias = torch.empty(N, device=dev())
    K.act_bwd(dout, pre, dpre, act=act, dbias=dbias)
    within(dpre, want, tol + rounding(want, BF) + 2.0 ** -130, "dpre")
    assert bool((whole[:, N:] == 7).all())
    depth = 32 + -(-M // 512) + 16
    within(dbias, want.sum(0), tol.sum(0) + depth * 2.0 ** -24 * (want.abs() + tol).sum(0), "dbias")
    over = dout if dtype == BF else pre
    K.act_bwd(dout, pre, over, act=act)
    assert torch.equal(over, dpre)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_every_bfloat16_value(act):
    """The activation and its slope over all finite bfloat16 pre-activations up to 2^60, by a product with one."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    v = bits[torch.isfinite(bits.float()) & (bits.float().abs() < 2.0 ** 60)].to(dev())
    n = v.numel() // 8 * 8
    v = v[-n:]
    x = torch.zeros(8, 64, dtype=BF, device=dev())
    x[:, 0] = 1
    w = torch.zeros(n, 64, dtype=BF, device=dev())
    w[:, 0] = v
    out, pre = torch.empty(8, n, device=dev()), torch.empty(8, n, dtype=BF, device=dev())
    K.gemm_act(x, w, out, act=act, pre=pre)
    assert torch.equal(pre[3], v)
    y = f(v.double(), act)
    # For negative x the value is x times an exponential e^-a (a = |x|, x^2 / 2 or |2 u|):
    # a passes up to four roundings of 2^-24 of itself on its way into the exponent
    # (products, the constant log2 e, the exponent), each of them as much of the value.
    # The rest is the 1e-6 above; below 2^-100 the exponential may be zero.
    x64 = v.double()
    a = {"silu": x64.abs(), "gelu": x64.square() / 2, "gelu_tanh": (1.5957691216057308 * (x64 + 0.044715 * x64 ** 3)).abs()}.get(
        act, torch.zeros_like(x64)).clamp_max(200) * (x64 < 0)
    within(out[5], y, (1.2e-6 + 4 * a * 2.0 ** -24) * y.abs() + 2.0 ** -100, "f")
    dout, dpre = torch.ones(8, n, dtype=torch.float32, device=dev()), torch.empty(8, n, dtype=BF, device=dev())
    K.act_bwd(dout, pre, dpre, act=act)
    s = slope(v.double(), act)
    s = torch.where(torch.isfinite(s), s, (v > 0).double())
    within(dpre[2], s, 2e-6 * (1 + v.double().abs().clamp_max(30)) + rounding(s, BF), "slope")


@pytest.mark.gpu
def test_gradients_against_differences():
    """A whole ungated MLP's weight and bias gradients from these calls, against differences of the float64 loss."""
    M, h, n = 24, 64, 128
    g = torch.Generator(device=dev()).manual_seed(9)
    x = torch.randn(M, h, generator=g, device=dev()).to(BF)
    w1 = (torch.randn(n, h, generator=g, device=dev()) / 8).to(BF)
    w2 = (torch.randn(h, n, generator=g, device=dev()) / 11).to(BF)
    b = torch.randn(n, generator=g, device=dev())
    target = torch.randn(M, h, generator=g, device=dev())
    for act in ACTS:
        hidden, pre = torch.empty(M, n, dtype=BF, device=dev()), torch.empty(M, n, dtype=BF, device=dev())
        K.gemm_act(x, w1, hidden, act=act, bias=b, pre=pre)
        y = torch.empty(M, h, device=dev())
        K.gemm("nt", hidden, w2, y, M=M, N=h, K=n)
        dy = (y - target).to(BF)
        dpre, db, dw = torch.empty(M, n, dtype=BF, device=dev()), torch.empty(n, device=dev()), torch.empty(n, h, device=dev())
        K.gemm_act_bwd(dy, w2, pre, dpre, act=act, dbias=db)
        K.gemm("tn", torch.nn.functional.pad(dpre, (0, 0, 0, 64 - M)), torch.nn.functional.pad(x, (0, 0, 0, 64 - M)), dw, M=n, N=h, K=64)

        def loss(b64, w64):
            return 0.5 * (f(x.double() @ w64.t() + b64, act) @ w2.double().t() - target.double()).square().sum()

        step = 1e-5
        scale_b, scale_w = float(db.double().norm()), float(dw.double().norm())
        for i in (0, 17, 101):
            e = torch.zeros(n, dtype=torch.float64, device=dev())
            e[i] = step
            d = float(loss(b.double() + e, w1.double()) - loss(b.double() - e, w1.double())) / (2 * step)
            # three bfloat16 roundings (hidden, dy, pre) of 2^-8 on every term of a sum of M
            assert abs(float(db[i]) - d) <= 4 * 2.0 ** -8 * (scale_b + abs(d)) + 1e-3
            e2 = torch.zeros(n, h, dtype=torch.float64, device=dev())
            e2[i, 5] = step
            d = float(loss(b.double(), w1.double() + e2) - loss(b.double(), w1.double() - e2)) / (2 * step)
            assert abs(float(dw[i, 5]) - d) <= 5 * 2.0 ** -8 * (scale_w + abs(d)) + 1e-3


@pytest.mark.gpu
def test_non_finite_values_stay_in_their_rows():
    M, N, Kd = 70, 136, 128
    g = torch.Generator(device=dev()).manual_seed(2)
    x = torch.randn(M, Kd, generator=g, device=dev()).to(BF)
    w = torch.randn(N, Kd, generator=g, device=dev()).to(BF)
    x[33, 5] = float("nan")
    x[34, 6] = float("inf")
    for act in ACTS:
        out = torch.empty(M, N, dtype=BF, device=dev())
        K.gemm_act(x, w, out, act=act)
        bad = ~torch.isfinite(out)
        assert bool(torch.isnan(out[33]).all()) and not bool(bad[:33].any()) and not bool(bad[35:].any())


@pytest.mark.gpu
def test_graph_and_streams():
    """A captured pair, replayed on new inputs; the same on two streams at once."""
    M, N, Kd = 257, 264, 6144  # cut along K: partials in the call's own workspace
    g = torch.Generator(device=dev()).manual_seed(4)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=dev()) * std).to(BF)
    x, w, dd, wd = rnd(M, Kd), rnd(N, Kd, std=0.02), rnd(M, Kd), rnd(Kd, N, std=0.02)
    new = lambda: (torch.empty(M, N, dtype=BF, device=dev()), torch.empty(M, N, dtype=BF, device=dev()),
                   torch.empty(M, N, dtype=BF, device=dev()), torch.empty(N, device=dev()))

    def both(o):
        K.gemm_act(x, w, o[0], act="gelu", pre=o[1])
        K.gemm_act_bwd(dd, wd, o[1], o[2], act="gelu", dbias=o[3])

    outs = new()
    both(outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(outs)
    side = torch.cuda.Stream()
    for _ in range(3):
        x.copy_(rnd(M, Kd))
        dd.copy_(rnd(M, Kd))
        want, other = new(), new()
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            both(other)
        both(want)
        torch.cuda.synchronize()
        for a, b, c in zip(outs, want, other):
            assert torch.equal(a, b) and torch.equal(a, c)


# ------------------------------------------------------------------- refusals --

P = ctypes.c_void_p


def test_forward_refusals_before_launch():
    lib = K.lib()

    def call(M=16, N=64, Kd=128, x=P(1 << 20), ldx=128, w=P(1 << 21), ldw=128, act=3, bias=P(1 << 22), r=None, ldr=0,
             c=P(1 << 23), dt=1, ldc=64, pre=P(1 << 24), ldp=64, ws=None, nws=0):
        return lib.mr_gemm_act(M, N, Kd, x, ldx, w, ldw, act, bias, r, ldr, c, dt, ldc, pre, ldp, ws, nws, None)

    for bad, word in ((dict(M=-1), b"negative"), (dict(act=5), b"activation"), (dict(act=-1), b"activation"),
                      (dict(x=None), b"null"), (dict(w=None), b"null"), (dict(c=None), b"null"), (dict(N=60), b"multiple"),
                      (dict(Kd=100), b"multiple"), (dict(Kd=0), b"multiple"), (dict(M=1 << 31), b"large"),
                      (dict(dt=2), b"fp32 or bf16"), (dict(r=P(1 << 25), ldr=64), b"residual"),
                      (dict(ldx=64), b"smaller"), (dict(ldw=64), b"smaller"), (dict(ldc=56), b"smaller"),
                      (dict(ldp=56), b"smaller"), (dict(ldx=1 << 23), b"above"), (dict(x=P((1 << 20) + 8)), b"aligned"),
                      (dict(ldw=132), b"aligned"), (dict(pre=P((1 << 24) + 2)), b"aligned"), (dict(ldc=68), b"aligned"),
                      (dict(bias=P((1 << 22) + 1)), b"aligned"), (dict(c=P((1 << 20) + 1024)), b"overlap"),
                      (dict(pre=P((1 << 23) + 64)), b"overlap"), (dict(c=P(1 << 22)), b"overlap"),
                      (dict(ws=P(1 << 24), nws=4096), b"overlap"),
                      (dict(dt=0, r=P((1 << 23) + 256), ldr=64), b"overlap"), (dict(ws=P((1 << 26) + 8), nws=64), b"workspace")):
        assert call(**bad) == -22, bad
        assert word in lib.mr_last_error(), (bad, lib.mr_last_error())


def test_backward_refusals_before_launch():
    lib = K.lib()

    def call(M=16, N=64, Kd=128, dd=P(1 << 20), ldd=128, w=P(1 << 21), ldw=64, pre=P(1 << 22), ldp=64, act=0, d=P(1 << 23),
             ldo=64, db=P(1 << 24), part=P(1 << 25), npart=4096, ws=None, nws=0):
        return lib.mr_gemm_act_bwd(M, N, Kd, dd, ldd, w, ldw, pre, ldp, act, d, ldo, db, part, npart, ws, nws, None)

    for bad, word in ((dict(N=-8), b"negative"), (dict(act=9), b"activation"), (dict(dd=None), b"null"), (dict(pre=None), b"null"),
                      (dict(d=None), b"null"), (dict(M=0), b"no rows"), (dict(N=12), b"multiple"), (dict(Kd=32), b"multiple"),
                      (dict(ldw=56), b"smaller"), (dict(ldp=32), b"smaller"), (dict(part=None), b"partials"),
                      (dict(npart=16), b"partials"), (dict(part=P((1 << 25) + 4)), b"aligned"), (dict(w=P((1 << 21) + 2)), b"aligned"),
                      (dict(d=P((1 << 22) + 16)), b"overlap"), (dict(d=P(1 << 22), ldo=72), b"overlap"),
                      (dict(db=P(1 << 25)), b"overlap"), (dict(part=P(1 << 21)), b"overlap")):
        assert call(**bad) == -22, bad
        assert word in lib.mr_last_error(), (bad, lib.mr_last_error())

    def last(M=16, N=64, dout=P(1 << 20), dt=0, ldo=64, pre=P(1 << 22), ldp=64, act=0, d=P(1 << 23), ldd=64, db=None, part=None,
             npart=0):
        return lib.mr_act_bwd(M, N, dout, dt, ldo, pre, ldp, act, d, ldd, db, part, npart, None)

    for bad, word in ((dict(M=-1), b"negative"), (dict(act=7), b"activation"), (dict(dt=2), b"dout"), (dict(dout=None), b"null"),
                      (dict(N=12), b"multiple"), (dict(M=1 << 22), b"large"), (dict(ldd=32), b"smaller"),
                      (dict(ldo=66), b"aligned"), (dict(db=P(1 << 24)), b"partials"), (dict(d=P(1 << 20)), b"overlap"),
                      (dict(M=0, db=P(1 << 24)), b"no rows")):
        assert last(**bad) == -22, bad
        assert word in lib.mr_last_error(), (bad, lib.mr_last_error())


def test_bindings_refuse_on_the_host():
    x, w, out = torch.zeros(4, 64, dtype=BF), torch.zeros(16, 64, dtype=BF), torch.zeros(4, 16, dtype=BF)
    with pytest.raises(KernelError, match="activation"):
        K.gemm_act(x, w, out, act="tanh")
    with pytest.raises(KernelError, match="w must be"):
        K.gemm_act(x, w.float(), out, act="silu")
    with pytest.raises(KernelError, match="out must be"):
        K.gemm_act(x, w, out[:3], act="silu")
    with pytest.raises(KernelError, match="bias"):
        K.gemm_act(x, w, out, act="silu", bias=torch.zeros(15))
    with pytest.raises(KernelError, match="resid"):
        K.gemm_act(x, w, out.float(), act="silu", resid=torch.zeros(4, 15))
    with pytest.raises(KernelError, match="ROCm device"):
        K.gemm_act(x, w, out, act="silu")
    with pytest.raises(KernelError, match="pre must be"):
        K.gemm_act_bwd(x, w.t().contiguous(), out.float(), out, act="silu")
    with pytest.raises(KernelError, match="dbias"):
        K.act_bwd(out.float(), out, out, act="silu", dbias=torch.zeros(3, device="cpu"))


def test_columns_past_a_launch_are_refused_before_it():
    """The bias gradient's sum takes 1024 threads for 64 columns, and a launch's threads are a 32-bit number."""
    lib, N = K.lib(), 1 << 28
    far = lambda n: P(n << 50)
    assert lib.mr_act_bwd(1, N, far(1), 0, N, far(2), N, 0, far(3), N, far(4), far(5), ctypes.c_size_t(4 * N), None) == -22
    assert b"large" in lib.mr_last_error()


@pytest.mark.gpu
def test_a_single_row_of_any_stride():
    """A single row's stride leads nowhere: rows of odd, of huge and of no distance give what a row of its own gives."""
    print("case act single row", file=sys.stderr, flush=True)
    N, Kd, g = 64, 128, torch.Generator().manual_seed(4)
    full = lambda n, dt: torch.randn(1, n, generator=g).to(dt).to(dev())
    x, w, r, pre0 = full(Kd, BF), torch.randn(N, Kd, generator=g).to(BF).to(dev()), full(N, torch.float32), full(N, BF)
    dd, wd = full(Kd, BF), torch.randn(Kd, N, generator=g).to(BF).to(dev())

    def row(t, stride):  # the same values, and a stride of its own
        return t.clone().as_strided(t.shape, (stride, 1))

    def outputs(at):
        out, pre = at(torch.zeros(1, N, device=dev())), at(torch.zeros(1, N, dtype=BF, device=dev()))
        K.gemm_act(at(x), w, out, act="silu", pre=pre, resid=at(r))
        d1, d2 = at(torch.zeros(1, N, dtype=BF, device=dev())), at(torch.zeros(1, N, dtype=BF, device=dev()))
        K.gemm_act_bwd(at(dd), wd, at(pre0), d1, act="gelu")
        K.act_bwd(at(r), at(pre0), d2, act="relu2")
        return out, pre, d1, d2

    want = outputs(lambda t: t.clone())
    for stride in (0, 131, 1 << 30):
        for got, ref in zip(outputs(lambda t: row(t, stride)), want):
            assert torch.equal(got, ref), stride
