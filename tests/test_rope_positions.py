"""Rotary positions of any layout (``rope_positions``) against the rotation in
float64, and what it refuses.

Bound of one element: the angle is off by half a unit of its distance from a
whole turn (2 pi 2^-26) and, far out, by 2^-53 of the turns (under 2^-22 at
2^31); sine and cosine by 2 units (2^-23); the scale, two products and a sum
round once each (2^-24): (|a| + |b|) s 2^-20 covers them twice over, and the
output rounds by half a unit of its type.
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

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def expected(x, positions, freq, *, n_heads, d, pairing, scale, backward):
    """(rotated heads [T, n_heads, d], bound) in float64 on the CPU."""
    r = 2 * freq.numel()
    x = x.cpu().double()[:, :n_heads * d].reshape(-1, n_heads, d)
    ang = positions.cpu().double()[:, None] * freq.cpu()[None]
    if backward:
        ang = -ang
    c, s = (ang.cos() * scale)[:, None], (ang.sin() * scale)[:, None]
    y, mag = x.clone(), torch.zeros_like(x)
    ia = torch.arange(r // 2) if pairing == "half" else 2 * torch.arange(r // 2)
    ib = ia + (r // 2 if pairing == "half" else 1)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * scale
    return y, mag


def check(got, y, mag, dtype):
    eps = torch.finfo(dtype).eps
    tol = mag * 2.0 ** -20 + y.abs() * (eps / 2) * (1 + 2.0 ** -10) * (mag > 0) + 2.0 ** -25 * (dtype == torch.float16)
    err = (got.cpu().double() - y).abs()
    assert bool((err <= tol).all()), f"worst {float((err - tol).max())} past its bound of {float(tol.max())}"


def frequencies(r, theta=10000.0):
    return theta ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)


CASES = [
    # T, heads, extra columns, d, r, pairing
    (1, 1, 0, 2, 2, "half"),
    (1, 32, 512, 128, 128, "half"),
    (7, 3, 0, 64, 32, "interleaved"),
    (129, 5, 8, 80, 32, "half"),
    (33, 2, 3, 96, 38, "half"),          # 19 pairs, rows off 16 bytes
    (33, 2, 3, 96, 38, "interleaved"),
    (50, 4, 1, 10, 6, "interleaved"),
    (50, 4, 1, 10, 6, "half"),
    (2500, 9, 3, 64, 64, "interleaved"),
    (1, 1, 0, 256, 64, "half"),
    (3, 1, 0, 4096, 4096, "half"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_rotation(case, backward, dtype):
    T, H, extra, d, r, pairing = case
    print("case rope", case, backward, dtype, file=sys.stderr, flush=True)
    g = torch.Generator().manual_seed(11)
    x = torch.randn(T, H * d + extra, generator=g).to(DT[dtype]).to(dev())
    pos = torch.randint(0, 1 << 20, (T,), generator=g, dtype=torch.int32).to(dev())
    freq = frequencies(r)
    kw = dict(n_heads=H, head_dim=d, pairing=pairing, scale=1.25, backward=backward)
    y, mag = expected(x, pos, freq, n_heads=H, d=d, pairing=pairing, scale=1.25, backward=backward)
    out = torch.full_like(x, 7.0)
    K.rope_positions(x, pos, freq.to(dev()), out=out, **kw)
    check(out[:, :H * d].reshape(T, H, d), y, mag, DT[dtype])
    assert bool((out[:, H * d:] == 7.0).all())  # columns past the heads are not written
    # in place: the same bits, and the columns past the heads kept
    before = x.clone()
    K.rope_positions(x, pos, freq.to(dev()), **kw)
    assert torch.equal(x[:, :H * d], out[:, :H * d]) and torch.equal(x[:, H * d:], before[:, H * d:])


@pytest.mark.gpu
@pytest.mark.parametrize("positions", [[0, 0, 0], [2**31 - 1, 2**31 - 2, 12345678], [-5, -(2**31), 3]])
def test_far_and_negative_positions(positions):
    print("case rope far", positions, file=sys.stderr, flush=True)
    x = torch.randn(3, 2 * 64, generator=torch.Generator().manual_seed(3)).to(dev())
    pos = torch.tensor(positions, dtype=torch.int32)
    freq = frequencies(64)
    y, mag = expected(x, pos, freq, n_heads=2, d=64, pairing="half", scale=1.0, backward=False)
    K.rope_positions(x, pos.to(dev()), freq.to(dev()), n_heads=2, head_dim=64)
    check(x.view(3, 2, 64), y, mag, torch.float32)


@pytest.mark.gpu
def test_unrotated_values_pass_as_they_are():
    """Infinities, NaN and negative zeros past the rotated part, and none from it."""
    x = torch.zeros(4, 64, device=dev())
    x[:, 33], x[:, 34], x[:, 35], x[:, 36] = math.inf, -math.inf, math.nan, -0.0
    x[:, :32] = 1.0
    for pairing in ("half", "interleaved"):
        out = torch.empty_like(x)
        K.rope_positions(x, torch.arange(4, dtype=torch.int32, device=dev()), frequencies(32).to(dev()), n_heads=1,
                         head_dim=64, pairing=pairing, out=out)
        assert torch.equal(out[:, 32:].view(torch.int32), x[:, 32:].view(torch.int32))
        assert bool(torch.isfinite(out[:, :32]).all())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    T, ld = 34000, 65600  # 4.46 GB of bfloat16
    x = torch.zeros(T, ld, dtype=torch.bfloat16, device=dev())
    rows = torch.tensor([0, T // 2, T - 1])
    vals = torch.randn(3, 128, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    x[rows, :128] = vals.to(dev())
    pos = torch.arange(T, dtype=torch.int32, device=dev())
    freq = frequencies(64)
    K.rope_positions(x, pos, freq.to(dev()), n_heads=2, head_dim=64)
    y, mag = expected(vals, rows, freq, n_heads=2, d=64, pairing="half", scale=1.0, backward=False)
    check(x[rows, :128].view(3, 2, 64), y, mag, torch.bfloat16)


@pytest.mark.gpu
def test_backward_is_the_gradient():
    """<g, R x> = <R^T g, x>, the rotation being linear, in float32."""
    gen = torch.Generator().manual_seed(8)
    x, g = (torch.randn(40, 4 * 96, generator=gen).to(dev()) for _ in range(2))
    pos = torch.randint(0, 5000, (40,), generator=gen, dtype=torch.int32).to(dev())
    for pairing in ("half", "interleaved"):
        kw = dict(n_heads=4, head_dim=96, pairing=pairing, scale=1.1)
        y, dx = torch.empty_like(x), torch.empty_like(x)
        K.rope_positions(x, pos, frequencies(48).to(dev()), out=y, **kw)
        K.rope_positions(g, pos, frequencies(48).to(dev()), out=dx, backward=True, **kw)
        lhs, rhs = float((g.double() * y.double()).sum()), float((dx.double() * x.double()).sum())
        # every element within 2^-20 of (|a| + |b|) s
        bound = 2 * 2.0 ** -20 * 1.1 * 2 * float(g.double().norm() * x.double().norm())
        assert abs(lhs - rhs) <= bound


@pytest.mark.gpu
def test_graph_and_stream():
    """Captured on a side stream and replayed with new inputs between eager work."""
    H, d, T = 6, 64, 70
    x, out = torch.zeros(T, H * d, device=dev(), dtype=torch.bfloat16), torch.empty(T, H * d, device=dev(), dtype=torch.bfloat16)
    pos = torch.zeros(T, dtype=torch.int32, device=dev())
    freq = frequencies(d).to(dev())
    kw = dict(n_heads=H, head_dim=d, pairing="interleaved")
    K.rope_positions(x, pos, freq, out=out, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.rope_positions(x, pos, freq, out=out, **kw)
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(T, H * d, generator=gen))
        pos.copy_(torch.randint(0, 10000, (T,), generator=gen, dtype=torch.int32))
        graph.replay()
        want = torch.empty_like(out)
        K.rope_positions(x, pos, freq, out=want, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_empty():
    K.rope_positions(torch.empty(0, 64, device=dev()), torch.empty(0, dtype=torch.int32, device=dev()),
                     frequencies(64).to(dev()), n_heads=1, head_dim=64)


def test_refusals_before_launch():
    lib, P = K.lib(), ctypes.c_void_p
    f = ctypes.c_float(1.0)

    def call(x=P(4096), dt=1, ldx=256, T=4, H=2, d=128, pos=P(1 << 20), freq=P(1 << 21), r=128, pair=0, out=P(1 << 22),
             ldo=256):
        return lib.mr_rope_positions(x, dt, ldx, T, H, d, pos, freq, r, pair, f, 0, out, ldo, None)

    for bad, word in ((dict(x=None), b"null"), (dict(pos=None), b"null"), (dict(freq=None), b"null"),
                      (dict(out=None), b"null"), (dict(dt=3), b"dtype"), (dict(pair=2), b"pairing"),
                      (dict(r=3), b"even"), (dict(r=130), b"even"), (dict(r=0), b"even"), (dict(ldx=255), b"leading"),
                      (dict(ldo=255), b"leading"), (dict(T=-1), b"sizes"), (dict(T=1 << 31), b"rows"),
                      (dict(d=5000, ldx=10000, ldo=10000, r=64), b"4096"), (dict(x=P(4097)), b"aligned"),
                      (dict(out=P(4096 + 512)), b"share"), (dict(out=P(4096), ldo=512), b"share"),
                      (dict(pos=P(1 << 22)), b"share"), (dict(freq=P((1 << 22) + 8)), b"share")):
        assert call(**bad) == -22, bad
        assert word in lib.mr_last_error(), (bad, lib.mr_last_error())


def test_binding_refuses_on_the_host():
    x = torch.zeros(4, 128)
    pos, freq = torch.zeros(4, dtype=torch.int32), frequencies(64)
    kw = dict(n_heads=2, head_dim=64)
    with pytest.raises(KernelError, match="pairing"):
        K.rope_positions(x, pos, freq, pairing="both", **kw)
    with pytest.raises(KernelError, match="int32"):
        K.rope_positions(x, pos.long(), freq, **kw)
    with pytest.raises(KernelError, match="float64"):
        K.rope_positions(x, pos, freq.float(), **kw)
    with pytest.raises(KernelError, match="one position each"):
        K.rope_positions(x, pos[:3], freq, **kw)
    with pytest.raises(KernelError, match="heads"):
        K.rope_positions(x, pos, freq, n_heads=3, head_dim=64)
    with pytest.raises(KernelError, match="dtype"):
        K.rope_positions(x, pos, freq, out=x.half(), **kw)
    with pytest.raises(KernelError, match="ROCm device"):
        K.rope_positions(x, pos, freq, **kw)


def test_rows_past_a_launch_are_refused_before_it():
    """A block takes some tokens, and blocks times threads is a 32-bit number: the first row too many of each kind."""
    lib, P = K.lib(), ctypes.c_void_p
    for d, tokens in ((4096, 1), (128, 4), (2, 256)):
        T = (((1 << 32) - 1) // 256) * tokens + 1
        if T > 0x7fffffff:
            T = 1 << 31
        assert lib.mr_rope_positions(P(1 << 50), 1, d, T, 1, d, P(2 << 50), P(3 << 50), d, 0, ctypes.c_float(1.0), 0,
                                     P(4 << 50), d, None) == -22, d
        assert b"too many rows" in lib.mr_last_error()


# rows enough for several tokens a block, the last block short of them, whole pieces of 16 bytes and not
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("case", [(4000, 16, 128, 64, 32, "interleaved"), (9001, 4, 0, 128, 64, "half"),
                                  (2049, 2, 64, 64, 64, "half"), (4099, 3, 0, 64, 16, "half"),
                                  (4099, 3, 0, 64, 16, "interleaved"), (3203, 2, 3, 80, 20, "half"),
                                  (20001, 1, 0, 32, 32, "interleaved"), (300003, 1, 0, 16, 2, "half")],
                         ids=lambda c: "x".join(map(str, c)))
def test_blocks_of_several_tokens(case, backward, dtype):
    test_rotation(case, backward, dtype)
