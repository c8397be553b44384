"""Decoder blocks whose rotation covers part of a head, pairs neighbours or is
scaled for long contexts, an ungated MLP, and the teacher objective, each along
the path that a user takes it: checkpoint configs, the block engine's forward
and backward, whole-model scoring.

Frequencies are held to Hugging Face transformers' own rope initialisation, run
as a library; blocks and losses to float64. Results that pass through bfloat16
operands are held to 1e-2 of their norm, as the other block tests hold them.
"""

from __future__ import annotations

import json
import math
import sys

import pytest
import torch

from mround_amd import api
from mround_amd import kernels as K
from mround_amd.exceptions import ArchitectureError, CalibrationError, SchemeError
from mround_amd.pipeline.block import (LAYERS, BlockEngine, BlockShape, BlockWeights, placements, rope_frequencies,
                                       rope_magnitude, unplace)
from mround_amd.pipeline.checkpoint import DecoderModel, block_shape, write_random_checkpoint
from mround_amd.schemes import QuantScheme, Symmetry
from oracle import block as OB
from oracle import causal_lm as OC
from tests.helpers import dev

BASE = {"model_type": "llama", "hidden_size": 512, "num_attention_heads": 8, "num_key_value_heads": 4,
        "intermediate_size": 1024, "rope_theta": 10000.0}


# --------------------------------------------------------------- configs (CPU) --

@pytest.mark.parametrize("extra", [{}, {"beta_fast": 16.0, "beta_slow": 2.0}, {"attention_factor": 1.25},
                                   {"mscale": 0.8, "mscale_all_dim": 0.5}, {"truncate": False}, {"factor": 1.0}])
def test_yarn_matches_the_rope_initialisation(extra):
    R = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import LlamaConfig

    scaling = {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096, **extra}
    shape = block_shape({**BASE, "head_dim": 128, "rope_scaling": scaling})
    cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, head_dim=128, rope_theta=10000.0, rope_scaling=dict(scaling),
                      max_position_embeddings=int(4096 * scaling["factor"]))
    inv, magnitude = R.ROPE_INIT_FUNCTIONS["yarn"](cfg, "cpu")
    got = rope_frequencies(128, 10000.0, shape.rope_scaling)
    # theirs is float32: a power, a division, a blend of two products
    assert torch.allclose(got, inv.double(), rtol=2.0 ** -20, atol=0)
    assert rope_magnitude(shape.rope_scaling) == pytest.approx(float(magnitude), rel=1e-12)


def test_configs_of_other_rotations():
    s = block_shape({**BASE, "partial_rotary_factor": 0.5, "rope_traditional": True})
    assert s.rotary_dim == 32 and s.rope_interleaved
    s = block_shape({**BASE, "rope_parameters": {"rope_theta": 5e5, "partial_rotary_factor": 0.25}})
    assert s.rotary_dim == 16 and s.rope_theta == 10000.0
    assert block_shape({**BASE, "partial_rotary_factor": 1.0}).rotary_dim == 0
    for bad in (0.0, 0.02, 1.5):
        with pytest.raises(ArchitectureError, match="partial_rotary_factor"):
            block_shape({**BASE, "partial_rotary_factor": bad})
    with pytest.raises(ArchitectureError, match="lacks"):
        block_shape({**BASE, "rope_scaling": {"rope_type": "yarn", "factor": 4.0}})
    with pytest.raises(ArchitectureError, match="rotated part"):
        BlockShape(hidden=512, n_heads=8, n_kv_heads=4, head_dim=64, intermediate=1024, rotary_dim=66).validate()
    with pytest.raises(SchemeError, match="sensitivity_objective"):
        api.plan_mixed_precision("nowhere", 3.0, sensitivity_objective="tokens")


# -------------------------------------------------------------- blocks (oracle) --

def rotate(shape):
    """The oracle's rotation of ``[B, H, S, d]`` for a block's shape."""
    r = shape.rotary_dim or shape.head_dim
    freq, mag = rope_frequencies(r, shape.rope_theta, shape.rope_scaling), rope_magnitude(shape.rope_scaling)

    def fn(x, *_):
        ang = torch.arange(x.shape[2], dtype=torch.float64)[:, None] * freq
        c, s = ang.cos() * mag, ang.sin() * mag
        y = x.clone()
        i = torch.arange(r // 2)
        ia, ib = (2 * i, 2 * i + 1) if shape.rope_interleaved else (i, i + r // 2)
        y[..., ia], y[..., ib] = x[..., ia] * c - x[..., ib] * s, x[..., ia] * s + x[..., ib] * c
        return y
    return fn


YARN = (("beta_fast", 32.0), ("factor", 4.0), ("original_max_position_embeddings", 64.0), ("rope_type", "yarn"))
FORMS = [dict(rotary_dim=32), dict(rope_interleaved=True), dict(rope_scaling=YARN),
         dict(rotary_dim=16, rope_interleaved=True, rope_scaling=YARN)]


def make_shape(form, **kw):
    return BlockShape(**{**dict(hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, intermediate=384, rope_theta=10000.0,
                                attn_bias=True), **form, **kw})


def oracle_shape(s):
    return OB.Shape(hidden=s.hidden, n_heads=s.n_heads, n_kv_heads=s.n_kv_heads, head_dim=s.head_dim,
                    intermediate=s.intermediate, norm_eps=s.norm_eps, rope_theta=s.rope_theta)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("form", FORMS, ids=["partial", "interleaved", "yarn", "all"])
def test_block_forward_and_backward(form, split, monkeypatch):
    shape = make_shape(form)
    print("case block form", form, split, file=sys.stderr, flush=True)
    w = BlockWeights.random(shape, dtype=torch.bfloat16, device=dev(), seed=4, std=0.05)
    B, S = 2, 128
    g = torch.Generator().manual_seed(7)
    x, dout = torch.randn(B, S, shape.hidden, generator=g), torch.randn(B, S, shape.hidden, generator=g) * 1e-2
    eng = BlockEngine(shape, batch=B, seq_len=S, device=dev(), split=split)
    eng.set_block(w)
    eng.load_dense(w.linears)
    out, dx = torch.empty(B * S, shape.hidden, device=dev()), torch.empty(B * S, shape.hidden, device=dev())
    eng.forward(x.view(B * S, -1).to(dev()), out, save=True)
    eng.grad_out.copy_(dout.view(B * S, -1))
    eng.backward(dx_out=dx)

    monkeypatch.setattr(OB, "rope", rotate(shape))
    lin = {n: t.cpu().double().requires_grad_() for n, t in w.linears.items()}
    xo = x.double().requires_grad_()
    ref = OB.block_forward(xo, lin, {n: b.cpu().double() for n, b in w.biases.items()},
                           (w.input_norm.cpu().double(), w.post_norm.cpu().double()), oracle_shape(shape))
    ref.backward(dout.double())
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())
    assert rel(out.view(B, S, -1) - x.to(dev()), ref.detach() - x.double()) < (1e-3 if split else 1e-2)
    assert rel(dx.view(B, S, -1), xo.grad) < 1e-2
    place = placements(shape)
    for n in LAYERS:
        got = unplace(eng.dw[place[n].operand], lin[n].shape[0], place[n])
        assert rel(got, lin[n].grad) < 1.5e-2, n


@pytest.mark.gpu
def test_the_plain_rotation_by_either_kernel():
    """Halves of whole heads: the block's table and the positions' angles agree to a rounding of bfloat16."""
    T, S, H, d = 256, 128, 6, 64
    x = torch.randn(T, H * d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev())
    a, b = x.clone(), x.clone()
    from mround_amd.pipeline.block import rope_table
    K.rope(a, seq_len=S, n_heads=H, head_dim=d, cos_sin=rope_table(S, d, 1e6, dev()))
    pos = torch.arange(S, dtype=torch.int32, device=dev()).repeat(T // S)
    K.rope_positions(b, pos, rope_frequencies(d, 1e6).to(dev()), n_heads=H, head_dim=d)
    # both are within 2^-20 (|a| + |b|) of the value before they round: a rounding may fall either way
    mag = x.float().view(T, H, 2, d // 2).abs().sum(2, keepdim=True).expand(T, H, 2, d // 2).reshape(T, H * d)
    assert bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * a.float().abs() + 2.0 ** -19 * mag).all())


# ---------------------------------------------------- one decoder, end to end --

@pytest.mark.gpu
def test_ungated_decoder_against_its_teacher():
    """Projections, a partial rotation, attention, an ungated MLP, the head and the loss against a teacher's
    list, run together and back: logits, loss and every weight's gradient against float64."""
    B, S, h, H, Hkv, d, mlp, V, k = 2, 128, 256, 4, 2, 64, 512, 1000, 24
    T, rows = B * S, (H + 2 * Hkv) * d
    g = torch.Generator().manual_seed(21)
    rnd = lambda *s, std=1.0: torch.randn(*s, generator=g) * std
    bf = torch.bfloat16
    w = {n: rnd(*s, std=s[1] ** -0.5).to(bf) for n, s in
         {"qkv": (rows, h), "o": (h, H * d), "up": (mlp, h), "down": (h, mlp), "head": (V, h)}.items()}
    bias = rnd(mlp, std=0.1)
    x = rnd(T, h)
    freq = rope_frequencies(32, 10000.0)
    pos = torch.arange(S, dtype=torch.int32).repeat(B)
    teacher = rnd(T, V, std=2.0).to(bf)

    # ---- the framework's calls
    to = lambda t: t.to(dev())
    e = lambda *s, dt=bf: torch.empty(*s, dtype=dt, device=dev())
    wd, f32 = {n: to(t) for n, t in w.items()}, torch.float32
    values, ids, lse = e(T, k, dt=f32), e(T, k, dt=torch.int32), e(T, dt=f32)
    K.top_logits(to(teacher), V=V, values=values, ids=ids, lse=lse)
    rope = dict(n_heads=H + Hkv, head_dim=d, pairing="interleaved")
    xd = to(x)
    xb = xd.to(bf)
    qkv, attn, lse_a = e(T, rows), e(T, H * d), e(B, H, S, dt=f32)
    K.gemm("nt", xb, wd["qkv"], qkv, M=T, N=rows, K=h)
    K.rope_positions(qkv, to(pos), to(freq), **rope)
    geo = dict(batch=B, seq_len=S, n_heads=H, n_kv_heads=Hkv, head_dim=d, scale=d ** -0.5)
    K.attn_fwd(qkv, out=attn, lse=lse_a, **geo)
    h1 = e(T, h, dt=f32)
    K.gemm("nt", attn, wd["o"], h1, M=T, N=h, K=H * d, resid=xd)
    h1b = h1.to(bf)
    hidden, pre = e(T, mlp), e(T, mlp)
    K.gemm_act(h1b, wd["up"], hidden, act="relu2", bias=to(bias), pre=pre)
    h2 = e(T, h, dt=f32)
    K.gemm("nt", hidden, wd["down"], h2, M=T, N=h, K=mlp, resid=h1)
    h2b, logits = h2.to(bf), e(T, V)
    K.gemm("nt", h2b, wd["head"], logits, M=T, N=V, K=h)
    row, loss, dlogits = e(T, dt=f32), e(1, dt=f32), e(T, V)
    K.distill_loss(logits, values, ids, V=V, scale=1.0 / T, row_loss=row, lse=lse, loss_out=loss, dlogits=dlogits)
    grads = {n: e(*t.shape, dt=f32) for n, t in w.items()}
    K.gemm("tn", dlogits, h2b, grads["head"], M=V, N=h, K=T)
    # (the head's rows, 1000, are not whole k-tiles: the product by a padded copy)
    pad = lambda t, n: torch.nn.functional.pad(t, (0, n - t.shape[1]))
    dh2 = e(T, h, dt=f32)
    K.gemm("nn", pad(dlogits, 1024), torch.nn.functional.pad(wd["head"], (0, 0, 0, 24)), dh2, M=T, N=h, K=1024)
    dh2b, dpre, db = dh2.to(bf), e(T, mlp), e(mlp, dt=f32)
    K.gemm("tn", dh2b, hidden, grads["down"], M=h, N=mlp, K=T)
    K.gemm_act_bwd(dh2b, wd["down"], pre, dpre, act="relu2", dbias=db)
    K.gemm("tn", dpre, h1b, grads["up"], M=mlp, N=h, K=T)
    dh1 = e(T, h, dt=f32)
    K.gemm("nn", dpre, wd["up"], dh1, M=T, N=h, K=mlp, resid=dh2)
    dh1b, dattn, dqkv, dsum = dh1.to(bf), e(T, H * d), e(T, rows), e(B, H, S, dt=f32)
    K.gemm("tn", dh1b, attn, grads["o"], M=h, N=H * d, K=T)
    K.gemm("nn", dh1b, wd["o"], dattn, M=T, N=H * d, K=h)
    K.attn_bwd(qkv, attn, dattn, lse_a, dsum, dqkv=dqkv, **geo)
    K.rope_positions(dqkv, to(pos), to(freq), backward=True, **rope)
    K.gemm("tn", dqkv, xb, grads["qkv"], M=rows, N=h, K=T)

    # ---- float64
    lw = {n: t.double().requires_grad_() for n, t in w.items()}
    bo = bias.double().requires_grad_()
    shape = BlockShape(hidden=h, n_heads=H, n_kv_heads=Hkv, head_dim=d, intermediate=mlp, rotary_dim=32, rope_interleaved=True)
    spin = rotate(shape)
    heads = (xb.cpu().double() @ lw["qkv"].t()).view(B, S, H + 2 * Hkv, d).transpose(1, 2)
    q, kk, v = spin(heads[:, :H]), spin(heads[:, H:H + Hkv]), heads[:, H + Hkv:]
    kk, v = kk.repeat_interleave(H // Hkv, 1), v.repeat_interleave(H // Hkv, 1)
    sc = (q @ kk.transpose(-1, -2)) * d ** -0.5
    sc = sc.masked_fill(~torch.ones(S, S, dtype=torch.bool).tril(), -math.inf)
    o = (torch.softmax(sc, -1) @ v).transpose(1, 2).reshape(T, H * d)
    r1 = x.double() + o @ lw["o"].t()
    r2 = r1 + torch.relu(r1 @ lw["up"].t() + bo).square() @ lw["down"].t()
    z = r2 @ lw["head"].t()
    tl = torch.log_softmax(teacher.double(), 1)
    on = torch.zeros(T, V, dtype=torch.bool).scatter_(1, ids.cpu().long(), True)
    lp = torch.log_softmax(z, 1)
    rest = lambda t: torch.logsumexp(t.masked_fill(on, -math.inf), 1)
    ref = (torch.where(on, tl.exp() * (tl - lp), 0.0).sum(1) + rest(tl).exp() * (rest(tl) - rest(lp))).mean()
    ref.backward()
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())
    assert rel(logits, z.detach()) < 1e-2
    assert float(loss) == pytest.approx(float(ref.detach()), rel=1e-2)
    assert rel(db, bo.grad) < 2e-2
    for n in w:
        assert rel(grads[n], lw[n].grad) < 2e-2, n


# -------------------------------------------------------- scoring by a teacher --

def tiny_model(form, layers=2, vocab=300, seed=3):
    from mround_amd.pipeline.runner import DecoderBlock

    shape = make_shape(form, attn_bias=False)
    blocks = [DecoderBlock(i, f"model.layers.{i}", shape, BlockWeights.random(shape, dtype=torch.bfloat16, device=dev(),
                                                                               seed=seed + i, std=0.05)) for i in range(layers)]
    g = torch.Generator().manual_seed(seed)
    embed = (torch.randn(vocab, shape.hidden, generator=g)).to(torch.bfloat16).to(dev())
    head = (torch.randn(vocab, shape.hidden, generator=g) * 0.15).to(torch.bfloat16).to(dev())
    model = DecoderModel({}, torch.bfloat16, embed, blocks, torch.ones(shape.hidden, device=dev()), head)
    om = OC.Model(oracle_shape(shape), embed.cpu().double(),
                  [(b.name, {n: t.cpu().double() for n, t in b.weights.linears.items()}, {},
                    (b.weights.input_norm.cpu().double(), b.weights.post_norm.cpu().double())) for b in blocks],
                  torch.ones(shape.hidden, dtype=torch.float64), head.cpu().double())
    return model, om


@pytest.mark.gpu
@pytest.mark.parametrize("form", [{}, dict(rotary_dim=32, rope_interleaved=True)], ids=["plain", "partial"])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_teacher_objective_of_a_model(form, temperature, monkeypatch):
    """The loss and the block gradients of the quantized model against its own list, a short batch in a larger
    engine, lengths of no whole tiles."""
    from mround_amd.pipeline.causal_lm import CausalLM
    from mround_amd.core.quantizer import mode_of

    model, om = tiny_model(form)
    monkeypatch.setattr(OB, "rope", rotate(model.blocks[0].shape))
    scheme = QuantScheme(bits=3, group_size=64, symmetry=Symmetry.ASYMMETRIC)
    tokens = torch.randint(0, 300, (2, 101), generator=torch.Generator().manual_seed(5))
    lm = CausalLM(model, batch=3, seq_len=101, device=dev())
    lm.set_weights({})
    teacher = lm.teacher_list(tokens, top=32, temperature=temperature)
    assert bool((teacher.ids.view(3, -1, 32)[:2, :100] >= 0).all()) and bool((teacher.ids.view(3, -1, 32)[:2, 100:] == -1).all())
    assert bool((teacher.ids.view(3, -1, 32)[2] == -1).all())
    same = float(lm.run(tokens, teacher=teacher))
    assert abs(same) < 1e-5  # the model against itself
    lm.set_weights({f"{b.name}.{n}": scheme for b in model.blocks for n in LAYERS})
    got = {}
    loss = float(lm.run(tokens, lambda b, dw: got.update({(b, k): v.clone() for k, v in dw.items()}), teacher))

    def logits(linears):
        x = om.embed[tokens[:, :-1]]
        for name, lin, biases, norms in om.blocks:
            x = OB.block_forward(x, {n: linears.get(f"{name}.{n}", lin[n]) for n in LAYERS}, biases, norms, om.shape)
        return (OB.rms_norm(x, om.norm, om.shape.norm_eps) @ om.head.t()).flatten(0, 1) / temperature

    leaves = {f"{name}.{n}": torch.from_numpy(OC.rtn(lin[n].float().numpy(), bits=3, group_size=64, mode=mode_of(scheme))).double()
              .requires_grad_() for name, lin, *_ in om.blocks for n in LAYERS}
    with torch.no_grad():
        tl = torch.log_softmax(logits({}), 1)
    lists = teacher.ids.view(3, -1, 32)[:2, :100].reshape(-1, 32).cpu().long()
    on = torch.zeros_like(tl, dtype=torch.bool).scatter_(1, lists, True)
    lp = torch.log_softmax(logits(leaves), 1)
    rest = lambda t: torch.logsumexp(t.masked_fill(on, -math.inf), 1)
    ref = (torch.where(on, tl.exp() * (tl - lp), 0.0).sum(1) + rest(tl).exp() * (rest(tl) - rest(lp))).mean()
    ref.backward()
    assert loss == pytest.approx(float(ref.detach()), rel=5e-2)
    place = placements(model.blocks[0].shape)
    for b, blk in enumerate(model.blocks):
        for n in LAYERS:
            want = leaves[f"{blk.name}.{n}"].grad
            have = unplace(got[b, place[n].operand], want.shape[0], place[n]).cpu().double()
            # the gradient is a difference of predictions that bfloat16 logits carry to 2^-8 of themselves
            assert float((have - want).norm() / want.norm()) < 6e-2, (b, n)


@pytest.mark.gpu
def test_scores_against_the_teacher():
    from mround_amd.pipeline.scoring import score_widths

    model, _ = tiny_model(dict(rope_scaling=YARN))
    tokens = torch.randint(0, 300, (4, 65), generator=torch.Generator().manual_seed(6), device="cpu").to(dev())
    base = QuantScheme(bits=4, group_size=64, symmetry=Symmetry.ASYMMETRIC)
    for source in ("own_width", "widest"):
        s = score_widths(model, [tokens[:3], tokens[3:]], [2, 4], base, gradient_source=source, objective="teacher",
                         teacher_top=16).scores
        assert all(math.isfinite(v[2]) and v[2] > v[4] > 0 for v in s.values())
    with pytest.raises(ValueError, match="objective"):
        score_widths(model, [tokens], [2], base, objective="text")


@pytest.mark.gpu
def test_plan_by_the_teacher(tmp_path):
    """A checkpoint whose config asks for a partial, neighbour-paired, scaled rotation, planned by the command."""
    from mround_amd.cli import main

    cfg = dict(BASE, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=256,
               num_hidden_layers=2, vocab_size=200, rms_norm_eps=1e-6, tie_word_embeddings=True, torch_dtype="bfloat16",
               partial_rotary_factor=0.5, rope_traditional=True,
               rope_scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64})
    path = write_random_checkpoint(tmp_path / "m", cfg, seed=1, device=dev())
    out = tmp_path / "plan.json"
    assert main(["plan", str(path), "--average-bits", "3", "--options", "2,4", "--asym", "--objective", "teacher",
                 "--scoring-samples", "4", "--scoring-seq-len", "65", "--write", str(out)]) == 0
    assert len(json.loads(out.read_text())) == 14


@pytest.mark.gpu
def test_a_list_of_another_batch_is_refused():
    from mround_amd.pipeline.causal_lm import CausalLM

    model, _ = tiny_model({})
    lm = CausalLM(model, batch=2, seq_len=65, device=dev())
    lm.set_weights({})
    tokens = torch.randint(0, 300, (2, 65))
    teacher = lm.teacher_list(tokens)
    with pytest.raises(CalibrationError, match="another batch"):
        lm.run(tokens[:1], teacher=teacher)
    with pytest.raises(CalibrationError, match="1 to 1024"):
        lm.teacher_list(tokens, top=0)


@pytest.mark.gpu
@pytest.mark.parametrize("form", [dict(partial_rotary_factor=0.5),
                                  dict(rope_traditional=True, rope_scaling={"rope_type": "yarn", "factor": 4.0,
                                                                            "original_max_position_embeddings": 64})],
                         ids=["partial", "interleaved-yarn"])
def test_quantize_blocks_of_other_forms(tmp_path, form):
    """The whole run: scores by the teacher, tuning (steps recorded and replayed), holdout, export."""
    from mround_amd.schemes import TuningConfig

    cfg = dict(BASE, hidden_size=128, num_attention_heads=2, num_key_value_heads=1, head_dim=64, intermediate_size=256,
               num_hidden_layers=2, vocab_size=200, rms_norm_eps=1e-6, tie_word_embeddings=True, torch_dtype="bfloat16", **form)
    src = write_random_checkpoint(tmp_path / "m", cfg, seed=2, std=0.05)
    tuning = TuningConfig(iters=24, batch_size=2, n_samples=8, seq_len=100)
    kw = dict(symmetry=Symmetry.ASYMMETRIC, tuning=tuning, seed=5, average_bits=3.0, candidate_bits=(2, 4),
              sensitivity_objective="teacher")
    res = api.quantize(src, output_dir=tmp_path / "q", **kw)
    again = api.quantize(src, output_dir=tmp_path / "q2", **kw)
    assert len(res.summary.blocks) == 2
    for a, b in zip(res.summary.blocks, again.summary.blocks):
        assert math.isfinite(a.initial_loss) and a.final_loss <= a.initial_loss
        assert (a.initial_loss, a.final_loss) == (b.initial_loss, b.final_loss)
    assert (tmp_path / "q" / "model.safetensors").read_bytes() == (tmp_path / "q2" / "model.safetensors").read_bytes()


def test_a_list_knows_its_batch():
    from mround_amd.pipeline.causal_lm import TeacherList

    def made_from(t):
        e = torch.empty(0)
        return TeacherList(e, e, e, 1.0, t, t.to(torch.int32, copy=True), None if t.is_inference() else t._version)

    tokens = torch.randint(0, 300, (2, 65))
    teacher = made_from(tokens)
    other = tokens.clone()
    other[1, 7] += 1
    assert teacher.belongs_to(tokens) and teacher.belongs_to(tokens.clone()) and teacher.belongs_to(tokens.int())
    assert not teacher.belongs_to(other) and not teacher.belongs_to(tokens[:1]) and not teacher.belongs_to(tokens[:, :64])
    tokens[0, 3] += 1  # the same tensor with other tokens, and as it was
    assert not teacher.belongs_to(tokens)
    tokens[0, 3] -= 1
    assert teacher.belongs_to(tokens)
    with torch.inference_mode():
        inside = torch.randint(0, 300, (2, 65))
        teacher = made_from(inside)
        assert teacher.belongs_to(inside)
        inside[0, 0] += 1
        assert not teacher.belongs_to(inside)


@pytest.mark.gpu
def test_a_list_of_other_tokens_is_refused():
    """Lists of batches of one shape, taken before either is run, as a scoring pass takes them."""
    from mround_amd.pipeline.causal_lm import CausalLM

    model, _ = tiny_model({})
    lm = CausalLM(model, batch=2, seq_len=65, device=dev())
    lm.set_weights({})
    first, second = torch.randint(0, 300, (2, 65)), torch.randint(0, 300, (2, 65), device=dev())
    lists = lm.teacher_list(first), lm.teacher_list(second)
    with pytest.raises(CalibrationError, match="another batch"):
        lm.run(first, teacher=lists[1])
    with pytest.raises(CalibrationError, match="another batch"):
        lm.run(second, teacher=lists[0])
    assert abs(float(lm.run(first, teacher=lists[0]))) < 1e-5
    assert abs(float(lm.run(second.clone(), teacher=lists[1]))) < 1e-5
    second[0, 0] = (second[0, 0] + 1) % 300
    with pytest.raises(CalibrationError, match="another batch"):
        lm.run(second, teacher=lists[1])


def test_an_objective_without_a_scoring_pass_is_refused(tmp_path):
    from mround_amd.exceptions import SchemeError

    cfg = dict(BASE, hidden_size=128, num_attention_heads=2, num_key_value_heads=1, head_dim=64, intermediate_size=256,
               num_hidden_layers=1, vocab_size=200, rms_norm_eps=1e-6, tie_word_embeddings=True, torch_dtype="bfloat16")
    src = write_random_checkpoint(tmp_path / "m", cfg, seed=2)
    plan = {f"model.layers.0.{n}": 2 for n in LAYERS}
    for kw in (dict(), dict(average_bits=2.0, candidate_bits=(2, 4), plan=plan)):
        with pytest.raises(SchemeError, match="scoring pass"):
            api.quantize(src, output_dir=tmp_path / "q", device="cpu", sensitivity_objective="teacher", **kw)
    with pytest.raises(SchemeError, match="must be 'labels' or 'teacher'"):
        api.quantize(src, output_dir=tmp_path / "q", device="cpu", sensitivity_objective="text")
    assert not (tmp_path / "q").exists()


def _small(tmp_path, device, **form):
    cfg = dict(BASE, hidden_size=128, num_attention_heads=2, num_key_value_heads=1, head_dim=64, intermediate_size=256,
               num_hidden_layers=1, vocab_size=200, rms_norm_eps=1e-6, tie_word_embeddings=True, torch_dtype="bfloat16", **form)
    return str(write_random_checkpoint(tmp_path / "m", cfg, seed=2, std=0.05, device=device))


def test_the_command_asks_for_an_objective(tmp_path, capsys):
    from mround_amd.cli import main

    src, out = _small(tmp_path, "cpu"), str(tmp_path / "q")
    dry = ["quantize", src, "-o", out, "--dry-run", "--memory-budget", "100"]
    said = []
    for objective in ("labels", "teacher"):
        assert main([*dry, "--average-bits", "3", "--objective", objective]) == 0
        said.append(capsys.readouterr().out.split("scoring ")[1].split(" ")[0])
    assert said[0] != said[1]  # (the teacher's lists)
    assert main([*dry, "--objective", "teacher"]) == 1
    assert "scoring pass" in capsys.readouterr().err


@pytest.mark.gpu
def test_the_command_quantizes_by_the_teacher(tmp_path):
    from mround_amd.cli import main

    src, out = _small(tmp_path, dev()), tmp_path / "q"
    assert main(["quantize", src, "-o", str(out), "--asym", "--average-bits", "3", "--options", "2,4", "--objective",
                 "teacher", "--iters", "4", "--samples", "4", "--seq-len", "100", "--batch-size", "2"]) == 0
    record = json.loads((out / api.RUN_RECORD).read_text())
    assert record["mixed"]["objective"] == "teacher" and record["mixed"]["source"] == "scored"
