"""The device-memory prediction against the peak a run actually allocates
(``torch.cuda.max_memory_allocated``: every device buffer of the run, the
library's workspaces included, is a torch allocation)."""

from __future__ import annotations

import json
import sys

import pytest
import torch

from mround_amd import api
from mround_amd.pipeline.checkpoint import write_random_checkpoint
from mround_amd.schemes import Symmetry, TuningConfig

pytestmark = pytest.mark.gpu

SMALL = dict(model_type="qwen2", hidden_size=512, num_attention_heads=8, num_key_value_heads=2,
             intermediate_size=1536, rms_norm_eps=1e-6, rope_theta=1e6, num_hidden_layers=3,
             vocab_size=4096, tie_word_embeddings=True)


# (mixed, quantized_inputs, holdout_batches, seq_len): the block loop holds
# three calibration streams with quantized inputs and the fused advance, two
# without quantized inputs (inputs, targets) or with held-out batches; 200
# tokens run on sequences padded to 256 rows.
CASES = [(False, True, 0, 256), (True, True, 0, 256), (False, False, 0, 256), (False, True, 1, 256),
         (False, True, 0, 200)]


@pytest.mark.parametrize("mixed,quantized_inputs,holdout,seq_len", CASES)
def test_prediction_bounds_the_measured_peak(tmp_path, mixed, quantized_inputs, holdout, seq_len):
    print("case memory", mixed, quantized_inputs, holdout, seq_len, flush=True, file=sys.stderr)
    src = write_random_checkpoint(tmp_path / "m", SMALL, seed=1)
    tuning = TuningConfig(iters=2, batch_size=4, n_samples=8, seq_len=seq_len)
    kw = dict(average_bits=3.0, candidate_bits=(2, 4), scoring_samples=8, scoring_seq_len=257) if mixed else {}
    res = api.quantize(src, output_dir=tmp_path / "q", bits=4, symmetry=Symmetry.ASYMMETRIC, tuning=tuning,
                       seed=2, quantized_inputs=quantized_inputs, holdout_batches=holdout, **kw)
    rec = json.loads(res.config_path.read_text())["memory"]
    predicted = rec["peak"]
    measured = rec["peak_allocated"]
    print(f"  predicted {predicted} measured {measured} ({measured / predicted:.3f}) in {rec['peak_stage']}",
          file=sys.stderr)
    assert rec["peak_stage"] == ("scoring" if mixed else "blocks")
    assert 0.85 * predicted <= measured <= 1.05 * predicted


def test_prediction_bounds_a_pass_by_the_teacher(tmp_path):
    """The lists of 65 scoring batches, the last one not full, beside the small model's engine."""
    print("case memory teacher", flush=True, file=sys.stderr)
    src = write_random_checkpoint(tmp_path / "m", SMALL, seed=1)
    res = api.quantize(src, output_dir=tmp_path / "q", bits=4, symmetry=Symmetry.ASYMMETRIC, seed=2, average_bits=3.0,
                       candidate_bits=(2, 4), tuning=TuningConfig(iters=2, batch_size=4, n_samples=8, seq_len=256),
                       scoring_samples=129, scoring_seq_len=1025, scoring_batch_size=2, sensitivity_objective="teacher")
    rec = json.loads(res.config_path.read_text())
    memory, predicted = rec["memory"], rec["memory"]["peak"]
    print(f"  predicted {predicted} measured {memory['peak_allocated']}", file=sys.stderr)
    assert rec["mixed"]["objective"] == "teacher" and memory["peak_stage"] == "scoring"
    assert 0.85 * predicted <= memory["peak_allocated"] <= 1.05 * predicted


def test_the_measured_peak_is_the_runs_own(tmp_path):
    """Tensors that the process has dropped in reference cycles, which a collection during the run would free, are not
    held by it."""
    print("case memory cycles", flush=True, file=sys.stderr)
    src = write_random_checkpoint(tmp_path / "m", SMALL, seed=1)

    class Cycle:
        pass

    def peak():
        res = api.quantize(src, output_dir=tmp_path / "q", bits=4, symmetry=Symmetry.ASYMMETRIC, seed=2,
                           tuning=TuningConfig(iters=2, batch_size=4, n_samples=8, seq_len=256))
        return json.loads(res.config_path.read_text())["memory"]["peak_allocated"]

    peak()  # (what a first run leaves with the process)
    want = peak()
    for _ in range(3):
        c = Cycle()
        c.itself, c.tensor = c, torch.empty(10 << 20, dtype=torch.uint8, device="cuda")
    del c
    assert peak() == want
