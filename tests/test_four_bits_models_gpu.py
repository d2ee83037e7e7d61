"""Every architecture that has attention or gated feed-forwards whose matrices four bits hold, served with them: the same logits as with the numbers that the codes stand for in plain matrices.
Whole prompts, portions, single tokens in captured steps, requests of different kinds in one step."""

import importlib

import pytest
import torch

import tiny_models
from harness import make_runner, run_mixed, run_portions, run_whole

pytestmark = pytest.mark.gpu

MODELS = [("godotar", "SHARP"), ("godotar", "WIDE"), ("gotivik", "SHARP"), ("gotivik", "WIDE"), ("kinanex", "SHARP"), ("kinanex", "WIDE"), ("kinanex", "RECURRENT"), ("nafazen", "WIDE"),
          ("tugodra", "WIDE"), ("zirurax", "SHARP"), ("zirurax", "WIDE")]


# (the SHARP ones' near one-hot attention turns a rounding of a score into another key, as the models' own tests say: their bfloat16 logits are up to half the largest from float32's, with plain matrices too)
@pytest.mark.parametrize("name,cfg,dtype", [(n, c, t) for n, c in MODELS for t in ("float32", "bfloat16") if t == "float32" or c != "SHARP"])
def test_the_same_logits_as_with_the_numbers(name, cfg, dtype, tmp_path, monkeypatch):
    """float32: sums in other orders, 1e-4 of the largest logit as in test_steps_against_the_plain_implementation; bfloat16: activations
    move logits by up to 2e-2 from those of float32, there, and these are two runs in bfloat16 (the plain one's numbers are rounded to it besides), each as far from float32's: 4e-2 from one another at most."""
    from lily_b200.csrc import ops
    models = importlib.import_module(f"{name}_models")
    cfg = getattr(models, cfg)
    path = models.write_model_dir(str(tmp_path / "m"), cfg, models.make_weights(cfg, 3))
    ids, other = tiny_models.random_tokens(45, cfg["vocab"], 1), tiny_models.random_tokens(20, cfg["vocab"], 2)

    def logits():
        runner = make_runner(path, dtype, "cuda", quantization="int4", quantization_group=32)
        mixed = run_mixed(runner, {"a": ids, "b": other}, [{"a": 30}, {"a": 1, "b": 12}, {"a": 1, "b": 1}, {"b": 7, "a": 1}, {"a": 12}])
        return [run_whole(runner, ids), run_portions(runner, ids, [17, 1, 1, 9]), mixed["a"], mixed["b"]], runner.model.weight_bytes(four_bits=True)
    four, held = logits()
    quantise = ops.quantize_weight4
    monkeypatch.setattr(ops, "quantize_weight4", lambda w, group: ops.weights4(quantise(w, group), torch.float32).to(w.dtype))
    plain, full = logits()
    assert held > 0 and full == 0                     # (bytes in four bits; a matrix of 32 columns takes a tile of 128, so that a small model may grow)
    for a, b in zip(four, plain):
        assert bool(torch.isfinite(a).all())
        off = float((a - b).abs().max()) / float(b.abs().max())
        assert off < (1e-4 if dtype == "float32" else 4e-2), off
