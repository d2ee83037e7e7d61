"""The engine around matrices and caches in four bits, what can be looked at without a GPU."""

import logging

import pytest
import torch

import kernel_refs
import nafazen_models
import tiny_models
from harness import make_runner, model_dir
from lily_b200.engine.scheduler import Scheduler
from lily_b200.models.assembled import AssembledModel
from lily_b200.parts.attention import AttentionSpec
from lily_b200.parts.base import BlockSpec, BuildContext, ModelSpec, ScheduleEntry
from lily_b200.parts.mlp import SwiGLUSpec
from lily_b200.parts.norm import RMSNormSpec
from lily_b200.sampling.params import SamplingParams


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    cfg = tiny_models.TINY_QWEN3
    return cfg, model_dir(cfg, 3, str(tmp_path_factory.mktemp("m")))[0]


def test_a_step_whose_4_bit_product_gave_up_a_wait_fails(model, monkeypatch):
    """What the tcgen05 product reports of a wait that ran out reaches the caller as an error, ahead of the step's tokens."""
    cfg, path = model
    runner = make_runner(path)
    s = Scheduler(runner, random_seed=7)
    reports = iter([0, 0, 3 << 24 | 5])
    monkeypatch.setattr(kernel_refs, "linear4_lost", lambda: next(reports), raising=False)
    s.add_request("r0", tiny_models.random_tokens(7, cfg["vocab_size"], 1), SamplingParams(max_new_tokens=8, ignore_eos=True))
    with pytest.raises(RuntimeError, match="code 3, block 5"):
        s.run_to_completion()
    assert next(reports, None) is None


def test_every_runner_hears_of_a_4_bit_product_that_gave_up(model, monkeypatch):
    """Each runner of the process raises once, whatever else it hears of at the same time, and one made afterwards does not."""
    path = model[1]
    runners = [make_runner(path) for _ in range(3)]
    reports, rows = iter([0, 1 << 24]), iter([0, 4])
    monkeypatch.setattr(kernel_refs, "linear4_lost", lambda: next(reports, 0), raising=False)
    monkeypatch.setattr(kernel_refs, "attention_decode_lost", lambda: next(rows, 0), raising=False)
    runners[0].check_waits()
    for r in (runners[1], runners[0], runners[2]):
        with pytest.raises(RuntimeError, match="4-bit weights"):
            r.check_waits()
        r.check_waits()
    make_runner(path).check_waits()


@pytest.mark.parametrize("cfg", [nafazen_models.SHARP, dict(nafazen_models.WIDE, layers=[dict(layer, mlp=nafazen_models.moe(ff=64, experts=8, top=4, shared=None)) for layer in nafazen_models.WIDE["layers"]])])
def test_architectures_without_such_matrices_are_refused(cfg, tmp_path):
    """Four bits hold the matrices of attention and gated feed-forwards: a model that has neither would be served in its dtype without a word."""
    path = nafazen_models.write_model_dir(str(tmp_path / "m"), cfg, nafazen_models.make_weights(cfg, 3))
    make_runner(path)
    with pytest.raises(ValueError, match="quantization = int4: .* held in four bits"):
        make_runner(path, quantization="int4", quantization_group=32)


def test_the_load_report_is_what_the_device_holds(tmp_path, monkeypatch, caplog):
    """Bytes of a quantised model are those it is held in, not those of the checkpoint, and the log says how many of them are in four bits."""
    from lily_b200.csrc import ops
    monkeypatch.setattr(kernel_refs, "quantize_weight4", ops.quantize_weight4, raising=False)
    cfg = dict(tiny_models.TINY_QWEN3, hidden_size=128, head_dim=64, intermediate_size=256)
    path, weights = model_dir(cfg, 3, str(tmp_path))
    full = make_runner(path)
    caplog.set_level(logging.INFO)
    four = make_runner(path, quantization="int4", quantization_group=64)
    names = [n for n in weights if any(f"{x}_proj.weight" in n for x in ("q", "k", "v", "o", "gate", "up", "down"))]
    numbers = sum(weights[n].numel() for n in names)
    held = four.model.weight_bytes(four_bits=True)
    # codes in whole tiles of 128 rows and columns, a bfloat16 scale a group: these matrices' sizes are whole tiles once q, k and v, and gate and up, are stacked
    assert held == numbers // 2 + numbers // 64 * 2
    assert full.weight_bytes == sum(w.numel() * 4 for w in weights.values()) and four.weight_bytes == full.weight_bytes - numbers * 4 + held
    said = [r.getMessage() for r in caplog.records if "four bits" in r.getMessage()]
    assert len(said) == 1 and f"{held / 1e9:.2f} GB" in said[0]


def test_runs_that_read_another_runs_4_bit_cache_are_refused():
    """When the model is put together, and not by its first step."""
    block = BlockSpec(prefix="l", mixer=AttentionSpec(64, 2, 1, 64), feed_forward=SwiGLUSpec(64, 128), norm_in=RMSNormSpec(64, 1e-6), norm_post=RMSNormSpec(64, 1e-6))
    build = lambda schedule, cache4: AssembledModel(ModelSpec(architecture="toy", vocab_size=32, hidden_size=64, blocks=[block], schedule=schedule, final_norm=RMSNormSpec(64, 1e-6), head_name=None,
                                                              max_position=64, eos_token_ids=[]), BuildContext(torch.device("cpu"), torch.float32, kernel_refs, cache4=cache4))
    lent = [ScheduleEntry(0), ScheduleEntry(0, reads=0)]
    build(lent, False), build([ScheduleEntry(0), ScheduleEntry(0)], True)
    with pytest.raises(ValueError, match="read by the run that writes it"):
        build(lent, True)
