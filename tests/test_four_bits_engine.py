"""The engine around matrices and caches in four bits, what can be looked at without a GPU."""

import pytest

import kernel_refs
import nafazen_models
import tiny_models
from harness import make_runner, model_dir
from lily_b200.engine.scheduler import Scheduler
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
