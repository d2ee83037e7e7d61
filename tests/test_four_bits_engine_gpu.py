"""The engine with its matrices, its cache, or both in four bits: every step against the plain implementation with the same numbers in place of the matrices, and keys and values as the cache
holds them; captured steps; generation."""

import pytest
import torch

import four_bits as fb
import plain_impl
import tiny_models
from harness import make_runner, model_dir, run_mixed, run_portions, run_whole

pytestmark = pytest.mark.gpu

QWEN = {**tiny_models.TINY_QWEN3, "hidden_size": 128, "head_dim": 64, "intermediate_size": 256}
LLAMA = {**tiny_models.TINY_LLAMA, "hidden_size": 256, "head_dim": 128, "num_attention_heads": 4, "num_key_value_heads": 1, "intermediate_size": 384}


def held(weights, group):
    """The checkpoint with the matrices that the engine holds in four bits replaced by the numbers they stand for."""
    from lily_b200.csrc import ops
    out = dict(weights)
    for name, w in weights.items():
        if any(part in name for part in ("q_proj.weight", "k_proj.weight", "v_proj.weight", "o_proj.weight", "gate_proj.weight", "up_proj.weight", "down_proj.weight")):
            out[name] = ops.weights4(ops.quantize_weight4(w.to("cuda"), group)).cpu()
    return out


def quantised_heads(monkeypatch):
    """Keys and values of the plain implementation as the cache holds them."""
    plain = plain_impl.causal_attention

    def values(x):
        codes, pairs = fb.hold(x)
        step, low = (pairs[..., i].float().repeat_interleave(64, -1) for i in range(2))
        return low + step * codes.float()
    monkeypatch.setattr(plain_impl, "causal_attention", lambda q, k, v, scale, window=None: plain(q, values(k), values(v), scale, window))


def near(got, want, cache4):
    """float32 sums in other orders (1e-4 of the largest logit); over a 4-bit cache a number next to the border of two codes may have the other one, a whole step off: few do (an error of 10^-6 of a
    step's place in 2 10^4 numbers), so nearly all rows are as near as without, and the others within what single codes move (a step is a tenth of a head's spread, one of 64 features of one place)."""
    scale = float(want.abs().max())
    off = (got - want).abs().amax(-1) / scale
    if not cache4:
        assert float(off.max()) < 1e-4, float(off.max())
    else:
        assert float(off.max()) < 2e-2 and float((off < 1e-3).float().mean()) > 0.7, off


@pytest.mark.parametrize("cfg", [QWEN, LLAMA])
@pytest.mark.parametrize("quantization,kv,group", [("int4", "auto", 128), ("int4", "auto", 32), (None, "int4", 128), ("int4", "int4", 64)])
def test_steps_against_the_plain_implementation(cfg, quantization, kv, group, tmp_path, monkeypatch):
    path, weights = model_dir(cfg, 3, str(tmp_path))
    if quantization:
        weights = held(weights, group)
    ids = tiny_models.random_tokens(45, cfg["vocab_size"], 1)
    other = tiny_models.random_tokens(20, cfg["vocab_size"], 2)
    if kv == "int4":
        quantised_heads(monkeypatch)
    want, want_other = plain_impl.all_logits(cfg, weights, ids), plain_impl.all_logits(cfg, weights, other)
    runner = make_runner(path, device="cuda", quantization=quantization, kv_cache_dtype=kv, quantization_group=group)
    near(run_whole(runner, ids), want, kv == "int4")
    near(run_portions(runner, ids, [17, 1, 1, 9]), want, kv == "int4")                                      # portions, then single tokens in captured steps
    got = run_mixed(runner, {"a": ids, "b": other}, [{"a": 30}, {"a": 1, "b": 12}, {"a": 1, "b": 1}, {"b": 7, "a": 1}, {"a": 12}])
    near(got["a"], want, kv == "int4")
    near(got["b"], want_other, kv == "int4")


@pytest.mark.parametrize("quantization,kv", [("int4", "auto"), (None, "int4"), ("int4", "int4")])
def test_bfloat16_against_the_plain_implementation_and_generation(quantization, kv, tmp_path, monkeypatch):
    """Logits within what bfloat16 activations move them by (2e-2 of the largest one, as without four bits; 5e-2 over a cache, where a key rounded by 2^-9 is at another code's side in some 2^-9 / (1 / 10)
    of all places), tokens that repeat.  The matrices that are quantised are the checkpoint's as bfloat16 holds them."""
    from lily_b200 import Engine, EngineConfig, SamplingParams
    path, weights = model_dir(QWEN, 4, str(tmp_path))
    weights = {k: v.to(torch.bfloat16).float() for k, v in weights.items()}
    if quantization:
        weights = held({k: v.to(torch.bfloat16) for k, v in weights.items()}, 128)
        weights = {k: v.float() for k, v in weights.items()}
    if kv == "int4":
        quantised_heads(monkeypatch)
    prompts = [tiny_models.random_tokens(n, QWEN["vocab_size"], n) for n in (5, 33, 150)]
    eng = Engine(EngineConfig(path, dtype="bfloat16", device="cuda:0", max_total_tokens=2048, server_args=dict(quantization=quantization, kv_cache_dtype=kv, page_size=16)))
    want, got = plain_impl.all_logits(QWEN, weights, prompts[2]), eng.all_prefill_logits(prompts[2]).float().cpu()
    assert float((got - want).abs().max()) < (5e-2 if kv == "int4" else 2e-2) * float(want.abs().max())
    params = SamplingParams(max_new_tokens=12, ignore_eos=True)
    first = [g["output_ids"] for g in eng.generate(prompts, params)]
    assert [g["output_ids"] for g in eng.generate(prompts, params)] == first and all(len(t) == 12 for t in first)


def test_memory(tmp_path):
    """Matrices at five bits a number and less, pages at 0.29 of bfloat16's bytes."""
    path, _ = model_dir(QWEN, 5, str(tmp_path), dtype=torch.bfloat16)
    full = make_runner(path, "bfloat16", "cuda")
    four = make_runner(path, "bfloat16", "cuda", quantization="int4", kv_cache_dtype="int4")
    matrices = 2 * 2 * (128 * (4 + 2 * 2) * 64 + 256 * 128 + 3 * 128 * 256)                 # bytes of two layers in bfloat16
    assert full.model.weight_bytes() - four.model.weight_bytes() > matrices * (1 - 5 / 16)
    bytes_of = lambda r: r.cache.groups[0].data.numel() * r.cache.groups[0].data.element_size()
    assert bytes_of(four) == bytes_of(full) * (32 + 4) / 128
