"""Serving in four bits, what can be looked at without a GPU: how matrices are packed and quantised, arguments and sizes, what is refused."""

import subprocess
import sys

import pytest
import torch

import four_bits as fb
import godotar_models
import kernel_refs
from harness import make_runner
from lily_b200.cache.key_budget import KeyBudget
from lily_b200.cache.kv_cache import KVCacheManager, bytes_per_token
from lily_b200.config.server_args import ServerArgs
from lily_b200.csrc import ops
from lily_b200.parts.attention import Attention, AttentionSpec
from lily_b200.parts.base import BuildContext, CacheNeed
from lily_b200.parts.mlp import SwiGLU, SwiGLUSpec


def unpacked(w):
    """The matrix of a ``Weight4`` in 64 bits, code by code from its place."""
    f = torch.arange(w.k)
    within = f % 128
    at = 4 * (4 * (within % 32 // 8) + within // 32) + within % 8 // 2
    rows = torch.arange(w.n)
    codes = (w.codes[(rows // 128)[:, None], f // 128, (rows % 128)[:, None], at].int() >> (4 * (f % 2)).int()) & 15
    held = lambda t: t[(rows // 128)[:, None], f // w.group, (rows % 128)[:, None]].double()
    return held(w.scales) * (codes.double() - (8.0 if w.zeros is None else held(w.zeros)))


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (130, 160, 32), (128, 128, 128), (300, 448, 64)])
@pytest.mark.parametrize("zeros", [False, True])
def test_packed_matrices_hold_their_codes(n, k, group, zeros):
    g = torch.Generator().manual_seed(n)
    codes, scales, z = fb.make_matrix(n, k, group, zeros, g)
    w = ops.pack_weight4(codes.long(), scales, z)
    assert w.shape == (n, k) and w.bytes() == sum(t.numel() * t.element_size() for t in (w.codes, w.scales, w.zeros) if t is not None)
    assert torch.equal(unpacked(w), fb.matrix_values(codes, scales, z))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantised_matrices_are_near(group, zeros):
    """No number is further off than its code's half step, what rounding the scale to bfloat16 (2^-8) moves the outer codes by, and half a step of the largest ones that are kept at 15."""
    g = torch.Generator().manual_seed(group)
    w = torch.randn(40, 256, generator=g) * torch.rand(40, 1, generator=g)
    w[3] = 0.0
    q = ops.quantize_weight4(w, group, zeros)
    steps = q.scales.transpose(1, 2).reshape(128, -1)[:40].double().repeat_interleave(group, 1)
    off = (unpacked(q) - w.double()).abs()
    assert bool((off <= steps * (0.5 + 0.5 + 16 / 256)).all()) and bool((unpacked(q)[3] == 0).all())
    assert float((off / steps.clamp(min=1e-9)).mean()) < 0.3


@pytest.mark.parametrize("call", [
    lambda: ops.pack_weight4(torch.zeros(4, 96, dtype=torch.uint8), torch.ones(4, 2)),                     # groups of 48
    lambda: ops.pack_weight4(torch.zeros(4, 96, dtype=torch.uint8), torch.ones(3, 3)),                     # scales of other rows
    lambda: ops.pack_weight4(torch.full((4, 64), 16, dtype=torch.uint8), torch.ones(4, 1)),                # a code of five bits
    lambda: ops.pack_weight4(torch.zeros(4, 64), torch.ones(4, 1)),                                        # codes that are no whole numbers
    lambda: ops.pack_weight4(torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1), torch.full((4, 1), 99)),
    lambda: ops.pack_weight4(torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1), torch.zeros(4, 2, dtype=torch.uint8)),
    lambda: ops.quantize_weight4(torch.zeros(4, 96), 64),
    lambda: ops.quantize_weight4(torch.zeros(4, 96), 48),
    lambda: ops.cache4_shape(2, 16, 96),
    lambda: ops.cache4_shape(2, 16, 320),
    lambda: ops.weights4(ops.Weight4(None, None, None, 1, 32, 32), torch.float16),
    lambda: ops.cache4_values(None, None, 1, 64, 16, torch.float16),
    lambda: ops.linear4(torch.zeros(2, 32, dtype=torch.bfloat16), ops.Weight4(None, None, None, 1, 32, 32), out_dtype=torch.float16),
])
def test_what_does_not_fit_is_refused(call):
    with pytest.raises(ops.KernelError):
        call()


def test_tensors_off_the_device_are_refused():
    from lily_b200.csrc import build
    try:
        ops.library(), ops._faces()
    except build.BuildError as exc:
        pytest.skip(f"no kernel library here: {exc}")
    g = torch.Generator().manual_seed(0)
    w = ops.pack_weight4(*fb.make_matrix(8, 32, 32, False, g))
    kv, i32 = torch.zeros(2, *ops.cache4_shape(1, 16, 64), dtype=torch.uint8), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.linear4(torch.zeros(2, 32), w), lambda: ops.weights4(w), lambda: ops.cache4_values(kv, i32.view(1, 1), 1, 64, 16),
                 lambda: ops.attention_decode4(torch.zeros(1, 64), kv, i32.view(1, 1), i32, 0, 1, 1, 64, 16, 0.1),
                 lambda: ops.qk_norm_rope_write4(torch.zeros(1, 192), None, None, 1e-6, None, None, i32, i32, i32.view(1, 1), kv, 1, 1, 64, 0, 16),
                 lambda: ops.attention_prefill4(torch.zeros(1, 64), kv, i32.view(1, 1), torch.tensor([0, 1], dtype=torch.int32), i32, [0], [1], 1, 1, 64, 16, 0.1)):
        with pytest.raises(ops.KernelError, match="CUDA device"):
            call()


def entry(name, kinds, *args):
    """How a kernels' own entry answers arguments that it refuses ahead of any launch, in a process of its own."""
    code = f"""
import ctypes
from lily_b200.csrc import ops
lib = ops.library()
fn = lib.{name}
fn.restype = ctypes.c_int
of = dict(p=ctypes.c_void_p, i=ctypes.c_int, f=ctypes.c_float, d=ctypes.c_double)
fn.argtypes = [of[k] for k in {kinds!r}]
print(fn(*{args!r}), lib.lily_last_error().decode())
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    return done.stdout.strip()


DECODE = "pppp" "i" "pp" "iiiiiii" "f" "ip"          # q, kv, out, table, width, lengths, scratch, requests, longest, nq, nkv, d, page, pages, scale, dtype, stream
LINEAR = "pi" "pppp" "i" "p" "iiiii" "p"             # x, dtype, codes, scales, zeros, bias, bias_f32, out, out_f32, m, n, k, group, stream


WRITE = "pii" "pp" "id" "pp" "i" "p" "i" "pp" "ii" "p" "i" "p" "iiiii" "p"      # qkv, dtype, ld, gains, their dtype, eps, tables, rows, positions, tokens, token_req, table, requests, width, kv, pages, q_out, nq, nkv, d, rd, page, stream


@pytest.mark.parametrize("name,kinds,args,said", [
    ("lily_qk_norm_rope_write4", WRITE, (16, 1, 256, 0, 0, 0, 1e-6, 16, 16, 0, 16, 1, 16, 16, 1, 1, 16, 2, 16, 2, 1, 64, 64, 16, 0), "tables of 0 positions"),
    ("lily_qk_norm_rope_write4", WRITE, (16, 1, 256, 16, 0, 0, 1e-6, 16, 16, 8, 16, 1, 16, 16, 1, 1, 16, 2, 16, 2, 1, 64, 64, 16, 0), "gains come together"),
    ("lily_qk_norm_rope_write4", WRITE, (16, 1, 256, 0, 0, 0, 1e-6, 16, 16, 8, 16, 1, 16, 16, 1, 1, 24, 2, 16, 2, 1, 64, 64, 16, 0), "sixteen bytes"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1, 16, 16, 1, 16, 3, 2, 64, 16, 2, 0.1, 1, 0), "query heads over"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1, 16, 16, 1, 16, 2, 0, 64, 16, 2, 0.1, 1, 0), "query heads over"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1, 16, 16, 1, 16, 2, 2, 80, 16, 2, 0.1, 1, 0), "not 80"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1, 16, 16, 1, 17, 2, 2, 64, 16, 2, 0.1, 1, 0), "up to 17 places"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1, 16, 16, 1, 16, 2, 2, 64, 0, 2, 0.1, 1, 0), "pages of 0"),
    ("lily_attention_decode4", DECODE, (24, 16, 16, 16, 1, 16, 16, 1, 16, 2, 2, 64, 16, 2, 0.1, 1, 0), "sixteen bytes"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1, 16, 24, 1, 16, 2, 2, 64, 16, 2, 0.1, 1, 0), "scratch"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1, 16, 0, 1, 16, 2, 2, 64, 16, 2, 0.1, 1, 0), "scratch"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1, 16, 16, 1, 16, 2, 2, 64, 16, 2, 0.0, 1, 0), "a scale of 0"),
    ("lily_attention_decode4", DECODE, (16, 16, 16, 16, 1 << 24, 16, 16, 65535, 1 << 27, 64, 64, 64, 16, 2, 0.1, 1, 0), "too many for one call"),
    ("lily_linear4", LINEAR, (16, 1, 16, 16, 0, 0, 0, 16, 0, 4, 8, 96, 64, 0), "in groups of 64"),
    ("lily_linear4", LINEAR, (16, 1, 16, 16, 0, 0, 0, 16, 0, 4, 8, 96, 48, 0), "in groups of 48"),
    ("lily_linear4", LINEAR, (16, 1, 16, 16, 0, 0, 0, 16, 0, 17, 8, 64, 64, 0), "17 tokens"),
    ("lily_linear4", LINEAR, (8, 1, 16, 16, 0, 0, 0, 16, 0, 4, 8, 64, 64, 0), "sixteen bytes"),
    ("lily_linear4", LINEAR, (16, 0, 16, 16, 0, 0, 0, 16, 0, 4, 8, 64, 64, 0), "keep float32"),
    ("lily_linear4_many", "p" + LINEAR[2:], (16, 16, 24, 0, 0, 0, 16, 0, 40, 8, 64, 64, 0), "sixteen bytes"),
    ("lily_linear4_many", "p" + LINEAR[2:], (16, 16, 16, 0, 0, 0, 16, 0, 40, 8, 64, 48, 0), "in groups of 48"),
    ("lily_weights4", "pppp" "iiiip", (16, 16, 0, 16, 1, 8, 32, 64, 0), "in groups of 64"),
])
def test_the_kernels_own_entries_refuse(name, kinds, args, said):
    from lily_b200.csrc import build
    try:
        ops.library()
    except build.BuildError as exc:
        pytest.skip(f"no kernel library here: {exc}")
    answer = entry(name, kinds, *args)
    assert not answer.startswith("0 ") and said in answer, answer


# ---- arguments, cache, parts ----

def test_server_arguments():
    args = ServerArgs.parse(["--quantization", "int4", "--quantization-group", "64", "--kv-cache-dtype", "int4"])
    assert (args.quantization, args.quantization_group, args.kv_cache_dtype) == ("int4", 64, "int4")
    assert ServerArgs().quantization is None and ServerArgs().kv_cache_dtype == "auto"
    for bad in (dict(quantization="int3"), dict(quantization_group=48), dict(kv_cache_dtype="fp8")):
        with pytest.raises(ValueError):
            ServerArgs(**bad)


def test_cache_in_four_bits():
    """A group's pages, what a token takes (0.28 of bfloat16's), what four bits do not hold."""
    need = CacheNeed(2, 128, four_bits=True)
    cache = KVCacheManager([(need, 3), (CacheNeed(2, 128), 1)], [], page_size=16, num_pages=4, max_requests=2, max_context=64, device=torch.device("cpu"))
    assert cache.groups[0].data.dtype == torch.uint8 and tuple(cache.groups[0].data.shape) == (3, 5, *ops.cache4_shape(2, 16, 128))
    assert cache.groups[1].data.dtype == torch.bfloat16
    assert bytes_per_token([(need, 3)], torch.bfloat16) == 3 * 2 * 2 * (64 + 8) and bytes_per_token([(CacheNeed(2, 128), 3)], torch.bfloat16) == 3 * 2 * 2 * 256
    for bad in (CacheNeed(2, 96, four_bits=True), CacheNeed(2, 128, window=64, four_bits=True), CacheNeed(2, 128, v_head_dim=64, four_bits=True),
                CacheNeed(1, 128, values_in_keys=True, four_bits=True)):
        with pytest.raises(ValueError):
            bytes_per_token([(bad, 1)], torch.bfloat16)


def test_what_goes_with_a_cache_in_four_bits():
    """Layers that begin on boundaries of sixteen bytes; no budget of places, whose keys are moved as numbers."""
    make = lambda need, layers, page, pages: KVCacheManager([(need, layers)], [], page_size=page, num_pages=pages, max_requests=2, max_context=8, device=torch.device("cpu"))
    need = CacheNeed(1, 64, four_bits=True)
    make(need, 1, 1, 4), make(need, 3, 1, 5), make(need, 3, 2, 4)
    with pytest.raises(ValueError, match="sixteen"):
        make(need, 3, 1, 4)
    with pytest.raises(ValueError, match="four bits"):
        KeyBudget(make(need, 1, 2, 4), keep=4, first=1, recent=1, slack=1, ops=kernel_refs)


def test_architectures_that_cache_something_else_are_refused(tmp_path):
    path = godotar_models.write_model_dir(str(tmp_path / "m"), godotar_models.WIDE, godotar_models.make_weights(godotar_models.WIDE, 3))
    with pytest.raises(ValueError, match="four bits"):
        make_runner(path, kv_cache_dtype="int4")


@pytest.mark.parametrize("more", [dict(window=32), dict(softcap=30.0), dict(v_head_dim=128), dict(head_dim=32), dict(sink=True), dict(talk=True), dict(v_norm=True), dict(conv_taps=2),
                                  dict(own_kv=False), dict(head_gate=True), dict(head_dim=320)])
def test_attention_that_four_bits_do_not_serve_is_refused(more):
    spec = AttentionSpec(**{**dict(hidden_size=64, num_heads=2, num_kv_heads=1, head_dim=64), **more})
    with pytest.raises(ValueError):
        Attention(spec, "a", BuildContext(torch.device("cpu"), torch.float32, kernel_refs, cache4=True))
    Attention(spec, "a", BuildContext(torch.device("cpu"), torch.float32, kernel_refs))


def test_widths_that_do_not_come_in_groups_are_refused():
    ctx = BuildContext(torch.device("cpu"), torch.float32, kernel_refs, weight_group=128)
    with pytest.raises(ValueError, match="groups of 128"):
        Attention(AttentionSpec(192, 2, 1, 64), "a", ctx)
    with pytest.raises(ValueError, match="groups of 128"):
        SwiGLU(SwiGLUSpec(128, 192), "m", ctx)
