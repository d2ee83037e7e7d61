"""What the operators of a budgeted cache refuse on the host, looked at without a GPU: each call in a process of its own where a mistake would
end it."""

import subprocess
import sys

import pytest
import torch


def kernels():
    """The package's operators with their library, where one can be built."""
    from lily_b200.csrc import build, ops
    try:
        ops.library(), ops._faces()
    except build.BuildError as exc:
        pytest.skip(f"no kernel library here: {exc}")
    return ops


def outcome(lines):
    """How a process that runs these lines ends: what it printed, or the signal that ended it."""
    done = subprocess.run([sys.executable, "-c", lines], capture_output=True, text=True, timeout=300)
    assert done.returncode >= 0, f"ended by signal {-done.returncode}"
    assert done.returncode == 0, done.stderr[-2000:]
    return done.stdout.strip()


@pytest.mark.parametrize("nq,nkv", [(0, 4), (0, 1), (3, 4), (-4, 4), (4, 0), (4, -4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_heads_that_do_not_fit_have_no_plan(nq, nkv, dtype):
    kernels()
    assert outcome(f"""
import torch
from lily_b200.csrc import ops
try:
    ops.key_weights_scratch_floats([0], [10], {nq}, {nkv}, 128, 16, 0.1, {dtype})
except ops.KernelError as exc:
    print("refused" if "query heads over" in str(exc) else exc)
""") == "refused"


@pytest.mark.parametrize("nq,nkv", [(0, 4), (3, 4), (4, 0), (129, 1)])
def test_the_kernels_own_entries_size_nothing_for_heads_that_do_not_fit(nq, nkv):
    kernels()
    assert outcome(f"""
import ctypes
from lily_b200.csrc import ops
one = (ctypes.c_int * 1)(10)
lib = ops.library()
for name, more in (("lily_key_weights_tc_floats", ()), ("lily_key_weights_floats", (1 << 28,))):
    size = getattr(lib, name)
    size.restype = ctypes.c_size_t
    print(size(1, one, one, 0, {nq}, {nkv}, *more) > 0, end=" ")
""") == ("False True" if (nq, nkv) == (129, 1) else "False False")


def answer(name, *args):
    """What a kernels' own entry says to arguments that it refuses ahead of any launch (addresses that nothing is read from)."""
    lib = kernels().library()
    assert getattr(lib, name)(*args) != 0
    return lib.lily_last_error().decode()


@pytest.mark.parametrize("off", [4, 8, 12])
def test_scratch_that_is_not_aligned_is_refused(off):
    import ctypes
    none, ten = (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(10)
    at = lambda x: ctypes.c_void_p(4096 + x)
    said = answer("lily_key_weights", at(0), at(0), at(0), at(0), 1, at(off), 1, none, ten, 0, 4, 2, 48, 16, ctypes.c_float(0.1), 0, 1 << 28, None)
    assert "16-byte aligned" in said
    said = answer("lily_key_weights_tc", at(0), 10, at(0), 1, at(0), at(0), 1, at(off), 1, none, ten, 0, 4, 2, 64, 16, ctypes.c_float(0.1), None)
    assert "16-byte aligned" in said
    said = answer("lily_attention_decode_weighed", at(0), at(0), at(0), at(0), at(0), 1, at(0), at(off), 1, 16, 4, 2, 48, 16, 1, ctypes.c_float(0.1), 0, 1, None)
    assert "16-byte aligned" in said


@pytest.mark.parametrize("page", [0, -16])
def test_pages_without_places_are_refused(page):
    """(The kernel divides by the size of a page.)"""
    import ctypes
    at, f = ctypes.c_void_p(4096), ctypes.c_float
    said = answer("lily_axes_rope_write", at, 1, 1, ctypes.c_size_t(0), 1024, None, None, 0, f(1e-6), at, at, 9, at, at, 1, 3, at, at, at, 1, 1, at, 0, at, 1, 4, 2, 128, 128, page, None)
    assert "pages of" in said
    said = answer("lily_attention_decode_weighed", at, at, at, at, at, 1, at, at, 1, 16, 4, 2, 64, page, 1, f(0.1), 1, 1, None)
    assert "pages of" in said
    said = answer("lily_key_weights", at, at, at, at, 1, at, 1, (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(10), 0, 4, 2, 48, page, f(0.1), 0, 1 << 28, None)
    assert "pages of" in said
    said = answer("lily_select_keys", at, at, 1, at, at, 1, 2, 1, 2, page, 0, 4, 1, 1, None)
    assert "page_size" in said
    said = answer("lily_move_keys", at, at, at, 1, at, 1, at, 1, 2, 1, 2, page, 256, 4, 1, None)
    assert "page_size" in said


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cached,new", [([2 ** 31 - 5], [100]), ([0], [2 ** 31 - 1]), ([2 ** 31 - 1], [2 ** 31 - 1]), ([0] * 3, [2 ** 30] * 3)])
def test_places_and_tokens_that_pass_32_bits_have_no_plan(cached, new, dtype):
    ops = kernels()
    with pytest.raises(ops.KernelError, match="32-bit"):
        ops.key_weights_scratch_floats(cached, new, 4, 4, 128, 16, 0.1, dtype)


def test_portions_of_more_tiles_than_can_be_numbered_have_no_plan():
    """A million tokens of 128 heads over one kv head: a tile of rows a token, each of up to 4,096 pieces of keys."""
    ops = kernels()
    floats = lambda n: ops.key_weights_scratch_floats([0], [n], 128, 1, 64, 64, 0.1, torch.bfloat16)
    assert floats(1 << 18) > 0
    for n in (1 << 20, 3 << 20):
        with pytest.raises(ops.KernelError, match="too many tiles"):
            floats(n)
