"""Threads of one process whose first call of all is one of the kernels'."""

import os
import subprocess
import sys
import threading

import pytest
import torch

from test_key_budget_gpu import BF16, DEV, pool, same

pytestmark = pytest.mark.gpu


def in_a_thread(call):
    """What ``call`` gives in a thread that has not called anything of CUDA yet."""
    got = []

    def run():
        try:
            got.append(call())
        except Exception as exc:
            got.append(exc)
    t = threading.Thread(target=run)
    t.start()
    t.join()
    return got[0]


@pytest.mark.parametrize("kind", ["decode weighed", "key weights", "decode", "product"])
def test_a_thread_may_begin_with_a_kernel_whose_tiles_come_by_tma(kind):
    """(Tensor maps are made by the driver, which wants a context of the calling thread.)  Everything has been called here before and all memory is given, so
    that the call does nothing else first."""
    from lily_b200.csrc import ops as o
    n, nq, nkv, d, page = 300, 8, 2, 128, 64
    kv, w, table = pool([n], nkv, page, d, BF16, 3)
    g = torch.Generator(device=DEV).manual_seed(1)
    q, x, a = (torch.randn(r, nq * d, device=DEV, generator=g).to(BF16) for r in (1, n, 256))
    seq, cu, pre = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([n], [0, n], [0]))
    start = w.clone()
    if kind == "decode weighed":
        out, room = torch.empty_like(q), torch.empty(o.decode_weighed_scratch_floats(1, nq, nkv, d, n, page, BF16), device=DEV)
        call = lambda: o.attention_decode_weighed(q, kv, w, table, seq, n, nq, nkv, d, page, 0.1, out=out, scratch=room)
    elif kind == "key weights":
        out, room = w, torch.empty(o.key_weights_scratch_floats([0], [n], nq, nkv, d, page, 0.1, BF16), device=DEV)
        call = lambda: o.attention_key_weights(x, kv, w, table, cu, pre, [0], [n], nq, nkv, d, page, 0.1, scratch=room)
    elif kind == "decode":
        plan = o.plan_decode_attention(BF16, 1, nq, nkv, d, n, fusable=False)
        out, room = torch.empty_like(q), torch.empty(max(1, plan.scratch_floats), device=DEV)
        call = lambda: o.attention_decode(q, kv, table, seq, out, room, plan.splits, nq, nkv, d, page, 0.1, stages=plan.stages)
    else:
        out = torch.empty(256, 256, dtype=BF16, device=DEV)
        call = lambda: out.copy_(o.gemm_tc(a, a[:, :nq * d]))
    call()
    want, given = out.clone(), w.clone()
    torch.cuda.synchronize()
    out.zero_()
    w.copy_(start)
    torch.cuda.synchronize()
    failed = in_a_thread(call)
    assert not isinstance(failed, Exception), failed
    torch.cuda.synchronize()
    assert same(out, want) and same(w, given)


FIRST_CALLS = """
import threading, torch
from lily_b200.csrc import ops
page, d, nq, nkv = {page}, {d}, 16, 4
ops.library(), ops._faces()
start, wrong, calls = threading.Barrier(12), [], []
for i in range(12):
    n = 256 << i % 4
    table = torch.arange(n // page, dtype=torch.int32, device="cuda")[None]
    calls.append((torch.randn(1, nq * d, device="cuda", dtype=torch.bfloat16), torch.randn(n // page, 2, nkv, page, d, device="cuda", dtype=torch.bfloat16),
                  torch.zeros(n // page, nkv, page, device="cuda"), table, torch.tensor([n], dtype=torch.int32, device="cuda"), n))
torch.cuda.synchronize()
def one(q, kv, w, table, lens, n):
    start.wait()
    try:
        ops.attention_decode_weighed(q, kv, w, table, lens, n, nq, nkv, d, page, d ** -0.5)
    except Exception as exc:
        wrong.append(str(exc))
threads = [threading.Thread(target=one, args=c) for c in calls]
[t.start() for t in threads], [t.join() for t in threads]
torch.cuda.synchronize()
sums = [float(c[2].sum()) for c in calls]
print(wrong or [s for s in sums if abs(s - nq) > 0.01] or "as asked")
"""


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_first_calls_of_several_threads_are_all_served(page, d):
    """Clusters of 2 to 16 blocks, whose launches raise the kernel's limit of shared memory, in a process that has launched none."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(page=page, d=d)], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    assert done.stdout.strip().endswith("as asked"), done.stdout[-2000:]
