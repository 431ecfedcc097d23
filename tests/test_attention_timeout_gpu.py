"""Bounded waits of the linear attention kernels, without a GPU fault.

With the host-side fault injection the producers leave loads out, so that waits cannot complete.  Every
role of every block must give up after the limit, wait for what it has in flight, free TMEM and
return; the call is reported by ``status()``, the context stays usable and the next call is right.
In a process of its own: the status word keeps the first code."""
import os
import subprocess
import sys

import pytest

from cutedsl_pingpong_gemm_b200 import CpgError, _lib, attention

CHILD = """
import sys, time
import torch
from cutedsl_pingpong_gemm_b200 import attention

def case(seed, lengths, h, dk, dv):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = sum(lengths)
    q, k, v, dy = (torch.randn(t, h, d, device="cuda", generator=g).bfloat16()
                   for d in (dk, dk, dv, dv))
    offsets = torch.tensor([0] + lengths, device="cuda").cumsum(0).int()
    return dy, q, k, v, -torch.rand(h, device="cuda", generator=g), offsets

def forward(final):
    return lambda dy, q, k, v, g, offsets: attention.linear_attention(q, k, v, g, offsets=offsets,
                                                                      final=final)

def backward(dy, q, k, v, g, offsets):
    state = torch.ones(len(offsets) - 1, len(g), q.shape[2], v.shape[2], device="cuda")
    return attention.linear_attention_backward(dy, q, k, v, g, offsets=offsets, state=state)

calls = [(forward(None), case(1, [300], 2, 64, 64)),             # two-part scores
         (forward(True), case(2, [300, 0, 513], 100, 128, 128)),  # exact states
         (forward(None), case(3, [300, 0, 513], 100, 64, 128)),
         (forward(True), case(4, [9001], 1, 128, 128)),           # segments
         (backward, case(5, [300, 140], 50, 128, 64))]
want = [f(*args) for f, args in calls]
torch.cuda.synchronize()
assert attention.status() == 0
for i, (f, args) in enumerate(calls):
    attention.set_timeout_ms(200)
    attention.set_fault_injection(int(sys.argv[1]))
    t0 = time.time()
    f(*args)
    torch.cuda.synchronize()
    took = time.time() - t0
    assert 0.19 < took < 10, (i, took)
    code = attention.status()
    assert code & ~0xff == 0x100 and 0x60 <= code & 0xff <= 0x66, hex(code)
    attention.set_fault_injection(0)
    attention.set_timeout_ms(10000)
    got = f(*args)
    for a, b in zip(got, want[i]):
        assert a is b is None or torch.equal(a, b), i
print("recovered", hex(code))
"""


@pytest.mark.gpu
@pytest.mark.parametrize("flags", [_lib.CPG_INJECT_SKIP_LOADS, _lib.CPG_INJECT_SKIP_VALUES])
def test_waits_that_run_out_are_reported_and_leave_the_gpu_usable(flags):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", CHILD, str(flags)], cwd=root, timeout=240,
                          env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True)
    assert done.returncode == 0 and "recovered" in done.stdout, done.stdout + done.stderr


def test_limits_and_flags_that_are_refused(lib):
    for ms in (0, -5):
        with pytest.raises(CpgError) as e:
            attention.set_timeout_ms(ms)
        assert e.value.code == _lib.CPG_ERR_INVALID_SHAPE
    for flags in (4, -1):
        with pytest.raises(CpgError) as e:
            attention.set_fault_injection(flags)
        assert e.value.code == _lib.CPG_ERR_INVALID_CONFIG
    attention.set_fault_injection(0)
    attention.set_timeout_ms(10000)
