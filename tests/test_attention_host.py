"""Norm with rotation and linear attention without a GPU: the oracle against the recurrence and
differences, and every bad argument of the C entry points refused before anything is launched."""
import ctypes

import pytest
import torch

from cutedsl_pingpong_gemm_b200 import _lib, attention
from oracle import attention_ref as ref

F32, BF16, I8 = _lib.CPG_DTYPE_F32, _lib.CPG_DTYPE_BF16, _lib.CPG_DTYPE_I8
ADDRESS = 4096  # never dereferenced: every call below fails or has nothing to do
S, N, A, D, C, U = (_lib.CPG_ERR_INVALID_SHAPE, _lib.CPG_ERR_NULL, _lib.CPG_ERR_ALIGNMENT,
                    _lib.CPG_ERR_DTYPE, _lib.CPG_ERR_INVALID_CONFIG, _lib.CPG_ERR_UNSUPPORTED)
BIG = 2 ** 31


# --------------------------------------------------------------------------------- the oracle
@pytest.mark.parametrize("n", [0, 1, 5, 128, 300])
@pytest.mark.parametrize("start", [False, True])
def test_oracle_pass_is_the_recurrence(n, start):
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, d, generator=g, dtype=torch.float64) for d in (6, 6, 4))
    s = torch.randn(6, 4, generator=g, dtype=torch.float64) if start else None
    for decay in (0.0, -0.01, -3.0, -float("inf")):
        if decay == -float("inf"):  # e^g = 0: only the token itself
            o = 0.5 * (q * k).sum(1, keepdim=True) * v
            final = torch.outer(k[-1], v[-1]) if n else (s if start else torch.zeros(6, 4))
        else:
            o, final = ref.tokens_pass(q, k, v, decay, 0.5, s)
        got = ref.sequence_pass(q, k, v, decay, 0.5, s)
        assert torch.allclose(got[0], o, rtol=1e-11, atol=1e-11)
        assert torch.allclose(got[3], final.double(), rtol=1e-11, atol=1e-11)


def test_oracle_gradients_are_the_recurrences():
    """The gradient's three passes against automatic differentiation of the recurrence, with shared
    heads, a starting state and a gradient of the final one; and that against differences."""
    g = torch.Generator().manual_seed(3)
    n, dk, dv, scale = 150, 4, 6, 0.7
    q = torch.randn(n, 1, dk, generator=g, dtype=torch.float64, requires_grad=True)
    k = torch.randn(n, 2, dk, generator=g, dtype=torch.float64, requires_grad=True)
    v = torch.randn(n, 2, dv, generator=g, dtype=torch.float64, requires_grad=True)
    s = torch.randn(1, 2, dk, dv, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(n, 2, dv, generator=g, dtype=torch.float64)
    df = torch.randn(1, 2, dk, dv, generator=g, dtype=torch.float64)
    decay = torch.tensor([-0.02, -0.6])

    def loss(q, k, v, s):
        total = 0.0
        for h in range(2):
            o, f = ref.tokens_pass(q[:, 0], k[:, h], v[:, h], float(decay[h].double()), scale,
                                   s[0, h])
            total = total + (o * dy[:, h]).sum() + (f * df[0, h]).sum()
        return total
    want = torch.autograd.grad(loss(q, k, v, s), (q, k, v, s))
    with torch.no_grad():
        grads, (ds, _) = ref.linear_attention_backward(dy, q, k, v, decay, scale, None, s, df)
        for got, w in zip([x[0] for x in grads] + [ds], want):
            assert torch.allclose(got, w, rtol=1e-10, atol=1e-10)
        step = 1e-5
        for x, w in zip((q, k, v, s), want):
            move = torch.randn(x.shape, generator=g, dtype=torch.float64)
            args = [y + step * move if y is x else y for y in (q, k, v, s)]
            back = [y - step * move if y is x else y for y in (q, k, v, s)]
            slope = (loss(*args) - loss(*back)) / (2 * step)
            assert abs(slope - (w * move).sum()) <= 1e-6 * (1 + abs(slope))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(8, 8), (10, 4), (6, 0)])
def test_oracle_norm_rope_gradient(interleaved, d, rot):
    g = torch.Generator().manual_seed(d + rot)
    x = torch.randn(5, 3, d, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(d, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(5, 3, d, generator=g, dtype=torch.float64)
    table = attention.rope_table(9, rot, device="cpu") if rot else None
    pos = torch.tensor([0, 8, 3, 3, 1], dtype=torch.int32)
    y, _ = ref.norm_rope(x, w, table, pos, 1e-6, interleaved)
    want = torch.autograd.grad((y * dy).sum(), (x, w))
    dx, _, dw, _ = ref.norm_rope_backward(dy, x.detach(), w.detach(), table, pos, 1e-6, interleaved)
    assert torch.allclose(dx, want[0], rtol=1e-10, atol=1e-12)
    assert torch.allclose(dw, want[1], rtol=1e-10, atol=1e-12)
    norms = x.detach().square().mean(-1) + 1e-6  # rotation keeps lengths
    if rot:
        one, _ = ref.norm_rope(x.detach(), None, table, pos, 1e-6, interleaved)
        assert torch.allclose(one.square().mean(-1), x.detach().square().mean(-1) / norms,
                              rtol=1e-6)


def test_rope_table():
    t = attention.rope_table(100000, 8, base=100.0, device="cpu")
    assert t.dtype == torch.float32 and t.shape == (100000, 8)
    angle = 99999 * torch.tensor(100.0, dtype=torch.float64) ** (-2 / 8)
    assert t[99999, 1] == torch.cos(angle).float() and t[99999, 5] == torch.sin(angle).float()
    for bad in ((4, 3), (4, 0), (-1, 4)):
        with pytest.raises(_lib.CpgError):
            attention.rope_table(*bad, device="cpu")


# ----------------------------------------------------------------------------------- refusals
def heads(p=ADDRESS, ts=64, hs=8, h=8, dtype=BF16):
    return ctypes.byref(_lib.HeadsC(p, ts, hs, h, dtype))


def test_norm_rope_refusals(lib):
    def forward(q=heads(), k=heads(), t=4, d=8, wq=ADDRESS, wk=ADDRESS, dw=BF16, eps=1e-6,
                table=ADDRESS, rows=16, ld=8, rot=8, pos=ADDRESS, qo=heads(), ko=heads()):
        return lib.cpg_norm_rope(q, k, t, d, wq, wk, dw, eps, table, rows, ld, rot, pos, 0, qo, ko,
                                 None)

    def backward(q=heads(), k=heads(), t=4, d=8, wq=ADDRESS, wk=ADDRESS, dw=BF16, eps=1e-6,
                 table=ADDRESS, rows=16, ld=8, rot=8, pos=ADDRESS, qo=heads(), ko=heads(),
                 dq=heads(), dk=heads(), dwq=ADDRESS, dwk=ADDRESS, ws=ADDRESS, n=1 << 30):
        return lib.cpg_norm_rope_backward(dq, dk, q, k, t, d, wq, wk, dw, eps, table, rows, ld, rot,
                                          pos, 0, qo, ko, dwq, dwk, ws, n, None)
    for f in (forward, backward):
        assert f(q=None) == N and f(qo=None) == N and f(k=None) == N and f(ko=None) == N
        assert f(t=-1) == S and f(t=BIG) == S and f(t=BIG // 8) == S
        assert f(d=0) == S and f(d=1) == S and f(d=257) == S
        assert f(rot=3) == S and f(rot=10) == S and f(rot=-2) == S
        assert f(dw=I8) == D and f(q=heads(dtype=I8)) == D and f(k=heads(dtype=F32)) == D
        assert f(qo=heads(dtype=F32)) == D and f(qo=heads(h=4)) == S and f(q=heads(h=0)) == S
        assert f(eps=-1.0) == C and f(eps=float("nan")) == C and f(eps=float("inf")) == C
        assert f(table=None) == N and f(pos=None) == N and f(ld=7) == S and f(rows=-1) == S
        assert f(q=heads(p=None)) == N and f(q=heads(p=4097)) == A and f(pos=4097) == A
        assert f(table=4098) == A and f(wq=4097) == A and f(wk=4097) == A
        assert f(qo=heads(hs=7)) == S and f(qo=heads(ts=63)) == S and f(qo=heads(hs=0)) == S
        assert f(q=heads(ts=-64)) == S and f(q=heads(hs=2 ** 41)) == S
        assert lib.cpg_last_error_message()
    assert forward(t=0, q=heads(p=None), table=None, pos=None) == _lib.CPG_OK
    assert backward(dq=None) == N and backward(dk=None) == N and backward(dq=heads(dtype=F32)) == D
    assert backward(dq=heads(h=2)) == S and backward(ws=None) == N and backward(n=16) == N
    assert backward(dwq=4097) == A and backward(ws=4104) == A
    assert backward(k=None, ko=None, dk=None) == N  # a gradient of k's weight without k
    size = ctypes.c_int64(-1)
    assert lib.cpg_norm_rope_workspace(4, 8, 0, 8, ctypes.byref(size)) == _lib.CPG_OK
    assert size.value > 0 and size.value % 32 == 0
    assert lib.cpg_norm_rope_workspace(4, 0, 1, 8, ctypes.byref(size)) == S
    assert lib.cpg_norm_rope_workspace(4, 1, -1, 8, ctypes.byref(size)) == S
    assert lib.cpg_norm_rope_workspace(4, 1, 1, 300, ctypes.byref(size)) == S
    assert lib.cpg_norm_rope_workspace(4, 1, 1, 8, None) == N


def problem(t=4, b=1, h=8, dk=8, dv=8, scale=1.0):
    return ctypes.byref(_lib.LinearProblemC(t, b, h, dk, dv, scale))


def states(p=ADDRESS, slots=None, places=1):
    return ctypes.byref(_lib.StatesC(p, slots, places))


def test_linear_attention_refusals(lib):
    def forward(p=problem(), q=heads(), k=heads(), v=heads(), g=ADDRESS, off=None, st=None, fin=None,
                out=heads(), ws=ADDRESS, n=1 << 40):
        return lib.cpg_linear_attention(p, q, k, v, g, off, st, fin, out, ws, n, None)

    def backward(p=problem(), q=heads(), k=heads(), v=heads(), g=ADDRESS, off=None, st=None,
                 fin=None, out=heads(), dq=heads(), dk=heads(), dv=heads(), ds=None, ws=ADDRESS,
                 n=1 << 40):
        return lib.cpg_linear_attention_backward(p, out, q, k, v, g, off, st, fin, dq, dk, dv, ds, 1,
                                                 ws, n, None)

    def step(p=problem(), q=heads(), k=heads(), v=heads(), g=ADDRESS, st=states(places=4),
             out=heads()):
        return lib.cpg_linear_attention_step(p, q, k, v, g, st, out, None)
    for f in (forward, backward, step):
        assert f(p=None) == N and f(q=None) == N and f(k=None) == N and f(v=None) == N
        assert f(out=None) == N and f(g=None) == N and f(g=4097) == A
        for bad in (dict(t=-1), dict(t=BIG), dict(h=0), dict(dk=0), dict(dk=7), dict(dk=12),
                    dict(dk=136), dict(dv=4), dict(dv=256), dict(b=-1)):
            assert f(p=problem(**bad)) == S, bad
        for bad in (0.0, float("nan"), float("inf"), 1e-39):
            assert f(p=problem(scale=bad)) == C
        assert f(q=heads(dtype=F32)) == D and f(v=heads(dtype=I8)) == D
        assert f(q=heads(h=3)) == S and f(k=heads(h=16)) == S and f(v=heads(h=0)) == S
        assert f(q=heads(ts=0)) == U and f(v=heads(hs=0)) == U  # give a shared head once
        assert f(q=heads(p=None)) == N and f(q=heads(p=4104)) == A
        assert f(k=heads(ts=68)) == A and f(v=heads(hs=12)) == A and f(out=heads(h=4)) == S
        assert f(st=states(p=None, places=9)) == N and f(st=states(p=4100, places=9)) == A
        assert f(st=states(slots=4097, places=9)) == A and f(st=states(places=-1)) == S
        assert f(st=states(places=0)) == S  # without slots: one place for every sequence
        assert lib.cpg_last_error_message()
    for f in (forward, backward):
        assert f(p=problem(b=2)) == N  # two sequences without offsets
        assert f(off=4097) == A and f(fin=states(places=0)) == S
        assert f(p=problem(b=BIG // 4), off=ADDRESS) == S
        assert f(ws=4104) == A
    assert forward(p=problem(b=0), off=ADDRESS) == _lib.CPG_OK
    assert forward(out=heads(hs=0)) == S and forward(out=heads(dtype=I8)) == D
    assert backward(out=heads(dtype=F32)) == D and backward(dq=heads(dtype=F32)) == D
    assert backward(dk=heads(h=4)) == S and backward(dv=None) == N
    # Shared heads need FP32 sums.
    assert backward(q=heads(h=4), dq=heads(h=4), ws=None) == N
    assert backward(q=heads(h=4), dq=heads(h=4), n=100) == N
    assert step(st=None) == N and step(p=problem(t=BIG // 8)) == S
    assert step(p=problem(t=0), q=heads(p=None)) == _lib.CPG_OK
    size = ctypes.c_int64(-1)
    args = (8, 8, 8, 0)
    assert lib.cpg_linear_attention_workspace(problem(), *args, ctypes.byref(size)) == _lib.CPG_OK
    assert size.value >= 0
    assert lib.cpg_linear_attention_workspace(problem(), 4, 8, 8, 1, ctypes.byref(size)) == _lib.CPG_OK
    assert size.value >= 4 * 8 * 8 * 4
    assert lib.cpg_linear_attention_workspace(problem(), *args, None) == N
    assert lib.cpg_linear_attention_workspace(None, *args, ctypes.byref(size)) == N
    assert lib.cpg_linear_attention_workspace(problem(), 0, 8, 8, 0, ctypes.byref(size)) == S


def test_linear_attention_refuses_heads_that_its_counts_do_not_hold(lib):
    """2^24 heads x 128 channels are 2^31 elements of a token; a workspace's bytes fit 64 bits."""
    size = ctypes.c_int64(-1)
    for h in (BIG - 1, 1 << 24, (1 << 20) + 1):
        p = problem(t=4, h=h, dk=128, dv=128)
        assert lib.cpg_linear_attention_workspace(p, 1, 1, 1, 1, ctypes.byref(size)) == S
        assert lib.cpg_linear_attention(p, heads(h=1), heads(h=1), heads(h=1), ADDRESS, None, None,
                                        None, heads(h=h, hs=128, ts=h * 128), None, 0, None) == S
    most = problem(t=BIG - 1, h=1 << 20, dk=128, dv=128)
    assert lib.cpg_linear_attention_workspace(most, 1, 1, 1, 1, ctypes.byref(size)) == _lib.CPG_OK
    assert size.value >= 3 * (BIG - 1) * (1 << 20) * 128 * 4


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 2, 8, dtype=torch.bfloat16)
    g = torch.zeros(2)
    for f in (lambda: attention.norm_rope(x, x, None, None, None, torch.zeros(4, dtype=torch.int32)),
              lambda: attention.linear_attention(x, x, x, g),
              lambda: attention.linear_attention_backward(x, x, x, x, g),
              lambda: attention.linear_attention_step(x, x, x, g, torch.zeros(4, 2, 8, 8))):
        with pytest.raises(_lib.CpgError) as e:
            f()
        assert e.value.code == _lib.CPG_ERR_NO_DEVICE
