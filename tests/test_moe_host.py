"""Host-side checks of the INT8 and expert operators' C entry points (no GPU): every bad argument is
an error code with a message before anything is launched, and the oracle's own pieces."""
import ctypes

import pytest
import torch

from cutedsl_pingpong_gemm_b200 import _lib, _tensors, moe
from oracle import moe_ref

F32, BF16, I8, E4M3 = (_lib.CPG_DTYPE_F32, _lib.CPG_DTYPE_BF16, _lib.CPG_DTYPE_I8,
                       _lib.CPG_DTYPE_E4M3)
P = ctypes.c_void_p(4096)  # never dereferenced: every call below fails or has nothing to do
ODD = ctypes.c_void_p(4097)
BIG = 2 ** 31


def config(**kw):
    base = dict(experts=8, k=2, scoring=0, groups=1, kept_groups=1, group_score=0, renormalize=1,
                scale=1.0)
    base.update(kw)
    return ctypes.byref(_lib.RouteConfigC(**base))


def test_route_refusals(lib):
    def route(cfg=None, logits=P, dtype=F32, tokens=4, ld=8, bias=None, ids=P, w=P):
        return lib.cpg_route(config() if cfg is None else cfg, logits, dtype, tokens, ld, bias,
                             ids, w, None)

    def back(cfg=None, dw=P, logits=P, dtype=F32, tokens=4, ld=8, ids=P, out=P, ldd=8):
        return lib.cpg_route_backward(config() if cfg is None else cfg, dw, logits, dtype, tokens,
                                      ld, ids, out, ldd, None)
    S, C = _lib.CPG_ERR_INVALID_SHAPE, _lib.CPG_ERR_INVALID_CONFIG
    for f in (route, back):
        for bad, code in [(dict(experts=0), S), (dict(experts=1025), S), (dict(k=0), S),
                          (dict(k=9), S), (dict(experts=100, k=33), S), (dict(scoring=2), C),
                          (dict(groups=0), C), (dict(groups=3), C), (dict(experts=64, groups=64), C),
                          (dict(kept_groups=0), C), (dict(kept_groups=2), C),
                          (dict(groups=8, kept_groups=1), C), (dict(group_score=7), C)]:
            assert f(config(**bad)) == code, bad
            assert lib.cpg_last_error_message()
        assert f(dtype=I8) == _lib.CPG_ERR_DTYPE
        assert f(tokens=-1) == S and f(tokens=BIG) == S and f(tokens=BIG // 2) == S
        assert f(ld=7) == S
        assert f(logits=None) == _lib.CPG_ERR_NULL and f(ids=None) == _lib.CPG_ERR_NULL
        assert f(logits=ODD) == _lib.CPG_ERR_ALIGNMENT and f(ids=ODD) == _lib.CPG_ERR_ALIGNMENT
        assert f(tokens=0, logits=None, ids=None) == _lib.CPG_OK
    assert lib.cpg_route(None, P, F32, 4, 8, None, P, P, None) == _lib.CPG_ERR_NULL
    assert route(bias=ODD) == _lib.CPG_ERR_ALIGNMENT and route(w=None) == _lib.CPG_ERR_NULL
    assert back(ldd=7) == S and back(dw=None) == _lib.CPG_ERR_NULL
    assert back(out=None) == _lib.CPG_ERR_NULL and back(out=ODD) == _lib.CPG_ERR_ALIGNMENT


def test_order_and_row_refusals(lib):
    S, N, A, D = (_lib.CPG_ERR_INVALID_SHAPE, _lib.CPG_ERR_NULL, _lib.CPG_ERR_ALIGNMENT,
                  _lib.CPG_ERR_DTYPE)

    def order(ids=P, tokens=4, k=2, experts=8, off=P, slots=P):
        return lib.cpg_expert_order(ids, tokens, k, experts, off, slots, None)
    assert order(tokens=-1) == S and order(k=0) == S and order(k=33) == S
    assert order(tokens=BIG // 2, k=2) == S and order(experts=0) == S and order(experts=1025) == S
    assert order(ids=None) == N and order(off=None) == N and order(slots=None) == N
    assert order(ids=ODD) == A and order(off=ODD) == A and order(slots=ODD) == A

    def rows(x=P, dt=BF16, tokens=4, cols=8, ldx=8, slots=P, k=2, out=P, dr=BF16, n=8, ldr=8, sc=P):
        return lib.cpg_dispatch_rows(x, dt, tokens, cols, ldx, slots, k, out, dr, n, ldr, sc, None)
    assert rows(dt=E4M3) == D and rows(dr=F32) == D and rows(dt=I8, dr=I8) == D
    assert rows(ldx=7) == S and rows(ldr=7) == S and rows(tokens=-1) == S and rows(n=-1) == S
    assert rows(cols=-1) == S and rows(k=0) == S
    assert rows(x=None) == N and rows(slots=None) == N and rows(out=None) == N
    assert rows(dr=I8, sc=None) == N
    assert rows(x=ODD) == A and rows(out=ODD) == A and rows(slots=ODD) == A and rows(sc=ODD) == A
    assert rows(tokens=0, x=None) == _lib.CPG_OK and rows(cols=0, x=None) == _lib.CPG_OK
    assert rows(n=0) == _lib.CPG_OK

    def combine(x=P, dt=F32, n=8, cols=8, ldr=8, slots=P, w=P, tokens=4, k=2, src=None, lds=0, y=P,
                ldy=8):
        return lib.cpg_combine_rows(x, dt, n, cols, ldr, slots, w, tokens, k, src, lds, y, ldy, None)
    assert combine(dt=I8) == D and combine(ldr=7) == S and combine(ldy=7) == S
    assert combine(src=P, lds=7) == S and combine(k=33) == S and combine(n=BIG) == S
    assert combine(x=None) == N and combine(slots=None) == N and combine(y=None) == N
    assert combine(x=ODD) == A and combine(y=ODD) == A and combine(src=ODD, lds=8) == A
    assert combine(w=ODD) == A
    assert combine(tokens=0) == _lib.CPG_OK and combine(cols=0) == _lib.CPG_OK

    def back(dy=P, dt=F32, tokens=4, cols=8, lddy=8, x=P, n=8, ldr=8, slots=P, w=P, k=2, dr=P,
             lddr=8, dw=P):
        return lib.cpg_combine_rows_backward(dy, dt, tokens, cols, lddy, x, n, ldr, slots, w, k, dr,
                                             lddr, dw, None)
    assert back(dt=I8) == D and back(lddy=7) == S and back(ldr=7) == S and back(lddr=7) == S
    assert back(k=0) == S and back(dy=None) == N and back(w=None) == N and back(dw=None) == N
    assert back(dr=None) == N and back(dy=ODD) == A and back(dw=ODD) == A
    assert back(tokens=0) == _lib.CPG_OK


def test_rows_of_too_many_columns(lib):
    """Columns are counted in 32 bits: 2^30 and more are refused by every row operator."""
    S, w = _lib.CPG_ERR_INVALID_SHAPE, 2 ** 30
    assert lib.cpg_dispatch_rows(P, BF16, 4, w, w, P, 2, P, BF16, 8, w, None, None) == S
    assert lib.cpg_combine_rows(P, F32, 8, w, w, P, P, 4, 2, None, 0, P, w, None) == S
    assert lib.cpg_combine_rows_backward(P, F32, 4, w, w, P, 8, w, P, P, 2, P, w, P, None) == S
    assert lib.cpg_quantize_int8(P, F32, 4, w, w, P, w, P, None) == S


def test_clear_refusals(lib):
    def clear(x=P, dt=F32, n=8, cols=8, ldr=8, slots=P, tokens=4, k=2):
        return lib.cpg_clear_unnamed_rows(x, dt, n, cols, ldr, slots, tokens, k, None)
    S, N, A = _lib.CPG_ERR_INVALID_SHAPE, _lib.CPG_ERR_NULL, _lib.CPG_ERR_ALIGNMENT
    assert clear(dt=I8) == _lib.CPG_ERR_DTYPE and clear(ldr=7) == S and clear(n=BIG) == S
    assert clear(k=0) == S and clear(k=33) == S and clear(tokens=-1) == S
    assert clear(cols=2 ** 30, ldr=2 ** 30) == S
    assert clear(x=None) == N and clear(slots=None) == N
    assert clear(x=ODD) == A and clear(slots=ODD) == A
    assert clear(n=0, x=None) == _lib.CPG_OK and clear(cols=0, x=None) == _lib.CPG_OK


def test_counts_that_32_bits_would_wrap():
    """More experts or choices than the C entry points' 32-bit counts hold are refused before they
    could be cut to another, valid number."""
    for experts in (2 ** 32 + 8, 2 ** 31, 2 ** 33 + 4):
        with pytest.raises(_lib.CpgError) as e:
            moe._route_config(experts, 2, "softmax", 1, 1, "max", True, 1.0)
        assert e.value.code == _lib.CPG_ERR_INVALID_SHAPE
    for k in (2 ** 32 + 2, 2 ** 31, 33):
        with pytest.raises(_lib.CpgError) as e:
            _tensors.pairs("ids", torch.empty(0, k, dtype=torch.int32))
        assert e.value.code == _lib.CPG_ERR_INVALID_SHAPE
    assert tuple(_tensors.pairs("ids", torch.empty(3, 32, dtype=torch.int32))) == (3, 32)


def test_quantize_refusals(lib):
    def quant(x=P, dt=F32, rows=4, cols=8, ldx=8, q=P, ldq=8, s=P):
        return lib.cpg_quantize_int8(x, dt, rows, cols, ldx, q, ldq, s, None)
    assert quant(dt=I8) == _lib.CPG_ERR_DTYPE and quant(rows=-1) == _lib.CPG_ERR_INVALID_SHAPE
    assert quant(rows=BIG) == _lib.CPG_ERR_INVALID_SHAPE
    assert quant(ldx=7) == _lib.CPG_ERR_INVALID_SHAPE and quant(ldq=7) == _lib.CPG_ERR_INVALID_SHAPE
    assert quant(x=None) == _lib.CPG_ERR_NULL and quant(q=None) == _lib.CPG_ERR_NULL
    assert quant(s=None) == _lib.CPG_ERR_NULL
    assert quant(x=ODD) == _lib.CPG_ERR_ALIGNMENT and quant(s=ODD) == _lib.CPG_ERR_ALIGNMENT
    assert quant(rows=0, x=None, q=None, s=None) == _lib.CPG_OK


def test_int8_plan_refusals(lib):
    """What cpg_gemm_create refuses about INT8 before it looks for a device."""
    cfg = _lib.GemmConfigC(128, 256, 128, 32, 2, 1, 1, 1, 1, 4, 2, 1, 0, 1, 0, 8, 0)

    def create(k=128, dtype=I8, dtype_d=BF16, lda=None):
        prob = _lib.GemmProblemC(64, 64, k, lda or -(-k // 16) * 16, -(-k // 16) * 16, 64, dtype,
                                 dtype_d, 0, 1)
        h = ctypes.c_void_p()
        return lib.cpg_gemm_create(ctypes.byref(cfg), ctypes.byref(prob), 0, ctypes.byref(h))
    assert create(k=131072) == _lib.CPG_ERR_INVALID_SHAPE
    assert b"131071" in lib.cpg_last_error_message()
    assert create(dtype=4) == _lib.CPG_ERR_DTYPE and create(dtype_d=I8) == _lib.CPG_ERR_DTYPE
    assert create(lda=136) == _lib.CPG_ERR_ALIGNMENT
    prob = _lib.GemmProblemC(64, 64, 128, 128, 128, 64, I8, BF16, 0, 1)
    assert lib.cpg_gemm_splitk_static(ctypes.byref(cfg), ctypes.byref(prob), P, P, P, None,
                                      None) == _lib.CPG_ERR_DTYPE
    out = ctypes.c_int32()
    assert lib.cpg_sched_plan_group_size(ctypes.byref(cfg), 8192, I8, ctypes.byref(out)) == 0


def test_oracle_quantise_and_route():
    """Known answers of the oracle's own forms."""
    q, s = moe_ref.quantize_int8(torch.tensor([[127.0, -63.5, 0.5, 1.5], [0.0, 0.0, 0.0, 0.0]]))
    assert q.tolist() == [[127, -64, 0, 2], [0, 0, 0, 0]] and s[0] == 1.0
    ids, w = moe_ref.route(torch.tensor([[0.0, 2.0, 2.0, 1.0]]), 2, renormalize=True)
    assert ids.tolist() == [[1, 2]] and torch.allclose(w, torch.tensor([[0.5, 0.5]]).double())
    ids, w = moe_ref.route(torch.tensor([[5.0, 0.0, 1.0, 4.0]]), 2, groups=2, kept_groups=1,
                           group_score="max")
    assert ids.tolist() == [[0, 1]]
    off, slots = moe_ref.expert_order(torch.tensor([[1, 0], [1, -1], [0, 1]]), 3)
    assert off.tolist() == [0, 2, 5, 5] and slots.tolist() == [[2, 0], [3, -1], [1, 4]]
    y, _ = moe_ref.combine(torch.tensor([[1.0], [2.0]]), torch.tensor([[1, 0], [5, -1]]),
                           torch.tensor([[0.5, 2.0], [1.0, 1.0]]))
    assert y.tolist() == [[3.0], [0.0]]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_oracle_route_backward_is_the_gradient(scoring, renorm):
    """The oracle's gradient formulas against autograd of the forward formulas, in 64 bits."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(5, 9, generator=g, dtype=torch.float64, requires_grad=True)
    dw = torch.randn(5, 3, generator=g, dtype=torch.float64)
    ids, _ = moe_ref.route(x.detach(), 3, scoring=scoring, renormalize=renorm)
    s = x.softmax(1) if scoring == "softmax" else x.sigmoid()
    w = s.gather(1, ids.long())
    if renorm:
        w = w / w.sum(1, keepdim=True)
    (1.5 * w * dw).sum().backward()
    got = moe_ref.route_backward(dw, x.detach(), ids, scoring, renorm, 1.5)
    assert (got - x.grad).abs().max() < 1e-13
