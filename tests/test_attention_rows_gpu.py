"""Rows of linear attention's outputs that belong to no sequence."""
import ctypes

import pytest
import torch

from cutedsl_pingpong_gemm_b200 import _lib, attention

BF, F32 = torch.bfloat16, torch.float32


def normal(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,first,t,hv,h,dv", [
    ([70, 0, 130], 3, 300, 4, 4, 64),      # short
    ([400, 300], 0, 1000, 50, 50, 128),    # chunks on more than every SM
    ([5000, 3001], 7, 8100, 1, 2, 72),     # segments
    ([], 0, 33, 2, 2, 8), ([0], 5, 33, 2, 2, 8), ([1], 40, 41, 3, 3, 8)])
def test_rows_outside_are_zero_in_an_output_that_is_allocated(lengths, first, t, hv, h, dv):
    """Whatever the memory held: a padded batch's output goes to the output projection whole, and NaN
    times the zero gradient of a padded row would spoil that projection's gradient."""
    q, k, v = normal(1, t, h, 64), normal(2, t, h, 64), normal(3, t, hv, dv)
    decay = -torch.linspace(0.01, 1, h, device="cuda")
    offsets = torch.tensor([first] + lengths, device="cuda").cumsum(0).int()
    end = first + sum(lengths)
    given = torch.full((t, h, dv), 5.0, dtype=BF, device="cuda")
    attention.linear_attention(q, k, v, decay, offsets=offsets, out=given)
    assert (given[:first] == 5).all() and (given[end:] == 5).all()
    torch.cuda.synchronize()
    for _ in range(2):
        held = torch.full((t, h, dv), float("nan"), dtype=BF, device="cuda")
        address = held.data_ptr()
        del held
        out, _ = attention.linear_attention(q, k, v, decay, offsets=offsets)
        assert out.data_ptr() == address  # else the test shows nothing
        assert torch.equal(out[first:end], given[first:end])
        assert not out[:first].any() and not out[end:].any()
        del out


@pytest.mark.gpu
def test_clear_leaves_everything_else():
    """Strided heads of both types; only the heads' own channels of the rows outside change."""
    lib = _lib.load()
    offsets = torch.tensor([2, 5, 9], dtype=torch.int32, device="cuda")
    for dtype in (BF, F32):
        x = torch.full((12, 5, 48), 3.0, dtype=dtype, device="cuda")
        part = x[:, 1:4, 8:32]
        p = _lib.LinearProblemC(12, 2, 3, 8, 24, 1.0)
        attention.call(lib.cpg_linear_attention_clear, "clear", x.device, ctypes.byref(p),
                       attention.same_heads("x", part, part.shape, dtype, x.device),
                       offsets.data_ptr())
        want = torch.full_like(x, 3.0)
        want[:2, 1:4, 8:32] = 0
        want[9:, 1:4, 8:32] = 0
        assert torch.equal(x, want)


def test_clear_refusals(lib):
    def clear(t=4, h=8, dv=8, out=True, p=4096, ts=64, hs=8, dtype=_lib.CPG_DTYPE_BF16, off=4096):
        problem = _lib.LinearProblemC(t, 1, h, 8, dv, 1.0)
        heads = ctypes.byref(_lib.HeadsC(p, ts, hs, h, dtype)) if out else None
        return lib.cpg_linear_attention_clear(ctypes.byref(problem), heads, off, None)
    S, N, A, D = (_lib.CPG_ERR_INVALID_SHAPE, _lib.CPG_ERR_NULL, _lib.CPG_ERR_ALIGNMENT,
                  _lib.CPG_ERR_DTYPE)
    assert clear(out=False) == N and clear(off=None) == N and clear(p=None) == N
    assert clear(t=-1) == S and clear(h=0) == S and clear(dv=12) == S and clear(hs=0) == S
    assert clear(p=4104) == A and clear(off=4098) == A and clear(hs=12, ts=96) == A
    assert clear(dtype=_lib.CPG_DTYPE_I8) == D
    assert lib.cpg_linear_attention_clear(None, None, 4096, None) == N
    assert clear(t=0, p=None) == _lib.CPG_OK


@pytest.mark.gpu
def test_tensors_without_heads_are_refused():
    """With the framework's own error, before an output is made."""
    q, decay = normal(1, 9, 2, 64), torch.zeros(2, device="cuda")
    state = torch.zeros(9, 2, 64, 64, device="cuda")
    none = q[:, :0]
    for a, b, c in ((none, q, q), (q, none, q), (q, q, none)):
        for call in (lambda: attention.linear_attention(a, b, c, decay),
                     lambda: attention.linear_attention_step(a, b, c, decay, state),
                     lambda: attention.linear_attention_backward(q, a, b, c, decay)):
            with pytest.raises(_lib.CpgError) as e:
                call()
            assert e.value.code == _lib.CPG_ERR_INVALID_SHAPE
    with pytest.raises(_lib.CpgError):
        attention.linear_attention(q, q, q, decay[:0])
    pos = torch.zeros(9, dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.CpgError):
        attention.norm_rope(none, q, None, None, None, pos)


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [[0, 140, 90], [50, 100, 0, 30], [60, 20, 190, 40], [5, 3],
                                     [-4, 70, 2 ** 31 - 1, 10]])
@pytest.mark.parametrize("share", [1, 2])
def test_rows_of_a_sequence_stay_where_offsets_decrease(offsets, share):
    """A sequence that would end before it starts is empty; clearing what is outside leaves the rows of
    the others, wherever they lie."""
    t, h = 200, 2
    q, k, v, dy = (normal(i, t, h if i == 3 else h // share, 64) for i in range(4))
    decay = torch.tensor([-0.1, -0.02], device="cuda")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    held = torch.full((t, h, 64), 7.0, dtype=BF, device="cuda")
    want, _ = attention.linear_attention(q, k, v, decay, offsets=off, out=held)
    out, _ = attention.linear_attention(q, k, v, decay, offsets=off)
    wants = [torch.full(q.shape, 7.0, dtype=BF, device="cuda") for _ in range(3)]
    attention.linear_attention_backward(dy, q, k, v, decay, offsets=off, out=tuple(wants))
    grads = attention.linear_attention_backward(dy, q, k, v, decay, offsets=off)
    inside = torch.zeros(t, dtype=torch.bool)
    for a, b in zip(offsets, offsets[1:]):
        inside[max(a, 0):max(b, 0)] = True
    assert 0 < int(inside.sum()) < t or offsets == [5, 3] or offsets[0] < 0
    for x, y in ((out, want), *zip(grads, wants)):
        assert torch.equal(x[inside], y[inside]) and not x[~inside].any()
        assert (y[~inside] == 7).all()
