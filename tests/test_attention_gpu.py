"""Norm with rotation and linear attention on the GPU against the 64-bit oracle.

Tolerances.  Half a step of a type is H = eps / 2 (BF16 2^-8, FP32 2^-24).  norm_rope: the output is
rounded once, after about ten FP32 operations on terms of size `size`: H |y| + 2^-19 size.  Linear
attention rounds scores and chunk states to BF16 (2^-8 of `near`, the sum of the terms made of
them), then the output (H |o|); the sums of products of up to 128 tokens and channels, and the
states' two BF16 parts, keep 2^-15 of the terms' sizes `far`.  States: three BF16 parts of every
addend and FP32 sums of at most a few hundred terms, 2^-17 of their sizes."""
import ctypes

import pytest
import torch

from cutedsl_pingpong_gemm_b200 import CpgError, GemmSM90, _lib, attention
from oracle import attention_ref as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=BF, mean=0.0):
    return (torch.randn(*shape, device="cuda", generator=g) + mean).to(dtype)


def within(got, want, tol, what=""):
    """Every element within its tolerance; NaN and infinities at the same places."""
    got, want = got.double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = (got - want).abs()
    # A term below the smallest normal FP32 number, 2^-126, may be lost (decays of e^-200 make terms
    # that no FP32 number holds); sums have at most 2^8 such terms that matter: 2^-118.
    bad = ~(same | (off <= tol + 2 ** -118))
    assert not bad.any(), (what, int(bad.sum()), float((off / tol)[bad].nan_to_num(1e30).max()))


def half(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------- norm and rotation
def rope_case(seed, t, hq, hk, d, rot, dtype, layout, w_dtype=None):
    g = gen(seed)
    if layout == "fused":
        rows = normal(g, t, hq + 2 * hk, d, dtype=dtype)
        q, k = rows[:, :hq], rows[:, hq:hq + hk]
    elif layout == "odd":  # unaligned starts and strides
        q = normal(g, t, hq, d + 3, dtype=dtype)[:, :, 1:1 + d]
        k = normal(g, hk, t, d + 1, dtype=dtype).transpose(0, 1)[:, :, :d]
    else:
        q, k = normal(g, t, hq, d, dtype=dtype), normal(g, t, hk, d, dtype=dtype)
    w_dtype = dtype if w_dtype is None else w_dtype
    wq, wk = (normal(g, d, dtype=w_dtype, mean=1.0) for _ in range(2))
    table = attention.rope_table(300, rot) if rot else None
    pos = torch.randint(0, 300, (t,), device="cuda", generator=g, dtype=torch.int32)
    return q, k, wq, wk, table, pos


ROPE = [
    # t, hq, hk, d, rot, interleaved, dtype, layout
    (1, 1, 1, 2, 2, False, BF, "plain"),
    (3, 2, 1, 2, 2, True, F32, "plain"),
    (16, 32, 8, 128, 128, False, BF, "fused"),
    (17, 4, 2, 128, 64, True, BF, "fused"),
    (5, 3, 3, 80, 40, True, F32, "plain"),
    (5, 3, 3, 80, 40, False, F32, "fused"),
    (7, 2, 5, 96, 20, False, BF, "plain"),
    (9, 3, 1, 250, 250, False, BF, "plain"),
    (9, 3, 1, 250, 124, True, F32, "odd"),
    (33, 1, 2, 256, 256, False, F32, "fused"),
    (33, 1, 2, 256, 128, True, BF, "odd"),
    (4, 2, 2, 255, 2, False, BF, "plain"),
    (4, 2, 2, 255, 254, True, F32, "plain"),
    (300, 2, 1, 64, 0, False, BF, "plain"),
    (2, 2, 2, 36, 12, False, BF, "plain"),
    (2, 2, 2, 36, 36, True, BF, "fused"),
    (1001, 4, 2, 12, 8, False, BF, "odd"),
]


@pytest.mark.parametrize("t,hq,hk,d,rot,interleaved,dtype,layout", ROPE)
def test_norm_rope(t, hq, hk, d, rot, interleaved, dtype, layout):
    q, k, wq, wk, table, pos = rope_case(t + d, t, hq, hk, d, rot, dtype, layout)
    qo, ko = attention.norm_rope(q, k, wq, wk, table, pos, eps=1e-5, interleaved=interleaved)
    for x, w, y in ((q, wq, qo), (k, wk, ko)):
        assert y.shape == x.shape and y.dtype == dtype
        want, size = ref.norm_rope(x, w, table, pos, 1e-5, interleaved)
        within(y, want, half(dtype) * want.abs() + 2 ** -19 * size)


@pytest.mark.parametrize("t,hq,hk,d,rot,interleaved,dtype,layout", ROPE)
def test_norm_rope_backward(t, hq, hk, d, rot, interleaved, dtype, layout):
    q, k, wq, wk, table, pos = rope_case(t + d, t, hq, hk, d, rot, dtype, layout)
    g = gen(1)
    dq, dk = normal(g, t, hq, d, dtype=dtype), normal(g, t, hk, d, dtype=dtype)
    args = (dq, dk, q, k, wq, wk, table, pos)
    got = attention.norm_rope_backward(*args, eps=1e-5, interleaved=interleaved)
    for x, w, dy, dx, dw in ((q, wq, dq, got[0], got[2]), (k, wk, dk, got[1], got[3])):
        assert dx.dtype == dtype and dw.dtype == F32
        want, size, dwant, dsize = ref.norm_rope_backward(dy, x, w, table, pos, 1e-5, interleaved)
        # Sums over up to 256 channels first: 2^-18 of the terms' sizes.
        within(dx, want, half(dtype) * want.abs() + 2 ** -18 * size, "dx")
        within(dw, dwant, 2 ** -17 * dsize, "dw")
    again = attention.norm_rope_backward(*args, eps=1e-5, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_norm_rope_gradient_against_differences():
    q, k, wq, wk, table, pos = rope_case(5, 6, 2, 1, 16, 8, F32, "plain")
    g = gen(2)
    dq, dk = normal(g, 6, 2, 16, dtype=F32), normal(g, 6, 1, 16, dtype=F32)
    got = attention.norm_rope_backward(dq, dk, q, k, wq, wk, table, pos)

    def loss(q, k, wq, wk):
        a, b = ref.norm_rope(q, wq, table, pos, 1e-6, False)[0], ref.norm_rope(k, wk, table, pos,
                                                                             1e-6, False)[0]
        return float((a * dq.double()).sum() + (b * dk.double()).sum())
    leaves = [x.double() for x in (q, k, wq, wk)]
    for i, grad in enumerate(got):
        move = torch.randn(leaves[i].shape, device="cuda", dtype=torch.float64, generator=g)
        up, down = ([x + s * 1e-5 * move if j == i else x for j, x in enumerate(leaves)]
                    for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / 2e-5
        assert abs(slope - float((grad.double() * move).sum())) <= 1e-4 * (1 + abs(slope))


def test_norm_rope_in_place_and_outputs():
    for dtype, layout in ((BF, "fused"), (F32, "odd"), (BF, "odd")):
        q, k, wq, wk, table, pos = rope_case(9, 50, 6, 2, 64, 32, dtype, layout)
        want = attention.norm_rope(q, k, wq, wk, table, pos)
        rows = torch.full((50, 9, 70), 7.0, dtype=dtype, device="cuda")
        out = (rows[:, :6, 2:66], rows[:, 6:8, 2:66])
        got = attention.norm_rope(q, k, wq, wk, table, pos, out=out)
        assert got[0] is out[0] and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert (rows[:, 8] == 7).all() and (rows[:, :, :2] == 7).all() and (rows[:, :, 66:] == 7).all()
        attention.norm_rope(q, k, wq, wk, table, pos, out=(q, k))
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_norm_rope_backward_in_place():
    q, k, wq, wk, table, pos = rope_case(9, 50, 6, 2, 64, 32, BF, "fused")
    g = gen(3)
    dq, dk = normal(g, 50, 6, 64), normal(g, 50, 2, 64)
    want = attention.norm_rope_backward(dq, dk, q, k, wq, wk, table, pos)
    got = attention.norm_rope_backward(dq, dk, q, k, wq, wk, table, pos, out=(dq, dk))
    assert got[0] is dq and all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_rope_parts():
    """Without keys, weights, rotation or rows; weights of the other type."""
    q, k, wq, wk, table, pos = rope_case(4, 12, 3, 2, 32, 32, BF, "plain")
    both = attention.norm_rope(q, k, wq, wk, table, pos)
    alone = attention.norm_rope(q, None, wq, None, table, pos)
    assert alone[1] is None and torch.equal(alone[0], both[0])
    bare = attention.norm_rope(q, k, None, None, table, pos)
    ones = torch.ones(32, device="cuda")
    assert all(torch.equal(a, b) for a, b in
               zip(bare, attention.norm_rope(q, k, ones, ones, table, pos)))
    wide = attention.norm_rope(q, k, wq.float(), wk.float(), table, pos)
    assert all(torch.equal(a, b) for a, b in zip(both, wide))
    still = attention.norm_rope(q, k, wq, wk, None, pos)
    want, size = ref.norm_rope(q, wq, None, pos, 1e-6, False)
    within(still[0], want, half(BF) * want.abs() + 2 ** -19 * size)
    dq, dk = q.clone(), k.clone()
    back = attention.norm_rope_backward(dq, None, q, None, None, None, table, pos)
    assert back[1] is None and back[2] is None and back[3] is None
    full = attention.norm_rope_backward(dq, dk, q, k, None, wk, table, pos)
    assert torch.equal(back[0], full[0]) and full[2] is None and full[3].shape == (32,)
    none = attention.norm_rope_backward(dq[:0], dk[:0], q[:0], k[:0], wq, wk, table, pos[:0])
    assert none[0].shape == (0, 3, 32) and not none[2].any() and not none[3].any()
    assert attention.norm_rope(q[:0], k[:0], wq, wk, table, pos[:0])[0].shape == (0, 3, 32)


def test_norm_rope_positions_outside_the_table():
    q, k, wq, wk, table, pos = rope_case(6, 5, 2, 2, 32, 16, BF, "plain")
    pos[:] = torch.tensor([0, -1, 300, 299, 2 ** 31 - 1], dtype=torch.int32)
    for y in attention.norm_rope(q, k, wq, wk, table, pos):
        assert y[[1, 2, 4], :, :16].isnan().all()
        assert y[[0, 3]].isfinite().all() and y[:, :, 16:].isfinite().all()


def test_norm_rope_extreme_rows():
    """Zero rows stay zero with eps, NaN stays in its head; a tiny eps of 0 with zeros is NaN."""
    q, k, wq, wk, table, pos = rope_case(6, 4, 2, 2, 32, 16, BF, "plain")
    q[0, 0] = 0
    q[1, 1, 3] = float("nan")
    a, _ = attention.norm_rope(q, k, wq, wk, table, pos)
    assert not a[0, 0].any() and a[1, 1].isnan().all()
    keep = torch.ones(4, 2, dtype=torch.bool)
    keep[1, 1] = False
    assert a[keep.cuda()].isfinite().all()


def test_norm_rope_refusals():
    q, k, wq, wk, table, pos = rope_case(6, 4, 2, 2, 32, 16, BF, "plain")
    bad = [((q.double(), None, None, None, table, pos), _lib.CPG_ERR_DTYPE),
           ((q, k.float(), wq, wk, table, pos), _lib.CPG_ERR_DTYPE),
           ((q, k[:3], wq, wk, table, pos), _lib.CPG_ERR_INVALID_SHAPE),
           ((q, k[..., :30], wq, wk, table, pos), _lib.CPG_ERR_INVALID_SHAPE),
           ((q, None, wq, wk, table, pos), _lib.CPG_ERR_NULL),
           ((q, k, wq, wk.float(), table, pos), _lib.CPG_ERR_DTYPE),
           ((q, k, wq[:30], wk, table, pos), _lib.CPG_ERR_INVALID_SHAPE),
           ((q, k, wq, wk, table.double(), pos), _lib.CPG_ERR_DTYPE),
           ((q, k, wq, wk, table[:, :15], pos), _lib.CPG_ERR_INVALID_SHAPE),
           ((q, k, wq, wk, attention.rope_table(4, 64), pos), _lib.CPG_ERR_INVALID_SHAPE),
           ((q, k, wq, wk, table, pos.long()), _lib.CPG_ERR_INVALID_SHAPE),
           ((q, k, wq, wk, table, None), _lib.CPG_ERR_NULL),
           ((q.transpose(1, 2), None, None, None, table, pos), _lib.CPG_ERR_UNSUPPORTED),
           ((q[0], None, None, None, table, pos), _lib.CPG_ERR_INVALID_SHAPE)]
    for args, code in bad:
        with pytest.raises(CpgError) as e:
            attention.norm_rope(*args)
        assert e.value.code == code, args
    with pytest.raises(CpgError):
        attention.norm_rope(q, k, wq, wk, table, pos, out=(q[:, :1].expand(4, 2, 32), k))
    with pytest.raises(CpgError):
        attention.norm_rope_backward(q.float(), k, q, k, wq, wk, table, pos)


# ---------------------------------------------------------------------------- linear attention
def offsets_of(lengths, first=0):
    return torch.tensor([first] + lengths, device="cuda").cumsum(0).int()


def linear_case(seed, lengths, hq, hk, hv, h, dk, dv, pad=0, first=0, layout="plain"):
    g = gen(seed)
    t = first + sum(lengths) + pad
    if layout == "fused":  # a projection's rows
        width = hq * dk + hk * dk + hv * dv
        rows = normal(g, t, width)
        a, b = hq * dk, hq * dk + hk * dk
        q, k, v = (rows[:, :a].unflatten(1, (hq, dk)), rows[:, a:b].unflatten(1, (hk, dk)),
                   rows[:, b:].unflatten(1, (hv, dv)))
    elif layout == "heads_first":
        q, k, v = (normal(g, n, t, d).transpose(0, 1) for n, d in ((hq, dk), (hk, dk), (hv, dv)))
    else:
        q, k, v = normal(g, t, hq, dk), normal(g, t, hk, dk), normal(g, t, hv, dv, mean=0.3)
    decay = -(2.0 ** -torch.linspace(0, 9, h, device="cuda"))
    decay[0] = 0.0 if h > 1 else -0.05
    return q, k, v, decay, offsets_of(lengths, first)


def check_forward(q, k, v, decay, offsets, scale, state_list, out, final=None, dtype=BF):
    o, near, far, want, size = ref.whole_pass(q, k, v, decay, scale, offsets, state_list)
    if out is not None:
        within(out, o, 2 ** -8 * near + half(dtype) * o.abs() + 2 ** -15 * far, "out")
    if final is not None:
        within(final, want, 2 ** -17 * size, "final")


LINEAR = [
    # lengths, hq, hk, hv, heads, dk, dv, layout
    ([1], 1, 1, 1, 1, 8, 8, "plain"),
    ([2], 2, 2, 2, 2, 64, 64, "plain"),
    ([37], 3, 3, 3, 3, 64, 64, "fused"),
    ([127, 128, 129], 2, 2, 2, 2, 128, 128, "plain"),
    ([0, 5, 0, 256, 1, 0], 2, 2, 2, 2, 128, 64, "plain"),
    ([300, 64], 1, 1, 4, 4, 64, 128, "plain"),
    ([515], 2, 1, 4, 4, 128, 128, "fused"),
    ([130, 257], 2, 2, 2, 2, 72, 40, "heads_first"),
    ([383, 1], 2, 2, 2, 2, 8, 128, "plain"),
    ([200], 3, 3, 3, 3, 120, 8, "fused"),
    ([1100, 3, 140], 1, 2, 1, 2, 96, 80, "plain"),
]


@pytest.mark.parametrize("lengths,hq,hk,hv,h,dk,dv,layout", LINEAR)
def test_linear_attention(lengths, hq, hk, hv, h, dk, dv, layout):
    q, k, v, decay, offsets = linear_case(dk + dv, lengths, hq, hk, hv, h, dk, dv, layout=layout)
    scale = dk ** -0.5
    out, final = attention.linear_attention(q, k, v, decay, scale=scale, offsets=offsets, final=True)
    assert out.dtype == BF and final.shape == (len(lengths), h, dk, dv)
    check_forward(q, k, v, decay, offsets, scale, None, out, final)
    alone, none = attention.linear_attention(q, k, v, decay, scale=scale, offsets=offsets)
    assert none is None
    check_forward(q, k, v, decay, offsets, scale, None, alone)
    again = attention.linear_attention(q, k, v, decay, scale=scale, offsets=offsets, final=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], final)


@pytest.mark.parametrize("lengths,hq,hk,hv,h,dk,dv,layout", LINEAR)
def test_linear_attention_from_states(lengths, hq, hk, hv, h, dk, dv, layout):
    """Rows before and behind the sequences, starting states, an FP32 output."""
    q, k, v, decay, offsets = linear_case(dk + dv, lengths, hq, hk, hv, h, dk, dv, pad=9, first=3,
                                          layout=layout)
    b = len(lengths)
    for x in (q, k, v):  # rows of no sequence reach nothing
        x[:3] = float("nan")
        x[3 + sum(lengths):] = float("inf")
    state = normal(gen(7), b, h, dk, dv, dtype=F32)
    kept = state.clone()
    out = torch.full((q.shape[0], h, dv), 5.0, dtype=F32, device="cuda")
    _, final = attention.linear_attention(q, k, v, decay, scale=-0.3, offsets=offsets, state=state,
                                          final=True, out=out)
    assert torch.equal(state, kept)
    assert (out[:3] == 5).all() and (out[3 + sum(lengths):] == 5).all()
    for x in (q, k, v):
        x[:3] = 0
        x[3 + sum(lengths):] = 0
    inside = slice(3, 3 + sum(lengths))
    out[:3] = 0
    out[3 + sum(lengths):] = 0
    assert out[inside].isfinite().all()
    check_forward(q, k, v, decay, offsets, -0.3, list(state), out, final, F32)


@pytest.mark.parametrize("lengths,hq,hk,hv,h,dk,dv,layout", LINEAR)
@pytest.mark.parametrize("states", [False, True])
def test_linear_attention_backward(lengths, hq, hk, hv, h, dk, dv, layout, states):
    q, k, v, decay, offsets = linear_case(dk + dv, lengths, hq, hk, hv, h, dk, dv, pad=2, first=1,
                                          layout=layout)
    g = gen(11)
    b = len(lengths)
    dy = normal(g, q.shape[0], h, dv)
    state = normal(g, b, h, dk, dv, dtype=F32) if states else None
    dfinal = normal(g, b, h, dk, dv, dtype=F32) if states else None
    scale = dk ** -0.5
    got = attention.linear_attention_backward(dy, q, k, v, decay, scale=scale, offsets=offsets,
                                              state=state, dfinal=dfinal)
    grads, (ds, size) = ref.linear_attention_backward(
        dy, q, k, v, decay, scale, offsets, list(state) if states else None,
        list(dfinal) if states else None)
    for name, x, like, (want, near, far) in zip(("dq", "dk", "dv"), got, (q, k, v), grads):
        assert x.shape == like.shape and x.dtype == BF
        within(x, want, 2 ** -8 * near + half(BF) * want.abs() + 2 ** -15 * far, name)
        assert not x[:1].any() and not x[1 + sum(lengths):].any()
    if states:
        within(got[3], ds, 2 ** -17 * size, "dstate")
    else:
        assert got[3] is None
    again = attention.linear_attention_backward(dy, q, k, v, decay, scale=scale, offsets=offsets,
                                                state=state, dfinal=dfinal)
    assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("lengths,dk,dv", [([1200, 1101], 64, 128), ([1200, 1101], 128, 40),
                                           ([1000, 9], 64, 128), ([1000, 9], 128, 40)])
def test_linear_attention_backward_of_two_widths(lengths, dk, dv):
    """dq and dk with dv, or before it."""
    q, k, v, decay, offsets = linear_case(6, lengths, 1, 2, 2, 2, dk, dv)
    dy = normal(gen(5), *v.shape)
    state = normal(gen(7), len(lengths), 2, dk, dv, dtype=F32)
    got = attention.linear_attention_backward(dy, q, k, v, decay, scale=0.2, offsets=offsets,
                                              state=state, dfinal=state)
    grads, (ds, size) = ref.linear_attention_backward(dy, q, k, v, decay, 0.2, offsets, list(state),
                                                      list(state))
    for x, (want, near, far) in zip(got, grads):
        within(x, want, 2 ** -8 * near + half(BF) * want.abs() + 2 ** -15 * far)
    within(got[3], ds, 2 ** -17 * size)


def test_linear_attention_backward_outputs():
    q, k, v, decay, offsets = linear_case(1, [70, 200], 2, 2, 2, 2, 64, 64, pad=3, first=2)
    dy = normal(gen(2), 275, 2, 64)
    want = attention.linear_attention_backward(dy, q, k, v, decay, offsets=offsets)
    out = tuple(torch.full((275, 5, 64), 3.0, dtype=BF, device="cuda") for _ in range(3))
    dstate = torch.empty(2, 2, 64, 64, device="cuda")
    got = attention.linear_attention_backward(dy, q, k, v, decay, offsets=offsets, dstate=dstate,
                                              out=tuple(x[:, 1:3] for x in out))
    assert got[3] is dstate
    # dstate makes the states of dv's pass FP32-exact, so that their BF16 copies may be rounded the
    # other way than without (see the tolerances above); asked for twice it gives the same bits.
    twice = attention.linear_attention_backward(dy, q, k, v, decay, offsets=offsets,
                                                dstate=torch.empty_like(dstate))
    assert torch.equal(twice[3], dstate)
    grads, _ = ref.linear_attention_backward(dy, q, k, v, decay, 1.0, offsets)
    for x, w, y, (g, near, far) in zip(out, want, twice, grads):
        assert torch.equal(x[2:272, 1:3], y[2:272])
        for z in (y, w):
            within(z, g, 2 ** -8 * near + half(BF) * g.abs() + 2 ** -15 * far)
        assert (x[:2] == 3).all() and (x[272:] == 3).all()
        assert (x[:, 0] == 3).all() and (x[:, 3:] == 3).all()
    _, (ds, size) = ref.linear_attention_backward(dy, q, k, v, decay, 1.0, offsets)
    within(dstate, ds, 2 ** -17 * size)


def test_linear_attention_gradient_against_differences():
    """<gradient, move> against differences of the 64-bit forward pass; BF16 gradients of values of
    size 1 are off by 2^-8 of their terms, which the sums of 400 values average."""
    q, k, v, decay, offsets = linear_case(8, [200], 2, 2, 2, 2, 8, 8)
    g = gen(4)
    dy = normal(g, 200, 2, 8)
    got = attention.linear_attention_backward(dy, q, k, v, decay, scale=0.4, offsets=offsets)
    leaves = [x.double() for x in (q, k, v)]

    def loss(q, k, v):
        return float((ref.whole_pass(q, k, v, decay, 0.4, offsets)[0] * dy.double()).sum())
    for i in range(3):
        move = torch.randn(leaves[i].shape, device="cuda", dtype=torch.float64, generator=g)
        up, down = ([x + s * 1e-4 * move if j == i else x for j, x in enumerate(leaves)]
                    for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / 2e-4
        grad = got[i].double()
        assert abs(slope - float((grad * move).sum())) <= 2 ** -7 * float((grad * move).norm()) * 4


@pytest.mark.parametrize("decay", [0.0, -1e-6, -0.69, -5.0, -40.0, -200.0, float("-inf")])
def test_linear_attention_decays(decay):
    """From no forgetting to keeping the token alone, in all directions."""
    q, k, v, _, offsets = linear_case(9, [140, 261], 1, 1, 1, 1, 64, 64)
    g = torch.tensor([decay], device="cuda")
    state = normal(gen(7), 2, 1, 64, 64, dtype=F32)
    out, final = attention.linear_attention(q, k, v, g, scale=0.2, offsets=offsets, state=state,
                                            final=True)
    check_forward(q, k, v, g, offsets, 0.2, list(state), out, final)
    dy = normal(gen(8), 401, 1, 64)
    got = attention.linear_attention_backward(dy, q, k, v, g, scale=0.2, offsets=offsets,
                                              state=state, dfinal=state)
    grads, (ds, size) = ref.linear_attention_backward(dy, q, k, v, g, 0.2, offsets, list(state),
                                                      list(state))
    for x, (want, near, far) in zip(got, grads):
        within(x, want, 2 ** -8 * near + half(BF) * want.abs() + 2 ** -15 * far)
    within(got[3], ds, 2 ** -17 * size)


@pytest.mark.parametrize("lengths,h,dk,dv,dtype", [
    ([1], 1, 8, 8, BF), ([2], 1, 64, 64, BF), ([5], 2, 128, 64, F32), ([1, 1, 1], 2, 64, 128, BF),
    ([1, 2, 1, 3] * 20, 4, 64, 64, BF), ([37], 3, 72, 40, BF), ([128], 1, 128, 128, F32), ([129, 3], 2, 128, 128, BF)])
def test_linear_attention_of_few_chunks(lengths, h, dk, dv, dtype):
    """Without a starting state and up to one chunk a sequence, only the output is rounded to BF16:
    scores are two BF16 parts, their sum to 2^-17 (half a step of the second, which is below 2^-8 of
    the score), and the sums of their products stay within 2^-15 of far.
    (Tokens of a second chunk also read a BF16 state.)"""
    q, k, v, decay, offsets = linear_case(11, lengths, h, h, h, h, dk, dv)
    out = torch.empty(*v.shape, dtype=dtype, device="cuda")
    attention.linear_attention(q, k, v, decay, scale=dk ** -0.5, offsets=offsets, out=out)
    o, near, far, _, _ = ref.whole_pass(q, k, v, decay, dk ** -0.5, offsets)
    tol = half(dtype) * o.abs() + 2 ** -15 * far
    first = 0
    for n in lengths:
        tol[first + 128:first + n] += 2 ** -8 * near[first + 128:first + n]
        first += n
    within(out, o, tol)
    # Against the order of the tokens, a gradient: dk = pass(v, dy, q) from behind.
    dy = normal(gen(12), *v.shape)
    dk_got = attention.linear_attention_backward(dy, q, k, v, decay, scale=dk ** -0.5,
                                                 offsets=offsets)[1]
    o, near, far, _, _ = ref.whole_pass(v, dy, q, decay, dk ** -0.5, offsets, reverse=True)
    tol = half(BF) * o.abs() + 2 ** -15 * far
    first = 0
    for n in lengths:  # (chunks are counted from the sequence's first token; the last has no state)
        tol[first:first + (n - 1) // 128 * 128] += 2 ** -8 * near[first:first + (n - 1) // 128 * 128]
        first += n
    within(dk_got, o, tol)


def test_linear_attention_one_sequence_without_offsets():
    q, k, v, decay, offsets = linear_case(3, [333], 2, 2, 2, 2, 64, 128)
    a = attention.linear_attention(q, k, v, decay, offsets=offsets, final=True)
    b = attention.linear_attention(q, k, v, decay, final=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    dy = normal(gen(2), 333, 2, 128)
    a = attention.linear_attention_backward(dy, q, k, v, decay, offsets=offsets)
    b = attention.linear_attention_backward(dy, q, k, v, decay)
    assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3]))


def test_linear_attention_pool_of_states():
    """States at slots, updated in place; slots outside the pool start from zeros and stay out."""
    lengths = [40, 0, 129, 7]
    q, k, v, decay, offsets = linear_case(3, lengths, 2, 2, 2, 2, 64, 32)
    pool = normal(gen(5), 9, 2, 64, 32, dtype=F32)
    before = pool.clone()
    slots = torch.tensor([8, 2, -1, 5], dtype=torch.int32, device="cuda")
    out, final = attention.linear_attention(q, k, v, decay, offsets=offsets, state=pool, slots=slots,
                                            final=pool)
    assert final is pool
    states = [before[8], before[2], torch.zeros_like(before[0]), before[5]]
    check_forward(q, k, v, decay, offsets, 1.0, states, out)
    _, _, _, want, size = ref.whole_pass(q, k, v, decay, 1.0, offsets, states)
    for s, b in ((8, 0), (2, 1), (5, 3)):
        within(pool[s], want[b], 2 ** -17 * size[b])
    rest = [i for i in range(9) if i not in (8, 2, 5)]
    assert torch.equal(pool[rest], before[rest])
    assert torch.equal(pool[2], before[2])  # an empty sequence's state is kept
    slots[3] = 9
    attention.linear_attention(q, k, v, decay, offsets=offsets, state=pool, slots=slots)


@pytest.mark.parametrize("lengths,h,dk,dv", [([9001], 1, 128, 128), ([6000, 0, 7001, 1], 2, 64, 128),
                                             ([12000], 3, 128, 40)])
def test_linear_attention_of_long_sequences(lengths, h, dk, dv):
    """Few heads and long sequences are worked on in segments, whose states are joined; a pool's
    states are read before they are written."""
    q, k, v, decay, offsets = linear_case(3, lengths, h, h, h, h, dk, dv, pad=1)
    b, g = len(lengths), gen(6)
    pool = normal(g, b + 2, h, dk, dv, dtype=F32)
    slots = torch.randperm(b + 2, device="cuda", generator=g)[:b].int()
    states = [pool[i].clone() for i in slots.tolist()]
    size = _lib.ctypes.c_int64()
    p = _lib.LinearProblemC(q.shape[0], b, h, dk, dv, 1.0)
    _lib.load().cpg_linear_attention_workspace(_lib.ctypes.byref(p), h, h, h, 0,
                                               _lib.ctypes.byref(size))
    assert size.value > 0  # they are cut
    first = attention.linear_attention(q, k, v, decay, scale=0.1, offsets=offsets)[0]
    check_forward(q[:-1], k[:-1], v[:-1], decay, offsets, 0.1, None, first[:-1])
    out, _ = attention.linear_attention(q, k, v, decay, scale=0.1, offsets=offsets, state=pool,
                                        slots=slots, final=pool)
    # FP32 sums and decays over 100 chunks: 2^-14 of the terms' sizes at most.
    o, near, far, want, sizes = ref.whole_pass(q, k, v, decay, 0.1, offsets, states)
    within(out[:-1], o[:-1], (2 ** -8 * near + half(BF) * o.abs() + 2 ** -14 * far)[:-1], "out")
    within(pool[slots.long()], want, 2 ** -14 * sizes, "final")
    dy = normal(g, q.shape[0], h, dv)
    state, dfinal = torch.stack(states), normal(g, b, h, dk, dv, dtype=F32)
    got = attention.linear_attention_backward(dy, q, k, v, decay, scale=0.1, offsets=offsets,
                                              state=state, dfinal=dfinal)
    grads, (ds, dsize) = ref.linear_attention_backward(dy, q, k, v, decay, 0.1, offsets, states,
                                                       list(dfinal))
    for name, x, (want, near, far) in zip(("dq", "dk", "dv"), got, grads):
        within(x, want, 2 ** -8 * near + half(BF) * want.abs() + 2 ** -14 * far, name)
    within(got[3], ds, 2 ** -14 * dsize, "dstate")


def test_linear_attention_nothing_to_do():
    q, k, v, decay, _ = linear_case(3, [4], 2, 2, 2, 2, 64, 64)
    empty = offsets_of([0, 0])
    state = normal(gen(1), 2, 2, 64, 64, dtype=F32)
    out, final = attention.linear_attention(q[:0], k[:0], v[:0], decay, offsets=empty, state=state,
                                            final=True)
    assert out.shape == (0, 2, 64) and torch.equal(final, state)
    out, final = attention.linear_attention(q, k, v, decay, offsets=empty, final=True)
    assert not final.any()
    _, final = attention.linear_attention(q[:0], k[:0], v[:0], decay, final=True)
    assert final.shape == (1, 2, 64, 64) and not final.any()
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, final = attention.linear_attention(q, k, v, decay, offsets=none, final=True)
    assert final.shape == (0, 2, 64, 64)
    got = attention.linear_attention_backward(v[:0], q[:0], k[:0], v[:0], decay, offsets=empty,
                                              state=state, dfinal=state)
    assert got[0].shape == (0, 2, 64) and torch.equal(got[3], state)
    got = attention.linear_attention_backward(v, q, k, v, decay, offsets=empty)
    assert not any(x.any() for x in got[:3])


@pytest.mark.parametrize("dk,dv", [(8, 8), (24, 128), (128, 40), (128, 128)])
def test_linear_attention_empty_sequences_hand_their_states_on(dk, dv):
    """Their final states are the starting ones, bit for bit, in place too; gradients likewise."""
    q, k, v, decay, offsets = linear_case(3, [0, 9, 0, 140, 0], 2, 2, 2, 2, dk, dv)
    state = normal(gen(4), 5, 2, dk, dv, dtype=F32)
    _, final = attention.linear_attention(q, k, v, decay, scale=0.3, offsets=offsets, state=state,
                                          final=True)
    pool = state.clone()
    attention.linear_attention(q, k, v, decay, scale=0.3, offsets=offsets, state=pool, final=pool)
    assert torch.equal(pool, final) and torch.equal(final[::2], state[::2])
    dy = normal(gen(5), *v.shape)
    dstate = attention.linear_attention_backward(dy, q, k, v, decay, offsets=offsets, state=state,
                                                 dfinal=state)[3]
    assert torch.equal(dstate[::2], state[::2])


def test_linear_attention_offsets_beyond_the_rows():
    """Offsets are cut to the rows there are; a sequence that would end before it starts is empty."""
    q, k, v, decay, _ = linear_case(3, [300], 2, 2, 2, 2, 64, 64)
    offsets = torch.tensor([-5, 140, 90, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    out, final = attention.linear_attention(q[:200], k[:200], v[:200], decay, offsets=offsets,
                                            final=True)
    for b, (x, e) in enumerate(((0, 140), (140, 140), (90, 200))):
        one, end = attention.linear_attention(q[x:e], k[x:e], v[x:e], decay, final=True)
        assert torch.equal(final[b], end[0])
        if b == 2:
            assert torch.equal(out[140:200], one[50:])


def test_linear_attention_offsets_that_decrease_stay_in_their_workspace():
    """Offsets that go back and forth name more segments than the rows have; those past the
    workspace are left out, and nothing behind it or in front of it changes."""
    h, n = 2, 64
    lib = _lib.load()
    for t, sequences in ((8192, 3), (65536, 9)):
        q, k, v, decay, _ = linear_case(3, [t], h, h, h, h, 64, 64)
        offsets = torch.tensor([0, t] * ((sequences + 1) // 2), dtype=torch.int32, device="cuda")
        p, problem, q_c, k_c, v_c = attention._linear_args(q, k, v, decay, 1.0, sequences)
        size = ctypes.c_int64()
        _lib.check(lib.cpg_linear_attention_workspace(p, h, h, h, 0, ctypes.byref(size)))
        assert size.value > sequences * h * 64 * 64 * 4  # the sequences are cut
        work = torch.full((n + size.value + n,), 7, dtype=torch.uint8, device="cuda")
        out, o_c = attention._attention_output(None, v, problem)
        final = torch.zeros(sequences, h, 64, 64, device="cuda")
        f_c = attention._states("final", final, problem, sequences, None, q.device)
        _lib.check(lib.cpg_linear_attention(
            p, q_c, k_c, v_c, decay.data_ptr(), offsets.data_ptr(), None, f_c, o_c,
            work.data_ptr() + n, size.value, torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert (work[:n] == 7).all() and (work[n + size.value:] == 7).all()
        assert attention.status() == 0


def test_linear_attention_keeps_sequences_and_times_apart():
    """NaN in one sequence or head reaches no other, and a later token no earlier chunk."""
    q, k, v, decay, offsets = linear_case(3, [150, 300, 150], 2, 2, 2, 2, 64, 64)
    want, _ = attention.linear_attention(q, k, v, decay, offsets=offsets)
    k2, v2 = k.clone(), v.clone()
    k2[150 + 200, 0] = float("nan")
    v2[150 + 250, 0] = float("inf")
    got, _ = attention.linear_attention(q, k2, v2, decay, offsets=offsets)
    assert torch.equal(got[:, 1], want[:, 1])
    assert torch.equal(got[:278, 0], want[:278, 0]) and torch.equal(got[450:], want[450:])
    assert got[350:450, 0].isnan().all()
    assert torch.equal(got[278:350, 0], want[278:350, 0])  # a NaN key spoils no earlier output


def test_linear_attention_backward_keeps_times_apart():
    """A NaN in an operand reaches the gradients that are made of it and no others."""
    q, k, v, decay, _ = linear_case(3, [300], 2, 2, 2, 2, 64, 64)
    dy = normal(gen(5), 300, 2, 64)
    f = attention.linear_attention_backward
    want = f(dy, q, k, v, decay)[:3]
    t = 200
    # Which rows of head 0 of (dq, dk, dv) a NaN at token t makes NaN, at least in one channel.
    later, earlier = set(range(t, 300)), set(range(t + 1))
    reach = {"q": (set(), earlier, earlier), "k": (later, set(), {t}), "v": (later, {t}, set()),
             "dy": ({t}, earlier, earlier)}
    for name, rows in reach.items():
        x = {"q": q, "k": k, "v": v, "dy": dy}
        x[name] = x[name].clone()
        x[name][t, 0, 5] = float("nan")
        got = f(x["dy"], x["q"], x["k"], x["v"], decay)[:3]
        for g, w, spoilt in zip(got, want, rows):
            assert torch.equal(g[:, 1], w[:, 1])
            keep = torch.tensor([i not in spoilt for i in range(300)])
            assert torch.equal(g[keep, 0], w[keep, 0]), name
            assert g[~keep, 0].isnan().any(dim=1).all(), name


def test_linear_attention_infinities_in_several_places():
    """Bad values in neighbouring chunks, in both boxes of channels and in two sequences of a block;
    each channel is NaN from its first on, in the final state too."""
    lengths = [300] * 3
    q, k, v, decay, offsets = linear_case(4, lengths, 100, 100, 100, 100, 64, 128)
    v = v.clone()
    bad = [(10, 3, 7), (140, 3, 7), (290, 3, 100), (300, 3, 64), (301, 50, 0), (899, 99, 127)]
    for t, h, c in bad:
        v[t, h, c] = float("inf") if t % 2 else float("nan")
    clean = torch.where(v.isfinite(), v, 0.0).bfloat16()
    want, wf = attention.linear_attention(q, k, clean, decay, offsets=offsets, final=True)
    got, gf = attention.linear_attention(q, k, v, decay, offsets=offsets, final=True)
    for t, h, c in bad:
        end = (t // 300 + 1) * 300
        want[t:end, h, c] = float("nan")
        wf[t // 300, h, :, c] = float("nan")
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(gf.isnan(), wf.isnan())
    assert torch.equal(got[~got.isnan()], want[~want.isnan()])
    assert torch.equal(gf[~gf.isnan()], wf[~wf.isnan()])


def test_linear_attention_of_many_short_sequences():
    lengths = [i % 4 for i in range(3000)]
    q, k, v, decay, offsets = linear_case(4, lengths, 2, 2, 2, 2, 16, 16)
    out, final = attention.linear_attention(q, k, v, decay, offsets=offsets, final=True)
    check_forward(q, k, v, decay, offsets, 1.0, None, out, final)
    some = offsets[:1501]  # few enough to be sorted by their lengths
    part, ends = attention.linear_attention(q, k, v, decay, offsets=some, final=True)
    n = int(some[-1])
    assert torch.equal(part[:n], out[:n]) and torch.equal(ends, final[:1500])


def test_rows_and_states_past_2_31_elements():
    """Tokens 2^30 elements apart, and a pool of states of more than 2^31."""
    wide = torch.empty(2 ** 31 + 4096, dtype=BF, device="cuda")
    far = lambda h, d, at: wide.as_strided((3, h, d), (2 ** 30, d, 1), at)  # noqa: E731
    g = gen(2)
    q, k, v, out = (far(2, 64, 256 * i) for i in range(4))
    near = [normal(g, 3, 2, 64) for _ in range(3)]
    for x, y in zip((q, k, v), near):
        x.copy_(y)
    decay = torch.tensor([-0.1, -1.0], device="cuda")
    attention.linear_attention(q, k, v, decay, out=out)
    assert torch.equal(out, attention.linear_attention(*near, decay)[0])
    dy = normal(g, 3, 2, 64)
    got = attention.linear_attention_backward(dy, q, k, v, decay, out=(q, k, out))
    want = attention.linear_attention_backward(dy, *near, decay)
    assert torch.equal(out, want[2])
    for x, y in zip((q, k), near):
        x.copy_(y)
    w = torch.ones(64, device="cuda")
    table, pos = attention.rope_table(8, 64), torch.arange(3, device="cuda").int()
    attention.norm_rope(q, k, w, w, table, pos, out=(q, k))
    for x, y in zip((q, k), attention.norm_rope(*near[:2], w, w, table, pos)):
        assert torch.equal(x, y)
    del wide, q, k, v, out, got
    places = 2 ** 31 // (32 * 128 * 128) + 2
    pool = torch.empty(places, 32, 128, 128, device="cuda")
    q, k, v = (normal(g, 2, 32, 128) for _ in range(3))
    decay = -torch.rand(32, device="cuda", generator=g)
    slots = torch.tensor([places - 1, 0], dtype=torch.int32, device="cuda")
    small = normal(g, 2, 32, 128, 128, dtype=F32)
    for f in (lambda s, slots: attention.linear_attention_step(q, k, v, decay, s, slots=slots),
              lambda s, slots: attention.linear_attention(
                  q, k, v, decay, offsets=torch.arange(3, device="cuda").int(), state=s, slots=slots,
                  final=s)[0]):
        pool[slots.long()] = small
        mine = small.clone()
        y = f(pool, slots)
        assert torch.equal(y, f(mine, torch.arange(2, device="cuda").int()))
        assert torch.equal(pool[slots.long()], mine)


def test_calls_on_two_streams():
    """The same operators at once on two streams, each with its own inputs."""
    cases = [linear_case(s, [700, 900], 8, 8, 8, 8, 128, 128) for s in (1, 2)]
    want = [attention.linear_attention(*c[:4], offsets=c[4], final=True) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(5):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i] = attention.linear_attention(*c[:4], offsets=c[4], final=True)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert attention.status() == 0


STEP = [(1, 1, 1, 1, 1, 8, 8), (4, 32, 32, 32, 32, 128, 128), (3, 2, 1, 4, 4, 64, 128),
        (7, 2, 2, 2, 2, 128, 40), (65, 1, 1, 2, 2, 72, 64), (300, 3, 3, 3, 3, 16, 24)]


@pytest.mark.parametrize("t,hq,hk,hv,h,dk,dv", STEP)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_attention_step(t, hq, hk, hv, h, dk, dv, dtype):
    """One token: each state element is one FP32 product and sum (2^-22 of its terms), the output a
    sum of dk of them (2^-16)."""
    q, k, v, decay, _ = linear_case(t, [t], hq, hk, hv, h, dk, dv)
    g = gen(3)
    pool = normal(g, t + 3, h, dk, dv, dtype=F32)
    slots = torch.randperm(t + 3, device="cuda", generator=g)[:t].int()
    if t > 3:
        slots[2], slots[3] = -1, t + 3
    before = pool.clone()
    out = torch.full((t, h, dv), 9.0, dtype=dtype, device="cuda")
    got = attention.linear_attention_step(q, k, v, decay, pool, scale=0.3, slots=slots, out=out)
    assert got is out
    untouched = set(range(t + 3))
    lam = decay.double().exp()[:, None, None]
    for i, s in enumerate(slots.tolist()):
        if not 0 <= s < t + 3:
            assert not out[i].any()
            continue
        untouched.discard(s)
        qi, ki, vi = (x[i].double().repeat_interleave(h // x.shape[1], dim=0) for x in (q, k, v))
        new = lam * before[s].double() + ki[:, :, None] * vi[:, None, :]
        size = lam * before[s].double().abs() + (ki[:, :, None] * vi[:, None, :]).abs()
        within(pool[s], new, 2 ** -22 * size, "state")
        o = 0.3 * (qi[:, None] @ new)[:, 0]
        within(out[i], o, half(dtype) * o.abs() + 2 ** -16 * 0.3 * (qi.abs()[:, None] @ size)[:, 0])
    rest = sorted(untouched)
    assert torch.equal(pool[rest], before[rest])


def test_steps_continue_a_prompt():
    """A prompt, then single tokens, against all tokens at once: states to FP32, outputs to BF16."""
    q, k, v, decay, _ = linear_case(5, [200], 2, 2, 2, 2, 64, 64)
    want, end = attention.linear_attention(q, k, v, decay, scale=0.1, final=True)
    n = 190
    out, state = attention.linear_attention(q[:n], k[:n], v[:n], decay, scale=0.1, final=True)
    rows = [out]
    for t in range(n, 200):
        rows.append(attention.linear_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], decay, state,
                                                    scale=0.1))
    o, near, far, final, size = ref.whole_pass(q, k, v, decay, 0.1, None)
    tol = 2 ** -8 * near + half(BF) * o.abs() + 2 ** -15 * far
    within(torch.cat(rows), o, tol)
    within(want, o, tol)
    within(state, final, 2 ** -17 * size)
    within(end, final, 2 ** -17 * size)


def test_prompt_in_pieces():
    q, k, v, decay, _ = linear_case(5, [700], 2, 2, 2, 2, 128, 128)
    state, rows = None, []
    for a, b in ((0, 1), (1, 130), (130, 130), (130, 500), (500, 700)):
        y, state = attention.linear_attention(q[a:b], k[a:b], v[a:b], decay, scale=0.1, state=state,
                                              final=True if state is None else state)
        rows.append(y)
    o, near, far, final, size = ref.whole_pass(q, k, v, decay, 0.1, None)
    # Chunks start elsewhere here, so terms may be rounded on either path: both sums of terms.
    within(torch.cat(rows), o, 2 ** -8 * (near + far / 4) + half(BF) * o.abs())
    within(state, final, 2 ** -16 * size)


def test_linear_attention_refusals():
    q, k, v, decay, offsets = linear_case(3, [20, 30], 2, 2, 2, 2, 64, 64)
    f = attention.linear_attention
    state = torch.zeros(2, 2, 64, 64, device="cuda")
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")
    S, D = _lib.CPG_ERR_INVALID_SHAPE, _lib.CPG_ERR_DTYPE
    bad = [(lambda: f(q.float(), k, v, decay), D), (lambda: f(q, k, v.half(), decay), D),
           (lambda: f(q, k, v, decay.double()), S), (lambda: f(q, k, v, decay[:1]), S),
           (lambda: f(q, k, v, None), S),
           (lambda: f(q, k[:, :, :56], v, decay), S), (lambda: f(q, k[:40], v, decay), S),
           (lambda: f(q[..., :60], k[..., :60], v, decay), S),
           (lambda: f(q[..., 4:60], k[..., 8:], v, decay), _lib.CPG_ERR_ALIGNMENT),
           (lambda: f(q, k, v, decay, offsets=offsets.long()), S),
           (lambda: f(q, k, v, decay, offsets=offsets[:0]), S),
           (lambda: f(q, k, v, decay, offsets=offsets, state=state[:1]), S),
           (lambda: f(q, k, v, decay, offsets=offsets, state=state.double()), S),
           (lambda: f(q, k, v, decay, offsets=offsets, state=state, slots=slots[:1]), S),
           (lambda: f(q, k, v, decay, offsets=offsets, slots=slots, final=True),
            _lib.CPG_ERR_UNSUPPORTED),
           (lambda: f(q, k, v, decay, scale=0.0), _lib.CPG_ERR_INVALID_CONFIG),
           (lambda: f(q, k, v, decay, out=torch.empty(50, 2, 64, device="cuda", dtype=torch.half)), D),
           (lambda: f(q, k, v, decay, out=torch.empty(50, 2, 56, device="cuda", dtype=BF)), S),
           (lambda: f(q, k, v, decay, out=q[:, :1].expand(50, 2, 64)), S),
           (lambda: attention.linear_attention_backward(v.float(), q, k, v, decay), D),
           (lambda: attention.linear_attention_backward(v[:, :1], q, k, v, decay), S),
           (lambda: attention.linear_attention_step(q, k, v, decay, state), S),
           (lambda: attention.linear_attention_step(q, k, v, decay, None), _lib.CPG_ERR_NULL),
           (lambda: attention.linear_attention_step(q, k, v, decay, state, slots=slots), S)]
    for i, (call, code) in enumerate(bad):
        with pytest.raises(CpgError) as e:
            call()
        assert e.value.code == code, (i, e.value)


# ------------------------------------------------------------------------------------ together
def test_streams_and_graphs():
    """On a stream of its own, and captured twice and replayed in turn on new inputs."""
    lengths = [100, 0, 333]
    q, k, v, decay, offsets = linear_case(3, lengths, 2, 4, 4, 4, 64, 64)
    _, _, wq, wk, table, pos = rope_case(6, sum(lengths), 2, 4, 64, 32, BF, "plain")
    dy = normal(gen(1), sum(lengths), 4, 64)

    def layer(q, k, v):
        a, b = attention.norm_rope(q, k, wq, wk, table, pos)
        y, final = attention.linear_attention(a, b, v, decay, scale=0.1, offsets=offsets, final=True)
        da, db, dv, _ = attention.linear_attention_backward(dy, a, b, v, decay, scale=0.1,
                                                            offsets=offsets)
        return (y, final, dv) + attention.norm_rope_backward(da, db, q, k, wq, wk, table, pos)
    want = layer(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(q, k, v)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, results = [], []
    inputs = [x.clone() for x in (q, k, v)]
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(layer(*inputs))
        graphs.append(graph)
    other = linear_case(33, lengths, 2, 4, 4, 4, 64, 64)[:3]
    wants = {0: want, 1: layer(*other)}
    for i, g in ((0, 0), (1, 1), (0, 1), (1, 0)):
        for x, new in zip(inputs, ((q, k, v), other)[i]):
            x.copy_(new)
        graphs[g].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results[g], wants[i])), (i, g)
    del graphs


def test_graph_of_segments_advances_a_pool_in_place():
    """Captured with the sequences cut into segments, states read from and written to one pool:
    each replay goes on from the last one's states, as eager calls do, bit for bit."""
    q, k, v, decay, offsets = linear_case(8, [5000, 0, 3000], 2, 2, 2, 2, 64, 128)
    slots = torch.tensor([3, 0, 1], dtype=torch.int32, device="cuda")
    first = normal(gen(2), 5, 2, 64, 128, dtype=F32)
    wants, pool = [], first.clone()
    for _ in range(3):
        out, _ = attention.linear_attention(q, k, v, decay, scale=0.1, offsets=offsets, state=pool,
                                            slots=slots, final=pool)
        wants.append((out, pool.clone()))
    assert torch.equal(wants[2][1][[0, 2, 4]], first[[0, 2, 4]])
    check_forward(q, k, v, decay, offsets, 0.1, [first[3], first[0], first[1]], wants[0][0],
                  wants[0][1][[3, 0, 1]])
    pool = first.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = attention.linear_attention(q, k, v, decay, scale=0.1, offsets=offsets, state=pool,
                                            slots=slots, final=pool)
    assert torch.equal(pool, first)
    for want in wants:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(pool, want[1])
    del graph


def test_layer_of_products_and_attention():
    """Projection, norm with rotation, linear attention, output projection, as a layer runs them,
    with every step against the 64-bit form of the values it was given, and its gradient."""
    t, dim, hq, hk, d = 333, 256, 4, 2, 64
    g = gen(0)
    x = normal(g, t, dim)
    w_in = (normal(g, (hq + 2 * hk) * d, dim, dtype=F32) * dim ** -0.5).bfloat16()
    w_out = (normal(g, dim, hq * d, dtype=F32) * (hq * d) ** -0.5).bfloat16()
    decay = -(2.0 ** -torch.arange(1, hq + 1, device="cuda").float())
    offsets = offsets_of([200, 133])
    table = attention.rope_table(256, d)
    pos = torch.cat([torch.arange(200), torch.arange(133)]).int().cuda()
    wq, wk = normal(g, d, mean=1.0), normal(g, d, mean=1.0)
    gemm = GemmSM90((128, 128), (128, 32), (1, 1, 1), (1, 1), ab_stage=4, reuse_ab=False,
                    is_persistent=True)
    rows = torch.empty(t, (hq + 2 * hk) * d, dtype=BF, device="cuda")
    gemm(x, w_in, rows, None)
    heads = rows.view(t, hq + 2 * hk, d)
    q, k = attention.norm_rope(heads[:, :hq], heads[:, hq:hq + hk], wq, wk, table, pos)
    v = heads[:, hq + hk:]
    y, _ = attention.linear_attention(q, k, v, decay, scale=d ** -0.5, offsets=offsets)
    out = torch.empty(t, dim, dtype=BF, device="cuda")
    gemm(y.view(t, hq * d), w_out, out, None)
    check_forward(q, k, v, decay, offsets, d ** -0.5, None, y)
    want = y.view(t, -1).double() @ w_out.double().T
    within(out, want, half(BF) * want.abs() + 2 ** -16 * (y.view(t, -1).double().abs()
                                                          @ w_out.double().abs().T))
    dout = normal(g, t, dim)
    dy = torch.empty(t, hq * d, dtype=BF, device="cuda")
    gemm(dout, w_out.T.contiguous(), dy, None)
    drows = torch.empty_like(heads)
    dq, dk, _, _ = attention.linear_attention_backward(
        dy.view(t, hq, d), q, k, v, decay, scale=d ** -0.5, offsets=offsets,
        out=(torch.empty_like(q), torch.empty_like(k), drows[:, hq + hk:]))
    got = attention.norm_rope_backward(dq, dk, heads[:, :hq], heads[:, hq:hq + hk], wq, wk, table,
                                       pos, out=(drows[:, :hq], drows[:, hq:hq + hk]))
    assert got[0].data_ptr() == drows.data_ptr()
    # The whole chain by automatic differentiation in 64 bits, to the accuracy of five roundings.
    leaf = heads.double().requires_grad_()
    a = ref.norm_rope(leaf[:, :hq], wq, table, pos, 1e-6, False)[0]
    b = ref.norm_rope(leaf[:, hq:hq + hk], wk, table, pos, 1e-6, False)[0]
    total = 0.0
    for s, (x0, e) in enumerate(((0, 200), (200, 333))):
        i = torch.arange(e - x0, device="cuda", dtype=torch.float64)
        ago = i[:, None] - i
        for h in range(hq):
            w = torch.where(ago >= 0, torch.exp(float(decay[h]) * ago.clamp(min=0)), 0.0) * d ** -0.5
            o = ((a[x0:e, h] @ b[x0:e, h // 2].T) * w) @ leaf[x0:e, hq + hk + h // 2]
            total = total + (o * dy.view(t, hq, d)[x0:e, h].double()).sum()
    grad, = torch.autograd.grad(total, leaf)
    assert float((drows.double() - grad).norm() / grad.norm()) < 5 * 2 ** -8
