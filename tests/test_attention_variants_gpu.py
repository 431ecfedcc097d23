"""The kernel variants that large calls run, against the 64-bit oracle.

Linear attention takes its scores in two parts in calls of no more chunks of 128 tokens than SMs and of up
to four tokens a sequence; the calls here have more, so that they run the variants for long work: outputs
alone, and outputs with exact states.  Each test asserts from the sizes, or from results that differ, which
variant it has.  Norm with rotation takes several heads at a time above 148 * 2048 * 4 threads.
Tolerances are those of the small cases (their derivation stands there)."""
import ctypes

import pytest
import torch

from cutedsl_pingpong_gemm_b200 import _lib, attention
from oracle import attention_ref as ref
from test_attention_gpu import gen, half, linear_case, normal, rope_case, within

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
WIDTHS = [(64, 64), (64, 128), (128, 64), (128, 128), (72, 40), (128, 24)]
RAGGED = [400, 0, 131, 257, 64]


def assert_long_and_uncut(lengths, h, dk, dv, backward=False):
    """By the sizes: more chunks than SMs, more than four tokens a sequence, no segments (the workspace
    has no room for states)."""
    t, b = sum(lengths), len(lengths)
    assert (t // 128 + b) * h > torch.cuda.get_device_properties(0).multi_processor_count
    assert t > 4 * b
    p = _lib.LinearProblemC(t, b, h, dk, dv, 1.0)
    size = ctypes.c_int64()
    _lib.check(_lib.load().cpg_linear_attention_workspace(ctypes.byref(p), h, h, h, int(backward),
                                                          ctypes.byref(size)))
    assert size.value < h * dk * dv * 4 + 64 * b


def check_out(out, want, tail=15):
    o, near, far = want[:3]
    within(out, o, 2 ** -8 * near + half(out.dtype) * o.abs() + 2 ** -tail * far, "out")


# ---------------------------------------------------------------------------- linear attention
@pytest.mark.parametrize("dk,dv", WIDTHS)
def test_outputs_of_whole_sequences(dk, dv):
    """Without states: every block walks several sequences, the longest first."""
    assert_long_and_uncut(RAGGED, 40, dk, dv)
    q, k, v, decay, offsets = linear_case(dk + dv, RAGGED, 40, 20, 8, 40, dk, dv, pad=3)
    out, _ = attention.linear_attention(q, k, v, decay, scale=dk ** -0.5, offsets=offsets)
    check_out(out, ref.whole_pass(q, k, v, decay, dk ** -0.5, offsets))
    # Short calls round less, so that some bits differ: this one is none.
    alone, _ = attention.linear_attention(q[:400, :2], k[:400, :1], v[:400, :1], decay[:2],
                                          scale=dk ** -0.5)
    assert not torch.equal(alone, out[:400, :2])


@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_outputs_and_states_of_whole_sequences(dk, dv, dtype):
    """From a pool of states and back into it."""
    assert_long_and_uncut(RAGGED, 40, dk, dv)
    q, k, v, decay, offsets = linear_case(dk - dv, RAGGED, 10, 40, 20, 40, dk, dv, layout="fused")
    pool = normal(gen(4), 7, 40, dk, dv, dtype=F32)
    slots = torch.tensor([6, 2, 0, 5, 3], dtype=torch.int32, device="cuda")
    states = [pool[i].clone() for i in slots.tolist()]
    want = ref.whole_pass(q, k, v, decay, -0.2, offsets, states)
    first = pool.clone()
    out = torch.empty(sum(RAGGED), 40, dv, dtype=dtype, device="cuda")
    attention.linear_attention(q, k, v, decay, scale=-0.2, offsets=offsets, state=pool, slots=slots,
                               final=pool, out=out)
    check_out(out, want)
    within(pool[slots.long()], want[3], 2 ** -17 * want[4], "final")
    assert torch.equal(pool[[1, 4]], first[[1, 4]]) and torch.equal(pool[2], first[2])
    # Without a starting state, and the same bits again.
    got = [attention.linear_attention(q, k, v, decay, scale=-0.2, offsets=offsets, final=True)
           for _ in range(2)]
    want = ref.whole_pass(q, k, v, decay, -0.2, offsets)
    check_out(got[0][0], want)
    within(got[0][1], want[3], 2 ** -17 * want[4], "final")
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    # A starting state alone asks for no exact ones.
    got, _ = attention.linear_attention(q, k, v, decay, scale=-0.2, offsets=offsets, state=first,
                                        slots=slots)
    check_out(got, ref.whole_pass(q, k, v, decay, -0.2, offsets, states))


@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("states", [False, True])
def test_gradients_of_whole_sequences(dk, dv, states):
    """Both orders of the tokens, with and without states that arrive and are handed out."""
    assert_long_and_uncut(RAGGED, 40, dk, dv, backward=True)
    q, k, v, decay, offsets = linear_case(dk * dv, RAGGED, 20, 40, 40, 40, dk, dv, pad=2, first=1)
    g = gen(9)
    dy = normal(g, q.shape[0], 40, dv)
    state, dfinal = (normal(g, 5, 40, dk, dv, dtype=F32) if states else None for _ in range(2))
    got = attention.linear_attention_backward(dy, q, k, v, decay, scale=0.3, offsets=offsets,
                                              state=state, dfinal=dfinal)
    grads, (ds, size) = ref.linear_attention_backward(
        dy, q, k, v, decay, 0.3, offsets, list(state) if states else None,
        list(dfinal) if states else None)
    for name, x, (want, near, far) in zip(("dq", "dk", "dv"), got, grads):
        within(x, want, 2 ** -8 * near + half(BF) * want.abs() + 2 ** -15 * far, name)
        assert not x[:1].any() and not x[1 + sum(RAGGED):].any()
    if states:
        within(got[3], ds, 2 ** -17 * size, "dstate")


@pytest.mark.parametrize("lengths,h,dk,dv", [([300], 150, 128, 128), ([6] * 2100, 1, 64, 64),
                                             ([7, 5] * 1100, 1, 128, 128)])
def test_whole_sequences_in_their_order(lengths, h, dk, dv):
    """One sequence of many heads, and more sequences than are sorted."""
    assert_long_and_uncut(lengths, h, dk, dv)
    q, k, v, decay, offsets = linear_case(5, lengths, h, h, h, h, dk, dv)
    want = ref.whole_pass(q, k, v, decay, 0.1, offsets)
    alone, _ = attention.linear_attention(q, k, v, decay, scale=0.1, offsets=offsets)
    check_out(alone, want)
    out, final = attention.linear_attention(q, k, v, decay, scale=0.1, offsets=offsets, final=True)
    check_out(out, want)
    within(final, want[3], 2 ** -17 * want[4], "final")


def test_bad_values_in_whole_sequences():
    """The channel of an infinity or a NaN in v is NaN from its token on and nothing else changes, where the
    tiles of v have one slot and where they have two."""
    q, k, v, decay, offsets = linear_case(4, [300] * 3, 100, 100, 100, 100, 128, 128)
    v = v.clone()
    bad = [(10, 3, 7), (140, 3, 7), (290, 3, 100), (300, 3, 64), (301, 50, 0), (899, 99, 127)]
    for t, h, c in bad:
        v[t, h, c] = float("inf") if t % 2 else float("nan")
    clean = torch.where(v.isfinite(), v, 0.0).bfloat16()
    for final in (None, True):
        want, wf = attention.linear_attention(q, k, clean, decay, offsets=offsets, final=final)
        got, gf = attention.linear_attention(q, k, v, decay, offsets=offsets, final=final)
        for t, h, c in bad:
            end = (t // 300 + 1) * 300
            want[t:end, h, c] = float("nan")
            if final:
                wf[t // 300, h, :, c] = float("nan")
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~got.isnan()], want[~want.isnan()])
        if final:
            assert torch.equal(gf.isnan(), wf.isnan())
            assert torch.equal(gf[~gf.isnan()], wf[~wf.isnan()])


@pytest.mark.parametrize("lengths,h,dk,dv,kind", [
    ([100], 2, 128, 128, "short"), ([300, 5, 129], 40, 128, 128, "whole"),
    ([300, 5, 129], 40, 64, 128, "whole"), ([300, 5, 129], 40, 128, 64, "whole"),
    ([9001], 1, 128, 128, "segments"), ([6000, 7001], 2, 64, 128, "segments")])
def test_states_are_exact(lengths, h, dk, dv, kind):
    """States that are handed out are off, in norm, by what FP32 sums of their terms are, not by more.

    The tensor cores cut off a sum's bits below its last every 16 tokens, on the average 0.36 * 2^-23 of it
    (half a step, of a mantissa spread evenly in its logarithm) = 4.3e-8.  With a decay of e^-0.02 a token,
    a cut 16 tokens ago counts e^-0.32, all of them 3.7 times one: 1.6e-7; FP32 decays and products add
    roundings of 2^-24 = 6e-8 that average out.  In one sum, the small parts would be cut 16 times more at
    the state's size: 6.9e-7 more; two parts alone would leave 2^-9 * 2^-9 * 0.72^2 / 3 = 6.6e-7 at
    least.  So the limit is 5e-7."""
    q, k, v, _, offsets = linear_case(8, lengths, h, h, h, h, dk, dv)
    decay = torch.full((h,), -0.02, device="cuda")
    if kind == "whole":
        assert_long_and_uncut(lengths, h, dk, dv)
    _, final = attention.linear_attention(q, k, v, decay, offsets=offsets, final=True)
    want = ref.whole_pass(q, k, v, decay, 1.0, offsets)[3]
    off = (final.double() - want).norm() / want.norm()
    dy = normal(gen(3), *v.shape)
    dstate = torch.empty(len(lengths), h, dk, dv, device="cuda")
    attention.linear_attention_backward(dy, q, k, v, decay, offsets=offsets, dstate=dstate)
    want = ref.whole_pass(k, q, dy, decay, 1.0, offsets, reverse=True)[3]
    back = (dstate.double() - want).norm() / want.norm()
    assert off <= 5e-7 and back <= 5e-7


# ------------------------------------------------------------------------- norm and rotation
MANY = [
    # t, hq, hk, d, rot, interleaved, dtype, layout, lanes a head
    (40001, 5, 3, 128, 128, False, BF, "fused", 8),
    (40000, 6, 2, 128, 64, True, BF, "plain", 8),
    (160001, 3, 2, 16, 16, False, BF, "plain", 4),
    (20001, 6, 3, 80, 40, True, F32, "plain", 16),
    (20000, 5, 3, 128, 64, False, F32, "fused", 16),
    (40001, 5, 2, 20, 20, False, BF, "plain", 8),
    (10000, 5, 3, 75, 30, False, BF, "plain", 32),
    (9001, 5, 3, 250, 250, False, BF, "odd", 32),
]


@pytest.mark.parametrize("t,hq,hk,d,rot,interleaved,dtype,layout,lanes", MANY)
def test_norm_rope_of_several_heads_at_a_time(t, hq, hk, d, rot, interleaved, dtype, layout, lanes):
    """Head counts that the groups of heads do not divide, with and without keys, in place too."""
    assert t * hq * lanes > 148 * 2048 * 4
    q, k, wq, wk, table, pos = rope_case(t + d, t, hq, hk, d, rot, dtype, layout)
    got = attention.norm_rope(q, k, wq, wk, table, pos, eps=1e-5, interleaved=interleaved)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        want, size = ref.norm_rope(x, w, table, pos, 1e-5, interleaved)
        within(y, want, half(dtype) * want.abs() + 2 ** -19 * size)
    alone, _ = attention.norm_rope(q, None, wq, None, table, pos, eps=1e-5, interleaved=interleaved)
    assert torch.equal(alone, got[0])
    attention.norm_rope(q, k, wq, wk, table, pos, eps=1e-5, interleaved=interleaved, out=(q, k))
    assert torch.equal(q, got[0]) and torch.equal(k, got[1])


@pytest.mark.parametrize("t,hq,hk,d,rot,interleaved,dtype,layout,lanes", MANY)
def test_norm_rope_backward_of_several_heads_at_a_time(t, hq, hk, d, rot, interleaved, dtype, layout,
                                                       lanes):
    assert t * hq * lanes > 148 * 2048 * 4
    q, k, wq, wk, table, pos = rope_case(t + d, t, hq, hk, d, rot, dtype, layout)
    g = gen(1)
    dq, dk = normal(g, t, hq, d, dtype=dtype), normal(g, t, hk, d, dtype=dtype)
    args = (q, k, wq, wk, table, pos)
    got = attention.norm_rope_backward(dq, dk, *args, eps=1e-5, interleaved=interleaved)
    for x, w, dy, dx, dw in ((q, wq, dq, got[0], got[2]), (k, wk, dk, got[1], got[3])):
        want, size, dwant, dsize = ref.norm_rope_backward(dy, x, w, table, pos, 1e-5, interleaved)
        within(dx, want, half(dtype) * want.abs() + 2 ** -18 * size, "dx")
        # A channel's sum: at most about 100 additions one after the other, of 2^-24 each.
        within(dw, dwant, 2 ** -17 * dsize, "dw")
    again = attention.norm_rope_backward(dq, dk, *args, eps=1e-5, interleaved=interleaved, out=(dq, dk))
    assert again[0] is dq and all(torch.equal(a, b) for a, b in zip(got, again))
