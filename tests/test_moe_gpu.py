"""Routing, dispatch and combine on the GPU, against plain 64-bit forms (oracle.moe_ref), alone and
as one MoE layer with INT8 experts.

Tolerances: FP32 weights and gradients are compared with the 64-bit formulas within a few tens of
fp32 half steps of the row's largest value (exp, division, k-term sums); whole numbers are equal.
"""
import math

import pytest
import torch

from cutedsl_pingpong_gemm_b200 import CpgError, GemmSM90, _lib
from cutedsl_pingpong_gemm_b200 import moe
from cutedsl_pingpong_gemm_b200.quant import quantize_int8
from oracle import moe_ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
# exp and the sigmoid are good to 2 ulp, a quotient to half an ulp, sums of up to 1024 positive
# terms by pairs or lanes to (32 + 5) half steps: below 64 half steps of the value altogether.
WEIGHT_REL = 64 * moe_ref.F32_HALF


def logits_of(t, e, dtype, seed, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(t, e, generator=g) * spread).to(dtype)


def check_route(lg, k, bias=None, **kw):
    ids, w = moe.route(lg.cuda(), k, bias=None if bias is None else bias.cuda(), **kw)
    torch.cuda.synchronize()
    rid, rw = moe_ref.route(lg, k, bias=bias, **kw)
    assert torch.equal(ids.cpu(), rid)
    nan = torch.isnan(rw)
    assert torch.equal(torch.isnan(w.cpu()), nan)
    err = (w.cpu().double() - rw).abs()
    assert (err[~nan] <= WEIGHT_REL * rw[~nan].abs() + 1e-37).all(), err[~nan].max()
    return ids, w


EXPERTS = [(1, 1), (2, 1), (8, 2), (31, 5), (33, 7), (64, 6), (100, 32), (128, 8), (256, 8),
           (384, 8), (512, 10), (1000, 3), (1024, 32)]


@pytest.mark.parametrize("e,k", EXPERTS)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_route(e, k, scoring, dtype):
    """BF16 logits of many experts hold equal ones: those go to the lowest index."""
    lg = logits_of(37, e, dtype, seed=e + k)
    for renorm in (True, False):
        check_route(lg, k, scoring=scoring, renormalize=renorm, scale=2.5)


@pytest.mark.parametrize("e,k,groups,kept", [(8, 2, 4, 2), (256, 8, 8, 4), (160, 6, 8, 3),
                                             (60, 4, 30, 7), (32, 3, 32, 5), (1024, 16, 16, 3),
                                             (96, 32, 3, 1), (40, 8, 2, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_route_groups_and_bias(e, k, groups, kept, scoring, dtype):
    lg = logits_of(33, e, dtype, seed=e * groups)
    g = torch.Generator().manual_seed(7)
    bias = torch.randn(e, generator=g) * (0.1 if scoring == "sigmoid" else 0.01)
    for b in (None, bias, torch.zeros(e)):
        for score in (None, "max", "top2"):
            check_route(lg, k, bias=b, scoring=scoring, groups=groups, kept_groups=kept,
                        group_score=score)


def test_route_near_ties():
    """Scores that 32 bits cannot tell apart: large logits under the sigmoid, biases one step apart,
    logits a few steps apart; ranked as their 64-bit values (or, with no bias, as the logits)."""
    e = 64
    g = torch.Generator().manual_seed(3)
    step = torch.arange(e).float()[torch.randperm(e, generator=g)]
    lg = torch.stack([20 + step * 0.25, 30 + step, 1 + step * 2.0 ** -23, 88 + step, -88 - step,
                      torch.full((e,), 3.0), 0.5 - step * 2.0 ** -24])
    for bias in (None, torch.zeros(e), torch.full((e,), 0.5), step.flip(0) * 2.0 ** -26,
                 1 + step.flip(0) * 2.0 ** -23):
        for scoring in ("softmax", "sigmoid"):
            check_route(lg, 9, bias=bias, scoring=scoring)
            check_route(lg, 9, bias=bias, scoring=scoring, groups=8, kept_groups=3,
                        group_score="top2")


@pytest.mark.parametrize("e", [8, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("level", [-23, -20, -18, -17, -16, -14])
def test_route_softmax_biases_that_cancel_the_scores(e, level):
    """Biases near the scores' negatives leave ranked values of 2^level of the largest score, about
    the 32-bit scores' error: still ranked as in 64 bits, alone and in groups."""
    g = torch.Generator().manual_seed(e - level)
    k = min(8, e)
    for spread in (0.1, 2.0):
        lg = torch.randn(1, e, generator=g) * spread
        p = lg.double().softmax(1)
        bias = (p.max() * 2.0 ** level * torch.randn(e, generator=g) - p[0]).float()
        check_route(lg.expand(5, e).contiguous(), k, bias=bias)
        for score in ("max", "top2"):
            check_route(lg, min(k, 4), bias=bias, groups=4, kept_groups=2, group_score=score)


def test_route_equal_scores_go_to_the_lowest_index():
    lg = torch.zeros(5, 96)
    ids, _ = check_route(lg, 7, scoring="sigmoid", bias=torch.zeros(96))
    assert (ids.cpu() == torch.arange(7)).all()
    ids, _ = check_route(lg, 7, groups=8, kept_groups=2, group_score="top2")
    assert (ids.cpu() == torch.arange(7)).all()


def test_route_small_sigmoid_scores():
    """Scores near and below the smallest normal number: shares keep their ratios, and so does their
    gradient."""
    lg = torch.tensor([[-59.0, -88.0, -95.0], [-16.0, -60.0, -60.5], [-17.5, -30.0, -62.0],
                       [-86.0, -89.0, -110.0], [-3.0, -40.0, -62.0], [-61.0, -87.5, -88.5],
                       [-200.0, -201.0, -230.0], [-45.0, -87.4, -88.6]])
    for dtype in DTYPES:
        x = lg.to(dtype)
        for renorm in (True, False):
            kw = dict(scoring="sigmoid", renormalize=renorm)
            ids, _ = check_route(x, 3, **kw)
            _, share = moe_ref.route(x, 3, **kw)
            for j in range(3):
                dw = torch.zeros(x.shape[0], 3)
                dw[:, j] = 1.0
                out = moe.route_backward(dw.cuda(), x.float().cuda(), ids, **kw).cpu().double()
                ref = moe_ref.route_backward(dw, x.float(), ids.cpu(), **kw)
                # Two shares multiply; the choice's own 1 - share is good to its share's error.
                size = ref.abs().scatter(1, ids.cpu().long()[:, j:j + 1], share[:, j:j + 1])
                assert ((out - ref).abs() <= 2 * WEIGHT_REL * size + 1e-37).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("with_bias", [True, False])
def test_route_masked_and_bad(scoring, renorm, with_bias):
    """Rows with masked experts, with all masked, with the type's lowest value, with infinities
    and NaN; biases of -inf and NaN."""
    inf = math.inf
    lg = logits_of(12, 40, torch.float32, seed=5)
    lg[0] = -inf
    lg[1, 3:] = -inf
    lg[2] = torch.finfo(torch.float32).min
    lg[3, 5] = math.nan
    lg[4, 6] = inf
    lg[5] = -1000.0
    lg[5, 9] = -1001.0
    lg[6] = -inf
    lg[6, 39] = 2.0
    lg[7, :] = math.nan
    lg[8] = torch.finfo(torch.float32).min
    lg[8, 7] = 0.0
    bias = None
    if with_bias:
        bias = torch.randn(40, generator=torch.Generator().manual_seed(2)) * 0.1
        bias[11] = -inf
        bias[12] = math.nan
        bias[13] = 5.0
    kw = dict(scoring=scoring, renormalize=renorm, bias=bias)
    check_route(lg, 4, **kw)
    check_route(lg, 4, groups=5, kept_groups=2, **kw)
    check_route(lg, 6, groups=5, kept_groups=2, group_score="top2", **kw)


def test_route_strides_outputs_and_sizes():
    """Row strides, unaligned rows, given outputs; one token and many; no token."""
    for t, e, off in [(1, 256, 0), (5, 64, 1), (4099, 16, 3), (0, 8, 0), (130, 130, 2)]:
        base = logits_of(t, e + 5, torch.float32, seed=t)
        view = base.cuda()[:, off:off + e]
        ids = torch.full((t, 3), -7, dtype=torch.int32, device="cuda")
        w = torch.full((t, 3), -7.0, device="cuda")
        a, b = moe.route(view, 3, ids=ids, weights=w)
        assert a is ids and b is w
        torch.cuda.synchronize()
        rid, rw = moe_ref.route(base[:, off:off + e], 3)
        assert torch.equal(ids.cpu(), rid)
        assert ((w.cpu().double() - rw).abs() <= WEIGHT_REL * rw).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups,kept", [(64, 8, 3), (40, 5, 2), (256, 8, 8)])
def test_route_biases_of_the_lowest_value(scoring, e, groups, kept):
    """Biases of the type's lowest value as masks: ranked last but not out, also where the sum of a
    group's two best passes the 32-bit range; infinite biases."""
    low = torch.finfo(torch.float32).min
    lg = logits_of(9, e, torch.float32, seed=e)
    for pattern in range(4):
        bias = torch.randn(e, generator=torch.Generator().manual_seed(pattern)) * 0.1
        if pattern == 0:
            bias[e // groups:] = low  # one group unmasked, the others wholly masked
        elif pattern == 1:
            bias[:] = low
        elif pattern == 2:
            bias[::2] = low
            bias[1] = -low
        else:
            bias[3] = math.inf
            bias[e // 2:] = -math.inf
        check_route(lg, 6, bias=bias, scoring=scoring)
        for score in ("max", "top2"):
            check_route(lg, 6, bias=bias, scoring=scoring, groups=groups, kept_groups=kept,
                        group_score=score)


@pytest.mark.parametrize("e", [128, 256])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_more_equal_candidates_than_lanes(e, scoring):
    """The last choice ties exactly with more experts than a warp has lanes, and behind those, past
    what 32 bits tell apart, stands the better one: a bias one step higher."""
    lg = torch.zeros(3, e)
    bias = torch.full((e,), 0.25)
    bias[e - 1] = 0.25 + 2.0 ** -25
    bias[e - 2] = 0.25 + 2.0 ** -26
    for k in (1, 8):
        check_route(lg, k, bias=bias, scoring=scoring)


@pytest.mark.parametrize("e,k", [(64, 8), (256, 32), (1000, 20)])
def test_route_many_equal_candidates(e, k):
    """More candidates near the last choice than lanes: a row of few distinct values."""
    g = torch.Generator().manual_seed(e)
    lg = torch.randint(0, 2, (17, e), generator=g).float()
    lg += torch.randint(0, 2, (17, e), generator=g) * 2.0 ** -23
    bias = torch.randint(0, 2, (e,), generator=g).float() * 2.0 ** -24
    for scoring in ("softmax", "sigmoid"):
        check_route(lg, k, scoring=scoring)
        check_route(lg, k, scoring=scoring, bias=bias)


# ---------------------------------------------------------------------------------- gradient
@pytest.mark.parametrize("e,k", [(1, 1), (8, 2), (33, 7), (100, 32), (128, 8), (256, 8), (512, 3),
                                 (1024, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_route_backward(e, k, scoring, renorm, dtype):
    t = 21
    lg = logits_of(t, e, dtype, seed=e - k)
    g = torch.Generator().manual_seed(k)
    lg[3] = -math.inf
    if e > 4:
        lg[4, 2:] = -math.inf
        lg[5, 1] = math.nan
    kw = dict(scoring=scoring, renormalize=renorm, scale=1.5)
    ids, _ = moe.route(lg.cuda(), k, scoring=scoring, renormalize=renorm)
    ids = ids.cpu()
    ids[6, 0] = -1
    if k > 1:
        ids[7, 1] = ids[7, 0]  # the same expert twice
        ids[8, 1] = e  # no expert
    dw = torch.randn(t, k, generator=g)
    out = moe.route_backward(dw.cuda(), lg.cuda(), ids.cuda(), **kw)
    torch.cuda.synchronize()
    ref = moe_ref.route_backward(dw, lg, ids, **kw)
    assert out.dtype == dtype
    got = out.cpu().double()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan)
    # Each entry: shares within WEIGHT_REL of sizes at most |g| summed over the choices.
    size = dw.abs().sum(1, keepdim=True).double() * 1.5
    half = moe_ref.BF16_HALF if dtype == torch.bfloat16 else 0.0
    tol = 2 * WEIGHT_REL * size + half * ref.abs() * 1.01
    assert ((got - ref).abs() <= tol)[~nan].all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_backward_against_differences(scoring, renorm):
    """The gradient of sum(g w) with the experts held, by central differences of the 64-bit weights
    (step h = 1e-5: a truncation of order h^2 and 64-bit rounding over h, below 1e-8)."""
    t, e, k, h = 3, 12, 4, 1e-5
    lg = logits_of(t, e, torch.float32, seed=9)
    ids, _ = moe.route(lg.cuda(), k, scoring=scoring, renormalize=renorm)
    g = torch.randn(t, k, generator=torch.Generator().manual_seed(1))
    out = moe.route_backward(g.cuda(), lg.cuda(), ids, scoring=scoring,
                             renormalize=renorm).cpu().double()
    at = ids.cpu().long()

    def loss(x):
        s = x.softmax(1) if scoring == "softmax" else x.sigmoid()
        w = s.gather(1, at)
        if renorm:
            w = w / w.sum(1, keepdim=True)
        return (w * g.double()).sum(1)

    for i in range(e):
        d = torch.zeros(t, e, dtype=torch.float64)
        d[:, i] = h
        diff = (loss(lg.double() + d) - loss(lg.double() - d)) / (2 * h)
        tol = 1e-8 + 2 * WEIGHT_REL * g.abs().sum(1).double()
        assert ((out[:, i] - diff).abs() <= tol).all(), i


# ---------------------------------------------------------------------------------- dispatch
def ids_of(t, k, e, seed, skip=0.1):
    g = torch.Generator().manual_seed(seed)
    pop = torch.rand(e, generator=g) + 0.05
    ids = torch.multinomial(pop.expand(max(t, 1), e), k, replacement=k > e,
                            generator=g)[:t].to(torch.int32)
    ids[torch.rand(t, k, generator=g) < skip] = -1
    return ids


@pytest.mark.parametrize("t,k,e", [(0, 2, 4), (1, 1, 1), (1, 8, 256), (16, 2, 8), (33, 3, 5),
                                   (100, 32, 40), (700, 8, 1024), (2049, 6, 64), (20000, 8, 256)])
def test_dispatch_order(t, k, e):
    ids = ids_of(t, k, e, seed=t + e)
    if t > 20:
        ids[5, 0] = e  # no expert
        ids[6, 0] = -2 ** 31
        ids[7] = ids[7, 0]  # the same expert several times
    x = torch.randn(t, 8, device="cuda").bfloat16()
    d = moe.dispatch(x, ids.cuda(), e)
    torch.cuda.synchronize()
    off, slots = moe_ref.expert_order(ids, e)
    assert torch.equal(d.offsets.cpu(), off) and torch.equal(d.slots.cpu(), slots)
    here = slots >= 0
    token = torch.arange(t)[:, None].expand(t, k)[here]
    assert torch.equal(d.rows.cpu()[slots[here].long()], x.cpu()[token])


def expected_order(ids, e):
    """Offsets and slots by a stable sort of the pairs by expert."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < e), flat, torch.full_like(flat, e))
    order = key.argsort(stable=True)
    off = torch.zeros(e + 1, dtype=torch.int64)
    off[1:] = torch.bincount(key, minlength=e + 1)[:e].cumsum(0)
    slots = torch.full_like(flat, -1)
    used = int(off[-1])
    slots[order[:used]] = torch.arange(used)
    return off.int(), slots.reshape(ids.shape).int()


# A cluster of 16 blocks (8 where 16 do not fit) holds 512 pairs of each of its warps; with more
# every warp walks its run twice.
@pytest.mark.parametrize("pairs", [131071, 131073, 262143, 262144, 262145, 300000, 1000003])
@pytest.mark.parametrize("e", [3, 16, 17, 64, 65, 256, 257, 1024])
def test_dispatch_order_of_many_pairs(pairs, e):
    g = torch.Generator().manual_seed(pairs + e)
    ids = torch.randint(-1, e, (pairs, 1), generator=g, dtype=torch.int32)
    ids[::3] = ids[::3].clamp(max=e // 4)  # some experts more often than others
    ids[100] = e  # no expert
    ids[5000:5040] = ids[5000]
    ids[pairs // 2:pairs // 2 + 3000] = -1
    x = torch.zeros(pairs, 1, device="cuda")
    d = moe.dispatch(x, ids.cuda(), e)
    torch.cuda.synchronize()
    off, slots = expected_order(ids, e)
    assert torch.equal(d.offsets.cpu(), off) and torch.equal(d.slots.cpu(), slots)


def test_dispatch_order_of_equal_choices():
    """528000 pairs: token t goes to expert 7 - t % 8 with each of its 8 choices."""
    t, k, e = 66000, 8, 8
    tok = torch.arange(t)
    d = moe.dispatch(torch.zeros(t, 1, device="cuda"),
                     (7 - tok % 8)[:, None].expand(t, k).int().contiguous().cuda(), e)
    torch.cuda.synchronize()
    assert torch.equal(d.offsets.cpu(), torch.arange(e + 1, dtype=torch.int32) * (t * k // e))
    first = (7 - tok % 8) * (t * k // e) + tok // 8 * k
    assert torch.equal(d.slots.cpu(), (first[:, None] + torch.arange(k)).int())


@pytest.mark.parametrize("cols", [1, 7, 64, 100, 1032, 4096, 5000, 16392, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("int8", [False, True])
def test_dispatch_rows(cols, dtype, int8):
    """Rows of many lengths; rows that no token goes to are left as they were."""
    t, k, e = 19, 3, 6
    ids = ids_of(t, k, e, seed=cols)
    x = torch.randn(t, cols, generator=torch.Generator().manual_seed(cols)).to(dtype)
    x[4] = 0
    out = torch.full((t * k, cols), 77, dtype=torch.int8 if int8 else dtype, device="cuda")
    scales = torch.full((t * k,), 77.0, device="cuda") if int8 else None
    d = moe.dispatch(x.cuda(), ids.cuda(), e, quantize="int8" if int8 else None, out=out,
                     scales=scales)
    torch.cuda.synchronize()
    assert d.rows is out
    off, slots = moe_ref.expert_order(ids, e)
    want = torch.full((t * k, cols), 77, dtype=out.dtype)
    wants = torch.full((t * k,), 77.0)
    q, s = moe_ref.quantize_int8(x) if int8 else (x, None)
    for i in range(t):
        for j in range(k):
            if slots[i, j] >= 0:
                want[slots[i, j]] = q[i]
                if int8:
                    wants[slots[i, j]] = s[i]
    assert torch.equal(out.cpu(), want)
    assert not int8 or torch.equal(scales.cpu(), wants)


@pytest.mark.parametrize("shift,extra", [(1, 2), (4, 4), (3, 0)])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dispatch_combine_strided_views(shift, extra, int8, dtype):
    t, k, e, cols = 23, 2, 4, 260
    ids = ids_of(t, k, e, seed=3, skip=0.0)
    base = torch.randn(t, cols + shift + extra, generator=torch.Generator().manual_seed(4)).to(dtype)
    x = base.cuda()[:, shift:shift + cols]
    buf = torch.zeros(t * k, cols + 2 * shift + 5, dtype=torch.int8 if int8 else dtype,
                      device="cuda")
    d = moe.dispatch(x, ids.cuda(), e, quantize="int8" if int8 else None,
                     out=buf[:, shift:shift + cols])
    _, slots = moe_ref.expert_order(ids, e)
    flat = slots.reshape(-1).long()
    src = base[:, shift:shift + cols].repeat_interleave(k, 0)
    if int8:
        q, s = moe_ref.quantize_int8(src)
        assert torch.equal(d.rows.cpu()[flat], q) and torch.equal(d.scales.cpu()[flat], s)
        return
    assert torch.equal(d.rows.cpu()[flat], src)
    assert (buf[:, :shift] == 0).all() and (buf[:, shift + cols:] == 0).all()
    w = torch.rand(t, k, generator=torch.Generator().manual_seed(5))
    ybuf = torch.full((t, cols + 9), 5.0, dtype=dtype, device="cuda")
    y = moe.combine(d.rows, d.slots, w.cuda(), source=x, out=ybuf[:, 1:1 + cols])
    torch.cuda.synchronize()
    ref, slack = moe_ref.combine(d.rows.cpu(), slots, w, x.cpu())
    assert moe_ref.within(y, ref, slack) <= 0
    assert (ybuf[:, 0] == 5).all() and (ybuf[:, 1 + cols:] == 5).all()


@pytest.mark.parametrize("d", [8, 100, 129])
@pytest.mark.parametrize("t", [1, 50])
def test_dispatched_rows_are_operands(d, t):
    """The rows that dispatch allocates go into the grouped product at every width, BF16 and INT8."""
    e, k, n = 4, 2, 72
    g = torch.Generator().manual_seed(d)
    x = torch.randn(t, d, generator=g).bfloat16()
    ids = ids_of(t, k, e, seed=d, skip=0.0)
    per = -(-d // 8) * 8
    b = torch.zeros(e, n, per, dtype=torch.bfloat16)
    b[..., :d] = (torch.randn(e, n, d, generator=g) * d ** -0.5).bfloat16()
    gemm = GemmSM90(tile_shape_mn=(128, 128), epi_tile_mn=(128, 32), cluster_shape_mnk=(1, 1, 1),
                    atom_layout_mn=(1, 1), ab_stage=3, reuse_ab=False, is_persistent=True)
    p = moe.dispatch(x.cuda(), ids.cuda(), e)
    y = torch.zeros(t * k, n, dtype=torch.bfloat16, device="cuda")
    gemm.grouped(p.rows, b.cuda()[..., :d], y, p.offsets)
    torch.cuda.synchronize()
    off, slots = moe_ref.expert_order(ids, e)
    for i in range(t):
        for j in range(k):
            ref = x[i].double() @ b[ids[i, j], :, :d].double().t()
            mag = x[i].double().abs() @ b[ids[i, j], :, :d].double().abs().t()
            # d products exact in fp32, at most d sums of it, one rounding to BF16.
            slack = d * moe_ref.F32_HALF * 2 * mag
            assert moe_ref.within(y[slots[i, j]], ref, slack) <= 0
    q = moe.dispatch(x.cuda(), ids.cuda(), e, quantize="int8")
    bq = torch.randint(-127, 128, (e, n, -(-d // 16) * 16), generator=g, dtype=torch.int8)
    gemm.grouped(q.rows, bq.cuda()[..., :d], y, q.offsets, scale_a=q.scales)
    torch.cuda.synchronize()
    for i in range(e):
        r = slice(int(off[i]), int(off[i + 1]))
        ref, slack = moe_ref.int8_product(q.rows[r].cpu(), bq[i, :, :d], q.scales[r].cpu())
        assert moe_ref.within(y[r], ref, slack) <= 0


@pytest.mark.parametrize("int8", [False, True])
def test_dispatch_into_given_outputs(int8):
    """With every output given, dispatch allocates nothing and returns them."""
    t, k, e, d = 30, 3, 8, 64
    ids = ids_of(t, k, e, seed=2)
    x = torch.randn(t, d, device="cuda").bfloat16()
    out = torch.zeros(t * k, d, dtype=torch.int8 if int8 else x.dtype, device="cuda")
    scales = torch.zeros(t * k, device="cuda") if int8 else None
    offsets = torch.full((e + 1,), -7, dtype=torch.int32, device="cuda")
    slots = torch.full((t, k), -7, dtype=torch.int32, device="cuda")
    on = ids.cuda()
    kw = dict(quantize="int8" if int8 else None, out=out, scales=scales, offsets=offsets,
              slots=slots)
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    p = moe.dispatch(x, on, e, **kw)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    torch.cuda.synchronize()
    assert p.rows is out and p.offsets is offsets and p.slots is slots and p.scales is scales
    off, want = moe_ref.expert_order(ids, e)
    assert torch.equal(offsets.cpu(), off) and torch.equal(slots.cpu(), want)
    again = moe.dispatch(x, on, e, quantize=kw["quantize"])
    used = int(off[-1])
    assert torch.equal(again.rows[:used], out[:used])
    for bad in (dict(offsets=offsets[:-1]), dict(offsets=offsets.long()), dict(slots=slots[:-1]),
                dict(slots=slots.t()), dict(slots=slots.cpu()), dict(offsets=offsets.cpu())):
        with pytest.raises(CpgError) as err:
            moe.dispatch(x, on, e, **bad)
        assert err.value.code == _lib.CPG_ERR_INVALID_SHAPE


# ----------------------------------------------------------------------------------- combine
COMBINE = [(1, 1, 1), (1, 8, 4096), (16, 2, 4096), (37, 5, 100), (64, 32, 24), (300, 8, 1032),
           (9, 3, 16385), (0, 2, 64)]


@pytest.mark.parametrize("t,k,cols", COMBINE)
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine(t, k, cols, dtype):
    e = 2 * k
    g = torch.Generator().manual_seed(t + k)
    ids = ids_of(t, k, e, seed=t * k)
    if t > 2:
        ids[2] = -1  # a token without experts
    _, slots = moe_ref.expert_order(ids, e)
    rows = torch.randn(t * k, cols, generator=g).to(dtype)
    used = slots[slots >= 0].long()
    rows[[i for i in range(t * k) if i not in set(used.tolist())]] = math.nan  # never read
    if t > 3:
        slots[3, 0] = t * k  # no row
    w = torch.rand(t, k, generator=g)
    src = torch.randn(t, cols, generator=g).to(dtype)
    for weights, source in ((w, None), (None, None), (w, src)):
        y = moe.combine(rows.cuda(), slots.cuda(), None if weights is None else weights.cuda(),
                        source=None if source is None else source.cuda())
        torch.cuda.synchronize()
        ref, slack = moe_ref.combine(rows, slots, weights, source)
        assert moe_ref.within(y, ref, slack) <= 0
    y = src.cuda()
    moe.combine(rows.cuda(), slots.cuda(), w.cuda(), source=y, out=y)  # in place
    torch.cuda.synchronize()
    ref, slack = moe_ref.combine(rows, slots, w, src)
    assert moe_ref.within(y, ref, slack) <= 0


@pytest.mark.parametrize("cols", [1, 2, 31, 63, 130, 258, 515, 1029, 2051])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_every_alignment(cols, dtype):
    """Copies, weighted sums and row gradients are the same bits whatever the rows' alignment (the
    sums of each element go in the order of the choices); what lies beyond a row stays."""
    t, k, e = 37, 5, 6
    g = torch.Generator().manual_seed(cols)
    ids = ids_of(t, k, e, seed=cols)
    w = torch.randn(t, k, generator=g).cuda()
    x0 = torch.randn(t, cols, generator=g).to(dtype)
    src0 = torch.randn(t, cols, generator=g).to(dtype)
    results = []
    for step in (16, 8, 4, 2):  # bytes the rows' addresses are multiples of
        unit = max(step // x0.element_size(), 1)
        ld = -(-(cols + 1) // unit) * unit
        if (ld // unit) % 2 == 0 and unit * x0.element_size() < 16:
            ld += unit  # and of no more

        def view(rows, fill=7.0):
            buf = torch.full((rows * ld + unit,), fill, dtype=dtype, device="cuda")
            v = buf[unit if unit * x0.element_size() < 16 else 0:][:rows * ld].view(rows, ld)
            return v, v[:, :cols]
        _, x = view(t)
        _, src = view(t)
        x.copy_(x0)
        src.copy_(src0)
        rows_all, rows = view(t * k)
        y_all, y = view(t)
        dr_all, dr = view(t * k)
        d = moe.dispatch(x, ids.cuda(), e, out=rows)
        moe.combine(rows, d.slots, w, source=src, out=y)
        _, dw = moe.combine_backward(x, rows, d.slots, w, drows=dr)
        torch.cuda.synchronize()
        for whole in (rows_all, y_all, dr_all):
            assert (whole[:, cols:] == 7).all()
        used = int(d.offsets[-1])
        assert (rows[used:] == 7).all() and (dr[used:] == 7).all()
        results.append((rows.clone(), y.clone(), dr.clone(), dw))
    for got in results[1:]:
        for a, b in zip(got[:3], results[0][:3]):
            assert torch.equal(a, b)
    ref, slack = moe_ref.combine(results[0][0].cpu(), d.slots.cpu(), w.cpu(), source=src0)
    assert moe_ref.within(results[0][1], ref, slack) <= 0
    # Each product of a dot product is rounded to at most half a step and so are its cols - 1 sums.
    rows64 = results[0][0].double().cpu()
    slot = d.slots.cpu().long()
    real = (slot >= 0)[..., None]
    prod = x0.double()[:, None, :] * rows64[slot.clamp(min=0)] * real
    bound = (cols + 1) * moe_ref.F32_HALF * prod.abs().sum(-1) * 1.01 + 1e-37
    for got in results:
        assert ((got[3].cpu().double() - prod.sum(-1)).abs() <= bound).all()


def launched_kernels(f):
    """Names of the kernels that f launches, from the graph of a captured call."""
    from cuda.bindings import driver

    def ok(result):
        assert result[0] == driver.CUresult.CUDA_SUCCESS, result
        return result[1]
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        f()
    names = []
    count = driver.cuGraphGetNodes(graph.raw_cuda_graph(), 0)[2]
    for node in ok(driver.cuGraphGetNodes(graph.raw_cuda_graph(), count)):
        if ok(driver.cuGraphNodeGetType(node)) == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            params = ok(driver.cuGraphKernelNodeGetParams(node))
            names.append(ok(driver.cuFuncGetName(params.func) if int(params.func)
                            else driver.cuKernelGetName(params.kern)).decode())
    return " ".join(names)


@pytest.mark.parametrize("cols", [4097, 260, 17])
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_is_read_as_its_memory_is_aligned(cols, dtype):
    """The row stride of one row is not used: a 16-byte aligned row takes the kernels of 16-byte
    accesses whatever its length, with the same bits."""
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(1, cols, generator=g).to(dtype).cuda()
    name = "13__nv_bfloat16" if dtype == torch.bfloat16 else "f"
    got = {}

    def quantise():
        got["q"] = quantize_int8(x)
    text = launched_kernels(quantise)
    assert f"rows_int8_vec_kernelI{name}Li16E" in text
    rq, rs = moe_ref.quantize_int8(x.cpu())
    quantise()
    assert torch.equal(got["q"][0].cpu(), rq) and torch.equal(got["q"][1].cpu(), rs)

    ids = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    w = torch.full((1, 1), 0.5, device="cuda")

    def chain():
        p = moe.dispatch(x, ids, 1)
        y = moe.combine(p.rows, p.slots, w, source=x)
        got["c"] = (p.rows, y, *moe.combine_backward(x, p.rows, p.slots, w))
    text = launched_kernels(chain)
    for kernel in ("rows_copy_kernel", "combine_kernel", "combine_grad_kernel"):
        assert f"{kernel}I{name}Li16E" in text, kernel
    chain()
    rows, y, drows, _ = got["c"]
    assert torch.equal(rows, x) and torch.equal(drows, (x.float() * 0.5).to(dtype))
    assert torch.equal(y, (x.float() * 1.5).to(dtype))

    q = torch.zeros(1, cols, dtype=torch.int8, device="cuda")
    text = launched_kernels(lambda: moe.dispatch(x, ids, 1, quantize="int8", out=q))
    assert f"rows_int8_vec_kernelI{name}Li16E" in text
    torch.cuda.synchronize()
    assert torch.equal(q.cpu(), rq)


@pytest.mark.parametrize("cols", [4096, 4097])
def test_rows_past_32_bit_offsets(cols):
    """Rows whose element offsets pass 2^31: token t goes to expert 7 - t % 8 with every choice, so
    the last rows are those of expert 7."""
    t, k, e = 66000, 8, 8
    assert t * k * cols > 2 ** 31
    tok = torch.arange(t, device="cuda")
    ids = ((7 - tok % 8)[:, None] + torch.zeros(k, dtype=torch.int64, device="cuda")).int()
    x = (tok % 251 - 125).to(torch.bfloat16)[:, None].expand(t, cols).contiguous()
    w = torch.full((t, k), 0.5, device="cuda")
    d = moe.dispatch(x, ids, e)
    q = moe.dispatch(x, ids, e, quantize="int8")
    torch.cuda.synchronize()
    assert torch.equal(q.slots, d.slots)
    of_row = torch.empty(t * k, dtype=torch.int64, device="cuda")
    of_row[d.slots.long().flatten()] = tok.repeat_interleave(k)
    for lo in range(0, t * k, 66000):
        want = x[of_row[lo:lo + 66000], :1]
        assert (d.rows[lo:lo + 66000] == want).all()
        assert (q.rows[lo:lo + 66000] == (127 * want.sign()).to(torch.int8)).all()
    del q
    # 8 halves of a whole number below 2^7: exact.
    assert torch.equal(moe.combine(d.rows, d.slots, w), 4 * x)
    drows, dw = moe.combine_backward(x, d.rows, d.slots, w, drows=d.rows.clone())
    torch.cuda.synchronize()
    for lo in range(0, t * k, 66000):
        assert (drows[lo:lo + 66000] == 0.5 * x[of_row[lo:lo + 66000], :1]).all()
    # cols squares below 2^14: their sums are whole numbers below 2^27, rounded where above 2^24.
    want = cols * x[:, 0].double() ** 2
    assert ((dw.double() - want[:, None]).abs() <= cols * moe_ref.F32_HALF * want[:, None]).all()


def test_combine_infinite_rows():
    """An infinity or NaN in a chosen row reaches its token and no other."""
    t, k, cols = 6, 2, 64
    slots = torch.arange(t * k, dtype=torch.int32).reshape(t, k)
    rows = torch.randn(t * k, cols, generator=torch.Generator().manual_seed(2))
    rows[3, 5] = math.inf
    rows[6, 7] = math.nan
    y = moe.combine(rows.cuda(), slots.cuda(), torch.full((t, k), 0.5, device="cuda")).cpu()
    bad = torch.zeros(t, cols, dtype=torch.bool)
    bad[1, 5] = bad[3, 7] = True
    assert torch.equal(torch.isfinite(y), ~bad)


@pytest.mark.parametrize("t,k,cols", COMBINE)
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine_backward(t, k, cols, dtype):
    e = 2 * k
    g = torch.Generator().manual_seed(t + k)
    ids = ids_of(t, k, e, seed=t * k)
    _, slots = moe_ref.expert_order(ids, e)
    if t > 3:
        slots[3, 0] = t * k
    rows = torch.randn(t * k, cols, generator=g).to(dtype)
    dy = torch.randn(t, cols, generator=g).to(dtype)
    w = torch.rand(t, k, generator=g)
    drows = torch.full((t * k, cols), math.nan, dtype=dtype, device="cuda")
    got, dw = moe.combine_backward(dy.cuda(), rows.cuda(), slots.cuda(), w.cuda(), drows=drows)
    torch.cuda.synchronize()
    assert got is drows
    rd, rw, slack = moe_ref.combine_backward(dy, rows, slots, w)
    assert moe_ref.within(drows, rd, moe_ref.F32_HALF * rd.abs()) <= 0
    assert ((dw.cpu().double() - rw).abs() <= slack + 1e-37).all()


@pytest.mark.parametrize("cols", [1, 64, 1031])
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine_backward_of_unused_rows(cols, dtype):
    """A row that enters no sum has the gradient 0 where the function makes the tensor, whatever its
    memory held before."""
    t, k, e = 40, 4, 6
    ids = ids_of(t, k, e, seed=cols, skip=0.4)
    ids[-3:] = -1
    _, slots = moe_ref.expert_order(ids, e)
    slots[0, 0] = t * k  # no row
    g = torch.Generator().manual_seed(cols)
    rows = torch.randn(t * k, cols, generator=g).to(dtype)
    dy = torch.randn(t, cols, generator=g).to(dtype)
    w = torch.rand(t, k, generator=g)
    args = dy.cuda(), rows.cuda(), slots.cuda(), w.cuda()
    stale = torch.full((t * k, cols), math.nan, dtype=dtype, device="cuda")
    del stale  # the allocator hands out its memory again
    drows, _ = moe.combine_backward(*args)
    torch.cuda.synchronize()
    ref, _, _ = moe_ref.combine_backward(dy, rows, slots, w)
    unused = torch.isnan(ref).all(1)
    assert unused.sum() > 10
    assert (drows.cpu()[unused] == 0).all()
    ref = ref.masked_fill(unused[:, None], 0.0)
    assert moe_ref.within(drows, ref, moe_ref.F32_HALF * ref.abs()) <= 0


@pytest.mark.parametrize("t,k,r,cols", [(0, 2, 5, 9), (1, 1, 1, 3), (3, 2, 20000, 130), (3, 32, 31, 8),
                                        (5, 1, 300001, 2), (20000, 8, 160000, 6),
                                        (9, 4, 4737, 1030)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_combine_backward_clears_what_no_slot_names(t, k, r, cols, dtype):
    """Any number of rows, more or fewer than pairs, and slots anywhere among them."""
    g = torch.Generator().manual_seed(r)
    slots = torch.randperm(max(r, t * k), generator=g)[:t * k].reshape(t, k).int()
    slots[torch.rand(t, k, generator=g) < 0.3] = -1
    if t:
        slots[0, 0] = 2 ** 31 - 1
    dy = torch.randn(t, cols, generator=g).to(dtype).cuda()
    w = torch.rand(t, k, generator=g).cuda()
    rows = torch.zeros(r, cols, dtype=dtype, device="cuda")
    stale = torch.full((r, cols), math.nan, dtype=dtype, device="cuda")
    del stale
    drows, _ = moe.combine_backward(dy, rows, slots.cuda(), w)
    torch.cuda.synchronize()
    want = torch.zeros(r, cols, dtype=dtype, device="cuda")
    on = slots.cuda().long()
    token, choice = ((on >= 0) & (on < r)).nonzero(as_tuple=True)
    want[on[token, choice]] = (w[token, choice, None] * dy[token].float()).to(dtype)
    assert torch.equal(drows, want)


def test_gradients_against_differences():
    """combine's gradients and dispatch's (a combine without weights) against central differences;
    both are linear, so with h = 1 the difference is exact up to fp32 rounding."""
    t, k, e, cols = 7, 3, 5, 40
    g = torch.Generator().manual_seed(8)
    ids = ids_of(t, k, e, seed=1)
    x = torch.randn(t, cols, generator=g)
    w = torch.rand(t, k, generator=g)
    d = moe.dispatch(x.cuda(), ids.cuda(), e, out=torch.zeros(t * k, cols, device="cuda"))
    gy = torch.randn(t, cols, generator=g)
    gr = torch.randn(t * k, cols, generator=g).cuda()
    dx = moe.combine(gr, d.slots).cpu().double()
    drows, dw = moe.combine_backward(gy.cuda(), d.rows, d.slots, w.cuda(),
                                     drows=torch.zeros(t * k, cols, device="cuda"))
    used = (d.slots >= 0).cpu()
    for i, j in [(0, 0), (3, 2), (6, 1)]:
        step = torch.zeros(t, cols)
        step[i, j] = 1.0

        def rows_of(v):
            return moe.dispatch(v.cuda(), ids.cuda(), e,
                                out=torch.zeros(t * k, cols, device="cuda")).rows
        diff = ((rows_of(x + step) - rows_of(x - step)).double() * gr.double()).sum() / 2
        assert abs(diff.item() - dx[i, j].item()) <= 1e-5 * max(1.0, abs(dx[i, j].item()))
        if used[i, j]:
            dwt = torch.zeros(t, k)
            dwt[i, j] = 1.0
            up = moe.combine(d.rows, d.slots, (w + dwt).cuda()).cpu().double()
            dn = moe.combine(d.rows, d.slots, (w - dwt).cuda()).cpu().double()
            diff = ((up - dn) * gy.double()).sum() / 2
            tol = 1e-5 * (gy.double().abs() * up.abs()).sum().item()
            assert abs(diff.item() - dw[i, j].item()) <= tol
            r = int(d.slots[i, j])
            bump = torch.zeros(t * k, cols, device="cuda")
            bump[r, 4] = 1.0
            up = moe.combine(d.rows + bump, d.slots, w.cuda()).cpu().double()
            dn = moe.combine(d.rows - bump, d.slots, w.cuda()).cpu().double()
            diff = ((up - dn) * gy.double()).sum() / 2
            assert abs(diff.item() - drows[r, 4].item()) <= 1e-5 * (1 + abs(drows[r, 4].item()))


# -------------------------------------------------------------------- streams, graphs, a layer
def test_streams_and_graph_replay():
    """The whole chain on a side stream, captured, and replayed on new inputs; two captured graphs
    that run at the same time do not share anything."""
    t, e, k, d = 300, 16, 4, 256
    graphs = []
    side = torch.cuda.Stream()
    for i in range(2):
        lg = torch.randn(t, e, device="cuda")
        x = torch.randn(t, d, device="cuda").bfloat16()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warm-up on another stream than the tensors'
            ids, w = moe.route(lg, k)
            moe.combine(moe.dispatch(x, ids, e).rows, moe.dispatch(x, ids, e).slots, w)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ids, w = moe.route(lg, k)
            p = moe.dispatch(x, ids, e)
            y = moe.combine(p.rows, p.slots, w)
            gr, gw = moe.combine_backward(y, p.rows, p.slots, w)
            gl = moe.route_backward(gw, lg, ids)
        graphs.append((graph, lg, x, ids, w, y, gw, gl))
    for graph, lg, x, *_ in graphs:
        lg.normal_()
        x.normal_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for (graph, *_), s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for _, lg, x, ids, w, y, gw, gl in graphs:
        rid, _ = moe_ref.route(lg.cpu(), k)
        assert torch.equal(ids.cpu(), rid)
        # Weights that sum to one over copies of one row give the row back.
        assert (y.float() - x.float()).abs().max() <= 2 ** -7 * x.float().abs().max()
        ref = moe_ref.route_backward(gw.cpu(), lg.cpu(), ids.cpu())
        assert ((gl.cpu().double() - ref).abs()
                <= 2 * WEIGHT_REL * gw.cpu().double().abs().sum(1, keepdim=True)).all()


@pytest.mark.parametrize("t", [1, 5, 700])
def test_moe_layer_int8(t):
    """route -> dispatch (int8) -> grouped gated product -> quantise -> grouped product -> combine,
    with some padded tokens, against the same steps in 64 bits from the kernel's own int8 rows."""
    e, k, d, f = 8, 2, 256, 320
    g = torch.Generator().manual_seed(t)
    x = torch.randn(t, d, generator=g).bfloat16()
    lg = torch.randn(t, e, generator=g)
    if t > 2:
        lg[-2:] = -math.inf
    wu, su = quantize_int8((torch.randn(e * 2 * f, d, generator=g) * d ** -0.5).cuda())
    wd, sd = quantize_int8((torch.randn(e * d, f, generator=g) * f ** -0.5).cuda())
    wu, su = wu.view(e, 2 * f, d), su.view(e, 2 * f)
    wd, sd = wd.view(e, d, f), sd.view(e, d)

    def gemm(n):
        return GemmSM90(tile_shape_mn=(128, n), epi_tile_mn=(128, 32), cluster_shape_mnk=(2, 1, 1),
                        atom_layout_mn=(1, 1), ab_stage=3, reuse_ab=False, is_persistent=True)
    ids, w = moe.route(lg.cuda(), k, scoring="sigmoid")
    p = moe.dispatch(x.cuda(), ids, e, quantize="int8",
                     out=torch.zeros(t * k, d, dtype=torch.int8, device="cuda"),
                     scales=torch.zeros(t * k, device="cuda"))
    h = torch.zeros(t * k, f, dtype=torch.bfloat16, device="cuda")
    gemm(512).grouped(p.rows, wu, h, p.offsets, scale_a=p.scales, scale_b=su, activation="silu",
                      gated=True)
    hq, hs = quantize_int8(h)
    o = torch.zeros(t * k, d, dtype=torch.bfloat16, device="cuda")
    gemm(256).grouped(hq, wd, o, p.offsets, scale_a=hs, scale_b=sd)
    y = moe.combine(o, p.slots, w)
    torch.cuda.synchronize()
    off = p.offsets.cpu().tolist()
    assert off[-1] == (t - 2 if t > 2 else t) * k
    for i in range(e):
        r = slice(off[i], off[i + 1])
        ref, slack = moe_ref.int8_product(p.rows[r].cpu(), wu[i].cpu(), p.scales[r].cpu(),
                                          su[i].cpu(), activation="silu", gated=True)
        assert moe_ref.within(h[r], ref, slack) <= 0
        ref, slack = moe_ref.int8_product(hq[r].cpu(), wd[i].cpu(), hs[r].cpu(), sd[i].cpu())
        assert moe_ref.within(o[r], ref, slack) <= 0
    ref, slack = moe_ref.combine(o.cpu(), p.slots.cpu(), w.cpu())
    assert moe_ref.within(y, ref, slack) <= 0
    if t > 2:
        assert (y[-2:] == 0).all()
    # And near the layer in full precision: the int8 steps are within half a step of 127 each, so
    # a relative error of about 1e-2 of the output's norm; 5e-2 leaves a factor of five.
    full = torch.zeros(t, d, dtype=torch.float64)
    wuf = wu.cpu().double() * su.cpu().double()[..., None]
    wdf = wd.cpu().double() * sd.cpu().double()[..., None]
    for i in range(t):
        for j in range(k):
            ex = int(ids[i, j])
            if ex >= 0:
                gu = wuf[ex] @ x[i].double()
                full[i] += float(w[i, j]) * (wdf[ex] @ (moe_ref.act("silu", gu[:f]) * gu[f:]))
    assert (y.cpu().double() - full).norm() <= 5e-2 * full.norm()


def test_refusals():
    lg = torch.randn(4, 8, device="cuda")
    x = torch.randn(4, 16, device="cuda")
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, 2, device="cuda")
    rows = torch.zeros(8, 16, device="cuda")
    S, C, D, U = (_lib.CPG_ERR_INVALID_SHAPE, _lib.CPG_ERR_INVALID_CONFIG, _lib.CPG_ERR_DTYPE,
                  _lib.CPG_ERR_UNSUPPORTED)
    for call, code in [
            (lambda: moe.route(lg, 0), S), (lambda: moe.route(lg, 9), S),
            (lambda: moe.route(lg, -1), S),
            (lambda: moe.route(torch.randn(2, 1025, device="cuda"), 2), S),
            (lambda: moe.route(lg, 2, groups=3), C),
            (lambda: moe.route(lg, 3, groups=4, kept_groups=1), C),
            (lambda: moe.route(lg, 2, groups=4, kept_groups=5), C),
            (lambda: moe.route(lg, 2, groups=0), C),
            (lambda: moe.route(lg, 2, scoring="tanh"), C),
            (lambda: moe.route(lg, 2, group_score="mean"), C),
            (lambda: moe.route(lg.double(), 2), D),
            (lambda: moe.route(lg[0], 2), S),
            (lambda: moe.route(lg.t(), 2), U),
            (lambda: moe.route(lg, 2, bias=torch.zeros(7, device="cuda")), S),
            (lambda: moe.route(lg, 2, bias=torch.zeros(8, device="cuda").half()), S),
            (lambda: moe.route(lg, 2, ids=ids.long()), S),
            (lambda: moe.route(lg.cpu(), 2), _lib.CPG_ERR_NO_DEVICE),
            (lambda: moe.route_backward(w, lg, ids[:3]), S),
            (lambda: moe.route_backward(w.double(), lg, ids), S),
            (lambda: moe.route_backward(w, lg, ids, out=torch.empty(4, 8, device="cuda").half()), D),
            (lambda: moe.dispatch(x, ids, 0), S), (lambda: moe.dispatch(x, ids, 1025), S),
            (lambda: moe.dispatch(x, ids.long(), 4), S),
            (lambda: moe.dispatch(x, ids[:, :0], 4), S),
            (lambda: moe.dispatch(x, ids, 4, quantize="int4"), U),
            (lambda: moe.dispatch(x, ids, 4, scales=torch.zeros(8, device="cuda")), U),
            (lambda: moe.dispatch(x, ids, 4, out=torch.zeros(7, 16, device="cuda")), S),
            (lambda: moe.dispatch(x, ids, 4, out=rows.bfloat16()), D),
            (lambda: moe.dispatch(x, ids, 4, out=torch.zeros(1, 16, device="cuda").expand(8, 16)), S),
            (lambda: moe.dispatch(x.half(), ids, 4), D),
            (lambda: moe.combine(rows, ids[0]), S),
            (lambda: moe.combine(rows, ids, w[:2]), S),
            (lambda: moe.combine(rows, ids, w, source=x[:2]), S),
            (lambda: moe.combine(rows, ids, w, source=x.bfloat16()), D),
            (lambda: moe.combine(rows.t(), ids, w), U),
            (lambda: moe.combine_backward(x, rows, ids, None), _lib.CPG_ERR_NULL),
            (lambda: moe.combine_backward(x, rows.bfloat16(), ids, w), D),
            (lambda: moe.combine_backward(x, rows[:, :8], ids, w), S)]:
        with pytest.raises(CpgError) as err:
            call()
        assert err.value.code == code, err.value
