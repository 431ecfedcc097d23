"""INT8 products (scales per token and per output channel) and the INT8 row quantiser on the GPU,
against plain 64-bit forms.

The integer sums are exact, so the tolerance counts only the roundings after them (see
oracle.moe_ref.int8_product): a handful of fp32 half steps plus one to the output type.
"""
import pytest
import torch

from cutedsl_pingpong_gemm_b200 import CpgError, GemmSM90, _lib, compile as cpg_compile
from cutedsl_pingpong_gemm_b200.quant import quantize_int8
from oracle import moe_ref

pytestmark = pytest.mark.gpu


def make_gemm(tile_n=256, cluster=(2, 1, 1), stages=4, dynamic=False, persistent=True):
    if tile_n == 512:  # what fits in shared memory
        stages = 3 if cluster[0] == 2 else 2
    return GemmSM90(tile_shape_mn=(128, tile_n), epi_tile_mn=(128, 32), cluster_shape_mnk=cluster,
                    atom_layout_mn=(1, 1), ab_stage=stages,
                    reuse_ab=False, is_persistent=persistent, dynamic_scheduler=dynamic)


def padded(t, per):
    """t in rows padded to `per` elements."""
    cols = t.shape[-1]
    out = torch.zeros(*t.shape[:-1], -(-cols // per) * per, dtype=t.dtype, device=t.device)
    out[..., :cols] = t
    return out[..., :cols]


def operands(m, n, k, seed, lead_a=(), lead_b=()):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-128, 128, (*lead_a, m, k), generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (*lead_b, n, k), generator=g, dtype=torch.int8)
    sa = torch.rand(*lead_a, m, generator=g) * 0.02 + 1e-3
    sb = torch.rand(*lead_b, n, generator=g) * 1e-2 + 1e-4
    return a, b, sa, sb


def output(m, n, dtype=torch.bfloat16, lead=()):
    per = 8 if dtype == torch.bfloat16 else 4
    ld = -(-n // per) * per
    return torch.full((*lead, m, ld), float("nan"), dtype=dtype, device="cuda")[..., :n]


SHAPES = [(1, 1, 1), (128, 256, 128), (129, 257, 131), (300, 1000, 1021), (513, 72, 4096),
          (1000, 520, 16)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("tile_n,cluster,dynamic", [(64, (1, 1, 1), False), (128, (2, 1, 1), False),
                                                    (256, (1, 2, 1), False), (256, (2, 1, 1), True),
                                                    (512, (2, 1, 1), True), (512, (1, 1, 1), False)])
def test_dense(m, n, k, tile_n, cluster, dynamic):
    a, b, sa, sb = operands(m, n, k, seed=m + n + k)
    d = output(m, n)
    make_gemm(tile_n, cluster, dynamic=dynamic)(
        padded(a.cuda(), 16), padded(b.cuda(), 16), d, scale_a=sa.cuda(), scale_b=sb.cuda())
    torch.cuda.synchronize()
    ref, slack = moe_ref.int8_product(a, b, sa, sb)
    assert moe_ref.within(d, ref, slack) <= 0


@pytest.mark.parametrize("which", ["none", "a_tensor", "b_tensor", "both_tensor", "a_rows", "b_rows"])
@pytest.mark.parametrize("m", [33, 200])
def test_scale_forms_fp32(which, m):
    """Every mix of no scale, one value and one per row, alpha and bias, FP32 output; M <= 128 runs
    the small-M kernel too."""
    n, k = 136, 272
    a, b, sa, sb = operands(m, n, k, seed=5)
    if which in ("a_tensor", "both_tensor"):
        sa = sa[:1]
    if which in ("b_tensor", "both_tensor"):
        sb = sb[:1]
    if which in ("none", "b_rows"):
        sa = None
    if which in ("none", "a_rows"):
        sb = None
    bias = torch.randn(n, generator=torch.Generator().manual_seed(6)).bfloat16()
    ref, slack = moe_ref.int8_product(a, b, sa, sb, alpha=0.375, bias=bias)
    for split in (1, -3) if m <= 128 else (1,):
        d = output(m, n, torch.float32)
        make_gemm()(a.cuda(), b.cuda(), d, bias=bias.cuda(), alpha=0.375, split_k=split,
                    scale_a=None if sa is None else sa.cuda(),
                    scale_b=None if sb is None else sb.cuda())
        torch.cuda.synchronize()
        assert moe_ref.within(d, ref, slack) <= 0, split


@pytest.mark.parametrize("m,split", [(130, 1), (7, -3)])
def test_sums_are_exact_integers(m, split):
    """No scales, FP32 output: the 32-bit integer sum itself, rounded once."""
    n, k = 260, 2048
    a, b, _, _ = operands(m, n, k, seed=8)
    d = output(m, n, torch.float32)
    make_gemm()(a.cuda(), b.cuda(), d, split_k=split)
    torch.cuda.synchronize()
    acc = a.long() @ b.long().t()
    assert torch.equal(d.cpu(), acc.float())


@pytest.mark.parametrize("m,split", [(129, 1), (3, -3), (128, -3)])
def test_largest_sums(m, split):
    """The longest K of the lowest value: sums of 131071 * 2^14 < 2^31, and the same negative."""
    k = 131071
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((16, k), -128, dtype=torch.int8, device="cuda")
    b[1::2] = 127
    d = output(m, 16, torch.float32)
    make_gemm()(padded(a, 16), padded(b, 16), d, split_k=split)
    torch.cuda.synchronize()
    want = torch.tensor([128 * 128 * k, -128 * 127 * k] * 8).float().expand(m, 16)
    assert torch.equal(d.cpu(), want)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 64, 100, 128])
@pytest.mark.parametrize("n,k", [(128, 128), (1000, 1021), (8192, 4096), (40, 20000)])
def test_small_m(m, n, k):
    a, b, sa, sb = operands(m, n, k, seed=m)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(6)).bfloat16()
    d = output(m, n)
    make_gemm()(padded(a.cuda(), 16), padded(b.cuda(), 16), d, bias=bias.cuda(), scale_a=sa.cuda(),
                scale_b=sb.cuda(), split_k=0)
    torch.cuda.synchronize()
    ref, slack = moe_ref.int8_product(a, b, sa, sb, bias=bias)
    assert moe_ref.within(d, ref, slack) <= 0


@pytest.mark.parametrize("split", [1, 3, -1, -2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_split_k(split, dtype):
    """K ranges and Stream-K: partial results are scaled and added in FP32 (one more rounding per
    range and addition; at most 8 ranges of a tile here)."""
    m, n, k = 300, 520, 5000
    a, b, sa, sb = operands(m, n, k, seed=12)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(6)).bfloat16()
    d = output(m, n, dtype)
    make_gemm(256, (1, 1, 1))(padded(a.cuda(), 16), padded(b.cuda(), 16), d, bias=bias.cuda(),
                              scale_a=sa.cuda(), scale_b=sb.cuda(), split_k=split)
    torch.cuda.synchronize()
    ref, slack = moe_ref.int8_product(a, b, sa, sb, bias=bias)
    parts = (a.double().abs() @ b.double().abs().t()) * sa.double()[:, None] * sb.double()
    ranges = -(-k // 128)  # no more ranges than k-blocks
    assert moe_ref.within(d, ref, slack + 2 * ranges * moe_ref.F32_HALF * (parts + ref.abs())) <= 0


@pytest.mark.parametrize("n", [1, 107, 130, 263])
@pytest.mark.parametrize("split", [0, 2, -1])
@pytest.mark.parametrize("lead", [(), (3,)])
@pytest.mark.parametrize("operand", [torch.int8, torch.bfloat16])
def test_split_k_into_bf16_of_any_width(n, split, lead, operand):
    """The FP32 workspace of a split has rows of its own padding: any N, as in one pass."""
    m, k = 310, 2240
    if operand == torch.int8:
        a, b, sa, sb = operands(m, n, k, 13, lead, lead)
    else:
        g = torch.Generator().manual_seed(13)
        a = torch.randn(*lead, m, k, generator=g).bfloat16()
        b = torch.randn(*lead, n, k, generator=g).bfloat16()
        sa = sb = None
    bias = torch.randn(n, generator=torch.Generator().manual_seed(6)).bfloat16()
    d = torch.full((*lead, m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    make_gemm(256, (1, 1, 1))(a.cuda(), b.cuda(), d, bias=bias.cuda(), split_k=split,
                              scale_a=None if sa is None else sa.cuda(),
                              scale_b=None if sb is None else sb.cuda())
    torch.cuda.synchronize()
    for i in range(lead[0]) if lead else (slice(None),):
        ref, slack = moe_ref.int8_product(a[i], b[i], None if sa is None else sa[i],
                                          None if sb is None else sb[i], bias=bias)
        mag = a[i].double().abs() @ b[i].double().abs().t()
        if sa is not None:
            mag = mag * sa[i].double()[:, None] * sb[i].double()
        # INT8: one rounding per range and addition; BF16: k fp32 additions of exact products.
        terms = 2 * -(-k // 128) if sa is not None else 2 * k
        assert moe_ref.within(d[i], ref, slack + terms * moe_ref.F32_HALF * (mag + ref.abs())) <= 0


@pytest.mark.parametrize("activation", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_epilogue(activation, dtype):
    m, n, k = 200, 328, 192
    a, b, sa, sb = operands(m, n, k, seed=21)
    sa = sa * 0.1
    g = torch.Generator().manual_seed(22)
    bias = torch.randn(n, generator=g).bfloat16()
    src = torch.randn(m, n, generator=g).to(dtype)
    d = output(m, n, dtype)
    make_gemm(128)(a.cuda(), b.cuda(), d, bias=bias.cuda(), scale_a=sa.cuda(), scale_b=sb.cuda(),
                   activation=activation, source=src.cuda(), beta=0.5, alpha=1.5)
    torch.cuda.synchronize()
    ref, slack = moe_ref.int8_product(a, b, sa, sb, alpha=1.5, bias=bias, source=src, beta=0.5,
                                      activation=activation)
    assert moe_ref.within(d, ref, slack) <= 0


@pytest.mark.parametrize("m,n,k", [(5, 8, 64), (257, 264, 300), (130, 1003, 128)])
@pytest.mark.parametrize("rows_b", [True, False])
def test_gated(m, n, k, rows_b):
    a, b, sa, sb = operands(m, 2 * n, k, seed=31)
    sa = sa * 0.1
    if not rows_b:
        sb = sb[:1]
    d = output(m, n)
    make_gemm(512)(padded(a.cuda(), 16), padded(b.cuda(), 16), d, scale_a=sa.cuda(),
                   scale_b=sb.cuda(), activation="silu", gated=True, split_k=0)
    torch.cuda.synchronize()
    ref, slack = moe_ref.int8_product(a, b, sa, sb, activation="silu", gated=True)
    assert moe_ref.within(d, ref, slack) <= 0


def test_batched():
    l, m, n, k = 3, 70, 201, 160
    a, b, sa, sb = operands(m, n, k, 41, (l,), (l,))
    d = output(m, n, lead=(l,))
    make_gemm(128, (1, 1, 1))(a.cuda(), b.cuda(), d, scale_a=sa.cuda(), scale_b=sb.cuda())
    torch.cuda.synchronize()
    for i in range(l):
        ref, slack = moe_ref.int8_product(a[i], b[i], sa[i], sb[i])
        assert moe_ref.within(d[i], ref, slack) <= 0, i


@pytest.mark.parametrize("tile_n,gated,dynamic", [(256, False, False), (512, True, True)])
@pytest.mark.parametrize("n", [264, 131])
def test_grouped(tile_n, gated, dynamic, n):
    sizes, k = [0, 37, 128, 300, 1, 0, 513, 90], 144
    start, tail = 16, 21
    t = start + sum(sizes) + tail
    rows_b = 2 * n if gated else n
    a, b, sa, sb = operands(t, rows_b, k, 51, (), (len(sizes),))
    sa = sa * 0.1
    off = [start]
    for s in sizes:
        off.append(off[-1] + s)
    d = output(t, n)
    make_gemm(tile_n, dynamic=dynamic).grouped(
        a.cuda(), b.cuda(), d, torch.tensor(off, dtype=torch.int32, device="cuda"),
        scale_a=sa.cuda(), scale_b=sb.cuda(), activation="silu" if gated else None, gated=gated)
    torch.cuda.synchronize()
    for g in range(len(sizes)):
        r = slice(off[g], off[g + 1])
        ref, slack = moe_ref.int8_product(a[r], b[g], sa[r], sb[g], gated=gated,
                                          activation="silu" if gated else None)
        assert moe_ref.within(d[r], ref, slack) <= 0, g
    assert torch.isnan(d[:start].float()).all() and torch.isnan(d[off[-1]:].float()).all()


def test_nan_scale_stays_in_its_row():
    """A row that could not be quantised (scale NaN) spoils its own row of D only."""
    m, n, k = 40, 256, 128
    a, b, sa, sb = operands(m, n, k, seed=61)
    sa[7] = float("nan")
    for split in (1, -3):
        d = output(m, n)
        make_gemm()(a.cuda(), b.cuda(), d, scale_a=sa.cuda(), scale_b=sb.cuda(), split_k=split)
        torch.cuda.synchronize()
        ref, slack = moe_ref.int8_product(a, b, sa, sb)
        assert moe_ref.within(d, ref, slack) <= 0


def test_unaligned_scales_compile_and_capture():
    """Scales at odd addresses, a second stream, and a captured graph replayed on new data."""
    m, n, k = 150, 260, 256
    a, b, sa, sb = operands(m, n, k, seed=71)
    da, db, d = a.cuda(), b.cuda(), output(m, n)
    both = torch.zeros(m + n + 1, device="cuda")
    dsa, dsb = both[1:m + 1], both[m + 1:]
    dsa.copy_(sa)
    dsb.copy_(sb)
    compiled = cpg_compile(make_gemm(), da, db, d, None, scale_a=dsa, scale_b=dsb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        compiled(da, db, d, None, scale_a=dsa, scale_b=dsb)
    side.synchronize()
    ref, slack = moe_ref.int8_product(a, b, sa, sb)
    assert moe_ref.within(d, ref, slack) <= 0
    x = torch.randn(m, k, device="cuda").bfloat16()
    with torch.cuda.stream(side):
        q, s = quantize_int8(x)
        compiled(q, db, d, None, scale_a=s, scale_b=dsb)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = quantize_int8(x)
        compiled(q, db, d, None, scale_a=s, scale_b=dsb)
    x.copy_(torch.randn(m, k, device="cuda") * 3)
    graph.replay()
    torch.cuda.synchronize()
    rq, rs = moe_ref.quantize_int8(x.cpu())
    assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)
    ref, slack = moe_ref.int8_product(rq, b, rs, sb)
    assert moe_ref.within(d, ref, slack) <= 0


def test_refusals():
    g = make_gemm(512)
    a, b, sa, sb = (t.cuda() for t in operands(64, 64, 128, seed=1))
    d = output(64, 64)
    cases = [
        (dict(scale_a=sa[:5], scale_b=sb), _lib.CPG_ERR_INVALID_SHAPE),
        (dict(scale_a=sa, scale_b=sb[:3]), _lib.CPG_ERR_INVALID_SHAPE),
        (dict(scale_a=sa.double(), scale_b=sb), _lib.CPG_ERR_INVALID_SHAPE),
        (dict(scale_a=sa, scale_b=sb, activation="silu", split_k=-3), _lib.CPG_ERR_UNSUPPORTED),
    ]
    for kw, code in cases:
        with pytest.raises(CpgError) as e:
            g(a, b, d, **kw)
        assert e.value.code == code, kw
    with pytest.raises(AssertionError):
        g(a, b.bfloat16(), d)
    with pytest.raises(CpgError) as e:  # K rows not 16-byte multiples
        g(a[:, :100].contiguous(), b[:, :100].contiguous(), d)
    assert e.value.code == _lib.CPG_ERR_ALIGNMENT
    long = torch.zeros(2, 131072, dtype=torch.int8, device="cuda")
    for split in (1, -3):
        with pytest.raises(CpgError) as e:
            g(long, long, output(2, 2), split_k=split)
        assert e.value.code == _lib.CPG_ERR_INVALID_SHAPE and "131071" in str(e.value)


def test_empty_rows():
    b = torch.ones(64, 128, dtype=torch.int8, device="cuda")
    x = torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda")
    q, s = quantize_int8(x)
    assert q.shape == (0, 128) and s.shape == (0,)
    make_gemm()(q, b, output(0, 64), scale_a=s, scale_b=torch.ones(64, device="cuda"))
    torch.cuda.synchronize()


@pytest.mark.parametrize("m,n,k", [(5, 8, 64), (257, 264, 300), (130, 1003, 128)])
@pytest.mark.parametrize("rows_b", [True, False])
@pytest.mark.parametrize("dynamic", [False, True])
def test_gated_fp32(m, n, k, rows_b, dynamic):
    a, b, sa, sb = operands(m, 2 * n, k, seed=33)
    sa = sa * 0.1
    if not rows_b:
        sb = sb[:1]
    d = output(m, n, torch.float32)
    make_gemm(512, dynamic=dynamic)(padded(a.cuda(), 16), padded(b.cuda(), 16), d,
                                    scale_a=sa.cuda(), scale_b=sb.cuda(), activation="silu",
                                    gated=True, split_k=0)
    torch.cuda.synchronize()
    ref, slack = moe_ref.int8_product(a, b, sa, sb, activation="silu", gated=True)
    assert moe_ref.within(d, ref, slack) <= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [130, 264])
def test_batched_gated(n, dtype):
    l, m, k = 3, 150, 160
    a, b, sa, sb = operands(m, 2 * n, k, 43, (l,), (l,))
    sa = sa * 0.1
    d = output(m, n, dtype, lead=(l,))
    make_gemm(512)(a.cuda(), b.cuda(), d, scale_a=sa.cuda(), scale_b=sb.cuda(), activation="silu",
                   gated=True)
    torch.cuda.synchronize()
    for i in range(l):
        ref, slack = moe_ref.int8_product(a[i], b[i], sa[i], sb[i], activation="silu", gated=True)
        assert moe_ref.within(d[i], ref, slack) <= 0, i


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("split", [0, 3])
def test_batched_split_k(dtype, split):
    """Every K range of every batch takes its batch's scales (tolerance as in test_split_k)."""
    l, m, n, k = 3, 200, 264, 5008
    a, b, sa, sb = operands(m, n, k, 44, (l,), (l,))
    bias = torch.randn(n, generator=torch.Generator().manual_seed(6)).bfloat16()
    d = output(m, n, dtype, lead=(l,))
    make_gemm(256, (1, 1, 1))(a.cuda(), b.cuda(), d, bias=bias.cuda(), scale_a=sa.cuda(),
                              scale_b=sb.cuda(), split_k=split)
    torch.cuda.synchronize()
    ranges = -(-k // 128)
    for i in range(l):
        ref, slack = moe_ref.int8_product(a[i], b[i], sa[i], sb[i], bias=bias)
        parts = (a[i].double().abs() @ b[i].double().abs().t()) * sa[i].double()[:, None]
        parts = parts * sb[i].double()
        slack = slack + 2 * ranges * moe_ref.F32_HALF * (parts + ref.abs())
        assert moe_ref.within(d[i], ref, slack) <= 0, i


@pytest.mark.parametrize("m", [1, 16, 100, 128])
@pytest.mark.parametrize("captured", [False, True])
def test_quantise_and_small_m_back_to_back(m, captured):
    """Each product is a dependent launch that may be set up while the quantiser before it still runs:
    every step reads the rows and scales of its own quantiser, though all steps share their buffers;
    eager and in a graph replayed on new inputs."""
    n, k, steps = 1024, 1040, 6
    _, b, _, sb = operands(m, n, k, seed=81)
    g = torch.Generator().manual_seed(m)
    xs = torch.zeros(steps, m, k, dtype=torch.bfloat16, device="cuda")
    db, dsb, gemm = b.cuda(), sb.cuda(), make_gemm()
    q = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    s = torch.zeros(m, device="cuda")
    outs = [output(m, n) for _ in range(steps)]

    def run():
        for i in range(steps):
            quantize_int8(xs[i], out=q, scales=s)
            gemm(q, db, outs[i], scale_a=s, scale_b=dsb, split_k=0)
    run()
    torch.cuda.synchronize()
    graph = None
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
    for _ in range(3):
        x = (torch.randn(steps, m, k, generator=g) * torch.rand(steps, m, 1, generator=g)).bfloat16()
        xs.copy_(x)
        run() if graph is None else graph.replay()
        torch.cuda.synchronize()
        for i in range(steps):
            rq, rs = moe_ref.quantize_int8(x[i])
            ref, slack = moe_ref.int8_product(rq, b, rs, sb)
            assert moe_ref.within(outs[i], ref, slack) <= 0, i


# --------------------------------------------------------------------------------- quantiser
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (33, 100), (4, 1024), (17, 1032),
                                       (2, 4096), (9, 8192), (2, 16384), (3, 16400), (2, 70001)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_matches_definition(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * cols)
    x = (torch.randn(rows, cols, generator=g) * torch.rand(rows, 1, generator=g) * 10).to(dtype)
    q, s = quantize_int8(x.cuda())
    rq, rs = moe_ref.quantize_int8(x)
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu(), rq)
    assert q.stride(0) % 16 == 0 or rows == 1


def test_quantize_at_rounding_borders():
    """Values whose quotients are half-integers or a few fp32 steps beside them: the fp32 quotient
    decides, as an IEEE division gives it."""
    s = torch.rand(64, generator=torch.Generator().manual_seed(3)) + 0.1
    half = torch.arange(-127, 127).float() + 0.5
    x = s[:, None] * half
    steps = torch.randint(-3, 4, x.shape, generator=torch.Generator().manual_seed(4),
                          dtype=torch.int32)
    x = (x.view(torch.int32) + steps).view(torch.float32)
    x = torch.cat([x, s[:, None] * 127], 1).contiguous()
    q, sc = quantize_int8(x.cuda())
    rq, rs = moe_ref.quantize_int8(x)
    assert torch.equal(sc.cpu(), rs) and torch.equal(q.cpu(), rq)


@pytest.mark.parametrize("cols", [64, 100, 5000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_special_rows(cols, dtype):
    x = torch.randn(8, cols, generator=torch.Generator().manual_seed(9)).to(dtype)
    x[0] = 0
    x[1, cols // 2] = float("inf")
    x[2, -1] = float("-inf")
    x[3, 0] = float("nan")
    x[4] *= 1e-30
    x[5] = torch.finfo(dtype).max
    x[6] = torch.finfo(dtype).tiny
    q, s = quantize_int8(x.cuda())
    rq, rs = moe_ref.quantize_int8(x)
    assert torch.equal(q.cpu(), rq)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(rs))
    assert torch.equal(s.cpu()[~torch.isnan(rs)], rs[~torch.isnan(rs)])
    assert torch.isnan(rs).tolist() == [False, True, True, True, False, False, False, False]


@pytest.mark.parametrize("shift,extra", [(0, 5), (1, 3), (8, 8), (3, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_strides_and_outputs(shift, extra, dtype):
    """Views at odd offsets with row strides of their own, given outputs, untouched surroundings."""
    rows, cols = 21, 250
    g = torch.Generator().manual_seed(17)
    base = torch.randn(rows, cols + shift + extra, generator=g).to(dtype).cuda()
    x = base[:, shift:shift + cols]
    qbase = torch.full((rows, cols + 2 * shift + 3), 77, dtype=torch.int8, device="cuda")
    out = qbase[:, shift:shift + cols]
    scales = torch.empty(rows, device="cuda")
    q, s = quantize_int8(x, out=out, scales=scales)
    assert q is out and s is scales
    rq, rs = moe_ref.quantize_int8(x.cpu())
    assert torch.equal(q.cpu(), rq) and torch.equal(s.cpu(), rs)
    assert (qbase[:, :shift] == 77).all() and (qbase[:, shift + cols:] == 77).all()


def test_quantize_refusals():
    x = torch.randn(4, 8, device="cuda")
    for bad, code in [(lambda: quantize_int8(x.double()), _lib.CPG_ERR_DTYPE),
                      (lambda: quantize_int8(x[0]), _lib.CPG_ERR_INVALID_SHAPE),
                      (lambda: quantize_int8(x.t()), _lib.CPG_ERR_UNSUPPORTED),
                      (lambda: quantize_int8(x, out=torch.empty(4, 8, device="cuda")),
                       _lib.CPG_ERR_DTYPE),
                      (lambda: quantize_int8(x, out=torch.empty(1, 8, dtype=torch.int8,
                                                                device="cuda").expand(4, 8)),
                       _lib.CPG_ERR_INVALID_SHAPE),
                      (lambda: quantize_int8(x, scales=torch.empty(5, device="cuda")),
                       _lib.CPG_ERR_INVALID_SHAPE)]:
        with pytest.raises(CpgError) as e:
            bad()
        assert e.value.code == code
