"""Cases and plain forms of the 8-bit integer products and of the expert routing operators.

Operators: ``linear`` (rows quantised to int8, int8 matrix product with a scale per row and per
column), ``experts`` (the same product grouped by expert, gated), ``route`` and its gradient,
``dispatch`` (rows put into expert order) and ``combine`` (their weighted sum) with its gradient.
``own`` false: elementary torch operations; ``own`` true: the framework's calls.
"""
import math

import numpy as np
import torch

own = False

FLOOR = 1e-12  # smallest row maximum a scale is made from


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One step of a 16-sequence decode batch through a square projection: weight-bound.
        dict(name="linear_decode", op="linear", m=16, n=8192, k=8192, gated=False, act="",
             bias=False, x="bf16"),
        # A ragged prefill of 1021 tokens into a gated feed-forward layer of odd width.
        dict(name="linear_gated_ragged", op="linear", m=1021, n=14333, k=4096, gated=True,
             act="silu", bias=False, x="bf16"),
        # A full batch of tokens through a square projection with a bias: compute-bound.
        dict(name="linear_large", op="linear", m=16384, n=8192, k=8192, gated=False, act="",
             bias=True, x="bf16"),
        # The gated up-projection of 8 experts over 16384 routed rows, groups of uneven size, one
        # of them empty.
        dict(name="experts_gated", op="experts", rows=16384, n=14336, k=4096, experts=8,
             gated=True, act="silu"),
        # A decode batch routed by sigmoid scores with a balance bias, 4 of 8 groups, top 8.
        dict(name="route_decode", op="route", tokens=16, experts=256, k=8, scoring="sigmoid",
             bias=True, groups=8, kept=4, renorm=True, pad=0, logits="fp32"),
        # The same router over a prefill or training batch, its last tokens padding.
        dict(name="route_prefill", op="route", tokens=16384, experts=256, k=8, scoring="sigmoid",
             bias=True, groups=8, kept=4, renorm=True, pad=37, logits="fp32"),
        # The gradient of a softmax router whose weights are not renormalised (every logit gets one).
        dict(name="route_backward", op="route_backward", tokens=16384, experts=128, k=8,
             scoring="softmax", renorm=False, pad=0, logits="fp32"),
        # A decode batch's rows into the order of 8 experts, top 2.
        dict(name="dispatch_decode", op="dispatch", tokens=16, d=4096, experts=8, k=2, int8=False,
             pad=0, x="bf16"),
        # A prefill batch's rows, quantised on the way, into the order of 256 experts, top 8.
        dict(name="dispatch_int8", op="dispatch", tokens=16384, d=4096, experts=256, k=8,
             int8=True, pad=100, x="bf16"),
        # The weighted sum of a decode batch's expert outputs.
        dict(name="combine_decode", op="combine", tokens=16, d=4096, experts=8, k=2, source=False,
             pad=0, x="bf16"),
        # The weighted sum of a prefill batch's expert outputs onto a shared expert's.
        dict(name="combine_prefill", op="combine", tokens=16384, d=4096, experts=256, k=8,
             source=True, pad=0, x="bf16"),
        # Its gradient in training: of the expert outputs and of the routing weights.
        dict(name="combine_backward", op="combine_backward", tokens=8191, d=4096, experts=8, k=2,
             pad=3, x="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "experts", "route", "route", "route_backward", "dispatch",
                     "dispatch", "combine", "combine_backward"])
    if op == "linear":
        gated = rng.random() < 0.3
        m = _log(rng, 1, 16384)
        case = dict(op=op, m=m, n=_log(rng, 64, 8192), k=_log(rng, 64, 8192), gated=gated,
                    act="silu" if gated else (rng.choice(["", "", "gelu"]) if m > 128 else ""),
                    bias=not gated and rng.random() < 0.5, x=rng.choice(["bf16", "bf16", "fp32"]))
        if gated and m > 8192:
            case["m"] = m // 2
        return case
    if op == "experts":
        experts = rng.choice([2, 5, 8, 16, 32, 64])
        gated = rng.random() < 0.6
        return dict(op=op, rows=_log(rng, 16, 16384), n=_log(rng, 64, 57344 // max(experts, 8)),
                    k=_log(rng, 64, 4096), experts=experts, gated=gated,
                    act="silu" if gated else "")
    x = rng.choice(["bf16", "bf16", "fp32"])
    tokens = _log(rng, 1, 16384)
    pad = rng.choice([0, 0, 1, 13]) if tokens > 13 else 0
    if op in ("route", "route_backward"):
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * rng.choice([2, 5, 8, 16, 20, 32]) if groups > 1 else _log(rng, 2, 256)
        kept = rng.randint(1, groups)
        k = rng.randint(1, min(16, kept * (experts // groups)))
        case = dict(op=op, tokens=tokens, experts=experts, k=k,
                    scoring=rng.choice(["softmax", "sigmoid"]), renorm=rng.random() < 0.7, pad=pad,
                    logits=x)
        if op == "route":
            case.update(bias=rng.random() < 0.5, groups=groups, kept=kept)
        return case
    experts = rng.choice([4, 8, 16, 60, 64, 128, 256])
    k = rng.randint(1, min(8, experts))
    case = dict(op=op, tokens=tokens, d=_log(rng, 64, 4096), experts=experts, k=k, pad=pad, x=x)
    if op == "dispatch":
        case["int8"] = rng.random() < 0.5
    if op == "combine":
        case["source"] = rng.random() < 0.3
    if x == "fp32":
        case["tokens"] = min(tokens, 8192)
    return case


# ----------------------------------------------------------------------------------- inputs
def _dtype(name):
    return {"bf16": torch.bfloat16, "fp32": torch.float32}[name]


def _padded(rows, cols, dtype, per, lead=()):
    """[*lead, rows, cols] zeros whose row stride is a multiple of `per` elements (16 bytes)."""
    ld = -(-cols // per) * per
    return torch.zeros(*lead, rows, ld, dtype=dtype, device="cuda")[..., :cols]


def _weights(g, rows, cols, lead=()):
    """int8 weights as a quantised layer holds them, rows padded to 16 bytes, and their scales."""
    w = _padded(rows, cols, torch.int8, 16, lead)
    w.copy_(torch.randn(*lead, rows, cols, device="cuda", generator=g, dtype=torch.float16)
            .mul_(32).round_().clamp_(-127, 127))
    s = torch.rand(*lead, rows, device="cuda", generator=g) * 1e-3 + 2e-4
    return w, s


def _activations(g, m, k, dtype):
    """Token rows whose channels differ in size, as activations do."""
    x = torch.randn(m, k, device="cuda", generator=g)
    return x.mul_(torch.randn(k, device="cuda", generator=g).mul_(0.5).exp_()).to(dtype)


def _chosen(g, case):
    """k distinct experts for each token, some experts more popular than others; -1 for padding."""
    t, e, k = case["tokens"], case["experts"], case["k"]
    liking = torch.randn(t, e, device="cuda", generator=g)
    liking += torch.randn(e, device="cuda", generator=g) * 0.5
    ids = liking.topk(k, dim=1).indices.to(torch.int32)
    if case["pad"]:
        ids[t - case["pad"]:] = -1
    return ids


def _slots(ids, experts):
    """Row of every (token, choice) in expert order, -1 for none, and the experts' offsets."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat >= 0, flat, experts)
    order = key.argsort(stable=True)
    slots = torch.empty_like(flat)
    slots[order] = torch.arange(flat.numel(), device=flat.device)
    slots = torch.where(flat >= 0, slots, -1)
    counts = (key[:, None] == torch.arange(experts, device=key.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return slots.view_as(ids).to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, st = case["op"], dict(case)
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        st["xs"] = _activations(g, m, k, _dtype(case["x"]))
        st["w"], st["sw"] = _weights(g, 2 * n if case["gated"] else n, k)
        st["b"] = torch.randn(n, device="cuda", generator=g).bfloat16() if case["bias"] else None
        st["out"] = _padded(m, n, torch.bfloat16, 8)
    elif op == "experts":
        rows, n, k, e = case["rows"], case["n"], case["k"], case["experts"]
        st["q"] = _padded(rows, k, torch.int8, 16)
        st["q"].copy_(torch.randn(rows, k, device="cuda", generator=g, dtype=torch.float16)
                      .mul_(35).round_().clamp_(-127, 127))
        st["sx"] = torch.rand(rows, device="cuda", generator=g) * 0.02 + 0.01
        st["w"], st["sw"] = _weights(g, 2 * n if case["gated"] else n, k, (e,))
        # Uneven groups, the second expert's empty: cuts at sorted random places.
        r = np.random.RandomState(seed % (1 << 31))
        cuts = np.sort(r.randint(0, rows + 1, e - 1))
        if e > 2:
            cuts[1] = cuts[0]
        off = np.concatenate([[0], cuts, [rows]]).astype(np.int32)
        st["sizes"] = np.diff(off).tolist()
        st["off"] = torch.from_numpy(off).cuda()
        st["out"] = _padded(rows, n, torch.bfloat16, 8)
    elif op in ("route", "route_backward"):
        t, e = case["tokens"], case["experts"]
        lg = torch.randn(t, e, device="cuda", generator=g) * 1.5
        lg += torch.randn(e, device="cuda", generator=g) * 0.5
        if case["pad"]:
            lg[t - case["pad"]:] = -math.inf
        st["lg"] = lg.to(_dtype(case["logits"]))
        if op == "route":
            st["b"] = torch.randn(e, device="cuda", generator=g) * 0.05 if case["bias"] else None
        else:
            st["ids"] = _chosen(g, case)
            st["dw"] = torch.randn(t, case["k"], device="cuda", generator=g)
    else:
        t, d, k = case["tokens"], case["d"], case["k"]
        dt = _dtype(case["x"])
        st["ids"] = _chosen(g, case)
        if op == "dispatch":
            st["xs"] = _activations(g, t, d, dt)
            st["out"] = torch.zeros(t * k, d, dtype=torch.int8 if case["int8"] else dt, device="cuda")
            st["sout"] = torch.zeros(t * k, device="cuda") if case["int8"] else None
        else:
            st["slots"], _ = _slots(st["ids"], case["experts"])
            st["rows"] = torch.randn(t * k, d, device="cuda", generator=g).to(dt)
            st["wt"] = torch.rand(t, k, device="cuda", generator=g)
            st["wt"] /= st["wt"].sum(1, keepdim=True)
            if op == "combine":
                st["src"] = (torch.randn(t, d, device="cuda", generator=g).to(dt)
                             if case["source"] else None)
                st["out"] = torch.empty(t, d, dtype=dt, device="cuda")
            else:
                st["dy"] = torch.randn(t, d, device="cuda", generator=g).to(dt)
                st["out"] = torch.zeros(t * k, d, dtype=dt, device="cuda")
    return st


# -------------------------------------------------------------------------------- plain forms
def _quantise(x):
    """Row scales amax / 127 and the rounded quotients, in 32 bits."""
    x = x.float()
    limit = torch.full((), 127.0, device=x.device)  # a tensor: a true division, not 1/127 times
    s = x.abs().amax(1).clamp_min(FLOOR) / limit
    return (x / s[:, None]).round(), s


def _act(name, v):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


def _product(q, s, w, sw, bias, gated, act):
    acc = (q.float() @ w.float().t()) * s[:, None] * sw[None, :]
    if bias is not None:
        acc = acc + bias.float()
    if gated:
        n = w.shape[0] // 2
        return (_act(act, acc[:, :n]) * acc[:, n:]).bfloat16()
    return _act(act, acc).bfloat16()


def _plain_route(st):
    x = st["lg"].double()
    t, e = x.shape
    some = x > -math.inf  # a masked logit is never chosen
    if st["scoring"] == "sigmoid":
        score = 1 / (1 + torch.exp(-x))
    else:
        top = torch.where(some, x, -1e300).amax(1, keepdim=True)
        score = torch.where(some, torch.exp(x - top), 0.0)
        score = score / score.sum(1, keepdim=True).clamp_min(1e-300)
    # Without a bias the score grows with the logit, so the logit itself ranks (two scores near 1
    # could be equal where the logits are not).
    choice = x if st["b"] is None else torch.where(some, score + st["b"].double(), -math.inf)
    if st["groups"] > 1:
        per = e // st["groups"]
        if st["b"] is None:
            value = x.view(t, -1, per).amax(2)
        else:
            best = choice.view(t, -1, per).sort(dim=2, descending=True).values[:, :, :2]
            value = best[:, :, 0] + torch.where(best[:, :, 1:] > -math.inf, best[:, :, 1:], 0.0).sum(2)
        order = value.sort(dim=1, descending=True, stable=True).indices[:, :st["kept"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, order, True)
        choice = torch.where(keep.repeat_interleave(per, 1), choice, -math.inf)
    best = choice.sort(dim=1, descending=True, stable=True)
    ids = best.indices[:, :st["k"]]
    there = best.values[:, :st["k"]] > -math.inf
    wt = torch.where(there, score.gather(1, ids), 0.0)
    if st["renorm"]:
        wt = wt / wt.sum(1, keepdim=True).clamp_min(1e-300)
    return torch.where(there, ids, -1).to(torch.int32), wt.float()


def _plain_route_backward(st):
    x = st["lg"].double()
    ids, dw = st["ids"].long(), st["dw"].double()
    there = ids >= 0
    at = ids.clamp_min(0)
    dw = torch.where(there, dw, 0.0)
    some = x > -math.inf
    if st["scoring"] == "sigmoid":
        score = 1 / (1 + torch.exp(-x))
    else:
        top = torch.where(some, x, -1e300).amax(1, keepdim=True)
        score = torch.where(some, torch.exp(x - top), 0.0)
        score = score / score.sum(1, keepdim=True).clamp_min(1e-300)
    mine = torch.where(there, score.gather(1, at), 0.0)
    if st["renorm"]:
        total = mine.sum(1, keepdim=True).clamp_min(1e-300)
        part = mine / total
        ds = torch.where(there, (dw - (dw * part).sum(1, keepdim=True)) / total, 0.0)
    else:
        ds = dw
    dscore = torch.zeros_like(x).scatter_add_(1, at, ds)
    if st["scoring"] == "sigmoid":
        dl = dscore * score * (1 - score)
    else:
        dl = score * (dscore - (dscore * score).sum(1, keepdim=True))
    return dl.to(st["lg"].dtype)


def _plain_dispatch(st):
    slots, offsets = _slots(st["ids"], st["experts"])
    flat = slots.view(-1).long()
    to = flat[flat >= 0]
    token = (torch.arange(flat.numel(), device="cuda") // st["k"])[flat >= 0]
    out = torch.zeros_like(st["out"])
    if not st["int8"]:
        out[to] = st["xs"][token]
        return out, offsets, slots
    q, s = _quantise(st["xs"])
    out[to] = q.to(torch.int8)[token]
    scales = torch.zeros_like(st["sout"])
    scales[to] = s[token]
    return out, offsets, slots, scales


def _gathered(rows, slots):
    got = rows.float()[slots.clamp_min(0).long()]
    return torch.where((slots >= 0)[..., None], got, 0.0)


def _plain(st):
    op = st["op"]
    if op == "linear":
        q, s = _quantise(st["xs"])
        return _product(q, s, st["w"], st["sw"], st["b"], st["gated"], st["act"])
    if op == "experts":
        parts = zip(st["q"].split(st["sizes"]), st["sx"].split(st["sizes"]), st["w"], st["sw"])
        return torch.cat([_product(q, s, w, sw, None, st["gated"], st["act"])
                          for q, s, w, sw in parts])
    if op == "route":
        return _plain_route(st)
    if op == "route_backward":
        return _plain_route_backward(st)
    if op == "dispatch":
        return _plain_dispatch(st)
    slots, wt = st["slots"], st["wt"]
    got = _gathered(st["rows"], slots)
    if op == "combine":
        y = (got * wt[..., None]).sum(1)
        return (y if st["src"] is None else y + st["src"].float()).to(st["rows"].dtype)
    dy = st["dy"].float()
    dwt = (got * dy[:, None, :]).sum(2)
    to = slots.view(-1).long()
    drows = torch.zeros_like(st["out"])
    drows[to[to >= 0]] = (wt[..., None] * dy[:, None, :]).view(-1, dy.shape[1]).to(dy.dtype)[
        to >= 0].to(drows.dtype)
    return drows, dwt


# ---------------------------------------------------------------------------- the framework's
_gemms = {}


def _gemm(tile_n):
    """The program's GEMM objects, one per tile width."""
    from cutedsl_pingpong_gemm_b200 import GemmSM90
    if tile_n not in _gemms:
        _gemms[tile_n] = GemmSM90(tile_shape_mn=(128, tile_n), epi_tile_mn=(128, 32),
                                  cluster_shape_mnk=(2, 1, 1), atom_layout_mn=(1, 1),
                                  ab_stage=3 if tile_n == 512 else 5, reuse_ab=False,
                                  is_persistent=True, dynamic_scheduler=True)
    return _gemms[tile_n]


def _own(st):
    op = st["op"]
    if op == "linear":
        from cutedsl_pingpong_gemm_b200.quant import quantize_int8
        q, s = quantize_int8(st["xs"])
        # Wide tiles where they fill the GPU, and for the gated form.
        m, n = st["out"].shape
        wide = st["gated"] or m * n >= 148 * 128 * 512
        _gemm(512 if wide else 256)(q, st["w"], st["out"], scale_a=s, scale_b=st["sw"],
                                    bias=st["b"], activation=st["act"] or None,
                                    gated=st["gated"], split_k=0)
        return st["out"]
    if op == "experts":
        _gemm(512).grouped(st["q"], st["w"], st["out"], st["off"], scale_a=st["sx"],
                           scale_b=st["sw"], activation=st["act"] or None, gated=st["gated"])
        return st["out"]
    from cutedsl_pingpong_gemm_b200 import moe
    if op == "route":
        return moe.route(st["lg"], st["k"], scoring=st["scoring"], bias=st["b"],
                         groups=st["groups"], kept_groups=st["kept"], renormalize=st["renorm"])
    if op == "route_backward":
        return moe.route_backward(st["dw"], st["lg"], st["ids"], scoring=st["scoring"],
                                  renormalize=st["renorm"])
    if op == "dispatch":
        got = moe.dispatch(st["xs"], st["ids"], st["experts"],
                           quantize="int8" if st["int8"] else None, out=st["out"],
                           scales=st["sout"])
        return ((got.rows, got.offsets, got.slots) if got.scales is None
                else (got.rows, got.offsets, got.slots, got.scales))
    if op == "combine":
        return moe.combine(st["rows"], st["slots"], st["wt"], source=st["src"], out=st["out"])
    return moe.combine_backward(st["dy"], st["rows"], st["slots"], st["wt"], drows=st["out"])


def run(state):
    return _own(state) if own else _plain(state)


# -------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "linear":
        m, k = case["m"], case["k"]
        nw = case["n"] * (2 if case["gated"] else 1)
        x = 2 if case["x"] == "bf16" else 4
        return {"bytes": m * k * x + nw * k + 4 * nw + (2 * case["n"] if case["bias"] else 0)
                + 2 * m * case["n"], "flops": 2 * m * nw * k}
    if op == "experts":
        t, k = case["rows"], case["k"]
        nw = case["n"] * (2 if case["gated"] else 1)
        return {"bytes": t * k + 4 * t + case["experts"] * nw * (k + 4) + 4 * (case["experts"] + 1)
                + 2 * t * case["n"], "flops": 2 * t * nw * k}
    t, e, k = case["tokens"], case["experts"], case["k"]
    if op in ("route", "route_backward"):
        size = 2 if case["logits"] == "bf16" else 4
        if op == "route":
            return {"bytes": t * e * size + 8 * t * k + (4 * e if case["bias"] else 0),
                    "flops": 8 * t * e}
        return {"bytes": 2 * t * e * size + 8 * t * k, "flops": 8 * t * e}
    d, size = case["d"], 2 if case["x"] == "bf16" else 4
    real = t - case["pad"]
    if op == "dispatch":
        return {"bytes": real * d * size + 8 * t * k + 4 * (e + 1)
                + real * k * (d + 4 if case["int8"] else d * size),
                "flops": 2 * real * d if case["int8"] else 0}
    if op == "combine":
        return {"bytes": real * k * d * size + t * d * size * (2 if case["source"] else 1)
                + 8 * t * k, "flops": 2 * real * k * d}
    return {"bytes": 2 * real * k * d * size + real * d * size + 12 * t * k,
            "flops": 3 * real * k * d}


# ------------------------------------------------------------------------------------- exact
def _exact_row_scales(x):
    """The scale is held in 32 bits by definition: the 64-bit quotient rounded once."""
    return (x.double().abs().max(dim=1).values.clamp_min(FLOOR) / torch.tensor(
        127.0, dtype=torch.float64, device=x.device)).float().double()


def _exact_product(a, sa, w, sw, bias, gated, act):
    def f(v):
        if act == "silu":
            return v * torch.sigmoid(v)
        if act == "gelu":
            return v * torch.special.ndtr(v)
        return v
    y = torch.einsum("mk,nk->mn", a, w.double())
    y *= sa.double().unsqueeze(1)
    y *= sw.double()
    if bias is not None:
        y += bias.double()
    if gated:
        gate, up = y.chunk(2, dim=1)
        return f(gate) * up
    return f(y)


def _exact_probabilities(case, x):
    """Scores of the rows of x (numpy, 64 bits); a fully masked row scores 0."""
    with np.errstate(all="ignore"):
        if case["scoring"] == "sigmoid":
            return np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))),
                            np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
        p = np.exp(x - x.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        return np.where(np.isnan(p), 0.0, p)


def _exact_route(case, st):
    x = st["lg"].double().cpu().numpy()
    t, e = x.shape
    p = _exact_probabilities(case, x)
    c = x.copy() if st["b"] is None else p + st["b"].double().cpu().numpy()
    c[np.isneginf(x)] = -np.inf
    if case["groups"] > 1:
        cg = c.reshape(t, case["groups"], -1)
        top = -np.sort(-cg, axis=2)
        if st["b"] is None or top.shape[2] == 1:
            value = top[:, :, 0]
        else:
            value = top[:, :, 0] + np.where(np.isneginf(top[:, :, 1]), 0.0, top[:, :, 1])
        rank = np.argsort(np.argsort(-value, axis=1, kind="stable"), axis=1, kind="stable")
        c = np.where((rank < case["kept"])[:, :, None], cg, -np.inf).reshape(t, e)
    ids = np.argsort(-c, axis=1, kind="stable")[:, :case["k"]]
    has = ~np.isneginf(np.take_along_axis(c, ids, 1))
    w = np.take_along_axis(p, ids, 1) * has
    if case["renorm"]:
        total = w.sum(axis=1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return torch.from_numpy(np.where(has, ids, -1).astype(np.int32)), torch.from_numpy(w)


def _exact_route_backward(case, st):
    x = st["lg"].double().cpu().numpy()
    ids, g = st["ids"].cpu().numpy(), st["dw"].double().cpu().numpy()
    t, e = x.shape
    p = _exact_probabilities(case, x)
    hot = np.zeros((t, e))
    rows, cols = np.nonzero(ids >= 0)
    np.add.at(hot, (rows, ids[rows, cols]), 1.0)
    grad = np.zeros((t, e))
    np.add.at(grad, (rows, ids[rows, cols]), g[rows, cols])
    if case["renorm"]:
        total = (hot * p).sum(axis=1, keepdims=True)
        total = np.where(total > 0, total, 1.0)
        grad = hot * (grad - (grad * p).sum(axis=1, keepdims=True) / total) / total
    if case["scoring"] == "sigmoid":
        return torch.from_numpy(grad * p * (1 - p))
    return torch.from_numpy(p * grad - p * (p * grad).sum(axis=1, keepdims=True))


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        s = _exact_row_scales(st["xs"])
        a = torch.round(st["xs"].double() / s.unsqueeze(1))
        return _exact_product(a, s, st["w"], st["sw"], st["b"], case["gated"], case["act"])
    if op == "experts":
        ends = np.cumsum(st["sizes"])
        y = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for i, end in enumerate(ends):
            part = slice(int(end) - st["sizes"][i], int(end))
            y[part] = _exact_product(st["q"][part].double(), st["sx"][part], st["w"][i],
                                     st["sw"][i], None, case["gated"], case["act"])
        return y
    if op == "route":
        return _exact_route(case, st)
    if op == "route_backward":
        return _exact_route_backward(case, st)
    ids = st["ids"].cpu().numpy().reshape(-1)
    order = np.argsort(ids, kind="stable")
    order = order[ids[order] >= 0]  # (token, choice) of each row, in expert order
    pair = torch.from_numpy(order).cuda()
    token = pair // case["k"]
    if op == "dispatch":
        slots = np.full(ids.shape, -1, np.int32)
        slots[order] = np.arange(order.size)
        offsets = np.concatenate([[0], np.cumsum(np.bincount(ids[ids >= 0],
                                                             minlength=case["experts"]))])
        slots = torch.from_numpy(slots.reshape(case["tokens"], case["k"]))
        offsets = torch.from_numpy(offsets.astype(np.int32))
        if not case["int8"]:
            y = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
            y[:order.size] = st["xs"].double()[token]
            return y, offsets, slots
        s = _exact_row_scales(st["xs"])
        q = torch.round(st["xs"].double() / s.unsqueeze(1)).to(torch.int8)
        y = torch.zeros(st["out"].shape, dtype=torch.int8, device="cuda")
        y[:order.size] = q[token]
        scales = torch.zeros(st["sout"].shape, dtype=torch.float64, device="cuda")
        scales[:order.size] = s[token]
        return y, offsets, slots, scales
    wt = st["wt"].double().view(-1)[pair].unsqueeze(1)
    if op == "combine":
        y = (torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
             if st["src"] is None else st["src"].double())
        return y.index_add_(0, token, st["rows"][:order.size].double() * wt)
    dy = st["dy"].double()[token]
    drows = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    drows[:order.size] = wt * dy
    dwt = torch.zeros(case["tokens"] * case["k"], dtype=torch.float64, device="cuda")
    dwt[pair] = (dy * st["rows"][:order.size].double()).sum(dim=1)
    return drows, dwt.view(case["tokens"], case["k"])
