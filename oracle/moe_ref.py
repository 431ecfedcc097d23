"""Plain 64-bit forms of the INT8 product and of the operators around the experts' products, on the
CPU -- TEST ORACLE ONLY.  Written from the formulas of include/cpgemm.h; the reference project has no
such operators."""
import math

import torch

BF16_HALF = torch.finfo(torch.bfloat16).eps / 2  # a rounding to BF16 is off by at most this much
F32_HALF = torch.finfo(torch.float32).eps / 2


def quantize_int8(x):
    """q (int8) and the fp32 scales of the rows of x, by the operator's definition: the fp32 scale
    max(amax, 1e-12) / 127 and the fp32 quotient rounded to the nearest even integer."""
    x = x.float()
    rows, cols = x.shape
    amax = x.abs().amax(1) if cols else torch.zeros(rows)
    bad = ~torch.isfinite(x).all(1)
    s = torch.maximum(amax, torch.tensor(1e-12)) / torch.tensor(127.0)
    s = torch.where(bad, torch.tensor(math.nan), s)
    q = torch.where(bad[:, None], torch.zeros(()), x / s[:, None]).round()
    return q.to(torch.int8), s


def act(name, y):
    if name in (None, "none"):
        return y
    if name == "relu":
        return y.clamp_min(0)
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def int8_product(a, b, sa=None, sb=None, alpha=1.0, bias=None, source=None, beta=1.0,
                 activation=None, gated=False):
    """(reference, its slack): the 64-bit result and how far fp32 arithmetic may be from it before
    the last rounding.  Roundings of a pre-activation value, each 2^-24 of its magnitude: the
    integer sum to fp32, alpha * s_a, its product with the sum, s_b; then the sum with the bias and
    beta * C (one more each, of the terms' magnitudes).  The activations are 1.13-Lipschitz (gelu's
    largest slope), their own fp32 evaluation is allowed 64 roundings of the value and of 1.0e-7."""
    acc = a.double() @ b.double().t()  # exact: |sum| < 2^31
    y = acc * alpha
    y = y * (1.0 if sa is None else sa.double().reshape(-1, 1))
    y = y * (1.0 if sb is None else sb.double().reshape(1, -1))
    slack = 4 * F32_HALF * y.abs()
    if gated:
        n = b.shape[0] // 2
        gate, up = y[:, :n], y[:, n:]
        g = act(activation, gate)
        g_slack = (1.13 * slack[:, :n] + (64 * F32_HALF * (g.abs() + 1.0)
                                          if activation else 0.0))
        ref = g * up
        return ref, (g_slack * up.abs() + g.abs() * slack[:, n:] + F32_HALF * ref.abs()) * 1.001
    mag = y.abs()
    for term in (None if bias is None else bias.double().reshape(1, -1),
                 None if source is None else beta * source.double()):
        if term is not None:
            y = y + term
            mag = mag + term.abs()
            slack = slack + 2 * F32_HALF * mag
    if activation:
        y = act(activation, y)
        slack = 1.13 * slack + 64 * F32_HALF * (y.abs() + 1.0)
    return y, slack * 1.001


def within(d, ref, slack):
    """Largest (error - tolerance) of d against ref: <= 0 when every element is within the slack
    plus one rounding to d's type."""
    half = BF16_HALF if d.dtype == torch.bfloat16 else 0.0
    d = d.double().cpu()
    ref, slack = ref.cpu(), slack.cpu()
    tol = slack + half * (ref.abs() + slack)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(d), nan), "NaN in other places"
    err = torch.where(nan, torch.zeros(()).double(), (d - ref).abs() - tol)
    return err.max().item() if err.numel() else 0.0


# ------------------------------------------------------------------------------------- routing
def route(logits, k, scoring="softmax", bias=None, groups=1, kept_groups=None, group_score=None,
          renormalize=True, scale=1.0):
    """ids, weights (64 bits), row by row in plain Python."""
    t, e = logits.shape
    kept_groups = groups if kept_groups is None else kept_groups
    group_score = group_score or ("max" if bias is None else "top2")
    by_logit = bias is None and (groups == 1 or group_score == "max")
    ids = torch.full((t, k), -1, dtype=torch.int32)
    w = torch.zeros(t, k, dtype=torch.float64)
    for r in range(t):
        l = [float(v) for v in logits[r].double()]
        spoiled = [math.isnan(v) or (scoring == "softmax" and v == math.inf) for v in l]
        ok = [v > -math.inf and not bad for v, bad in zip(l, spoiled)]
        s = scores(l, ok, scoring)
        c = [(l[i] if by_logit else s[i] + (0.0 if bias is None else float(bias[i]))) if ok[i]
             else -math.inf for i in range(e)]
        c = [-math.inf if math.isnan(v) else v for v in c]
        if groups > 1:
            per = e // groups
            value = []
            for g in range(groups):
                best = sorted(c[g * per:(g + 1) * per], reverse=True)
                v = best[0]
                if group_score == "top2" and per > 1 and best[1] > -math.inf:
                    v += best[1]
                value.append(v)
            kept = sorted(range(groups), key=lambda g: (-value[g], g))[:kept_groups]
            c = [c[i] if i // per in kept else -math.inf for i in range(e)]
        order = [i for i in sorted(range(e), key=lambda i: (-c[i], i)) if c[i] > -math.inf][:k]
        part = shares([l[i] for i in order], [s[i] for i in order], scoring, renormalize)
        for j, i in enumerate(order):
            ids[r, j] = i
            w[r, j] = scale * part[j]
        if any(spoiled):
            w[r] = math.nan
    return ids, w


def sigmoid(v):
    return 1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v) / (1 + math.exp(v))


def scores(l, ok, scoring):
    if scoring == "sigmoid":
        return [sigmoid(v) if o else 0.0 for v, o in zip(l, ok)]
    top = max((v for v, o in zip(l, ok) if o), default=0.0)
    p = [math.exp(v - top) if o else 0.0 for v, o in zip(l, ok)]
    total = math.fsum(p)
    return [v / total if total else 0.0 for v in p]


def shares(l, s, scoring, renormalize):
    """Shares of the chosen logits l with scores s; sums that underflow by their logarithms."""
    if not renormalize or not l:
        return s
    if scoring == "sigmoid" and max(l) >= -700:
        total = math.fsum(s)
        return [v / total for v in s]
    top = max(l)
    p = [math.exp(v - top) for v in l]
    return [v / math.fsum(p) for v in p]


def route_backward(dweights, logits, ids, scoring="softmax", renormalize=True, scale=1.0):
    """dlogits (64 bits) by the formulas, row by row."""
    t, e = logits.shape
    out = torch.zeros(t, e, dtype=torch.float64)
    for r in range(t):
        l = [float(v) for v in logits[r].double()]
        if any(math.isnan(v) or (scoring == "softmax" and v == math.inf) for v in l):
            out[r] = math.nan
            continue
        s = scores(l, [v > -math.inf for v in l], scoring)
        pairs = [(int(i), float(g)) for i, g in zip(ids[r], dweights[r].double())
                 if 0 <= int(i) < e and l[int(i)] > -math.inf]
        part = shares([l[i] for i, _ in pairs], [s[i] for i, _ in pairs], scoring, renormalize)
        mean = math.fsum(g * p for (_, g), p in zip(pairs, part))
        if scoring == "softmax" and not renormalize:
            for i in range(e):
                out[r, i] = -s[i] * mean * scale
        for (i, g), p in zip(pairs, part):
            v = p * (g - mean) if renormalize else p * g
            if scoring == "sigmoid":
                v *= sigmoid(-l[i])
            out[r, i] += scale * v
    return out


def expert_order(ids, experts):
    """offsets [experts + 1] and slots of ids [T, k]."""
    flat = [int(i) for i in ids.reshape(-1)]
    counts = [0] * experts
    for i in flat:
        if 0 <= i < experts:
            counts[i] += 1
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    at = offsets[:-1].copy()
    slots = []
    for i in flat:
        if 0 <= i < experts:
            slots.append(at[i])
            at[i] += 1
        else:
            slots.append(-1)
    return (torch.tensor(offsets, dtype=torch.int32),
            torch.tensor(slots, dtype=torch.int32).reshape(ids.shape))


def combine(rows, slots, weights=None, source=None):
    """(y, slack): 64-bit sums; fp32 sums of k terms in order are within (k + 1) roundings of the
    terms' magnitudes."""
    t, k = slots.shape
    here = (slots >= 0) & (slots < rows.shape[0])
    got = rows.double()[slots.clamp(0, max(rows.shape[0] - 1, 0)).long()] if rows.shape[0] else \
        torch.zeros(t, k, rows.shape[1], dtype=torch.float64)
    w = torch.ones(t, k, dtype=torch.float64) if weights is None else weights.double()
    terms = torch.where(here[..., None], got * w[..., None], torch.zeros(()).double())
    y, mag = terms.sum(1), terms.abs().sum(1)
    if source is not None:
        y, mag = y + source.double(), mag + source.double().abs()
    return y, (k + 1) * F32_HALF * mag


def combine_backward(dy, rows, slots, weights):
    """(drows, dweights, slack of dweights): rows no slot names are NaN in drows."""
    t, k = slots.shape
    d = dy.shape[1]
    drows = torch.full((rows.shape[0], d), math.nan, dtype=torch.float64)
    dw = torch.zeros(t, k, dtype=torch.float64)
    mag = torch.zeros(t, k, dtype=torch.float64)
    for i in range(t):
        for j in range(k):
            r = int(slots[i, j])
            if 0 <= r < rows.shape[0]:
                drows[r] = float(weights[i, j]) * dy[i].double()
                prod = dy[i].double() * rows[r].double()
                dw[i, j] = prod.sum()
                mag[i, j] = prod.abs().sum()
    return drows, dw, (d + 1) * F32_HALF * mag
