"""Cases and plain forms of the operators between a layer's projections when its tokens are mixed by
linear attention: ``norm_rope`` (norm and rotation of every query and key head) with its gradient,
and ``linear_attention`` (one decay per head) as a chunked product over packed sequences, with its
gradient, and as the recurrent ``step`` of single tokens.
``own`` false: elementary torch operations; ``own`` true: the framework's calls.

    norm_rope:         y = rotate(x / sqrt(mean(x^2) + eps) * weight, angles of the token's position)
    linear_attention:  S_t = exp(log_decay) S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t
"""
import math

import torch

own = False

EPS = 1e-6
CHUNK = 128  # tokens of a chunk in the plain form


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One step of a 16-sequence decode batch: query and key heads of a fused projection's rows.
        dict(name="norm_rope_decode", op="norm_rope", tokens=16, hq=32, hk=8, d=128, rot=128,
             interleaved=False, fused=True, x="bf16"),
        # The same heads over a prefill or training batch.
        dict(name="norm_rope_prefill", op="norm_rope", tokens=16384, hq=32, hk=8, d=128, rot=128,
             interleaved=False, fused=True, x="bf16"),
        # Heads of 80 channels, half of them rotated in neighbouring pairs, in FP32, an odd count.
        dict(name="norm_rope_fp32", op="norm_rope", tokens=4099, hq=20, hk=20, d=80, rot=40,
             interleaved=True, fused=False, x="fp32"),
        # The gradient in training, half of the channels rotated.
        dict(name="norm_rope_backward", op="norm_rope_backward", tokens=8191, hq=32, hk=8, d=128,
             rot=64, interleaved=False, fused=True, x="bf16"),
        # One short prompt into a fresh state: latency counts.
        dict(name="attention_short", op="attention", tokens=37, seqs=1, hq=16, hv=16, dk=64, dv=64,
             pad=0, ragged=False, state=False, final=True),
        # A prefill batch of 16 ragged requests that continue states kept in a pool.
        dict(name="attention_prefill", op="attention", tokens=8191, seqs=16, hq=32, hv=32, dk=128,
             dv=128, pad=5, ragged=True, state=True, final=True),
        # One long document through few heads.
        dict(name="attention_long", op="attention", tokens=65536, seqs=1, hq=16, hv=16, dk=128,
             dv=128, pad=0, ragged=False, state=False, final=True),
        # A training batch of 8 sequences, forward.
        dict(name="attention_train", op="attention", tokens=16384, seqs=8, hq=64, hv=64, dk=128,
             dv=128, pad=0, ragged=False, state=False, final=False),
        # Its gradient, with half of the heads.
        dict(name="attention_backward", op="attention_backward", tokens=16384, seqs=8, hq=32, hv=32,
             dk=128, dv=128, pad=0, ragged=False, state=False),
        # The gradient where queries and keys are shared by four value heads each, narrower than
        # them, over ragged sequences that start from a state, whose gradient is wanted too.
        dict(name="attention_backward_shared", op="attention_backward", tokens=4097, seqs=5, hq=4,
             hv=16, dk=64, dv=128, pad=3, ragged=True, state=True),
        # A decode step of 4 sequences: latency counts.
        dict(name="step_decode", op="step", tokens=4, hq=32, hv=32, dk=128, dv=128, pad=0),
        # A decode step of a full batch, some of its rows padding: every state read and written.
        dict(name="step_large", op="step", tokens=256, hq=64, hv=64, dk=128, dv=128, pad=3),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope", "norm_rope_backward", "attention", "attention",
                     "attention", "attention_backward", "attention_backward", "step", "step"])
    if op.startswith("norm_rope"):
        d = rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256, rng.randrange(6, 256, 2)])
        rot = rng.choice([d, d, d // 4 * 2, rng.randrange(2, d + 1, 2)])
        hk = rng.choice([1, 2, 5, 8, 16])
        hq = hk * rng.choice([1, 1, 2, 4])
        tokens = _log(rng, 1, 16384)
        return dict(op=op, tokens=max(1, min(tokens, (16384 * 40 * 128) // ((hq + hk) * d))), hq=hq,
                    hk=hk, d=d, rot=rot, interleaved=rng.random() < 0.4, fused=rng.random() < 0.5,
                    x=rng.choice(["bf16", "bf16", "fp32"]))
    share = rng.choice([1, 1, 1, 2, 4])
    hq = rng.choice([1, 2, 4, 5, 8, 12, 16])
    hv = hq * share
    dk = rng.choice([128, 128, 64, 64, 8 * rng.randint(1, 16)])
    dv = rng.choice([dk, dk, 128, 8 * rng.randint(1, 16)])
    if op == "step":
        tokens = _log(rng, 1, 512)
        return dict(op=op, tokens=tokens, hq=hq, hv=hv, dk=dk, dv=dv,
                    pad=rng.choice([0, 0, 1, 5]) if tokens > 5 else 0)
    tokens = _log(rng, 1, 32768)
    tokens = max(1, min(tokens, (16384 * 32) // hv))
    seqs = min(tokens, _log(rng, 1, 64))
    case = dict(op=op, tokens=tokens, seqs=seqs, hq=hq, hv=hv, dk=dk, dv=dv,
                pad=rng.choice([0, 0, 1, 77]), ragged=rng.random() < 0.7,
                state=rng.random() < 0.4)
    if op == "attention":
        case["final"] = rng.random() < 0.5
    return case


# ----------------------------------------------------------------------------------- inputs
def _dtype(name):
    return {"bf16": torch.bfloat16, "fp32": torch.float32}[name]


def _lengths(case, g):
    """Tokens of every sequence; ragged ones differ and one of several is empty."""
    n, t = case["seqs"], case["tokens"]
    if not case["ragged"]:
        return [t // n + (i < t % n) for i in range(n)]
    shares = torch.rand(n, generator=g, device="cuda").mul_(3).exp_().cpu().double()
    if n > 2:
        shares[n // 2] = 0
    ends = (shares.cumsum(0) / shares.sum() * t).round().long().tolist()
    ends[-1] = t
    return [b - a for a, b in zip([0] + ends, ends)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def normal(*shape, dtype=torch.bfloat16, size=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * size + mean).to(dtype)

    st = dict(case=case)
    if op.startswith("norm_rope"):
        t, hq, hk, d, dtype = (case["tokens"], case["hq"], case["hk"], case["d"], _dtype(case["x"]))
        channels = (torch.rand(d, device="cuda", generator=g) * 2 - 1).exp()  # channels differ
        if case["fused"]:  # rows of a fused query, key and value projection
            rows = torch.empty(t, hq + 2 * hk, d, dtype=dtype, device="cuda")
            q, k = rows[:, :hq], rows[:, hq:hq + hk]
        else:
            q = torch.empty(t, hq, d, dtype=dtype, device="cuda")
            k = torch.empty(t, hk, d, dtype=dtype, device="cuda")
        q.copy_(normal(t, hq, d, dtype=torch.float32) * channels)
        k.copy_(normal(t, hk, d, dtype=torch.float32) * channels)
        half = case["rot"] // 2
        angles = (torch.arange(32768, device="cuda", dtype=torch.float64)[:, None]
                  * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
        st.update(q=q, k=k, wq=normal(d, dtype=dtype, size=0.2, mean=1.0),
                  wk=normal(d, dtype=dtype, size=0.2, mean=1.0),
                  table=torch.cat([angles.cos(), angles.sin()], dim=1).float(),
                  positions=torch.randint(0, 32768, (t,), device="cuda", generator=g,
                                          dtype=torch.int32))
        if op == "norm_rope_backward":
            st.update(dq=normal(t, hq, d, dtype=dtype), dk=normal(t, hk, d, dtype=dtype))
        return st
    t, pad, hq, hv, dk, dv = (case[n] for n in ("tokens", "pad", "hq", "hv", "dk", "dv"))
    # Heads that forget at rates from half a token to hundreds of tokens.
    slopes = 2.0 ** (-8.0 * torch.arange(1, hv + 1, device="cuda") / hv)
    st["log_decay"] = -slopes * (0.75 + 0.5 * torch.rand(hv, device="cuda", generator=g))
    st["scale"] = dk ** -0.5
    st.update(q=normal(t + pad, hq, dk), k=normal(t + pad, hq, dk),
              v=normal(t + pad, hv, dv, mean=0.1))
    if op == "step":
        places = t + pad + 2
        slots = torch.randperm(places, device="cuda", generator=g)[:t + pad].int()
        slots[t:] = -1  # padding of the batch
        st.update(slots=slots, state=normal(places, hv, dk, dv, dtype=torch.float32, size=2.0))
        return st
    lengths = _lengths(case, g)
    ends = torch.tensor([0] + lengths).cumsum(0)
    st["lengths"] = lengths
    st["offsets"] = ends.int().cuda()
    if op == "attention":
        st["out"] = torch.zeros(t + pad, hv, dv, dtype=torch.bfloat16, device="cuda")
    seqs = case["seqs"]
    if case["state"] and op == "attention":  # a pool with places for more requests
        st["slots"] = torch.randperm(seqs + 3, device="cuda", generator=g)[:seqs].int()
        st["state"] = normal(seqs + 3, hv, dk, dv, dtype=torch.float32, size=2.0)
        if case["final"]:
            st["final"] = torch.zeros_like(st["state"])
    elif case["state"]:
        st["state"] = normal(seqs, hv, dk, dv, dtype=torch.float32, size=2.0)
        st["dfinal"] = normal(seqs, hv, dk, dv, dtype=torch.float32, size=0.1)
    if op == "attention_backward":
        st["dy"] = normal(t + pad, hv, dv)
    # Where each chunk's rows lie (-1: behind its sequence's end), which sequence it is of, how many
    # of the sequence's tokens precede it.
    first, seq, before = [], [], []
    for i, n in enumerate(lengths):
        for c in range(0, n, CHUNK):
            first.append(int(ends[i]) + c)
            seq.append(i)
            before.append(c)
    first, seq, before = (torch.tensor(x, dtype=torch.int64, device="cuda")
                          for x in (first, seq, before))
    rows = first[:, None] + torch.arange(CHUNK, device="cuda")
    rows = torch.where(rows < ends.cuda()[1:][seq][:, None], rows, -1)
    st.update(rows=rows, seq=seq, before=before)
    return st


# ------------------------------------------------------------------------------- plain forms
def _rotate(y, cos, sin, rot, interleaved):
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, y[..., rot:]], dim=-1)


def _plain_norm_rope(st, x, w):
    c = st["case"]
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * w.float()
    cs = st["table"][st["positions"].long()].unsqueeze(1)
    half = c["rot"] // 2
    return _rotate(y, cs[..., :half], cs[..., half:], c["rot"], c["interleaved"])


def _plain_norm_rope_backward(st, dy, x, w):
    c = st["case"]
    x, w = x.float(), w.float()
    r = torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS)
    cs = st["table"][st["positions"].long()].unsqueeze(1)
    half = c["rot"] // 2
    g = _rotate(dy.float(), cs[..., :half], -cs[..., half:], c["rot"], c["interleaved"])
    xn = x * r
    u = g * w
    dx = r * (u - xn * (u * xn).mean(dim=-1, keepdim=True))
    return dx, (g * xn).sum(dim=(0, 1))


def _powers(log_decay, n):
    """exp(n * log_decay) [H, *n.shape], and 0 where n is negative."""
    e = n.double() * log_decay.double().view(-1, *[1] * n.dim())
    return torch.where(n >= 0, e.exp(), 0.0).float()


def _plain_attention(st, q, k, v, state):
    """o [T, H, dv] in FP32 (0 outside the sequences) and the states after every sequence."""
    c, g = st["case"], st["log_decay"]
    share = c["hv"] // c["hq"]
    rows, seq, before = st["rows"], st["seq"], st["before"]
    valid = rows >= 0
    at = rows.clamp(min=0)

    def chunks(x, times):  # [chunks, H, CHUNK, d]
        x = torch.where(valid[..., None, None], x[at], 0.0)
        return x.repeat_interleave(times, dim=2).transpose(1, 2)

    q, k, v = chunks(q * st["scale"], share), chunks(k, share), chunks(v, 1)
    i = torch.arange(CHUNK, device="cuda")
    length = valid.sum(dim=1)
    o = ((q @ k.transpose(-1, -2)) * _powers(g, i[:, None] - i)) @ v
    # What each chunk adds to the state, and the state before each chunk: the earlier chunks of its
    # sequence, each decayed by the tokens between.
    left = _powers(g, length[:, None] - 1 - i).transpose(0, 1)  # [chunks, H, CHUNK]
    added = (k * left.unsqueeze(-1)).transpose(-1, -2) @ v
    between = before[:, None] - before - length
    between = torch.where(seq[:, None] == seq, between, -1)
    n = added.shape[0]
    flat = added.transpose(0, 1).reshape(c["hv"], n, -1)
    start = (_powers(g, between) @ flat).view(c["hv"], n, c["dk"], c["dv"]).transpose(0, 1)
    if state is not None:
        start = start + state[seq] * _powers(g, before).transpose(0, 1)[..., None, None]
    o = o + (q @ start) * _powers(g, i + 1).unsqueeze(-1)
    y = torch.zeros(c["tokens"] + c["pad"], c["hv"], c["dv"], device="cuda")
    y = y.index_put((at[valid],), o.transpose(1, 2)[valid])
    lengths = torch.tensor(st["lengths"], device="cuda")
    rest = lengths[:, None] - before - length
    rest = torch.where(seq == torch.arange(len(lengths), device="cuda")[:, None], rest, -1)
    final = (_powers(g, rest) @ flat).view(c["hv"], -1, c["dk"], c["dv"]).transpose(0, 1)
    if state is not None:
        final = final + state * _powers(g, lengths).transpose(0, 1)[..., None, None]
    return y, final


def _run_plain(st):
    c = st["case"]
    op = c["op"]
    if op == "norm_rope":
        return (_plain_norm_rope(st, st["q"], st["wq"]).to(st["q"].dtype),
                _plain_norm_rope(st, st["k"], st["wk"]).to(st["k"].dtype))
    if op == "norm_rope_backward":
        dq, dwq = _plain_norm_rope_backward(st, st["dq"], st["q"], st["wq"])
        dk, dwk = _plain_norm_rope_backward(st, st["dk"], st["k"], st["wk"])
        return dq.to(st["q"].dtype), dk.to(st["k"].dtype), dwq, dwk
    if op == "step":
        share = c["hv"] // c["hq"]
        used = st["slots"] >= 0
        slots = st["slots"][used].long()
        q, k = (st[n][used].float().repeat_interleave(share, dim=1) for n in "qk")
        s = st["state"][slots] * st["log_decay"].exp()[:, None, None]
        s = s + k.unsqueeze(-1) * st["v"][used].float().unsqueeze(-2)
        st["state"][slots] = s
        y = torch.zeros(st["v"].shape, device="cuda")
        y[used] = st["scale"] * (q.unsqueeze(-2) @ s).squeeze(-2)
        return y.bfloat16(), st["state"]
    state = st.get("state")
    if state is not None and "slots" in st:
        state = state[st["slots"].long()]
    if op == "attention":
        y, final = _plain_attention(st, st["q"].float(), st["k"].float(), st["v"].float(), state)
        st["out"][:c["tokens"]] = y[:c["tokens"]]
        if not c["final"]:
            return (st["out"],)
        if "final" in st:
            st["final"][st["slots"].long()] = final
            final = st["final"]
        return st["out"], final
    leaves = [st[n].float().requires_grad_() for n in "qkv"]
    if state is not None:
        leaves.append(state.clone().requires_grad_())
    y, final = _plain_attention(st, *leaves[:3], leaves[3] if state is not None else None)
    outs, grads = [y], [st["dy"].float()]
    if state is not None:
        outs.append(final)
        grads.append(st["dfinal"])
    d = torch.autograd.grad(outs, leaves, grads)
    return tuple(x.bfloat16() for x in d[:3]) + tuple(d[3:])


# ------------------------------------------------------------------------------------- a pass
def _run_own(st):
    from cutedsl_pingpong_gemm_b200 import attention

    c = st["case"]
    op = c["op"]
    if op == "norm_rope":
        return attention.norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["table"],
                                   st["positions"], eps=EPS, interleaved=c["interleaved"])
    if op == "norm_rope_backward":
        return attention.norm_rope_backward(st["dq"], st["dk"], st["q"], st["k"], st["wq"],
                                            st["wk"], st["table"], st["positions"], eps=EPS,
                                            interleaved=c["interleaved"])
    if op == "step":
        y = attention.linear_attention_step(st["q"], st["k"], st["v"], st["log_decay"],
                                            st["state"], scale=st["scale"], slots=st["slots"])
        return y, st["state"]
    if op == "attention":
        y, final = attention.linear_attention(
            st["q"], st["k"], st["v"], st["log_decay"], scale=st["scale"], offsets=st["offsets"],
            state=st.get("state"), slots=st.get("slots"),
            final=st.get("final", True) if c["final"] else None, out=st["out"])
        return (y, final) if c["final"] else (y,)
    dq, dk, dv, dstate = attention.linear_attention_backward(
        st["dy"], st["q"], st["k"], st["v"], st["log_decay"], scale=st["scale"],
        offsets=st["offsets"], state=st.get("state"), dfinal=st.get("dfinal"))
    return (dq, dk, dv, dstate) if c["state"] else (dq, dk, dv)


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


def work(case):
    op, t = case["op"], case["tokens"]
    if op.startswith("norm_rope"):
        eb = 4 if case["x"] == "fp32" else 2
        n = t * (case["hq"] + case["hk"]) * case["d"]
        back = op == "norm_rope_backward"
        table = min(t, 32768) * case["rot"] * 4 + 4 * t
        weights = 2 * case["d"] * (eb + (4 if back else 0))
        return {"bytes": n * eb * (3 if back else 2) + table + weights, "flops": n * (16 if back else 8)}
    hq, hv, dk, dv = (case[n] for n in ("hq", "hv", "dk", "dv"))
    qk, v = t * hq * dk * 2, t * hv * dv * 2
    if op == "step":
        return {"bytes": 2 * qk + 2 * v + 8 * t * hv * dk * dv, "flops": 5 * t * hv * dk * dv}
    states = 4 * case["seqs"] * hv * dk * dv
    if op == "attention":
        return {"bytes": 2 * qk + 2 * v + states * (case["state"] + case["final"]),
                "flops": 4 * t * hv * dk * dv}
    return {"bytes": 4 * qk + 3 * v + 3 * states * case["state"], "flops": 12 * t * hv * dk * dv}


# -------------------------------------------------------------------------- 64-bit definition
def _exact_norm_rope(st, x, w):
    """Through complex numbers: the rotated pairs are multiplied by e^(i angle)."""
    c = st["case"]
    half = c["rot"] // 2
    x = x.double()
    y = w.double() * x / (x.pow(2).sum(dim=-1, keepdim=True) / c["d"] + EPS).sqrt()
    cs = st["table"].double()[st["positions"].long()][:, None]
    turn = torch.complex(cs[..., :half], cs[..., half:])
    out = y.clone()
    first = slice(0, c["rot"], 2) if c["interleaved"] else slice(0, half)
    second = slice(1, c["rot"], 2) if c["interleaved"] else slice(half, c["rot"])
    z = torch.complex(y[..., first], y[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_attention(st, dy=None):
    """By the sum over all earlier tokens of the sequence, in blocks of rows, without chunk states:
    o_t = scale * sum_{j <= t} e^(g (t - j)) (q_t . k_j) v_j + scale * e^(g (t + 1)) S^T q_t."""
    c = st["case"]
    hv, share = c["hv"], c["hv"] // c["hq"]
    q, k, v = (st[n].double() for n in "qkv")
    scale, rows, seqs = st["scale"], c["tokens"] + c["pad"], c["seqs"]
    state = st.get("state")
    if state is not None:
        state = state.double()
        if "slots" in st:
            state = state[st["slots"].long()]
    made = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    o, final = made(rows, hv, c["dv"]), made(seqs, hv, c["dk"], c["dv"])
    if dy is not None:
        dy = dy.double()
        dq, dk, dv, ds = (made(*q.shape), made(*k.shape), made(*v.shape), made(*final.shape))
    starts = st["offsets"].tolist()
    for s in range(seqs):
        a, n = starts[s], starts[s + 1] - starts[s]
        place = torch.arange(n, device="cuda", dtype=torch.float64)
        for h in range(hv):
            g, hs = float(st["log_decay"][h].double()), h // share
            qh, kh, vh = q[a:a + n, hs], k[a:a + n, hs], v[a:a + n, h]
            left = torch.exp(g * (n - 1 - place))[:, None]
            final[s, h] = (kh * left).T @ vh
            since = torch.exp(g * (place + 1))[:, None]
            if state is not None:
                final[s, h] += math.exp(g * n) * state[s, h]
            if dy is not None:
                doh = dy[a:a + n, h]
                if state is not None:
                    df = st["dfinal"][s, h].double()
                    dk[a:a + n, hs] += left * (vh @ df.T)
                    dv[a:a + n, h] += left * (kh @ df)
                    ds[s, h] = scale * (qh * since).T @ doh + math.exp(g * n) * df
                    dq[a:a + n, hs] += scale * since * (doh @ state[s, h].T)
            elif state is not None:
                o[a:a + n, h] = scale * since * (qh @ state[s, h])
            for b in range(0, n, 4096):
                e = min(n, b + 4096)
                ago = place[b:e, None] - place[None, :e]
                w = torch.where(ago >= 0, torch.exp(g * ago.clamp(min=0)), 0.0).mul_(scale)
                p = (qh[b:e] @ kh[:e].T).mul_(w)
                if dy is None:
                    o[a + b:a + e, h] += p @ vh[:e]
                    continue
                dv[a:a + e, h] += p.T @ doh[b:e]
                dp = (doh[b:e] @ vh[:e].T).mul_(w)
                dq[a + b:a + e, hs] += dp @ kh[:e]
                dk[a:a + e, hs] += dp.T @ qh[b:e]
    if dy is None:
        return o, final
    return (dq, dk, dv, ds) if state is not None else (dq, dk, dv)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm_rope":
        return _exact_norm_rope(st, st["q"], st["wq"]), _exact_norm_rope(st, st["k"], st["wk"])
    if op == "norm_rope_backward":
        dx, dw = [], []
        for n in "qk":
            x = st[n].double().requires_grad_()
            w = st["w" + n].double().requires_grad_()
            y = _exact_norm_rope(st, x, w)
            a, b = torch.autograd.grad(y, (x, w), st["d" + n].double())
            dx.append(a)
            dw.append(b)
        return (*dx, *dw)
    if op == "step":
        y = torch.zeros(st["v"].shape, dtype=torch.float64, device="cuda")
        s = st["state"].double()
        for i, slot in enumerate(st["slots"].tolist()):
            if slot < 0:
                continue
            q, k = (torch.repeat_interleave(st[n][i].double(), case["hv"] // case["hq"], dim=0)
                    for n in "qk")
            s[slot] *= torch.exp(st["log_decay"].double())[:, None, None]
            s[slot] += torch.einsum("hk,hv->hkv", k, st["v"][i].double())
            y[i] = st["scale"] * torch.einsum("hk,hkv->hv", q, s[slot])
        return y, s
    if op == "attention_backward":
        return _exact_attention(st, st["dy"])
    y, final = _exact_attention(st)
    if not case["final"]:
        return (y,)
    if "final" in st:
        whole = torch.zeros(st["final"].shape, dtype=torch.float64, device="cuda")
        whole[st["slots"].long()] = final
        final = whole
    return y, final
