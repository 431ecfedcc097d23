"""Norm with rotation and linear attention in 64 bits, with the magnitudes that rounding errors of
the operators scale with."""
import torch


# ------------------------------------------------------------------------- norm and rotation
def _turn(y, cos, sin, interleaved):
    """Turn the first 2 * cos.shape[-1] channels of y [T, H, d] by the angles [T, 1, R / 2]."""
    half = cos.shape[-1]
    out = y.clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = y[..., first], y[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = a * sin + b * cos
    return out


def _angles(table, positions):
    """Cosines and sines [T, 1, R / 2] of the positions, NaN outside the table."""
    t = table.double()
    half = t.shape[1] // 2
    p = positions.long()
    known = (p >= 0) & (p < t.shape[0])
    rows = torch.full((len(p), t.shape[1]), float("nan"), dtype=torch.float64, device=t.device)
    rows[known] = t[p[known]]
    return rows[:, None, :half], rows[:, None, half:]


def norm_rope(x, w, table, positions, eps, interleaved):
    """``(y, size)``: size bounds the terms that a channel of y is the sum of."""
    x = x.double()
    n = x / (x.square().mean(dim=-1, keepdim=True) + eps).sqrt()
    if w is not None:
        n = n * w.double()
    if table is None or table.shape[1] == 0:
        return n, n.abs()
    cos, sin = _angles(table, positions)
    return _turn(n, cos, sin, interleaved), _turn(n.abs(), cos.abs(), sin.abs(), interleaved).abs() \
        + 2 * n.abs()


def norm_rope_backward(dy, x, w, table, positions, eps, interleaved):
    """``(dx, size of its terms, dw, size of its terms)``."""
    x, g = x.double(), dy.double()
    d = x.shape[-1]
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    size_g = g.abs()
    if table is not None and table.shape[1]:
        cos, sin = _angles(table, positions)
        half = cos.shape[-1]
        g = _turn(g, cos, -sin, interleaved)
        norm = size_g.clone()  # a turned pair's terms
        first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
        second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
        norm[..., first] = size_g[..., first] + size_g[..., second]
        norm[..., second] = norm[..., first]
        size_g = norm
    r = 1 / (x.square().mean(dim=-1, keepdim=True) + eps).sqrt()
    n = x * r
    u = g * w
    dx = r * (u - n * (u * n).mean(dim=-1, keepdim=True))
    size_u = size_g * w.abs()
    size = r * (size_u + n.abs() * (size_u * n.abs()).mean(dim=-1, keepdim=True))
    return dx, size, (g * n).sum(dim=(0, 1)), (size_g * n.abs()).sum(dim=(0, 1))


# ---------------------------------------------------------------------------- linear attention
def tokens_pass(q, k, v, g, scale, state=None):
    """The recurrence itself, token by token, of one sequence and head: q, k [n, dk], v [n, dv].
    ``(o, final)``."""
    s = torch.zeros(q.shape[1], v.shape[1], dtype=torch.float64) if state is None else state.double()
    o = []
    for t in range(len(q)):
        s = torch.exp(torch.as_tensor(g, dtype=torch.float64)) * s + torch.outer(k[t].double(),
                                                                                v[t].double())
        o.append(scale * (q[t].double() @ s))
    return (torch.stack(o) if o else torch.zeros(0, v.shape[1], dtype=torch.float64)), s


def _power(g, n):
    """e^(g n), 1 for n = 0 whatever g."""
    return torch.where(n == 0, 1.0, torch.exp(g * n))


def sequence_pass(a, b, c, g, scale, state=None, reverse=False, chunk=128):
    """One sequence and head: ``o_t = scale * sum_j e^(g |t - j|) (a_t . b_j) c_j`` over j <= t
    (reverse: j >= t) and what a starting state adds, in chunks counted from the first token.

    Returns ``(o, near, far, final, size)``: near and far bound the sums of the terms of o that
    are made of scores and chunk states as they are rounded (near) and of single products (far);
    final is the state that leaves, size bounds its terms.  A state arrives at a reversed pass
    without the decay of a token, and leaves it with that of its last one."""
    a, b, c = a.double(), b.double(), c.double()
    n, da = a.shape
    dc = c.shape[1]
    dev = a.device
    g = torch.as_tensor(float(g), dtype=torch.float64, device=dev)
    s = torch.zeros(da, dc, dtype=torch.float64, device=dev) if state is None else state.double()
    size = s.abs()
    o, near, far = (torch.zeros(n, dc, dtype=torch.float64, device=dev) for _ in range(3))
    starts = list(range(0, n, chunk))
    for x in reversed(starts) if reverse else starts:
        e = min(n, x + chunk)
        m = e - x
        i = torch.arange(m, device=dev, dtype=torch.float64)
        ago = i[None, :] - i[:, None] if reverse else i[:, None] - i[None, :]
        w = torch.where(ago >= 0, _power(g, ago.clamp(min=0)), 0.0)
        since = _power(g, m - 1 - i if reverse else i + 1)[:, None]
        left = _power(g, i + 1 if reverse else m - 1 - i)[:, None]
        aa, bb, cc = a[x:e], b[x:e], c[x:e]
        p = (aa @ bb.T) * w
        o[x:e] = p @ cc + since * (aa @ s)
        near[x:e] = p.abs() @ cc.abs() + since * (aa.abs() @ s.abs())
        far[x:e] = ((aa.abs() @ bb.abs().T) * w) @ cc.abs() + since * (aa.abs() @ size)
        s = _power(g, torch.tensor(float(m), device=dev)) * s + (bb * left).T @ cc
        size = _power(g, torch.tensor(float(m), device=dev)) * size + (bb * left).abs().T @ cc.abs()
    return o * scale, near * abs(scale), far * abs(scale), s, size


def _spans(offsets, tokens):
    if offsets is None:
        return [(0, tokens)]
    e = [min(max(int(x), 0), tokens) for x in offsets.tolist()]
    return [(x, max(x, y)) for x, y in zip(e, e[1:])]


def whole_pass(a, b, c, log_decay, scale, offsets, states=None, reverse=False):
    """``sequence_pass`` of every sequence and head of [T, heads, d] tensors whose heads divide
    those of log_decay; ``states``: a list of [H, da, dc] or None.  The outputs [T, H, dc], 0
    outside the sequences, and [B, H, da, dc]."""
    t, h = a.shape[0], len(log_decay)
    dev = a.device
    spans = _spans(offsets, t)
    made = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)  # noqa: E731
    o, near, far = (made(t, h, c.shape[2]) for _ in range(3))
    final, size = (made(len(spans), h, a.shape[2], c.shape[2]) for _ in range(2))
    for s, (x, e) in enumerate(spans):
        for j in range(h):
            pick = lambda m: m[x:e, j // (h // m.shape[1])]  # noqa: E731
            st = None if states is None or states[s] is None else states[s][j]
            r = sequence_pass(pick(a), pick(b), pick(c), float(log_decay[j].double()), scale, st,
                              reverse)
            o[x:e, j], near[x:e, j], far[x:e, j], final[s, j], size[s, j] = r
    return o, near, far, final, size


def shared(x, heads):
    """Sums over the heads that read one of ``heads``."""
    return x.view(x.shape[0], heads, -1, x.shape[2]).sum(dim=2)


def linear_attention_backward(dy, q, k, v, log_decay, scale, offsets, states=None, dfinal=None):
    """``[(gradient, near, far)] of q, k, v`` (shared heads summed) and ``(dstate, size)``."""
    turned = None if states is None else [s.transpose(1, 2) for s in states]
    dturned = None if dfinal is None else [s.double().transpose(1, 2) / scale for s in dfinal]
    df = None if dfinal is None else [s.double() / scale for s in dfinal]
    dq = whole_pass(dy, v, k, log_decay, scale, offsets, turned)
    dk = whole_pass(v, dy, q, log_decay, scale, offsets, dturned, reverse=True)
    dv = whole_pass(k, q, dy, log_decay, scale, offsets, df, reverse=True)
    grads = [tuple(shared(x, like.shape[1]) for x in r[:3])
             for r, like in ((dq, q), (dk, k), (dv, v))]
    return grads, (dv[3] * scale, dv[4] * abs(scale))
