"""What lies between a layer's query, key and value projections and its output projection when its
tokens are mixed by linear attention, on the GPU alone (C ABI: cpg_norm_rope, cpg_linear_attention,
cpg_linear_attention_step and their gradients).

    qkv = (x @ w_qkv.T).view(T, heads, d)                       # GemmSM90
    q, k = norm_rope(qkv[:, :Hq], qkv[:, Hq:Hq + Hk], w_q, w_k, table, positions)
    y, _ = linear_attention(q, k, qkv[:, Hq + Hk:], log_decay, scale=d ** -0.5, offsets=offsets)
    ...                                                         # output projection
    y = linear_attention_step(q, k, v, log_decay, states, slots=slots)   # decoding

Heads are [T, heads, channels] tensors with unit channel stride and any other strides, such as
slices of a projection's rows.  Nothing synchronises with the host; every function runs on the
current stream of its tensors' device and keeps nothing between calls, so calls on several streams
and captured graphs are independent.  Outputs must not overlap inputs, but where it is said.  The
reference has no such operators.
"""
import ctypes

import torch

from . import _lib
from ._tensors import (FLOAT_CODES, call, error, float_code, fresh_heads, heads, matrix, ptr,
                       same_heads, vector)


def rope_table(length: int, rotary: int, *, base: float = 10000.0, device="cuda"):
    """Table [length, rotary] (FP32) for ``norm_rope``: the cosines, then the sines of the angles
    ``position * base ** (-2 i / rotary)`` (i < rotary / 2), made in 64 bits."""
    if rotary < 2 or rotary % 2 or length < 0:
        raise error(_lib.CPG_ERR_INVALID_SHAPE, f"rotary {rotary} must be even, length {length}")
    rates = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    angles = torch.arange(length, dtype=torch.float64, device=device)[:, None] * rates
    return torch.cat([angles.cos(), angles.sin()], dim=1).float()


def _weight(name, w, d, device):
    if w is None:
        return None
    float_code(name, w)
    return vector(name, w, (d,), w.dtype, device)


def _norm_rope_args(q, k, q_weight, k_weight, table, positions, eps, interleaved):
    """Checked arguments of both directions, up to the outputs."""
    t, _, d, q_c = heads("q", q)
    float_code("q", q)
    dev = q.device
    k_c = None
    if k is not None:
        if k.dtype != q.dtype:
            raise error(_lib.CPG_ERR_DTYPE, f"k must be {q.dtype} like q, got {k.dtype}")
        _, _, _, k_c = heads("k", k, dev, tokens=t, channels=d)
    elif k_weight is not None:
        raise error(_lib.CPG_ERR_NULL, "k_weight without k")
    given = [w for w in (q_weight, k_weight) if w is not None]
    if len(given) == 2 and given[0].dtype != given[1].dtype:
        raise error(_lib.CPG_ERR_DTYPE, "q_weight and k_weight must have one type")
    wq, wk = _weight("q_weight", q_weight, d, dev), _weight("k_weight", k_weight, d, dev)
    w_code = FLOAT_CODES[given[0].dtype] if given else _lib.CPG_DTYPE_F32
    rows, rotary, ld = 0, 0, 0
    if table is not None:
        rows, rotary, ld = matrix("table", table, None, dev)
        if table.dtype != torch.float32:
            raise error(_lib.CPG_ERR_DTYPE, f"table must be FP32, got {table.dtype}")
        if rotary > d or rotary % 2:
            raise error(_lib.CPG_ERR_INVALID_SHAPE,
                        f"table has {rotary} columns: an even number, at most {d}")
    vector("positions", positions, (t,), torch.int32, dev)
    return t, d, q_c, k_c, (t, d, wq, wk, w_code, float(eps), ptr(table), rows, ld, rotary,
                            ptr(positions), 1 if interleaved else 0)


def _pair_outputs(out, q, k, q_name, k_name):
    """Outputs like q and k (k may be None) and their descriptions."""
    if out is None:
        q_out, qo = fresh_heads(q)
        k_out, ko = (None, None) if k is None else fresh_heads(k)
    else:
        q_out, k_out = out
        qo = same_heads(q_name, q_out, q.shape, q.dtype, q.device)
        ko = None if k is None else same_heads(k_name, k_out, k.shape, k.dtype, q.device)
    return q_out, k_out, qo, ko


def norm_rope(q, k, q_weight, k_weight, table, positions, *, eps: float = 1e-6,
              interleaved: bool = False, out=None):
    """Norm and rotation of every head: ``y = R(x / sqrt(mean(x^2) + eps) * weight)``.

    ``q`` [T, Hq, d] and ``k`` [T, Hk, d] (or None), BF16 or FP32, 2 <= d <= 256; their weights [d],
    BF16 or FP32, or None for ones.  ``table`` FP32 [P, R] (``rope_table``; None: no rotation)
    holds R / 2 cosines and R / 2 sines for every position; R turns channels i and i + R / 2 into
    one another, or 2i and 2i + 1 when ``interleaved``, and leaves the channels from R on.
    ``positions`` int32 [T]; one outside [0, P) makes the turned channels of its heads NaN.
    Returns ``(q_out, k_out)``, contiguous unless given as ``out``; ``out`` may be ``(q, k)``."""
    t, d, q_c, k_c, args = _norm_rope_args(q, k, q_weight, k_weight, table, positions, eps,
                                           interleaved)
    q_out, k_out, qo, ko = _pair_outputs(out, q, k, "q's output", "k's output")
    call(_lib.load().cpg_norm_rope, "norm_rope", q.device, q_c, k_c, *args, qo, ko)
    return q_out, k_out if k is not None else None


def norm_rope_backward(dq, dk, q, k, q_weight, k_weight, table, positions, *, eps: float = 1e-6,
                       interleaved: bool = False, out=None):
    """Gradient of ``norm_rope`` (same arguments) from ``dq`` and ``dk``, the gradients of its
    outputs.  Returns ``(dq_in, dk_in, dq_weight, dk_weight)``: the first two in q's type (``out``:
    a pair to write them to, which may be ``(dq, dk)``), the weights' in FP32 [d], None for weights
    that are None.  The weights' sums run in a fixed order."""
    t, d, q_c, k_c, args = _norm_rope_args(q, k, q_weight, k_weight, table, positions, eps,
                                           interleaved)
    dev = q.device
    dq_c = same_heads("dq", dq, q.shape, q.dtype, dev)
    dk_c = None if k is None else same_heads("dk", dk, k.shape, k.dtype, dev)
    dq_in, dk_in, qo, ko = _pair_outputs(out, q, k, "dq_in", "dk_in")
    dwq = None if q_weight is None else torch.empty(d, dtype=torch.float32, device=dev)
    dwk = None if k_weight is None else torch.empty(d, dtype=torch.float32, device=dev)
    lib = _lib.load()
    size = ctypes.c_int64()
    _lib.check(lib.cpg_norm_rope_workspace(t, q.shape[1], 0 if k is None else k.shape[1], d,
                                           ctypes.byref(size)), "norm_rope_backward")
    work = torch.empty(size.value, dtype=torch.uint8, device=dev)
    call(lib.cpg_norm_rope_backward, "norm_rope_backward", dev, dq_c, dk_c, q_c, k_c, *args, qo, ko,
         ptr(dwq), ptr(dwk), ptr(work), size.value)
    return dq_in, dk_in if k is not None else None, dwq, dwk


def _linear_args(q, k, v, log_decay, scale, sequences):
    """The problem and the operands of ``linear_attention``."""
    t, _, dk, q_c = heads("q", q)
    dev = q.device
    _, _, _, k_c = heads("k", k, dev, tokens=t, channels=dk)
    _, _, dv, v_c = heads("v", v, dev, tokens=t)
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.dtype != torch.bfloat16:
            raise error(_lib.CPG_ERR_DTYPE, f"{name} must be BF16, got {x.dtype}")
    if log_decay is None or log_decay.dim() != 1:
        raise error(_lib.CPG_ERR_INVALID_SHAPE, "log_decay must be FP32 [heads]")
    h = log_decay.shape[0]
    vector("log_decay", log_decay, (h,), torch.float32, dev)
    for what, n in (("sequences", sequences), ("heads", h)):
        if n >= 1 << 31:  # ctypes would wrap it
            raise error(_lib.CPG_ERR_INVALID_SHAPE, f"{n} {what}")
    problem = _lib.LinearProblemC(t, sequences, h, dk, dv, float(scale))
    return ctypes.byref(problem), problem, q_c, k_c, v_c


def _sequences(offsets, device):
    if offsets is None:
        return 1
    if offsets.dim() != 1 or offsets.shape[0] < 1:
        raise error(_lib.CPG_ERR_INVALID_SHAPE, "offsets must be int32 [sequences + 1]")
    vector("offsets", offsets, tuple(offsets.shape), torch.int32, device)
    return offsets.shape[0] - 1


def _slots(slots, n, device):
    return None if slots is None else vector("slots", slots, (n,), torch.int32, device)


def _attention_output(out, v, problem):
    """``out`` [tokens, heads, dv], or a new one in v's type, and its description."""
    if out is None:
        return fresh_heads(v, heads=problem.heads)
    if out.dtype not in FLOAT_CODES:
        raise error(_lib.CPG_ERR_DTYPE, f"out must be BF16 or FP32, got {out.dtype}")
    shape = (problem.tokens, problem.heads, problem.dv)
    return out, same_heads("out", out, shape, out.dtype, v.device)


def _states(name, s, problem, n, slots, device):
    """A pool of FP32 states [places, heads, dk, dv] (places = n without slots)."""
    if s is None:
        return None
    places = n if slots is None else (s.shape[0] if s.dim() == 4 else 0)
    vector(name, s, (places, problem.heads, problem.dk, problem.dv), torch.float32, device)
    return ctypes.byref(_lib.StatesC(ptr(s), ptr(slots), places))


def linear_attention(q, k, v, log_decay, *, scale: float = 1.0, offsets=None, state=None,
                     slots=None, final=None, out=None):
    """Linear attention with one decay per head over packed sequences, each head and sequence apart:
    ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T``, ``o_t = scale * S_t^T q_t`` (S in FP32).

    ``q``, ``k`` [T, Hq, dk] and [T, Hk, dk], ``v`` [T, Hv, dv], BF16; ``log_decay`` FP32 [H], at
    most 0 (-inf: no state is kept); Hq, Hk and Hv divide H (at most 2^20), and head h reads head
    h // (H // Hx) of each.  dk and dv are
    multiples of 8 up to 128, addresses and strides multiples of 16 bytes.
    ``offsets`` int32 [B + 1], read on the device: sequence b is the rows
    ``offsets[b] <= t < offsets[b + 1]`` (None: one sequence of all rows), cut to the rows that
    there are and empty where it would end before it starts; no two may overlap.  Rows outside are
    0 in an ``out`` that is allocated here and left as they were in one that is given.
    ``state`` FP32 [B, H, dk, dv]: where the sequences start (None: zeros); ``final``: True, or a
    tensor like it, gets the states after their last tokens.  With ``slots`` (int32 [B]) both are
    pools [places, H, dk, dv] and sequence b is at ``slots[b]``; one outside the pool starts from
    zeros and is not written.  ``final`` may be ``state``; no two sequences may share a place there.
    Returns ``(out, final)``: ``out`` [T, H, dv] BF16 (FP32 if it is given so).
    Products are taken of BF16 values: the decayed scores (two parts of each in calls of few chunks
    of 128 tokens or of sequences of up to four tokens) and the state before each 128 tokens are
    rounded to BF16 for them, all sums and the states kept are FP32.  An infinity or a NaN in ``v``
    makes its channel NaN from its token on, and no output before it."""
    dev = q.device
    b = _sequences(offsets, dev)
    p, problem, q_c, k_c, v_c = _linear_args(q, k, v, log_decay, scale, b)
    _slots(slots, b, dev)
    fresh = out is None
    out, o_c = _attention_output(out, v, problem)
    if final is True:
        if slots is not None:
            raise error(_lib.CPG_ERR_UNSUPPORTED, "with slots, final must be a pool to write to")
        final = torch.empty((b, problem.heads, problem.dk, problem.dv), dtype=torch.float32,
                            device=dev)
    elif final is False:
        final = None
    s_c = _states("state", state, problem, b, slots, dev)
    f_c = _states("final", final, problem, b, slots, dev)
    lib = _lib.load()
    size = ctypes.c_int64()
    _lib.check(lib.cpg_linear_attention_workspace(p, q.shape[1], k.shape[1], v.shape[1], 0,
                                                  ctypes.byref(size)), "linear_attention")
    work = torch.empty(size.value, dtype=torch.uint8, device=dev) if size.value else None
    call(lib.cpg_linear_attention, "linear_attention", dev, p, q_c, k_c, v_c, ptr(log_decay),
         ptr(offsets), s_c, f_c, o_c, ptr(work), size.value)
    if fresh and offsets is not None:
        call(lib.cpg_linear_attention_clear, "linear_attention", dev, p, o_c, ptr(offsets))
    return out, final


def linear_attention_backward(dy, q, k, v, log_decay, *, scale: float = 1.0, offsets=None,
                              state=None, dfinal=None, dstate=None, out=None):
    """Gradient of ``linear_attention`` (same q, k, v, log_decay, scale, offsets and state, without
    slots) from ``dy`` (BF16 [T, H, dv]) and, where final states were used, ``dfinal`` (FP32
    [B, H, dk, dv]).  Returns ``(dq, dk, dv, dstate)``: BF16 gradients shaped like q, k and v,
    summed in FP32 over the heads that share one and rounded once; ``dstate`` FP32 like ``state``,
    None if there is neither a ``state`` nor a ``dstate`` to write to.  Rows outside the sequences
    get the gradient 0; in tensors given as ``out`` (a triple) they are left as they were.  The
    decays are constants of the layer and get no gradient."""
    dev = q.device
    b = _sequences(offsets, dev)
    p, problem, q_c, k_c, v_c = _linear_args(q, k, v, log_decay, scale, b)
    y_c = same_heads("dy", dy, (problem.tokens, problem.heads, problem.dv), torch.bfloat16, dev)
    fresh = out is None
    if fresh:
        out, outs = zip(*(fresh_heads(x) for x in (q, k, v)))
    else:
        outs = [same_heads(name, x, like.shape, torch.bfloat16, dev)
                for name, x, like in zip(("dq", "dk", "dv"), out, (q, k, v))]
    if dstate is None and state is not None:
        dstate = torch.empty((b, problem.heads, problem.dk, problem.dv), dtype=torch.float32,
                             device=dev)
    s_c = _states("state", state, problem, b, None, dev)
    f_c = _states("dfinal", dfinal, problem, b, None, dev)
    d_c = _states("dstate", dstate, problem, b, None, dev)
    lib = _lib.load()
    size = ctypes.c_int64()
    _lib.check(lib.cpg_linear_attention_workspace(p, q.shape[1], k.shape[1], v.shape[1], 1,
                                                  ctypes.byref(size)), "linear_attention_backward")
    work = torch.empty(size.value, dtype=torch.uint8, device=dev) if size.value else None
    call(lib.cpg_linear_attention_backward, "linear_attention_backward", dev, p, y_c, q_c, k_c, v_c,
         ptr(log_decay), ptr(offsets), s_c, f_c, *outs, d_c, 1 if fresh else 0, ptr(work),
         size.value)
    return (*out, dstate)


def status(device=None) -> int:
    """0, or the code of the first wait within a linear attention kernel that ever ran out on this
    CUDA device (None: the current one); the outputs of that call are not valid.  Synchronises."""
    code = ctypes.c_int32()
    with torch.cuda.device(device):
        _lib.check(_lib.load().cpg_attention_status(ctypes.byref(code)), "status")
    return code.value


def set_timeout_ms(ms: int) -> None:
    """Limit of every wait within the linear attention kernels that this process launches from now on
    (10 s, or CPG_WAIT_TIMEOUT_MS from the environment)."""
    _lib.check(_lib.load().cpg_attention_set_timeout_ms(int(ms)), "set_timeout_ms")


def set_fault_injection(flags: int) -> None:
    """Test hook (see cpg_attention_set_fault_injection): 1 = no loads, 2 = none of v's tiles."""
    _lib.check(_lib.load().cpg_attention_set_fault_injection(int(flags)), "set_fault_injection")


def linear_attention_step(q, k, v, log_decay, state, *, scale: float = 1.0, slots=None, out=None):
    """One token of each of T sequences: ``state`` (FP32 [T, H, dk, dv], or with ``slots`` int32 [T]
    a pool [places, H, dk, dv]) is updated in place by ``S <- exp(log_decay) S + k v^T`` and
    ``o = scale * S^T q`` [T, H, dv] is returned (BF16, or ``out``, BF16 or FP32).  Heads, sizes and
    alignment as for ``linear_attention``.  A token whose slot is outside the pool is padding: its
    out is 0.  No two tokens may name the same slot."""
    dev = q.device
    p, problem, q_c, k_c, v_c = _linear_args(q, k, v, log_decay, scale, 0)
    t = problem.tokens
    _slots(slots, t, dev)
    out, o_c = _attention_output(out, v, problem)
    if state is None:
        raise error(_lib.CPG_ERR_NULL, "state must be given")
    s_c = _states("state", state, problem, t, slots, dev)
    call(_lib.load().cpg_linear_attention_step, "linear_attention_step", dev, p, q_c, k_c, v_c,
         ptr(log_decay), s_c, o_c)
    return out
