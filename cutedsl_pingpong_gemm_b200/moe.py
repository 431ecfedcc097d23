"""What surrounds the experts' products of an MoE layer (``GemmSM90.grouped``), on the GPU alone (C
ABI: cpg_route, cpg_expert_order, cpg_dispatch_rows, cpg_combine_rows and their gradients).

    ids, weights = route(logits, k)                      # experts and weights of every token
    d = dispatch(x, ids, experts, quantize="int8")       # rows in expert order, group offsets
    gemm.grouped(d.rows, w_up, h, d.offsets, scale_a=d.scales, scale_b=s_up, ...)
    ...
    y = combine(out, d.slots, weights)                   # weighted sum back per token

Nothing synchronises with the host: offsets and slots stay on the device.  Every function runs on
the current stream of its tensors' device and keeps nothing between calls, so calls on several
streams and captured graphs are independent.  Outputs must not overlap inputs, but for ``combine``'s
``source``, which may be ``out``.  Rows may have any alignment and stride (and fewer than 2**30
columns).  Gradients: ``route_backward``, ``combine_backward``; the gradient of ``dispatch`` is
``combine`` of the rows' gradients without weights (a quantised dispatch: of the rows it stands for,
rounding ignored).  The reference has no such operators.
"""
import ctypes
import functools
from collections import namedtuple
from typing import Optional

import torch

from . import _lib
from ._tensors import call, error, float_code, matrix, output, pairs, ptr, vector
from .quant import alloc_operand_rows

Dispatched = namedtuple("Dispatched", "rows offsets slots scales")


@functools.lru_cache(maxsize=256)
def _route_config(experts, k, scoring, groups, kept_groups, group_score, renormalize, scale):
    if scoring not in _lib.ROUTE_SCORINGS:
        raise error(_lib.CPG_ERR_INVALID_CONFIG, f"unknown scoring {scoring!r}")
    if group_score not in _lib.ROUTE_GROUP_SCORES:
        raise error(_lib.CPG_ERR_INVALID_CONFIG, f"unknown group_score {group_score!r}")
    for name, v in (("experts", experts), ("k", k), ("groups", groups),
                    ("kept_groups", kept_groups)):
        if abs(v) >= 1 << 31:  # ctypes would wrap it
            raise error(_lib.CPG_ERR_INVALID_SHAPE, f"{name} = {v}")
    return ctypes.byref(_lib.RouteConfigC(
        experts, k, _lib.ROUTE_SCORINGS[scoring], groups, kept_groups,
        _lib.ROUTE_GROUP_SCORES[group_score], 1 if renormalize else 0, scale))


def route(logits, k: int, *, scoring: str = "softmax", bias=None, groups: int = 1,
          kept_groups: Optional[int] = None, group_score: Optional[str] = None,
          renormalize: bool = True, scale: float = 1.0, ids=None, weights=None):
    """Choose ``k`` of the E experts for every row of ``logits`` [T, E] (BF16 or FP32).

    Returns ``(ids, weights)``, int32 and FP32 [T, k], best first: the experts with the largest
    ``scoring(logits) + bias`` ("softmax" over all experts, or "sigmoid"; ties to the lowest index)
    and ``scale * score``, over the sum of the chosen scores when ``renormalize``.  ``bias`` (FP32
    [E]) only ranks.  ``groups`` > 1 first keeps the best ``kept_groups`` groups of E / groups
    consecutive experts, a group counting as its best expert ("max") or its two best ("top2";
    the default with a bias).  A logit of -inf masks an expert; where fewer than k are left the
    last ids are -1 with weight 0.  A NaN logit makes the row's weights NaN (under the softmax
    +inf too).  E <= 1024, k and groups <= 32.  ``ids`` / ``weights`` may be given as outputs."""
    t, e, ld = matrix("logits", logits)
    code = float_code("logits", logits)
    dev = logits.device
    k = int(k)
    if group_score is None:
        group_score = "top2" if bias is not None else "max"
    cfg = _route_config(e, k, scoring, int(groups),
                        int(groups if kept_groups is None else kept_groups), group_score,
                        bool(renormalize), float(scale))
    if bias is not None:
        vector("bias", bias, (e,), torch.float32, dev)
    shape = (t, max(k, 0))
    if ids is None:
        ids = torch.empty(shape, dtype=torch.int32, device=dev)
    else:
        vector("ids", ids, shape, torch.int32, dev)
    if weights is None:
        weights = torch.empty(shape, dtype=torch.float32, device=dev)
    else:
        vector("weights", weights, shape, torch.float32, dev)
    call(_lib.load().cpg_route, "route", dev, cfg, ptr(logits), code, t, ld, ptr(bias),
          ptr(ids), ptr(weights))
    return ids, weights


def route_backward(dweights, logits, ids, *, scoring: str = "softmax", renormalize: bool = True,
                   scale: float = 1.0, out=None):
    """Gradient of ``route``'s weights: ``dlogits`` [T, E] in the logits' type from ``dweights``
    (FP32 [T, k]) for the choices ``ids`` of the forward call (same scoring, renormalize, scale).
    Entries of ``ids`` that are no expert take no part; an expert given twice counts twice."""
    t, e, ld = matrix("logits", logits)
    code = float_code("logits", logits)
    dev = logits.device
    _, k = pairs("ids", ids)
    vector("ids", ids, (t, k), torch.int32, dev)
    vector("dweights", dweights, (t, k), torch.float32, dev)
    cfg = _route_config(e, k, scoring, 1, 1, "max", bool(renormalize), float(scale))
    if out is None:
        out, ldd = torch.empty((t, e), dtype=logits.dtype, device=dev), e
    else:
        ldd = output("out", out, (t, e), logits.dtype, dev)
    call(_lib.load().cpg_route_backward, "route_backward", dev, cfg, ptr(dweights),
          ptr(logits), code, t, ld, ptr(ids), ptr(out), ldd)
    return out


def dispatch(x, ids, experts: int, *, quantize: Optional[str] = None, out=None, scales=None,
             offsets=None, slots=None):
    """Rows of ``x`` [T, D] (BF16 or FP32) in expert order, for ``GemmSM90.grouped``.

    ``ids`` int32 [T, k] gives each token's experts (entries outside [0, experts) are skipped).
    Returns ``Dispatched(rows, offsets, slots, scales)``: ``rows`` [T * k, D] holds the rows of
    expert e at ``offsets[e] <= r < offsets[e + 1]`` (int32 [experts + 1]) in token order, ``slots``
    int32 [T, k] the row of every (token, choice), -1 if skipped.  Rows from ``offsets[experts]``
    on are not written (undefined without a given ``out``).  BF16 and INT8 rows that it allocates
    are padded to 16 bytes, as the product needs.  ``quantize="int8"`` makes ``rows`` the int8 rows
    and ``scales`` (FP32 [T * k]) the scales of ``quant.quantize_int8``; otherwise ``scales`` is
    None.  ``out`` / ``scales`` / ``offsets`` / ``slots`` may be given as outputs.  experts <= 1024,
    k <= 32."""
    t, d, ldx = matrix("x", x)
    code = float_code("x", x)
    dev = x.device
    if quantize not in (None, "int8"):
        raise error(_lib.CPG_ERR_UNSUPPORTED, f"quantize must be None or 'int8', got {quantize!r}")
    _, k = pairs("ids", ids)
    vector("ids", ids, (t, k), torch.int32, dev)
    experts = int(experts)
    if experts < 1 or experts > _lib.CPG_ROUTE_MAX_EXPERTS:
        raise error(_lib.CPG_ERR_INVALID_SHAPE,
                     f"1 <= experts <= {_lib.CPG_ROUTE_MAX_EXPERTS}, got {experts}")
    int8 = quantize == "int8"
    dtype = torch.int8 if int8 else x.dtype
    if out is None:
        # FP32 rows are no operand of a product: without padding.
        out = (torch.empty((t * k, d), dtype=dtype, device=dev) if dtype == torch.float32
               else alloc_operand_rows(t * k, d, dtype, dev))
    ldr = output("out", out, (t * k, d), dtype, dev)
    if int8:
        if scales is None:
            scales = torch.empty(t * k, dtype=torch.float32, device=dev)
        else:
            vector("scales", scales, (t * k,), torch.float32, dev)
    elif scales is not None:
        raise error(_lib.CPG_ERR_UNSUPPORTED, "scales only with quantize='int8'")
    if offsets is None:
        offsets = torch.empty(experts + 1, dtype=torch.int32, device=dev)
    else:
        vector("offsets", offsets, (experts + 1,), torch.int32, dev)
    if slots is None:
        slots = torch.empty((t, k), dtype=torch.int32, device=dev)
    else:
        vector("slots", slots, (t, k), torch.int32, dev)
    slots_ptr = ptr(slots)
    lib = _lib.load()
    call(lib.cpg_expert_order, "dispatch", dev, ptr(ids), t, k, experts, offsets.data_ptr(),
         slots_ptr)
    call(lib.cpg_dispatch_rows, "dispatch", dev, ptr(x), code, t, d, ldx, slots_ptr, k, ptr(out),
         _lib.CPG_DTYPE_I8 if int8 else code, t * k, ldr, ptr(scales))
    return Dispatched(out, offsets, slots, scales)


def combine(rows, slots, weights=None, *, source=None, out=None):
    """``y[t] = source[t] + sum_j weights[t, j] * rows[slots[t, j]]`` (FP32 sums, rounded once).

    ``rows`` [R, D] BF16 or FP32, ``slots`` int32 [T, k] (entries outside [0, R) are not read),
    ``weights`` FP32 [T, k] or None for ones, ``source`` an optional [T, D] of the rows' type
    (it may be ``out``), such as a shared expert's output."""
    r, d, ldr = matrix("rows", rows)
    code = float_code("rows", rows)
    dev = rows.device
    t, k = pairs("slots", slots)
    vector("slots", slots, (t, k), torch.int32, dev)
    if weights is not None:
        vector("weights", weights, (t, k), torch.float32, dev)
    lds = 0
    if source is not None:
        _, _, lds = matrix("source", source, (t, d), dev)
        if source.dtype != rows.dtype:
            raise error(_lib.CPG_ERR_DTYPE, f"source must be {rows.dtype} like rows")
    if out is None:
        out, ldy = torch.empty((t, d), dtype=rows.dtype, device=dev), d
    else:
        ldy = output("out", out, (t, d), rows.dtype, dev)
    call(_lib.load().cpg_combine_rows, "combine", dev, ptr(rows), code, r, d, ldr, ptr(slots),
          ptr(weights), t, k, ptr(source), lds, ptr(out), ldy)
    return out


def combine_backward(dy, rows, slots, weights, *, drows=None, dweights=None):
    """Gradients of ``combine``: ``drows[slots[t, j]] = weights[t, j] * dy[t]`` [R, D], 0 in the rows
    that no slot names, and ``dweights[t, j] = <dy[t], rows[slots[t, j]]>`` FP32 [T, k].  No two
    slots may be the same row (``dispatch`` makes none).  ``drows`` / ``dweights`` may be given as
    outputs; rows of a given ``drows`` that no slot names are left as they were."""
    t, d, lddy = matrix("dy", dy)
    code = float_code("dy", dy)
    dev = dy.device
    r, cols, ldr = matrix("rows", rows, None, dev)
    if cols != d or rows.dtype != dy.dtype:
        raise error(_lib.CPG_ERR_INVALID_SHAPE if cols != d else _lib.CPG_ERR_DTYPE,
                     f"rows must be [R, {d}] {dy.dtype} like dy, got {tuple(rows.shape)} "
                     f"{rows.dtype}")
    _, k = pairs("slots", slots)
    vector("slots", slots, (t, k), torch.int32, dev)
    vector("weights", weights, (t, k), torch.float32, dev)
    fresh = drows is None
    if fresh:
        drows, lddr = torch.empty((r, d), dtype=dy.dtype, device=dev), d
    else:
        lddr = output("drows", drows, (r, d), dy.dtype, dev)
    if dweights is None:
        dweights = torch.empty((t, k), dtype=torch.float32, device=dev)
    else:
        vector("dweights", dweights, (t, k), torch.float32, dev)
    lib = _lib.load()
    if fresh:
        call(lib.cpg_clear_unnamed_rows, "combine_backward", dev, ptr(drows), code, r, d, lddr,
             ptr(slots), t, k)
    call(lib.cpg_combine_rows_backward, "combine_backward", dev, ptr(dy), code, t, d,
          lddy, ptr(rows), r, ldr, ptr(slots), ptr(weights), k, ptr(drows), lddr,
          ptr(dweights))
    return drows, dweights
