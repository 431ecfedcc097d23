"""FP8 E4M3 and INT8 quantisation and FP32 -> BF16 cast on the GPU (C ABI: cpg_quantize_e4m3,
cpg_quantize_int8, cpg_cast_f32_bf16).

``quantize_e4m3(x, block=None)`` returns ``(q, scales)`` with ``s = amax(|x|) / 448`` per tensor
(``block=None``), per 1 x 128 block (``block=(1, 128)``, the A operand of block-scaled FP8
GEMM) or per 128 x 128 block (``block=(128, 128)``, the B operand), and ``q = e4m3(x / s)``.
Scale layouts are described in ``include/cpgemm.h``.

``quantize_int8(x)`` returns ``(q, scales)`` with one scale per row, ``s = amax(|x|) / 127``, and
``q = rint(x / s)``: the scales of the tokens of A, or of the output channels of a weight B.
"""
from typing import Optional, Tuple

import torch

from . import _lib
from ._tensors import call, float_code, matrix, output, ptr, vector


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def quantize_e4m3(x, block: Optional[Tuple[int, int]] = None):
    if not x.is_cuda or x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float32):
        raise _lib.CpgError(_lib.CPG_ERR_DTYPE, "x must be a 2-D BF16 or FP32 CUDA tensor")
    if x.numel() and x.stride(1) != 1:
        raise _lib.CpgError(_lib.CPG_ERR_UNSUPPORTED, "x must have unit column stride")
    rows, cols = x.shape
    q = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device=x.device)
    br, bc = (0, 0) if block is None else block
    if (br, bc) == (0, 0):
        scales = torch.empty(1, dtype=torch.float32, device=x.device)
    elif (br, bc) == (1, 128):
        scales = torch.empty(-(-cols // 128), rows, dtype=torch.float32, device=x.device)
    elif (br, bc) == (128, 128):
        scales = torch.empty(-(-rows // 128), -(-cols // 128), dtype=torch.float32, device=x.device)
    else:
        raise _lib.CpgError(_lib.CPG_ERR_UNSUPPORTED, f"block {block} not supported")
    dt = _lib.CPG_DTYPE_BF16 if x.dtype == torch.bfloat16 else _lib.CPG_DTYPE_F32
    ldx = x.stride(0) if rows > 1 else cols
    lib = _lib.load()
    _lib.check(lib.cpg_quantize_e4m3(x.data_ptr() if x.numel() else None, dt, rows, cols, ldx,
                                     q.data_ptr() if q.numel() else None, cols, scales.data_ptr(),
                                     br, bc, _stream(x)), "quantize_e4m3")
    return q, scales


def alloc_operand_rows(rows: int, cols: int, dtype, device):
    """[rows, cols] whose rows start on 16 bytes, as the GEMM's loads need."""
    per16 = 16 // dtype.itemsize
    if cols % per16 == 0:
        return torch.empty((rows, cols), dtype=dtype, device=device)
    return torch.empty((rows, -(-cols // per16) * per16), dtype=dtype, device=device)[:, :cols]


def quantize_int8(x, out=None, scales=None):
    """INT8 rows of a 2-D BF16 or FP32 CUDA tensor and their FP32 scales [rows], on the current
    stream.  ``q`` has rows padded to 16 bytes, ready for the GEMM; ``out`` (int8, x's shape, unit
    column stride) and ``scales`` may be given as outputs.  Rows of zeros get q = 0 and a tiny
    scale; a row that holds an infinity or NaN gets q = 0 and the scale NaN."""
    code = float_code("x", x)
    rows, cols, ldx = matrix("x", x)
    device = x.device
    if out is None:
        out = alloc_operand_rows(rows, cols, torch.int8, device)
        ldq = out.stride(0) if rows > 1 else cols
    else:
        ldq = output("out", out, (rows, cols), torch.int8, device)
    if scales is None:
        scales = torch.empty(rows, dtype=torch.float32, device=device)
    else:
        vector("scales", scales, (rows,), torch.float32, device)
    call(_lib.load().cpg_quantize_int8, "quantize_int8", device, ptr(x),
              code, rows, cols, ldx, ptr(out), ldq, ptr(scales))
    return out, scales


def cast_f32_bf16(x, bias=None, out=None, stream=None):
    """out = bf16(x + bias) for a 2-D FP32 CUDA tensor x (on ``stream``, default current)."""
    if not x.is_cuda or x.dim() != 2 or x.dtype != torch.float32:
        raise _lib.CpgError(_lib.CPG_ERR_DTYPE, "x must be a 2-D FP32 CUDA tensor")
    rows, cols = x.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=torch.bfloat16, device=x.device)
    elif out.dtype != torch.bfloat16 or out.shape != x.shape or out.device != x.device:
        raise _lib.CpgError(_lib.CPG_ERR_INVALID_SHAPE,
                            f"out must be BF16 of shape {tuple(x.shape)} on {x.device}")
    for name, t in (("x", x), ("out", out)):
        if t.numel() and cols > 1 and t.stride(1) != 1:
            raise _lib.CpgError(_lib.CPG_ERR_UNSUPPORTED, f"{name} must have unit column stride")
    if bias is not None and not (bias.dtype == torch.bfloat16 and bias.numel() == cols
                                 and bias.device == x.device and bias.is_contiguous()):
        raise _lib.CpgError(_lib.CPG_ERR_INVALID_SHAPE,
                            f"bias must be a contiguous BF16 tensor of length {cols} on {x.device}")
    ldx = x.stride(0) if rows > 1 else cols
    ldy = out.stride(0) if rows > 1 else cols
    lib = _lib.load()
    from .gemm_base import _stream_handle
    st = _stream_handle(stream, x.device)
    _lib.check(lib.cpg_cast_f32_bf16(x.data_ptr() if x.numel() else None, rows, cols, ldx,
                                     out.data_ptr() if out.numel() else None, ldy,
                                     None if bias is None else bias.data_ptr(), st),
               "cast_f32_bf16")
    return out
