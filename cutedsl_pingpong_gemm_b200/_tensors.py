"""Checks of tensor arguments and the call into the C ABI on the current stream, shared by the
operators that allocate their outputs (``quant``, ``moe``, ``attention``)."""
import ctypes

import torch

from . import _lib

FLOAT_CODES = {torch.bfloat16: _lib.CPG_DTYPE_BF16, torch.float32: _lib.CPG_DTYPE_F32}


def error(code, message):
    return _lib.CpgError(code, message)


def float_code(name, t):
    code = FLOAT_CODES.get(t.dtype)
    if code is None:
        raise error(_lib.CPG_ERR_DTYPE, f"{name} must be BF16 or FP32, got {t.dtype}")
    return code


def matrix(name, t, shape=None, device=None):
    """A 2-D CUDA tensor with unit column stride (of ``shape``, on ``device``): its rows, columns
    and row stride."""
    if not t.is_cuda:
        raise error(_lib.CPG_ERR_NO_DEVICE, f"{name} must be a CUDA tensor")
    size = t.shape
    if len(size) != 2 or (shape is not None and size != shape):
        raise error(_lib.CPG_ERR_INVALID_SHAPE,
                    f"{name} must be 2-D{'' if shape is None else ' of shape ' + str(tuple(shape))}"
                    f", got {tuple(size)}")
    rows, cols = size
    ld, step = t.stride()
    if step != 1 and rows > 0 and cols > 1:
        raise error(_lib.CPG_ERR_UNSUPPORTED, f"{name} must have unit column stride")
    if device is not None and t.device != device:
        raise other_device(name, t, device)
    return rows, cols, ld if rows > 1 else cols


def other_device(name, t, device):
    return error(_lib.CPG_ERR_NO_DEVICE, f"{name} is on {t.device}, the others on {device}")


def output(name, t, shape, dtype, device):
    """Row stride of a matrix that is written: its rows must not overlap."""
    rows, cols, ld = matrix(name, t, shape, device)
    if t.dtype != dtype:
        raise error(_lib.CPG_ERR_DTYPE, f"{name} must be {dtype}, got {t.dtype}")
    if ld < cols:
        raise error(_lib.CPG_ERR_INVALID_SHAPE, f"{name}'s rows overlap (row stride {ld})")
    return ld


def vector(name, t, shape, dtype, device):
    """A contiguous tensor of this shape and type; its address."""
    if t is None:
        raise error(_lib.CPG_ERR_NULL, f"{name} must be given")
    if not (t.is_cuda and t.dtype == dtype and t.shape == shape and t.is_contiguous()):
        raise error(_lib.CPG_ERR_INVALID_SHAPE,
                    f"{name} must be a contiguous {dtype} CUDA tensor of shape {tuple(shape)}, "
                    f"got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise other_device(name, t, device)
    return t.data_ptr() or None


def pairs(name, t):
    """T and k of the choices [T, k]."""
    size = t.shape
    if len(size) != 2:
        raise error(_lib.CPG_ERR_INVALID_SHAPE, f"{name} must be [T, k], got {tuple(size)}")
    if size[1] > _lib.CPG_ROUTE_MAX_K:  # here: ctypes would wrap a k past 32 bits
        raise error(_lib.CPG_ERR_INVALID_SHAPE,
                    f"{name}: at most {_lib.CPG_ROUTE_MAX_K} choices, got {size[1]}")
    return size


def heads(name, t, device=None, tokens=None, channels=None):
    """Heads [T, H, d] with unit channel stride: T, H, d and the C description."""
    if t is None:
        raise error(_lib.CPG_ERR_NULL, f"{name} must be given")
    if not t.is_cuda:
        raise error(_lib.CPG_ERR_NO_DEVICE, f"{name} must be a CUDA tensor")
    size = t.shape
    if (len(size) != 3 or (tokens is not None and size[0] != tokens)
            or (channels is not None and size[2] != channels)):
        raise error(_lib.CPG_ERR_INVALID_SHAPE,
                    f"{name} must be [{'T' if tokens is None else tokens}, heads, "
                    f"{'channels' if channels is None else channels}], got {tuple(size)}")
    if size[1] >= 1 << 31 or size[2] >= 1 << 31:  # ctypes would wrap it
        raise error(_lib.CPG_ERR_INVALID_SHAPE, f"{name} is {tuple(size)}")
    step = t.stride()
    if step[2] != 1 and size[2] > 1 and size[0] > 0:
        raise error(_lib.CPG_ERR_UNSUPPORTED, f"{name} must have unit channel stride")
    if device is not None and t.device != device:
        raise other_device(name, t, device)
    code = FLOAT_CODES.get(t.dtype, -1)
    return size[0], size[1], size[2], ctypes.byref(
        _lib.HeadsC(t.data_ptr() or None, step[0], step[1], size[1], code))


def fresh_heads(like, heads=None):
    """A contiguous tensor of this shape and type (with another number of heads) and its C
    description."""
    t, h, d = like.shape
    h = h if heads is None else heads
    x = torch.empty((t, h, d), dtype=like.dtype, device=like.device)
    return x, ctypes.byref(_lib.HeadsC(x.data_ptr() or None, h * d, d, h, FLOAT_CODES[x.dtype]))


def same_heads(name, t, shape, dtype, device):
    """C description of heads of this shape and type."""
    if t is None:
        raise error(_lib.CPG_ERR_NULL, f"{name} must be given")
    if t.dtype != dtype:
        raise error(_lib.CPG_ERR_DTYPE, f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise error(_lib.CPG_ERR_INVALID_SHAPE,
                    f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    return heads(name, t, device)[3]


def ptr(t):
    """Address of a tensor; None without one or for an empty one."""
    return None if t is None else t.data_ptr() or None


def call(fn, what, device, *args):
    """Call a C entry point on the current stream of ``device`` (made current for the call)."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc != _lib.CPG_OK:
        _lib.check(rc, what)
