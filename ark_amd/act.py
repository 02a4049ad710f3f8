"""Activations kept in 8 bits for the backward pass (include/ark_act.h) for
torch tensors, and the weight gradient that reads them.

``pack(x)`` keeps a layer's input as an ``Act8`` of half the bytes (a quarter
of fp32's); ``weight_grad(kept, dy)`` is the weight gradient x^T dy from it, in
fp32, written to or added into the gradients an optimizer steps on;
``unpack(kept)`` gives the values back.  No call records an autograd graph: they
take the values of tensors that require grad, and their results are the parts
of a backward pass that its caller writes (an ``autograd.Function``, say).
"""
import ctypes as C
import functools

import torch

from . import _abi
from ._lib import check, lib

_TYPES = {torch.float16: _abi.ACT_F16, torch.bfloat16: _abi.ACT_BF16,
          torch.float32: _abi.ACT_F32}


# By the calls that are not public where this torch has them: a Stream object costs
# as much as queueing a kernel, the public current_device twice as much as this.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _queue(t, call, *args):
    """call(*args, the current stream of t's device) on that device: the library
    launches on the current one, and a default stream is any device's."""
    dev = t.get_device()
    if dev == _device():
        check(call(*args, _raw_stream(dev)))
    else:
        with torch.cuda.device(dev):
            check(call(*args, _raw_stream(dev)))


def _code(t, what):
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} holds {t.dtype}: float16, bfloat16 and float32 are taken")
    return code


def _rows(t, what):
    """(address, row stride) of a 2-D device tensor whose rows are contiguous."""
    if t.dim() != 2:
        raise ValueError(f"{what} has {t.dim()} dimensions, not 2")
    if not t.is_cuda:
        raise ValueError(f"{what} is not a device tensor")
    stride, one = t.stride()
    if one != 1 and t.shape[1] > 1:
        raise ValueError(f"{what}: the values of a row do not follow one another")
    return t.data_ptr(), stride


class Act8:
    """The 8-bit form of a (tokens, columns) array of ``dtype``: ``data`` holds
    33 bytes for every 32 tokens of a column."""

    __slots__ = ("tokens", "columns", "dtype", "data")

    def __init__(self, tokens, columns, dtype, device=None, data=None):
        if dtype not in _TYPES:
            raise ValueError(f"dtype {dtype}: float16, bfloat16 and float32 are taken")
        if tokens < 0 or columns < 0:
            raise ValueError(f"sizes {tokens} x {columns}")
        n = -(-tokens // _abi.ACT_GROUP) * columns * (_abi.ACT_GROUP + 1)
        if data is None:
            data = torch.empty(n, dtype=torch.uint8, device="cuda" if device is None else device)
        elif data.dtype != torch.uint8 or not data.is_contiguous() or data.numel() != n:
            raise ValueError(f"data must be {n} contiguous uint8")
        self.tokens, self.columns, self.dtype, self.data = tokens, columns, dtype, data

    @classmethod
    def _of(cls, tokens, columns, like):
        """A new one of the type and on the device of ``like``."""
        self = cls.__new__(cls)
        self.tokens, self.columns, self.dtype = tokens, columns, like.dtype
        self.data = like.new_empty(-(-tokens // _abi.ACT_GROUP) * columns * (_abi.ACT_GROUP + 1),
                                   dtype=torch.uint8)
        return self

    @property
    def nbytes(self):
        return self.data.numel()


def pack(x, out=None):
    """The 8-bit form of x (tokens x columns, rows of any stride), in ``out``
    (an Act8 of the same sizes and type) or a new one."""
    code = _code(x, "x")
    p, stride = _rows(x, "x")
    t, c = x.shape
    if out is None:
        out = Act8._of(t, c, x)
    elif (out.tokens, out.columns, out.dtype) != (t, c, x.dtype) or out.data.device != x.device:
        raise ValueError(f"out is {out.tokens} x {out.columns} {out.dtype}, x {t} x {c} {x.dtype}")
    _queue(x, lib().ark_act_pack, p, stride, code, t, c, out.data.data_ptr())
    return out


def unpack(kept, out=None):
    """The values of an Act8, in ``out`` (tokens x columns, rows of any stride)
    or a new tensor of the type they were packed from."""
    if out is None:
        out = kept.data.new_empty((kept.tokens, kept.columns), dtype=kept.dtype)
    elif tuple(out.shape) != (kept.tokens, kept.columns) or out.device != kept.data.device:
        raise ValueError(f"out is {tuple(out.shape)}, the activation {kept.tokens} x "
                         f"{kept.columns}")
    p, stride = _rows(out, "out")
    _queue(out, lib().ark_act_unpack, kept.data.data_ptr(), kept.tokens, kept.columns,
           _code(out, "out"), p, stride)
    return out


@functools.lru_cache(maxsize=256)
def _workspace(tokens, columns, dy_stride, outputs):
    need = C.c_uint64()
    check(lib().ark_act_weight_grad_workspace(tokens, columns, dy_stride, outputs, C.byref(need)))
    return need.value


def weight_grad(kept, dy, dw=None, accumulate=False, layout="in_out"):
    """dw (+)= x^T dy from the Act8 ``kept`` of x (tokens x columns) and dy
    (tokens x outputs; float16 for an activation packed from float16, bfloat16
    for any).  dw is float32, columns x outputs ("in_out") or outputs x columns
    ("out_in"), rows of any stride; a new tensor when None.  accumulate adds to
    it."""
    if layout not in ("in_out", "out_in"):
        raise ValueError(f"layout {layout!r}: 'in_out' or 'out_in'")
    dp, dstride = _rows(dy, "dy")
    if dy.shape[0] != kept.tokens or dy.device != kept.data.device:
        raise ValueError(f"dy has {dy.shape[0]} rows, the activation {kept.tokens}")
    n = dy.shape[1]
    shape = (kept.columns, n) if layout == "in_out" else (n, kept.columns)
    if dw is None:
        if accumulate:
            raise ValueError("accumulate needs a dw")
        dw = dy.new_empty(shape, dtype=torch.float32)
    elif tuple(dw.shape) != shape or dw.dtype != torch.float32 or dw.device != dy.device:
        raise ValueError(f"dw is {tuple(dw.shape)} {dw.dtype}, not {shape} float32")
    wp, wstride = _rows(dw, "dw")
    flags = (_abi.ACT_ACCUMULATE if accumulate else 0) | (
        _abi.ACT_TRANSPOSED if layout == "out_in" else 0)
    need = _workspace(kept.tokens, kept.columns, dstride, n)
    # torch's allocator hands a stream's memory back to it without waiting
    ws = dy.new_empty(need, dtype=torch.uint8) if need else None
    _queue(dy, lib().ark_act_weight_grad_noalloc, kept.data.data_ptr(), _TYPES[kept.dtype],
           kept.tokens, kept.columns, dp, dstride, _code(dy, "dy"), n, wp, wstride, flags,
           ws.data_ptr() if need else None, need)
    return dw
