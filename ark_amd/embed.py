"""The lookup of tokens in an embedding table and its gradient
(include/ark_embed.h) for torch tensors.

``lookup(table, tokens, scale)`` gives the tokens' rows, scaled;
``lookup_grad(dy, tokens, vocab, scale)`` the table's gradient in float32, new or
added into the gradients an optimizer steps on.  Tokens outside the table (-1 for
padding, say) have rows of zeros and give no gradient.  No call records an
autograd graph: ``lookup`` refuses a table that requires grad while one is
recorded.
"""
import ctypes as C
import functools

import torch

from . import _abi
from ._lib import check, lib
from .act import _code, _queue, _rows
from .rope import _no_graph

_INTEGERS = {torch.int32: 4, torch.int64: 8}


def _tokens(tokens, device):
    size = _INTEGERS.get(tokens.dtype)
    if size is None or tokens.device != device or not tokens.is_contiguous():
        raise ValueError(f"tokens must be contiguous int32 or int64 on {device}, not "
                         f"{tokens.dtype} on {tokens.device} of strides {tokens.stride()}")
    return tokens.data_ptr(), size, tokens.numel()


def _flat(t, shape, what):
    """t, of ``shape`` and one more dimension, as (address, stride) of its rows."""
    if not t.dim() or t.shape[:-1] != shape:
        raise ValueError(f"{what} is {tuple(t.shape)}, the tokens {tuple(shape)}")
    if t.dim() != 2:
        try:
            t = t.view(shape.numel(), t.shape[-1])
        except RuntimeError:
            raise ValueError(f"{what}: rows of {tuple(t.shape)} at strides {t.stride()} are not one "
                             "stride apart: pass a contiguous copy") from None
    return _rows(t, what)


def lookup(table, tokens, scale=1.0, dtype=None, out=None):
    """scale * table[tokens], contiguous tokens of any shape: (*tokens.shape, columns)
    of the table's type or ``dtype``, in ``out`` (its rows one stride apart) or a new
    tensor."""
    if table.requires_grad:
        _no_graph("lookup")
    tp, tstride = _rows(table, "table")
    kp, size, n = _tokens(tokens, table.device)
    vocab, columns = table.shape
    if out is None:
        out = table.new_empty((*tokens.shape, columns), dtype=dtype or table.dtype)
        op, ostride = out.data_ptr(), columns
    elif (out.shape[-1:] != (columns,) or out.device != table.device
          or dtype not in (None, out.dtype)):
        raise ValueError(f"out is {tuple(out.shape)} {out.dtype} on {out.device}")
    else:
        op, ostride = _flat(out, tokens.shape, "out")
    _queue(table, lib().ark_embed_lookup, tp, tstride, _code(table, "table"), vocab, columns, kp,
           size, n, scale, op, ostride, _code(out, "out"))
    return out


@functools.lru_cache(maxsize=256)
def _workspace(n, vocab, columns):
    need = C.c_uint64()
    check(lib().ark_embed_grad_workspace(n, vocab, columns, C.byref(need)))
    return need.value


def lookup_grad(dy, tokens, vocab, scale=1.0, dw=None, accumulate=False):
    """dw (+)= scale * the sums of dy's rows (*tokens.shape, columns) by token:
    float32 (vocab, columns), rows of any stride; a new tensor when None.  (dy's rows
    are one stride apart, whatever the tokens' shape.)  Rows of tokens that do not
    occur become zeros, or stay with ``accumulate``."""
    kp, size, n = _tokens(tokens, dy.device)
    yp, ystride = _flat(dy, tokens.shape, "dy")
    columns = dy.shape[-1]
    if dw is None:
        if accumulate:
            raise ValueError("accumulate needs a dw")
        dw = dy.new_empty((vocab, columns), dtype=torch.float32)
        wp, wstride = dw.data_ptr(), columns
    elif tuple(dw.shape) != (vocab, columns) or dw.dtype != torch.float32 or dw.device != dy.device:
        raise ValueError(f"dw is {tuple(dw.shape)} {dw.dtype}, not {(vocab, columns)} float32")
    else:
        wp, wstride = _rows(dw, "dw")
    need = _workspace(n, vocab, columns)
    ws = dy.new_empty(need, dtype=torch.uint8)
    _queue(dy, lib().ark_embed_grad, yp, ystride, _code(dy, "dy"), kp, size, n, vocab, columns,
           scale, wp, wstride, _abi.EMBED_ACCUMULATE if accumulate else 0, ws.data_ptr(), need)
    return dw
