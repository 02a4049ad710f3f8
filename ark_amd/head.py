"""The loss over a vocabulary from the last hidden rows and the output layer
(include/ark_head.h) for torch tensors, with its gradients, and distillation
from a teacher's top logits.  The logits are never in memory; with gradients
their gradient is, in 16 bits, in pieces of at most 1 GiB.

``cross_entropy(x, w, targets)`` is the loss of every token; with
``cross_entropy_grad`` come the gradients of x and of w (the tied embedding),
the latter into an optimizer's fp32 gradients or in w's own type.  ``distill``
and ``distill_grad`` do the same for the divergence from a teacher.

x is (tokens, columns) and w (vocab, columns), float16 or bfloat16 both, rows of
any stride.  No call records an autograd graph: ``cross_entropy`` and
``distill`` refuse inputs that require grad while one is recorded, and the other
two return what a backward pass needs.
"""
import ctypes as C
import functools

import torch

from . import _abi
from ._lib import check, lib
from .act import _code, _queue, _rows
from .rope import _no_graph

_INTEGERS = {torch.int32: 4, torch.int64: 8}


@functools.lru_cache(maxsize=256)
def _workspace(aligned, w_stride, tokens, columns, vocab, top, dw_dtype, grad):
    need = C.c_uint64()
    check(lib().ark_head_workspace(None if aligned else 2, w_stride, tokens, columns, vocab, top,
                                   dw_dtype, grad, C.byref(need)))
    return need.value


def _inputs(x, w):
    """What a call's arguments begin with."""
    code = _code(x, "x")
    if code == _abi.HEAD_F32 or w.dtype != x.dtype:
        raise ValueError(f"x holds {x.dtype} and w {w.dtype}: both float16, or both bfloat16")
    xp, xs = _rows(x, "x")
    wp, ws = _rows(w, "w")
    if w.shape[1] != x.shape[1] or w.device != x.device:
        raise ValueError(f"x is {tuple(x.shape)} on {x.device}, w {tuple(w.shape)} on {w.device}")
    return xp, xs, wp, ws, code, x.shape[0], x.shape[1], w.shape[0]


def _entries(t, x, what):
    """(address, row stride) of a teacher's indices or logits."""
    if t.dim() != 2 or t.shape[0] != x.shape[0] or t.device != x.device:
        raise ValueError(f"{what} is {tuple(t.shape)} on {t.device}: {x.shape[0]} rows on "
                         f"{x.device}")
    return _rows(t, what)


def _targets(targets, x):
    size = _INTEGERS.get(targets.dtype)
    if (size is None or targets.device != x.device or targets.numel() != x.shape[0]
            or not targets.is_contiguous()):
        raise ValueError(f"targets must be {x.shape[0]} contiguous int32 or int64 on {x.device}, not "
                         f"{tuple(targets.shape)} {targets.dtype} on {targets.device} of strides "
                         f"{targets.stride()}")
    return targets.data_ptr(), size


def _ignored(ignore):
    if not -2 ** 31 <= ignore < 2 ** 31:
        raise ValueError(f"ignore = {ignore} is not an int32")
    return ignore


def _teacher(index, logits, x, temperature):
    size = _INTEGERS.get(index.dtype)
    if size is None:
        raise ValueError(f"index holds {index.dtype}: int32 or int64")
    ip, istride = _entries(index, x, "index")
    lp, lstride = _entries(logits, x, "logits")
    if index.shape != logits.shape:
        raise ValueError(f"index is {tuple(index.shape)}, logits {tuple(logits.shape)}")
    return (ip, size, istride, lp, _code(logits, "logits"), lstride, index.shape[1],
            float(temperature))


def _loss(x, w, call, top, args):
    head = _inputs(x, w)
    need = _workspace(head[2] % 16 == 0, *head[3:4], *head[5:8], top, _abi.HEAD_F32, 0)
    loss = x.new_empty(x.shape[0], dtype=torch.float32)
    ws = x.new_empty(need, dtype=torch.uint8)
    _queue(x, call, *head, *args, loss.data_ptr(), ws.data_ptr(), need)
    return loss


def _loss_grad(x, w, call, top, args, grad, dx, dw, accumulate):
    head = _inputs(x, w)
    grads = None
    if isinstance(grad, torch.Tensor):
        if (grad.dtype != torch.float32 or grad.device != x.device or not grad.is_contiguous()
                or grad.numel() != x.shape[0]):
            raise ValueError(f"grad must be a number or {x.shape[0]} contiguous float32 on "
                             f"{x.device}")
        grads, grad = grad.data_ptr(), 0.0
    if dx is None:
        dx = x.new_empty(x.shape)
    elif dx is not False and (dx.shape != x.shape or dx.dtype != x.dtype or dx.device != x.device):
        raise ValueError(f"dx is {tuple(dx.shape)} {dx.dtype}, x {tuple(x.shape)} {x.dtype}")
    if dw is None:
        if accumulate:
            raise ValueError("accumulate needs a dw")
        dw = w.new_empty(w.shape)
    elif dw is not False and (dw.shape != w.shape or dw.device != x.device
                              or dw.dtype not in (w.dtype, torch.float32)):
        raise ValueError(f"dw is {tuple(dw.shape)} {dw.dtype}, not {tuple(w.shape)} float32 or "
                         f"{w.dtype}")
    xp, xs = (None, 0) if dx is False else _rows(dx, "dx")
    wp, wstride = (None, 0) if dw is False else _rows(dw, "dw")
    code = _abi.HEAD_F32 if dw is False else _code(dw, "dw")
    need = _workspace(head[2] % 16 == 0, *head[3:4], *head[5:8], top, code,
                      _abi.HEAD_GRAD | (0 if dx is False else _abi.HEAD_DX)
                      | (0 if dw is False else _abi.HEAD_DW))
    loss = x.new_empty(x.shape[0], dtype=torch.float32)
    # torch's allocator hands a stream's memory back to it without waiting
    ws = x.new_empty(need, dtype=torch.uint8)
    _queue(x, call, *head, *args, grad, grads, loss.data_ptr(), xp, xs, wp, code, wstride,
           _abi.HEAD_ACCUMULATE if accumulate else 0, ws.data_ptr(), need)
    return loss, None if dx is False else dx, None if dw is False else dw


def cross_entropy(x, w, targets, scale=1.0, ignore=-100):
    """The loss -log softmax(scale * x w^T)[target] of every token, float32.
    Tokens whose target is ``ignore``, or outside the vocabulary, have loss 0."""
    if x.requires_grad or w.requires_grad:
        _no_graph("cross_entropy")
    return _loss(x, w, lib().ark_head_cross_entropy, 1, (*_targets(targets, x), _ignored(ignore), scale))


def cross_entropy_grad(x, w, targets, grad=1.0, scale=1.0, ignore=-100, dx=None, dw=None,
                       accumulate=False):
    """The loss of every token, and the gradients of x and w for the sum of the
    losses times ``grad``: a number (a loss scale over the number of tokens, say)
    or float32 numbers, one a token.  dx is of x's type and dw of w's, or
    float32, where ``accumulate`` adds to it; new tensors when None, not formed
    when False.  Returns (loss, dx, dw)."""
    return _loss_grad(x, w, lib().ark_head_cross_entropy_grad, 1,
                      (*_targets(targets, x), _ignored(ignore), scale), grad, dx, dw, accumulate)


def distill(x, w, index, logits, temperature=1.0):
    """The divergence, float32 for every token, of softmax(x w^T / temperature)
    from a teacher's distribution: the softmax of its ``logits`` (tokens, top) /
    temperature at the vocabulary's ``index``.  Entries of an index outside the
    vocabulary (-1, say) are left out; tokens without any have 0."""
    if x.requires_grad or w.requires_grad or logits.requires_grad:
        _no_graph("distill")
    args = _teacher(index, logits, x, temperature)
    return _loss(x, w, lib().ark_head_distill, args[6], args)


def distill_grad(x, w, index, logits, grad=1.0, temperature=1.0, dx=None, dw=None,
                 accumulate=False):
    """As ``cross_entropy_grad``, of ``distill``'s divergence.  Returns (loss, dx,
    dw).  (Multiply ``grad`` by temperature squared to keep gradients' sizes
    alike over temperatures.)"""
    args = _teacher(index, logits, x, temperature)
    return _loss_grad(x, w, lib().ark_head_distill_grad, args[6], args, grad, dx, dw, accumulate)
