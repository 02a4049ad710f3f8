"""Rotary positions, and the RMS norm of every query and key head with the
rotation in the same pass (include/ark_rope.h), for torch tensors.

``Rope`` is a model's rotation; ``apply`` rotates queries and keys (or, with
``inverse``, their gradients back), ``norm`` normalises every head and rotates,
``norm_backward`` gives the gradients.  Queries and keys are (tokens, heads,
head_dim) or (batch, tokens, heads, head_dim) tensors of any strides whose
head_dim values follow one another: slices of a fused projection and
transposed (batch, heads, tokens, head_dim) arrays are taken as they are.

No call records an autograd graph.  ``apply`` and ``norm`` refuse inputs that
require grad while one is recorded: call them under ``torch.no_grad()``, or from
an ``autograd.Function`` whose backward calls ``apply(inverse=True)`` or
``norm_backward``.
"""
import ctypes as C

import torch

from . import _abi
from ._lib import check, lib
from .act import Act8, _code, _raw_stream

_LAYOUTS = {"half": _abi.ROPE_HALF, "interleaved": _abi.ROPE_INTERLEAVED}
_SCALINGS = {"linear": (_abi.ROPE_SCALE_LINEAR, ("factor",), {}),
             "ntk": (_abi.ROPE_SCALE_NTK, ("factor",), {}),
             "yarn": (_abi.ROPE_SCALE_YARN, ("factor", "original", "fast", "slow"),
                      {"fast": 32.0, "slow": 1.0}),
             "bands": (_abi.ROPE_SCALE_BANDS, ("factor", "original", "low", "high"),
                       {"low": 1.0, "high": 4.0})}
_U64x4 = C.c_uint64 * 4
_POSITIONS = {torch.int32: 4, torch.int64: 8}
_like = torch.empty_like


def _meta(t):
    """What a plan depends on; the last is the device's number."""
    return t.shape, t.stride(), t.dtype, t.get_device()


def _no_graph(what):
    """For inputs of which some require grad."""
    if torch.is_grad_enabled():
        raise ValueError(f"an input of {what} requires grad, and its result would have no graph: "
                         "use torch.no_grad(), or an autograd.Function over it and its backward "
                         "call")


def frequencies(rotary_dim, base=10000.0, scaling=None):
    """(inverse frequency of every pair, magnitude) of a rotation; ``scaling``
    is None or a dict with "kind" ("linear", "ntk", "yarn", "bands") and its
    parameters: factor; yarn also original, fast, slow; bands also original,
    low, high."""
    code, params = _abi.ROPE_SCALE_NONE, []
    if scaling is not None:
        given = dict(scaling)
        kind = given.pop("kind", None)
        if kind not in _SCALINGS:
            raise ValueError(f"scaling kind {kind!r}: one of {sorted(_SCALINGS)}")
        code, names, defaults = _SCALINGS[kind]
        if set(given) - set(names) or set(names) - set(given) - set(defaults):
            raise ValueError(f"scaling {kind} takes {names}, got {sorted(given)}")
        params = [float(given.get(n, defaults.get(n))) for n in names]
    freq = (C.c_double * max(1, rotary_dim // 2))()
    size = C.c_double()
    check(lib().ark_rope_frequencies(rotary_dim, base, code,
                                     (C.c_double * len(params))(*params) if params else None,
                                     freq, C.byref(size)))
    return list(freq)[:rotary_dim // 2], size.value


class Rope:
    """A model's rotation, on torch's current device: ``rotary_dim`` of the
    ``head_dim`` values of a head (all of them by default), pairs in halves or
    ``"interleaved"``, frequencies ``base ** (-2 i / rotary_dim)`` scaled as
    ``frequencies`` says, or given outright as ``inv_freq`` (with their
    ``magnitude``)."""

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, layout="half", scaling=None,
                 inv_freq=None, magnitude=1.0):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in _LAYOUTS:
            raise ValueError(f"layout {layout!r}: one of {sorted(_LAYOUTS)}")
        if inv_freq is None:
            inv_freq, magnitude = frequencies(rotary_dim, base, scaling)
        elif scaling is not None or len(inv_freq) != rotary_dim // 2:
            raise ValueError("inv_freq holds one value a pair and takes no scaling")
        self._h = None
        self._plans = {}
        self.device = torch.device("cuda", torch.cuda.current_device())
        h = C.c_void_p()
        check(lib().ark_rope_create(head_dim, rotary_dim, _LAYOUTS[layout],
                                    (C.c_double * max(1, len(inv_freq)))(*inv_freq), magnitude,
                                    C.byref(h)))
        self._h = h
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        self.inv_freq, self.magnitude = tuple(inv_freq), magnitude

    def close(self):
        if self._h:
            check(lib().ark_rope_destroy(self._h))
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- arguments --------------------------------------------------------

    def _layout(self, t, what):
        """The layout of a query or key tensor as the library takes it."""
        s, st, n = t.shape, t.stride(), t.dim()
        if n not in (3, 4):
            raise ValueError(f"{what} has {n} dimensions: (batch,) tokens, heads, head_dim")
        if s[-1] != self.head_dim:
            raise ValueError(f"{what} is {tuple(s)}: its heads must have {self.head_dim} values")
        if st[-1] != 1 and s[-1] > 1:
            raise ValueError(f"{what}: the values of a head do not follow one another")
        return _U64x4(s[-2], st[0] if n == 4 else 0, st[-3], st[-2])

    def _beside(self, t, like, what):
        """The layout of a tensor whose sizes but the heads must be ``like``'s."""
        if (t.shape[:-2] != like.shape[:-2] or t.dtype != like.dtype
                or t.device != like.device):
            raise ValueError(f"{what} is {tuple(t.shape)} {t.dtype} on {t.device}, not "
                             f"{tuple(like.shape[:-2])} x heads x {self.head_dim} {like.dtype} on "
                             f"{like.device}")
        return self._layout(t, what)

    def _into(self, out, t, what):
        """The layout of a result's tensor that the caller gives."""
        if out.shape != t.shape:
            raise ValueError(f"{what} is {tuple(out.shape)}, not {tuple(t.shape)}")
        return self._beside(out, t, what)

    def _plan(self, q, k, positions, gains, key):
        """What a call's sizes, strides and types come to, checked once for each
        combination met: the numbers it begins with, the size of a position, the
        gains' type, and the layouts of q and k and of new results for them."""
        code = _code(q, "q")
        if not q.is_cuda:
            raise ValueError(f"q is on {q.device}, not a GPU")
        if q.device != self.device:
            raise ValueError(f"q is on {q.device}, the rotation on {self.device}: make a Rope "
                             f"there")
        lq = self._layout(q, "q")
        batch, tokens = q.shape[0] if q.dim() == 4 else 1, q.shape[-3]
        lk = None if k is None else self._beside(k, q, "k")
        size = 0
        if positions is not None:
            size = _POSITIONS.get(positions.dtype)
            if (size is None or positions.device != q.device or not positions.is_contiguous()
                    or positions.numel() != batch * tokens):
                raise ValueError(f"positions must be {batch * tokens} contiguous int32 or int64 "
                                 f"on {q.device}")
        gcode = None
        if gains is not None:
            gcode = _code(gains[0], "gain_q")
            for g in gains:
                if (g.dtype != gains[0].dtype or not g.is_contiguous()
                        or g.numel() != self.head_dim or g.device != q.device):
                    raise ValueError(f"gains must be {self.head_dim} contiguous "
                                     f"{gains[0].dtype} on {q.device}")
        if len(self._plans) >= 256:
            self._plans.clear()
        found = self._plans[key] = (
            code, batch, tokens, size, gcode, lq, lk, self._layout(_like(q), "out"),
            None if k is None else self._layout(_like(k), "out"))
        return found

    def _kept(self, a, like, rows, heads):
        if ((a.tokens, a.columns, a.dtype) != (rows, heads * self.head_dim, like.dtype)
                or a.data.device != like.device):
            raise ValueError(f"kept is {a.tokens} x {a.columns} {a.dtype}, not {rows} x "
                             f"{heads * self.head_dim} {like.dtype}")

    # ---- calls ------------------------------------------------------------

    def apply(self, q, k=None, positions=None, start=0, inverse=False, out=None):
        """q and k rotated by their positions (int32 or int64, one for each batch
        and token; None: start, start + 1, ...), into ``out`` (a tensor, or a
        pair with k; q itself to rotate in place) or new tensors.  inverse
        rotates back, as the gradients of the results are.  Returns the pair, or
        one tensor without k."""
        if q.requires_grad or (k is not None and k.requires_grad):
            _no_graph("apply")
        key = _meta(q), k if k is None else _meta(k), positions if positions is None else _meta(
            positions)
        code, batch, tokens, size, _, lq, lk, loq, lok = (
            self._plans.get(key) or self._plan(q, k, positions, None, key))
        pos = None if positions is None else positions.data_ptr()
        flag = 1 if inverse else 0
        if k is None:
            if out is None:
                out = _like(q)
            else:
                loq = self._into(out, q, "out")
            check(lib().ark_rope_apply(self._h, code, batch, tokens, pos, size, start,
                                       q.data_ptr(), lq, out.data_ptr(), loq, None, None, None,
                                       None, flag, _raw_stream(key[0][-1])))
            return out
        oq, ok = (None, None) if out is None else out
        if oq is None:
            oq = _like(q)
        else:
            loq = self._into(oq, q, "out")
        if ok is None:
            ok = _like(k)
        else:
            lok = self._into(ok, k, "out")
        check(lib().ark_rope_apply(self._h, code, batch, tokens, pos, size, start, q.data_ptr(),
                                   lq, oq.data_ptr(), loq, k.data_ptr(), lk, ok.data_ptr(), lok,
                                   flag, _raw_stream(key[0][-1])))
        return oq, ok

    def norm(self, q, k, gain_q, gain_k, positions=None, start=0, eps=1e-5, out=None,
             keep8=False):
        """Every head of q and k divided by its root mean square, times the gain,
        rotated; into ``out`` (a pair) or new tensors.  keep8 also writes the
        8-bit forms of q and k in the same pass, for norm_backward: True for new
        ones, or a pair of Act8 of batch * tokens rows.  Returns (q, k) or (q,
        k, kept_q, kept_k)."""
        if (q.requires_grad or k.requires_grad or gain_q.requires_grad
                or gain_k.requires_grad):
            _no_graph("norm")
        key = (_meta(q), _meta(k), positions if positions is None else _meta(positions),
               _meta(gain_q), _meta(gain_k))
        code, batch, tokens, size, gcode, lq, lk, loq, lok = (
            self._plans.get(key) or self._plan(q, k, positions, (gain_q, gain_k), key))
        oq, ok = (None, None) if out is None else out
        if oq is None:
            oq = _like(q)
        else:
            loq = self._into(oq, q, "out")
        if ok is None:
            ok = _like(k)
        else:
            lok = self._into(ok, k, "out")
        aq = ak = dq = dk = None
        if keep8:
            rows, d = batch * tokens, self.head_dim
            if keep8 is True:
                aq, ak = Act8._of(rows, q.shape[-2] * d, q), Act8._of(rows, k.shape[-2] * d, q)
            else:
                aq, ak = keep8
                self._kept(aq, q, rows, q.shape[-2]), self._kept(ak, q, rows, k.shape[-2])
            dq, dk = aq.data.data_ptr(), ak.data.data_ptr()
        check(lib().ark_rope_norm(self._h, code, batch, tokens,
                                  None if positions is None else positions.data_ptr(), size, start,
                                  eps, gain_q.data_ptr(), gain_k.data_ptr(), gcode, q.data_ptr(),
                                  lq, oq.data_ptr(), loq, dq, k.data_ptr(), lk, ok.data_ptr(), lok,
                                  dk, _raw_stream(key[0][-1])))
        return (oq, ok, aq, ak) if keep8 else (oq, ok)

    def norm_backward(self, dq, dk, q, k, gain_q, gain_k, positions=None, start=0, eps=1e-5,
                      out=None, dgain_q=None, dgain_k=None, accumulate=False):
        """From the gradients dq and dk of norm's results, and its inputs q and k
        (tensors, or the Act8 that keep8 gave): the gradients of q and k, into
        ``out`` (a pair; dq and dk themselves for in place) or new tensors, and
        of the gains, float32, into dgain_q and dgain_k (added with accumulate)
        or new ones.  Returns (q_grad, k_grad, dgain_q, dgain_k)."""
        key = (_meta(dq), _meta(dk), positions if positions is None else _meta(positions),
               _meta(gain_q), _meta(gain_k))
        code, batch, tokens, size, gcode, lq, lk, loq, lok = (
            self._plans.get(key) or self._plan(dq, dk, positions, (gain_q, gain_k), key))
        oq, ok = (None, None) if out is None else out
        args, outs, grads = [], [], []
        for dy, ldy, x, o, lo, dgain in ((dq, lq, q, oq, loq, dgain_q),
                                         (dk, lk, k, ok, lok, dgain_k)):
            if isinstance(x, Act8):
                self._kept(x, dq, batch * tokens, dy.shape[-2])
                args += dy.data_ptr(), ldy, None, None, x.data.data_ptr()
            else:
                if x.shape != dy.shape:
                    raise ValueError(f"input is {tuple(x.shape)}, its gradient {tuple(dy.shape)}")
                args += dy.data_ptr(), ldy, x.data_ptr(), self._beside(x, dq, "input"), None
            if o is None:
                o = _like(dy)
            else:
                lo = self._into(o, dy, "out")
            if dgain is None:
                if accumulate:
                    raise ValueError("accumulate needs dgain_q and dgain_k")
                dgain = dq.new_empty(self.head_dim, dtype=torch.float32)
            elif (dgain.dtype != torch.float32 or not dgain.is_contiguous()
                  or dgain.numel() != self.head_dim or dgain.device != dq.device):
                raise ValueError(f"dgain must be {self.head_dim} contiguous float32")
            args += o.data_ptr(), lo, dgain.data_ptr()
            outs.append(o)
            grads.append(dgain)
        check(lib().ark_rope_norm_backward(
            self._h, code, batch, tokens, None if positions is None else positions.data_ptr(), size,
            start, eps, gain_q.data_ptr(), gain_k.data_ptr(), gcode, *args, 1 if accumulate else 0,
            _raw_stream(key[0][-1])))
        return outs[0], outs[1], grads[0], grads[1]
