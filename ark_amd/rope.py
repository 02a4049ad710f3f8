"""Rotary positions, and the RMS norm of every query and key head with the
rotation in the same pass (include/ark_rope.h), for torch tensors.

``Rope`` is a model's rotation; ``apply`` rotates queries and keys (or, with
``inverse``, their gradients back), ``norm`` normalises every head and rotates,
``norm_backward`` gives the gradients.  Queries and keys are (tokens, heads,
head_dim) or (batch, tokens, heads, head_dim) tensors of any strides whose
head_dim values follow one another: slices of a fused projection and
transposed (batch, heads, tokens, head_dim) arrays are taken as they are.
"""
import ctypes as C

import torch

from . import _abi
from ._lib import check, lib, current_stream as _stream
from .act import Act8, _code

_LAYOUTS = {"half": _abi.ROPE_HALF, "interleaved": _abi.ROPE_INTERLEAVED}
_SCALINGS = {"linear": (_abi.ROPE_SCALE_LINEAR, ("factor",), {}),
             "ntk": (_abi.ROPE_SCALE_NTK, ("factor",), {}),
             "yarn": (_abi.ROPE_SCALE_YARN, ("factor", "original", "fast", "slow"),
                      {"fast": 32.0, "slow": 1.0}),
             "bands": (_abi.ROPE_SCALE_BANDS, ("factor", "original", "low", "high"),
                       {"low": 1.0, "high": 4.0})}
_U64x4 = C.c_uint64 * 4
_POSITIONS = {torch.int32: 4, torch.int64: 8}


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
        self._layouts = {}
        torch.cuda.current_device()
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
        """The layout of a query or key tensor as the library takes it, one for
        every shape and strides met."""
        key = t.shape, t.stride()
        found = self._layouts.get(key)
        if found is not None:
            return found
        (s, st), n = key, t.dim()
        if n not in (3, 4):
            raise ValueError(f"{what} has {n} dimensions: (batch,) tokens, heads, head_dim")
        if s[-1] != self.head_dim:
            raise ValueError(f"{what} is {tuple(s)}: its heads must have {self.head_dim} values")
        if st[-1] != 1 and s[-1] > 1:
            raise ValueError(f"{what}: the values of a head do not follow one another")
        if len(self._layouts) >= 256:
            self._layouts.clear()
        found = self._layouts[key] = _U64x4(s[-2], st[0] if n == 4 else 0, st[-3], st[-2])
        return found

    def _array(self, t, like, what):
        """(address, layout) of a query or key tensor, whose sizes but the heads
        must be those of ``like``."""
        if t is not like and (t.shape[:-2] != like.shape[:-2] or t.dtype != like.dtype
                              or t.device != like.device):
            raise ValueError(f"{what} is {tuple(t.shape)} {t.dtype} on {t.device}, not "
                             f"{tuple(like.shape[:-2])} x heads x {self.head_dim} {like.dtype} on "
                             f"{like.device}")
        return t.data_ptr(), self._layout(t, what)

    def _call(self, like, positions, start):
        """The arguments every call begins with."""
        code = _code(like, "q")
        if not like.is_cuda:
            raise ValueError(f"q is on {like.device}, not a GPU")
        s = like.shape
        if len(s) not in (3, 4):
            raise ValueError(f"q has {len(s)} dimensions: (batch,) tokens, heads, head_dim")
        batch, tokens = s[0] if len(s) == 4 else 1, s[-3]
        if positions is None:
            return self._h, code, batch, tokens, None, 0, start
        size = _POSITIONS.get(positions.dtype)
        if (size is None or positions.device != like.device or not positions.is_contiguous()
                or positions.numel() != batch * tokens):
            raise ValueError(f"positions must be {batch * tokens} contiguous int32 or int64 on "
                             f"{like.device}")
        return self._h, code, batch, tokens, positions.data_ptr(), size, start

    def _gains(self, gq, gk, like):
        code = _code(gq, "gain_q")
        for g in (gq, gk):
            if (g.dtype != gq.dtype or not g.is_contiguous() or g.numel() != self.head_dim
                    or g.device != like.device):
                raise ValueError(f"gains must be {self.head_dim} contiguous {gq.dtype} on "
                                 f"{like.device}")
        return gq.data_ptr(), gk.data_ptr(), code

    def _out(self, t, out, what):
        """(the result's tensor, its address, its layout)."""
        if out is None:
            out = torch.empty_like(t)
            return out, out.data_ptr(), self._layout(out, what)
        if out.shape != t.shape:
            raise ValueError(f"{what} is {tuple(out.shape)}, not {tuple(t.shape)}")
        return out, *self._array(out, t, what)

    # ---- calls ------------------------------------------------------------

    def apply(self, q, k=None, positions=None, start=0, inverse=False, out=None):
        """q and k rotated by their positions (int32 or int64, one for each batch
        and token; None: start, start + 1, ...), into ``out`` (a tensor, or a
        pair with k; q itself to rotate in place) or new tensors.  inverse
        rotates back, as the gradients of the results are.  Returns the pair, or
        one tensor without k."""
        head = self._call(q, positions, start)
        qa = self._array(q, q, "q")
        if k is None:
            oq, *oa = self._out(q, out, "out")
            check(lib().ark_rope_apply(*head, *qa, *oa, None, None, None, None, int(bool(inverse)),
                                       _stream(q)))
            return oq
        oq, ok = (None, None) if out is None else out
        oq, *oa = self._out(q, oq, "out")
        ok, *ob = self._out(k, ok, "out")
        check(lib().ark_rope_apply(*head, *qa, *oa, *self._array(k, q, "k"), *ob,
                                   int(bool(inverse)), _stream(q)))
        return oq, ok

    def norm(self, q, k, gain_q, gain_k, positions=None, start=0, eps=1e-5, out=None,
             keep8=False):
        """Every head of q and k divided by its root mean square, times the gain,
        rotated; into ``out`` (a pair) or new tensors.  keep8 also writes the
        8-bit forms of q and k in the same pass, for norm_backward: True for new
        ones, or a pair of Act8 of batch * tokens rows.  Returns (q, k) or (q,
        k, kept_q, kept_k)."""
        head = self._call(q, positions, start)
        gains = self._gains(gain_q, gain_k, q)
        qa, ka = self._array(q, q, "q"), self._array(k, q, "k")
        oq, ok = (None, None) if out is None else out
        oq, *oa = self._out(q, oq, "out")
        ok, *ob = self._out(k, ok, "out")
        if not keep8:
            check(lib().ark_rope_norm(*head, eps, *gains, *qa, *oa, None, *ka, *ob, None,
                                      _stream(q)))
            return oq, ok
        rows, d = head[2] * head[3], self.head_dim
        if keep8 is True:
            aq = Act8(rows, q.shape[-2] * d, q.dtype, q.device)
            ak = Act8(rows, k.shape[-2] * d, q.dtype, q.device)
        else:
            aq, ak = keep8
            self._kept(aq, q, rows, q.shape[-2]), self._kept(ak, q, rows, k.shape[-2])
        check(lib().ark_rope_norm(*head, eps, *gains, *qa, *oa, aq.data.data_ptr(), *ka, *ob,
                                  ak.data.data_ptr(), _stream(q)))
        return oq, ok, aq, ak

    def _kept(self, a, like, rows, heads):
        if ((a.tokens, a.columns, a.dtype) != (rows, heads * self.head_dim, like.dtype)
                or a.data.device != like.device):
            raise ValueError(f"kept is {a.tokens} x {a.columns} {a.dtype}, not {rows} x "
                             f"{heads * self.head_dim} {like.dtype}")

    def norm_backward(self, dq, dk, q, k, gain_q, gain_k, positions=None, start=0, eps=1e-5,
                      out=None, dgain_q=None, dgain_k=None, accumulate=False):
        """From the gradients dq and dk of norm's results, and its inputs q and k
        (tensors, or the Act8 that keep8 gave): the gradients of q and k, into
        ``out`` (a pair; dq and dk themselves for in place) or new tensors, and
        of the gains, float32, into dgain_q and dgain_k (added with accumulate)
        or new ones.  Returns (q_grad, k_grad, dgain_q, dgain_k)."""
        head = self._call(dq, positions, start)
        gains = self._gains(gain_q, gain_k, dq)
        args, outs, grads = [], [], []
        for dy, x, o, dgain in ((dq, q, None if out is None else out[0], dgain_q),
                                (dk, k, None if out is None else out[1], dgain_k)):
            args += self._array(dy, dq, "gradient")
            if isinstance(x, Act8):
                self._kept(x, dq, head[2] * head[3], dy.shape[-2])
                args += [None, None, x.data.data_ptr()]
            else:
                if x.shape != dy.shape:
                    raise ValueError(f"input is {tuple(x.shape)}, its gradient {tuple(dy.shape)}")
                args += [*self._array(x, dq, "input"), None]
            o, *oa = self._out(dy, o, "out")
            if dgain is None:
                if accumulate:
                    raise ValueError("accumulate needs dgain_q and dgain_k")
                dgain = dq.new_empty(self.head_dim, dtype=torch.float32)
            elif (dgain.dtype != torch.float32 or not dgain.is_contiguous()
                  or dgain.numel() != self.head_dim or dgain.device != dq.device):
                raise ValueError(f"dgain must be {self.head_dim} contiguous float32")
            args += [*oa, dgain.data_ptr()]
            outs.append(o)
            grads.append(dgain)
        check(lib().ark_rope_norm_backward(*head, eps, *gains, *args, int(bool(accumulate)),
                                           _stream(dq)))
        return outs[0], outs[1], grads[0], grads[1]
