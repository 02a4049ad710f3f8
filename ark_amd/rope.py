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
        import torch
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

    def _array(self, t, like, what):
        """(address, layout) of a query or key tensor, whose sizes but the heads
        must be those of ``like``."""
        n = t.dim()
        if n != like.dim() or n not in (3, 4):
            raise ValueError(f"{what} has {n} dimensions: (batch,) tokens, heads, head_dim")
        if not t.is_cuda or t.device != like.device or t.dtype != like.dtype:
            raise ValueError(f"{what} is {t.dtype} on {t.device}, not {like.dtype} on "
                             f"{like.device}")
        s, st = t.shape, t.stride()
        if s[-1] != self.head_dim or s[:-2] != like.shape[:-2]:
            raise ValueError(f"{what} is {tuple(s)}, not {tuple(like.shape[:-2])} x heads x "
                             f"{self.head_dim}")
        if st[-1] != 1 and s[-1] > 1:
            raise ValueError(f"{what}: the values of a head do not follow one another")
        return t.data_ptr(), _U64x4(s[-2], st[0] if n == 4 else 0, st[-3], st[-2])

    def _call(self, like, positions, start):
        """The arguments every call begins with."""
        code = _code(like, "q")
        batch = like.shape[0] if like.dim() == 4 else 1
        tokens = like.shape[-3] if like.dim() >= 3 else 0
        if positions is None:
            return (self._h, code, batch, tokens, None, 0, start)
        if (not positions.is_cuda or not positions.is_contiguous()
                or positions.is_floating_point() or positions.element_size() not in (4, 8)
                or positions.numel() != batch * tokens or positions.device != like.device):
            raise ValueError(f"positions must be {batch * tokens} contiguous int32 or int64 on "
                             f"{like.device}")
        return (self._h, code, batch, tokens, positions.data_ptr(), positions.element_size(),
                start)

    def _gains(self, gq, gk, like):
        code = _code(gq, "gain_q")
        for g in (gq, gk):
            if g is not None and (not g.is_cuda or g.dtype != gq.dtype or not g.is_contiguous()
                                  or g.numel() != self.head_dim or g.device != like.device):
                raise ValueError(f"gains must be {self.head_dim} contiguous {gq.dtype} on "
                                 f"{like.device}")
        return gq.data_ptr(), None if gk is None else gk.data_ptr(), code

    def _out(self, t, out, what):
        import torch
        if out is None:
            out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        elif out.shape != t.shape:
            raise ValueError(f"{what} is {tuple(out.shape)}, not {tuple(t.shape)}")
        return out

    # ---- calls ------------------------------------------------------------

    def apply(self, q, k=None, positions=None, start=0, inverse=False, out=None):
        """q and k rotated by their positions (int32 or int64, one for each batch
        and token; None: start, start + 1, ...), into ``out`` (a tensor, or a
        pair with k; q itself to rotate in place) or new tensors.  inverse
        rotates back, as the gradients of the results are.  Returns the pair, or
        one tensor without k."""
        oq, ok = (out if k is not None and out is not None else (out, None))
        oq = self._out(q, oq, "out")
        head = self._call(q, positions, start)
        qp, ql = self._array(q, q, "q")
        op, ol = self._array(oq, q, "out")
        if k is None:
            check(lib().ark_rope_apply(*head, qp, ql, op, ol, None, None, None, None,
                                       int(bool(inverse)), _stream(q)))
            return oq
        ok = self._out(k, ok, "out")
        kp, kl = self._array(k, q, "k")
        okp, okl = self._array(ok, q, "out")
        check(lib().ark_rope_apply(*head, qp, ql, op, ol, kp, kl, okp, okl, int(bool(inverse)),
                                   _stream(q)))
        return oq, ok

    def norm(self, q, k, gain_q, gain_k, positions=None, start=0, eps=1e-5, out=None,
             keep8=False):
        """Every head of q and k divided by its root mean square, times the gain,
        rotated; into ``out`` (a pair) or new tensors.  keep8 also writes the
        8-bit forms of q and k in the same pass, for norm_backward: True for new
        ones, or a pair of Act8 of batch * tokens rows.  Returns (q, k) or (q,
        k, kept_q, kept_k)."""
        oq, ok = (None, None) if out is None else out
        oq, ok = self._out(q, oq, "out"), self._out(k, ok, "out")
        head = self._call(q, positions, start)
        qp, ql = self._array(q, q, "q")
        kp, kl = self._array(k, q, "k")
        oqp, oql = self._array(oq, q, "out")
        okp, okl = self._array(ok, q, "out")
        aq = ak = None
        if keep8:
            rows, d = head[2] * head[3], self.head_dim
            if keep8 is True:
                aq = Act8(rows, q.shape[-2] * d, q.dtype, q.device)
                ak = Act8(rows, k.shape[-2] * d, q.dtype, q.device)
            else:
                aq, ak = keep8
                self._kept(aq, q, rows, q.shape[-2]), self._kept(ak, q, rows, k.shape[-2])
        check(lib().ark_rope_norm(*head, eps, *self._gains(gain_q, gain_k, q), qp, ql, oqp, oql,
                                  aq.data.data_ptr() if keep8 else None, kp, kl, okp, okl,
                                  ak.data.data_ptr() if keep8 else None, _stream(q)))
        return (oq, ok, aq, ak) if keep8 else (oq, ok)

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
        import torch
        oq, ok = (None, None) if out is None else out
        oq, ok = self._out(dq, oq, "out"), self._out(dk, ok, "out")
        head = self._call(dq, positions, start)
        args, grads = [], []
        for dy, x, o, dgain in ((dq, q, oq, dgain_q), (dk, k, ok, dgain_k)):
            args += self._array(dy, dq, "gradient")
            if isinstance(x, Act8):
                self._kept(x, dq, head[2] * head[3], dy.shape[-2])
                args += [None, None, x.data.data_ptr()]
            else:
                if x.shape != dy.shape:
                    raise ValueError(f"input is {tuple(x.shape)}, its gradient {tuple(dy.shape)}")
                args += [*self._array(x, dq, "input"), None]
            args += self._array(o, dq, "out")
            if dgain is None:
                if accumulate:
                    raise ValueError("accumulate needs dgain_q and dgain_k")
                dgain = torch.empty(self.head_dim, dtype=torch.float32, device=dq.device)
            elif (dgain.dtype != torch.float32 or not dgain.is_contiguous()
                  or dgain.numel() != self.head_dim or dgain.device != dq.device):
                raise ValueError(f"dgain must be {self.head_dim} contiguous float32")
            args.append(dgain.data_ptr())
            grads.append(dgain)
        check(lib().ark_rope_norm_backward(*head, eps, *self._gains(gain_q, gain_k, dq), *args,
                                           int(bool(accumulate)), _stream(dq)))
        return oq, ok, grads[0], grads[1]
