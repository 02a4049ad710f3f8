"""The vocabulary loss's and the embedding's entry points on the CPU (no device):
refusals before any device call, and sizes of workspaces."""
import ctypes as C

import pytest

from ark_amd import _abi, _lib

GB = 1 << 40  # addresses far from one another
F16, BF16, F32 = _abi.HEAD_F16, _abi.HEAD_BF16, _abi.HEAD_F32


def _msg():
    return _lib.lib().ark_opt_last_error().decode()


def _need(tokens=64, columns=64, vocab=100, top=1, dw=F32, grad=7, w=GB, stride=64):
    out = C.c_uint64(7)
    rc = _lib.lib().ark_head_workspace(w, stride, tokens, columns, vocab, top, dw, grad,
                                       C.byref(out))
    return rc, out.value


def test_workspace_of_the_loss():
    assert _need()[0] == _abi.OK
    # a call's share of dz is bounded, whatever the tokens
    few, many = _need(16384, 64, 32000)[1], _need(1 << 20, 64, 32000)[1]
    assert many < 1.1 * few < 1.3 * 2 ** 30
    assert _need(1 << 20, 64, 1 << 21)[1] < 3 * 2 ** 30
    assert _need(grad=0)[1] < _need(grad=4)[1] < _need(grad=5)[1] <= _need()[1]
    assert _need(grad=8) == (_abi.EINVAL, 0)
    # a copy of w where its rows are not whole 16-byte pieces
    assert _need(stride=66)[1] >= _need()[1] + 100 * 64 * 2
    assert _need(w=GB + 2)[1] == _need(stride=66)[1]
    assert _need(tokens=0)[0] == _abi.OK


@pytest.mark.parametrize("what", [dict(tokens=1 << 31), dict(columns=0), dict(columns=65537),
                                  dict(vocab=0), dict(vocab=(1 << 21) + 1), dict(top=0),
                                  dict(top=257), dict(dw=3)])
def test_workspace_refusals(what):
    assert _need(**what) == (_abi.EINVAL, 0)
    assert _lib.lib().ark_head_workspace(GB, 64, 1, 1, 1, 1, F32, 1, None) == _abi.EINVAL


def _grad(x=GB, xs=64, w=2 * GB, ws=64, dtype=F16, t=64, d=64, v=100, y=3 * GB, yb=8, ignore=-100,
          scale=1.0, g=1.0, gs=None, loss=4 * GB, dx=5 * GB, dxs=64, dw=6 * GB, dwt=F32, dws=64,
          flags=0, wk=7 * GB, wkb=1 << 36):
    return _lib.lib().ark_head_cross_entropy_grad(x, xs, w, ws, dtype, t, d, v, y, yb, ignore,
                                                  scale, g, gs, loss, dx, dxs, dw, dwt, dws, flags,
                                                  wk, wkb, None)


@pytest.mark.parametrize("what,says", [
    (dict(dtype=F32), "fp16 or bf16"), (dict(dtype=9), "fp16 or bf16"), (dict(d=0), "columns"),
    (dict(v=0), "vocab"), (dict(t=1 << 40), "tokens"), (dict(dwt=BF16), "dw_dtype"),
    (dict(dwt=7), "dw_dtype"), (dict(flags=2), "flags"), (dict(flags=1, dwt=F16), "fp32 dw"),
    (dict(yb=2), "4 or 8"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=-1.0), "scale"), (dict(ws=1 << 22), "stride"),
    (dict(xs=1 << 32), "stride"), (dict(dxs=63), "rows"), (dict(dws=63), "rows"),
    (dict(x=GB + 1), "aligned"), (dict(dw=6 * GB + 2), "aligned"), (dict(y=3 * GB + 4), "aligned"),
    (dict(loss=4 * GB + 2), "aligned"), (dict(gs=8 * GB + 1), "aligned"), (dict(wkb=100), "needed"),
    (dict(wk=7 * GB + 8), "16-byte"), (dict(dx=GB), "overlap"), (dict(dw=2 * GB), "overlap"),
    (dict(dx=6 * GB + 64), "overlap"), (dict(loss=GB + 128), "overlap"),
    (dict(wk=6 * GB), "overlap"), (dict(wk=2 * GB - 4096), "overlap"),
    (dict(loss=3 * GB + 256), "overlap"), (dict(gs=4 * GB), "overlap")])
def test_loss_refusals(what, says):
    assert _grad(**what) == _abi.EINVAL and says in _msg(), _msg()


def test_not_memory_is_refused():
    assert _grad() != _abi.OK and "overlap" not in _msg()
    assert _grad(dx=None, dw=None) != _abi.OK
    assert _grad(t=0, dw=None) == _abi.OK
    assert _grad(t=0, flags=1) == _abi.OK
    assert _grad(t=0) != _abi.OK  # dw's zeros


def test_distill_refusals():
    def call(index=3 * GB, ib=8, istride=4, logits=4 * GB, ldt=F32, lstride=4, top=4, tau=1.0):
        return _lib.lib().ark_head_distill(GB, 64, 2 * GB, 64, F16, 64, 64, 100, index, ib, istride,
                                           logits, ldt, lstride, top, tau, 5 * GB, 7 * GB, 1 << 36,
                                           None)
    for what, says in ((dict(ib=3), "4 or 8"), (dict(ldt=3), "logits_dtype"), (dict(top=0), "top"),
                       (dict(top=257), "top"), (dict(tau=0.0), "temperature"),
                       (dict(tau=-2.0), "temperature"), (dict(tau=float("inf")), "temperature"),
                       (dict(tau=float("nan")), "temperature"), (dict(tau=1e-45), "temperature"),
                       (dict(index=3 * GB + 4), "aligned"), (dict(logits=4 * GB + 2), "aligned"),
                       (dict(istride=1 << 33), "stride"), (dict(logits=5 * GB), "overlap")):
        assert call(**what) == _abi.EINVAL and says in _msg(), _msg()
    assert call() != _abi.OK and "overlap" not in _msg()


def test_lookup_refusals():
    def call(table=GB, ts=8, tt=F16, v=100, d=8, tok=2 * GB, tb=8, n=5, out=3 * GB, os=8, ot=F16):
        return _lib.lib().ark_embed_lookup(table, ts, tt, v, d, tok, tb, n, 1.0, out, os, ot, None)
    for what, says in ((dict(tt=3), "dtype"), (dict(ot=3), "dtype"), (dict(tb=1), "4 or 8"),
                       (dict(v=0), "vocab"), (dict(v=1 << 31), "vocab"), (dict(d=0), "columns"),
                       (dict(d=65537), "columns"), (dict(n=1 << 31), "n ="),
                       (dict(ts=1 << 31), "stride"), (dict(os=7), "rows"),
                       (dict(table=GB + 1), "aligned"), (dict(tok=2 * GB + 4), "aligned"),
                       (dict(out=3 * GB + 2, ot=F32), "aligned"), (dict(out=GB + 64), "overlap"),
                       (dict(out=2 * GB), "overlap")):
        assert call(**what) == _abi.EINVAL and says in _msg(), _msg()
    assert call(n=0) == _abi.OK
    assert call() != _abi.OK and "overlap" not in _msg()


def test_lookup_gradient_refusals():
    L = _lib.lib()

    def call(dy=GB, ys=8, yt=F16, tok=2 * GB, tb=8, n=5, v=100, d=8, dw=3 * GB, ws=8, flags=0,
             wk=4 * GB, wkb=1 << 30):
        return L.ark_embed_grad(dy, ys, yt, tok, tb, n, v, d, 1.0, dw, ws, flags, wk, wkb, None)
    for what, says in ((dict(yt=3), "dtype"), (dict(tb=2), "4 or 8"), (dict(v=0), "vocab"),
                       (dict(d=0), "columns"), (dict(n=1 << 31), "n ="), (dict(flags=2), "flags"),
                       (dict(ws=7), "rows"), (dict(dy=GB + 1), "aligned"),
                       (dict(dw=3 * GB + 2), "aligned"), (dict(wkb=16), "needed"),
                       (dict(wk=4 * GB + 4), "16-byte"), (dict(dw=GB), "overlap"),
                       (dict(dw=2 * GB), "overlap"), (dict(wk=3 * GB), "overlap"),
                       (dict(wk=GB), "overlap")):
        assert call(**what) == _abi.EINVAL and says in _msg(), _msg()
    assert call(n=0, flags=1) == _abi.OK
    assert call() != _abi.OK and "overlap" not in _msg()
    out = C.c_uint64(7)
    assert L.ark_embed_grad_workspace(5, 100, 8, None) == _abi.EINVAL
    assert L.ark_embed_grad_workspace(5, 0, 8, C.byref(out)) == _abi.EINVAL and out.value == 0
    assert L.ark_embed_grad_workspace(5, 100, 8, C.byref(out)) == _abi.OK and out.value > 0


def test_strides_whose_bytes_wrap_are_refused():
    """(tokens - 1) * stride * 8 is past 64 bits: no array, whatever it wraps to."""
    L = _lib.lib()
    assert L.ark_head_distill(GB, 64, 2 * GB, 64, F16, 1 << 30, 64, 100, 3 * GB, 8, (1 << 32) - 1,
                              4 * GB, F32, 4, 4, 1.0, 6 * GB, 9 * GB, 1 << 36,
                              None) == _abi.EINVAL and "stride" in _msg()
    assert _grad(t=1 << 30, xs=(1 << 32) - 1) == _abi.EINVAL and "stride" in _msg()
    assert L.ark_embed_lookup(GB, 8, F16, 100, 8, 8 * GB, 8, (1 << 31) - 1, 1.0, 3 * GB,
                              (1 << 31) - 1, F32, None) == _abi.EINVAL and "stride" in _msg()


def test_the_largest_table():
    out = C.c_uint64(7)
    L = _lib.lib()
    assert L.ark_embed_grad_workspace(5, 1 << 28, 1, C.byref(out)) == _abi.OK and out.value > 1 << 30
    assert L.ark_embed_grad_workspace(5, (1 << 28) + 1, 1, C.byref(out)) == _abi.EINVAL


@pytest.mark.parametrize("tokens", [16384, 1 << 20])
def test_workspace_of_the_loss_alone_of_a_large_vocabulary(tokens):
    """The spans' sums of a piece are bounded as dz is, whatever the vocabulary."""
    for vocab in (1 << 19, 1 << 20, (1 << 21) - 5, 1 << 21):
        assert _need(tokens, 64, vocab, grad=0)[1] < 1.1 * 2 ** 30
