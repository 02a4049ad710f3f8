"""The 8-bit activation and rotation entry points on the CPU (no device):
refusals before any device call, sizes, and the frequencies of every scaling
against their formulas."""
import ctypes as C
import math

import pytest

from ark_amd import _abi, _lib
from ark_amd.rope import frequencies

MB = 1 << 20
F16, BF16, F32 = _abi.ACT_F16, _abi.ACT_BF16, _abi.ACT_F32


def _msg():
    return _lib.lib().ark_opt_last_error().decode()


@pytest.mark.parametrize("tokens,columns,want", [(0, 5, 0), (5, 0, 0), (1, 1, 33), (32, 7, 231),
                                                 (33, 7, 462), (4096, 768, 33 * 128 * 768)])
def test_bytes(tokens, columns, want):
    out = C.c_uint64(7)
    assert _lib.lib().ark_act_bytes(tokens, columns, C.byref(out)) == _abi.OK
    assert out.value == want


def test_bytes_refusals():
    L = _lib.lib()
    out = C.c_uint64(7)
    assert L.ark_act_bytes(1, 1, None) == _abi.EINVAL
    for t, c in ((2 ** 40, 1), (1, 2 ** 31), (2 ** 39, 2 ** 30), (2 ** 64 - 1, 2 ** 64 - 1)):
        assert L.ark_act_bytes(t, c, C.byref(out)) == _abi.EINVAL and "too large" in _msg()


def test_pack_and_unpack_refusals():
    L = _lib.lib()
    pack = lambda x, st, dt, t, c, a: L.ark_act_pack(x, st, dt, t, c, a, None)
    unpack = lambda x, st, dt, t, c, a: L.ark_act_unpack(a, t, c, dt, x, st, None)
    for f in (pack, unpack):
        assert f(None, 0, F16, 0, 8, None) == _abi.OK          # no rows
        assert f(None, 0, F16, 8, 0, None) == _abi.OK          # no columns
        assert f(MB, 8, 3, 8, 8, 2 * MB) == _abi.EINVAL and "dtype" in _msg()
        assert f(MB + 1, 8, F16, 8, 8, 2 * MB) == _abi.EINVAL and "aligned" in _msg()
        assert f(MB + 2, 8, F32, 8, 8, 2 * MB) == _abi.EINVAL and "aligned" in _msg()
        assert f(MB, 8, F16, 8, 8, 2 * MB + 8) == _abi.EINVAL and "16-byte" in _msg()
        assert f(MB, 8, F16, 8, 8, MB + 64) == _abi.EINVAL and "overlap" in _msg()
        assert f(MB, 8, F16, 64, 8, MB - 500) == _abi.EINVAL and "overlap" in _msg()
        assert f(MB, 2 ** 60, F16, 9, 8, 2 * MB) == _abi.EINVAL and "too large" in _msg()
        assert f(MB, 8, F16, 8, 8, 2 * MB) != _abi.OK           # not memory
        assert "overlap" not in _msg()
    assert unpack(MB, 7, F16, 8, 8, 2 * MB) == _abi.EINVAL and "rows" in _msg()
    assert pack(MB, 7, F16, 8, 8, 2 * MB) != _abi.OK and "rows" not in _msg()  # may be read


def test_weight_grad_refusals():
    L = _lib.lib()

    def wg(act=MB, adt=F16, t=64, c=8, dy=2 * MB, dst=16, ddt=F16, n=16, dw=3 * MB, wst=16,
           flags=0):
        return L.ark_act_weight_grad(act, adt, t, c, dy, dst, ddt, n, dw, wst, flags, None)

    assert wg(adt=9) == _abi.EINVAL and "act_dtype" in _msg()
    assert wg(ddt=F32) == _abi.EINVAL and "dy_dtype" in _msg()
    assert wg(adt=BF16, ddt=F16) == _abi.EINVAL and "fp16 dy" in _msg()
    assert wg(adt=F32, ddt=F16) == _abi.EINVAL and "fp16 dy" in _msg()
    assert wg(flags=4) == _abi.EINVAL and "flags" in _msg()
    assert wg(c=2 ** 31) == _abi.EINVAL and "too large" in _msg()
    assert wg(n=2 ** 31) == _abi.EINVAL and "too large" in _msg()
    assert wg(dy=2 * MB + 1) == _abi.EINVAL and "aligned" in _msg()
    assert wg(dw=3 * MB + 2) == _abi.EINVAL and "aligned" in _msg()
    assert wg(wst=15) == _abi.EINVAL and "rows" in _msg()
    assert wg(wst=8, flags=_abi.ACT_TRANSPOSED) != _abi.OK and "rows" not in _msg()
    assert wg(dw=MB + 512) == _abi.EINVAL and "overlaps" in _msg()
    assert wg(dw=2 * MB + 1024) == _abi.EINVAL and "overlaps" in _msg()
    assert wg(act=MB + 4) == _abi.EINVAL and "16-byte" in _msg()
    assert wg(c=0) == _abi.OK and wg(n=0) == _abi.OK
    assert wg(t=0, flags=_abi.ACT_ACCUMULATE) == _abi.OK


def test_rope_refusals_without_a_handle():
    L = _lib.lib()
    lay = (C.c_uint64 * 4)(1, 0, 8, 8)
    h = C.c_void_p(5)
    f = (C.c_double * 4)(1, 1, 1, 1)
    assert L.ark_rope_create(8, 8, 0, f, 1.0, None) == _abi.EINVAL
    for head, rot, layout, fr, mag, word in [(0, 0, 0, f, 1.0, "head_dim"),
                                             (513, 8, 0, f, 1.0, "head_dim"),
                                             (8, 3, 0, f, 1.0, "rotary_dim"),
                                             (8, 10, 0, f, 1.0, "rotary_dim"),
                                             (8, 8, 2, f, 1.0, "layout"),
                                             (8, 8, 0, None, 1.0, "inv_freq"),
                                             (8, 8, 0, f, float("inf"), "magnitude"),
                                             (8, 8, 0, (C.c_double * 4)(1, float("nan"), 1, 1),
                                              1.0, "inv_freq[1]")]:
        h.value = 5
        assert L.ark_rope_create(head, rot, layout, fr, mag, C.byref(h)) == _abi.EINVAL
        assert word in _msg() and h.value is None, _msg()
    assert L.ark_rope_destroy(None) == _abi.OK
    nine = (MB, lay, 2 * MB, lay)
    assert L.ark_rope_apply(None, F16, 1, 1, None, 0, 0, *nine, *nine, 0, None) == _abi.EINVAL
    assert "rope is NULL" in _msg()
    assert L.ark_rope_norm(None, F16, 1, 1, None, 0, 0, 1e-5, MB, MB, F16, *nine, None, *nine,
                           None, None) == _abi.EINVAL
    back = (MB, lay, MB, lay, None, 2 * MB, lay, 3 * MB)
    assert L.ark_rope_norm_backward(None, F16, 1, 1, None, 0, 0, 1e-5, MB, MB, F16, *back, *back,
                                    0, None) == _abi.EINVAL


def test_frequency_refusals():
    L = _lib.lib()
    f, m = (C.c_double * 256)(), C.c_double()
    p = lambda *v: (C.c_double * len(v))(*v)
    call = lambda r, b, s, q: L.ark_rope_frequencies(r, b, s, q, f, C.byref(m))
    assert L.ark_rope_frequencies(8, 1e4, 0, None, None, C.byref(m)) == _abi.EINVAL
    assert call(7, 1e4, 0, None) == _abi.EINVAL and "rotary_dim" in _msg()
    assert call(8, -1.0, 0, None) == _abi.EINVAL and "base" in _msg()
    assert call(8, 1e4, 5, None) == _abi.EINVAL and "scaling" in _msg()
    assert call(8, 1e4, 1, None) == _abi.EINVAL and "params" in _msg()
    assert call(8, 1e4, 1, p(0.0)) == _abi.EINVAL and "parameter 0" in _msg()
    assert call(8, 1e4, 3, p(2.0, 100.0, 1.0, 32.0)) == _abi.EINVAL and "fast" in _msg()
    assert call(8, 1e4, 4, p(2.0, 100.0, 4.0, 4.0)) == _abi.EINVAL and "low < high" in _msg()
    for bad in ({"kind": "other"}, {"kind": "linear"}, {"kind": "linear", "factor": 2, "low": 1}):
        with pytest.raises(ValueError):
            frequencies(8, scaling=bad)


@pytest.mark.parametrize("r", [2, 4, 64, 126, 128])
@pytest.mark.parametrize("kind", ["none", "linear", "ntk", "yarn", "bands"])
def test_frequencies(r, kind):
    base, f, length = 10000.0, 8.0, 4096.0
    sc = {"none": None, "linear": {"kind": kind, "factor": f}, "ntk": {"kind": kind, "factor": f},
          "yarn": {"kind": kind, "factor": f, "original": length},
          "bands": {"kind": kind, "factor": f, "original": length, "low": 1.0, "high": 4.0}}[kind]
    got, size = frequencies(r, base, sc)
    assert len(got) == r // 2
    pair = lambda turns: r * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))
    lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
    for i, g in enumerate(got):
        w = base ** (-2 * i / r)
        if kind == "linear":
            w /= f
        elif kind == "ntk" and r > 2:
            w = (base * f ** (r / (r - 2))) ** (-2 * i / r)
        elif kind == "yarn":
            s = min(max((i - lo) / max(hi - lo, 1e-3), 0), 1)
            w = w * (1 - s) + w / f * s
        elif kind == "bands":
            wave = 2 * math.pi / w
            if wave > length:
                w /= f
            elif wave > length / 4:
                s = (length / wave - 1) / 3
                w = (1 - s) * w / f + s * w
        assert abs(g - w) <= 1e-13 * w, (i, g, w)
    assert size == (pytest.approx(0.1 * math.log(f) + 1, abs=1e-15) if kind == "yarn" else 1.0)
