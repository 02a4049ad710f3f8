"""Rotary positions and head norms (include/ark_rope.h) at values and constants
where a kernel's spare lanes and padded rows could show: eps = 0, and non-finite
values beside ones that the call does not mix with them."""
import numpy as np
import pytest

from ark_amd import act
from ark_amd.rope import Rope
from tests.test_gpu_act import _dt, _f64, _torch
from tests.test_gpu_rope import U, Turn, _gains, _qk, _round_to

pytestmark = pytest.mark.gpu


def _near(got, want, bound, name="f32"):
    """Within the bound; a NaN is not."""
    got = _f64(got)
    good = np.abs(got - want) <= _round_to(bound, want, name)
    assert good.all(), (int((~good).sum()), float(np.abs(got - want).max()))


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("name,d,r", [("f16", 64, 64), ("bf16", 128, 64), ("f32", 66, 66),
                                      ("f16", 510, 38), ("f32", 512, 512)])
def test_no_eps(name, d, r, keep8):
    """eps = 0: rows of the input are all there is, whatever a wave pads with.
    The bounds are the norm's (a sum of D squares under a root, the mean's
    magnitudes, one rounding a row for the gain), with r = 1 / rms."""
    torch = _torch()
    rope = Rope(d, r)
    for shape, heads, kv in (((1,), 1, 1), ((33,), 3, 1), ((2, 35), 4, 2)):
        q, k = _qk(shape, heads, kv, d, name)
        dq, dk = _qk(shape, heads, kv, d, name, 1)
        gains = _gains(d, "f32")
        turn = Turn(np.broadcast_to(np.arange(shape[-1]), shape), d, r, "half")
        fwd = rope.norm(q, k, *gains, eps=0.0, keep8=keep8)
        kept = fwd[2:] if keep8 else (q, k)
        back = rope.norm_backward(dq, dk, *kept, *gains, eps=0.0)
        for i, (x, dy, g) in enumerate(((q, dq, gains[0]), (k, dk, gains[1]))):
            x, dy, g = _f64(x), _f64(dy), _f64(g)
            n = x / np.sqrt((x * x).mean(-1, keepdims=True)) * g
            _near(fwd[i], turn(n), (d / 2 + 18) * U * turn.size(n), name)
            if keep8:
                x = _f64(act.unpack(kept[i])).reshape(x.shape)
            s = 1 / np.sqrt((x * x).mean(-1, keepdims=True))
            h, dn, size = x * s, turn(dy, True), turn.size(dy)
            w, w_size = dn * g, size * np.abs(g)
            dx = s * (w - h * (w * h).mean(-1, keepdims=True))
            bound = (2 * d + 50) * U * s * (w_size + np.abs(h)
                                            * (w_size * np.abs(h)).mean(-1, keepdims=True))
            _near(back[i], dx, bound, name)
            axes = tuple(range(len(shape) + 1))
            rows = np.prod([x.shape[j] for j in axes])
            _near(back[2 + i], (dn * h).sum(axes),
                  (rows + d / 2 + 24) * U * (size * np.abs(h)).sum(axes))
