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


PARTIAL = [(64, 48), (64, 0), (80, 32), (192, 128), (66, 34), (33, 6), (5, 4), (7, 0), (510, 38)]


def _tail(d, r, name, layout, inverse):
    """q whose values past the rotary ones hold -0, inf, NaN and numbers, and
    its rotation."""
    torch = _torch()
    q, k = _qk((37,), 3, 1, d, name)
    g = torch.Generator(device="cuda").manual_seed(d + r)
    odd = torch.tensor([-0.0, 0.0, float("inf"), float("-inf"), float("nan"), 1.0, -1.0, -2.0],
                       device="cuda").to(_dt(name))
    for x in (q, k):
        at = torch.randint(0, 8, x[..., r:].shape, generator=g, device="cuda")
        x[..., r:] = odd[at]
    rope = Rope(d, r, layout=layout)
    pos = torch.randint(1, 5000, (37,), generator=g, device="cuda")
    return (q, k), rope.apply(q, k, positions=pos, inverse=inverse), pos


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", PARTIAL)
@pytest.mark.parametrize("name", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("inverse", [False, True])
def test_values_past_the_rotary_ones_stay_as_they_are(d, r, name, layout, inverse):
    torch = _torch()
    xs, ys, pos = _tail(d, r, name, layout, inverse)
    turn = Turn(pos.cpu().numpy(), d, r, layout)
    for x, y in zip(xs, ys):
        a, b = x[..., r:], y[..., r:]
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        a, b = (torch.where(torch.isnan(v), torch.ones_like(v), v) for v in (a, b))
        assert torch.equal(a, b) and torch.equal(torch.signbit(a), torch.signbit(b))
        head = _f64(x)
        head[..., r:] = 0.0
        _near(y[..., :r], turn(head, inverse)[..., :r], 8 * U * turn.size(head)[..., :r], name)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", PARTIAL)
@pytest.mark.parametrize("name", ["f16", "bf16", "f32"])
def test_an_infinite_value_past_the_rotary_ones_stays_alone(d, r, name, layout):
    """x[j] = inf makes the row's mean infinite: inf / inf at j, 0 elsewhere.
    dy[j] = inf makes the gain's gradient infinite at j alone."""
    torch = _torch()
    rope = Rope(d, r, layout=layout)
    gains = _gains(d, "f32")
    for j in {r, (r + d) // 2, d - 1}:
        q, k = _qk((37,), 3, 1, d, name)
        clean = q.clone()
        q[5, 1, j] = float("inf")
        for keep8 in (False, True):
            y = rope.norm(q, k, *gains, keep8=keep8)[0]
            row = y[5, 1].clone()
            assert torch.isnan(row[j])
            row[j] = 0
            assert not row.any()
            y[5, 1] = 0
            assert torch.isfinite(y).all()
        dq, dk = _qk((37,), 3, 1, d, name, 1)
        dq[7, 2, j] = float("inf")
        for kept in ((clean, k), rope.norm(clean, k, *gains, keep8=True)[2:]):
            dg = rope.norm_backward(dq, dk, *kept, *gains)[2]
            assert not torch.isfinite(dg[j])
            dg[j] = 0
            assert torch.isfinite(dg).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_an_infinite_gain_reaches_its_own_values_alone(layout):
    """Heads of odd sizes: the last value has no partner at all."""
    torch = _torch()
    for d, r in ((5, 4), (33, 6), (7, 0)):
        rope = Rope(d, r, layout=layout)
        gains = _gains(d, "f32")
        gains[0][d - 1] = float("inf")
        gains[1][0] = float("inf")
        q, k = _qk((9,), 2, 2, d, "f32")
        for keep8 in (False, True):
            y = rope.norm(q, k, *gains, keep8=keep8)
            assert not torch.isfinite(y[0][..., d - 1]).any()
            assert torch.isfinite(y[0][..., :d - 1]).all()
            assert torch.isfinite(y[1][..., r if r else 1:]).all()
