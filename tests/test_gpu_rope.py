"""Rotary positions and the norms of queries and keys (include/ark_rope.h)
against their definitions in 64 bits.

With u = 2^-24, a result of the rotation may be off by 8 u of the magnitudes it
mixes (cosine and sine within 4 u, two products and a sum), the norm's factor
by (D / 2 + 8) u of itself (a sum of D squares under a root), the backward
pass's mean by (D + 16) u of the mean of its magnitudes, a gain's gradient by
one rounding a row; then one rounding to the result's type."""
import numpy as np
import pytest

from ark_amd import act
from ark_amd._lib import ArkOptError
from ark_amd.rope import Rope, frequencies
from tests.test_gpu_act import _dt, _f64, _torch, eight

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5


def _round_to(bound, y, name):
    """bound widened by one rounding of y to the type."""
    half = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}[name]
    tiny = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}[name]
    return bound + half * (np.abs(y) + bound) + tiny


class Turn:
    """The rotation of positions (a numpy array) over a head of d, in 64 bits."""

    def __init__(self, positions, d, r, layout, scaling=None, base=10000.0, freq=None):
        self.d = d
        f, self.m = frequencies(r, base, scaling) if freq is None else (freq, 1.0)
        i = np.arange(r // 2)
        u, v = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
        a = positions.astype(np.float64)[..., None] * np.array(f)
        self.c, self.s = np.ones(positions.shape + (d,)), np.zeros(positions.shape + (d,))
        self.partner = np.arange(d)
        if r:
            self.c[..., u] = self.c[..., v] = self.m * np.cos(a)
            self.s[..., u], self.s[..., v] = -self.m * np.sin(a), self.m * np.sin(a)
            self.partner[u], self.partner[v] = v, u
        self.c, self.s = self.c[..., None, :], self.s[..., None, :]

    def __call__(self, x, back=False):
        return x * self.c + x[..., self.partner] * (-self.s if back else self.s)

    def size(self, x):
        """The magnitudes a result mixes."""
        return max(self.m, 1.0) * (np.abs(x) + np.abs(x[..., self.partner]))


def _near(got, want, bound, name="f32"):
    got = _f64(got)
    bad = np.abs(got - want) > _round_to(bound, want, name)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want).max()))


def _qk(shape, heads, kv, d, name, seed=0):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn((*shape, h, d), generator=g, device="cuda").to(_dt(name))
            for h in (heads, kv)]


# head_dim, rotary_dim: whole heads of the models here, parts, odd sizes, the
# largest, one pair, none
HEADS = [(64, 64), (128, 128), (128, 64), (256, 256), (80, 32), (96, 96), (66, 66), (40, 10),
         (5, 4), (33, 6), (2, 2), (1, 0), (512, 512), (510, 38), (64, 0), (192, 128)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", HEADS)
@pytest.mark.parametrize("name", ["f16", "bf16", "f32"])
def test_apply(d, r, layout, name):
    torch = _torch()
    rope = Rope(d, r, layout=layout)
    for tokens, heads, kv in ((1, 1, 1), (7, 3, 1), (67, 12, 4)):
        q, k = _qk((tokens,), heads, kv, d, name, tokens)
        pos = torch.randint(0, 5000, (tokens,), device="cuda")
        turn = Turn(pos.cpu().numpy(), d, r, layout)
        for back in (False, True):
            for x, y in zip((q, k), rope.apply(q, k, positions=pos, inverse=back)):
                _near(y, turn(_f64(x), back), 8 * U * turn.size(_f64(x)), name)


@pytest.mark.parametrize("scaling", [{"kind": "linear", "factor": 8},
                                     {"kind": "ntk", "factor": 8},
                                     {"kind": "yarn", "factor": 32, "original": 4096},
                                     {"kind": "bands", "factor": 8, "original": 8192}])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_scaled_for_long_contexts(scaling, layout):
    torch = _torch()
    rope = Rope(128, 96, layout=layout, scaling=scaling)
    q, k = _qk((300,), 4, 2, 128, "f32")
    pos = torch.randint(0, 1 << 20, (300,), device="cuda")
    turn = Turn(pos.cpu().numpy(), 128, 96, layout, scaling)
    # 64-bit angles themselves are off by 2^-53 of themselves
    for x, y in zip((q, k), rope.apply(q, k, positions=pos)):
        _near(y, turn(_f64(x)), 8 * U * turn.size(_f64(x)))


def test_far_and_negative_positions():
    """Angles at positions up to 2^40: frequencies that are whole fractions of a
    turn, so that the exact angle is known; theirs, a double's, may be off by
    2^-53 of itself, and the angle by that times the position."""
    torch = _torch()
    freq = [2 * np.pi * w for w in (0.125, 0.25, 0.375, 2.0 ** -20)]
    rope = Rope(8, inv_freq=freq)
    pos = torch.tensor([0, 1, -1, 7, -7, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 3, -2 ** 40 - 5],
                       device="cuda")
    q, k = _qk((9,), 3, 1, 8, "f32")
    p = pos.cpu().numpy()
    turn = Turn(p, 8, 8, "half", freq=freq)
    a = 2 * np.pi * (np.remainder(p[:, None] * np.array([2 ** 17, 2 ** 18, 3 * 2 ** 17, 1]),
                                  2 ** 20) / 2 ** 20)
    c, s = np.cos(a), np.sin(a)
    turn.c, turn.s = np.concatenate([c, c], 1)[:, None], np.concatenate([-s, s], 1)[:, None]
    off = np.abs(p[:, None] * np.array(freq)) * 2.0 ** -53
    off = np.concatenate([off, off], 1)[:, None]
    for x, y in zip((q, k), rope.apply(q, k, positions=pos)):
        _near(y, turn(_f64(x)), (8 * U + off) * turn.size(_f64(x)))
    small = pos.clamp(-2 ** 31, 2 ** 31 - 1).int()
    a, b = rope.apply(q, k, positions=small), rope.apply(q, k, positions=small.long())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_positions_that_follow_a_start():
    torch = _torch()
    rope = Rope(64)
    q, k = _qk((3, 50), 4, 2, 64, "f16")
    pos = (torch.arange(50, device="cuda") + 1234).expand(3, 50).contiguous()
    a, b = rope.apply(q, k, start=1234), rope.apply(q, k, positions=pos)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    zero = rope.apply(q[:, :1], start=0)
    assert torch.equal(zero, q[:, :1])          # position 0 turns nothing


def test_every_quarter_of_a_turn():
    """The sine and cosine over a fine grid of angles and at the quarters'
    edges, through q = (1, 0)."""
    torch = _torch()
    n = 1 << 16
    rope = Rope(2, inv_freq=[2 * np.pi / n])
    pos = torch.arange(-5, n + 5, device="cuda")
    q = torch.zeros((n + 10, 1, 2), device="cuda")
    q[..., 0] = 1.0
    y = _f64(rope.apply(q, positions=pos))[:, 0]
    a = 2 * np.pi * np.arange(-5, n + 5) / n
    assert np.abs(y[:, 0] - np.cos(a)).max() <= 4 * U
    assert np.abs(y[:, 1] - np.sin(a)).max() <= 4 * U


def _strided(x, how):
    """x's values in another memory order."""
    torch = _torch()
    if how == "fused":        # a slice of a wider row
        big = torch.full((*x.shape[:-2], x.shape[-2] * x.shape[-1] + 24), 3.0, dtype=x.dtype,
                         device="cuda")
        v = big[..., 8:8 + x.shape[-2] * x.shape[-1]].unflatten(-1, x.shape[-2:])
    elif how == "odd":        # a slice at an odd offset
        big = torch.full((*x.shape[:-2], x.shape[-2] * x.shape[-1] + 3), 3.0, dtype=x.dtype,
                         device="cuda")
        v = big[..., 1:1 + x.shape[-2] * x.shape[-1]].unflatten(-1, x.shape[-2:])
    else:                     # heads before tokens
        big = torch.empty((*x.shape[:-3], x.shape[-2], x.shape[-3], x.shape[-1]), dtype=x.dtype,
                          device="cuda")
        v = big.transpose(-2, -3)
    v.copy_(x)
    return v


@pytest.mark.parametrize("how", ["fused", "odd", "heads first"])
@pytest.mark.parametrize("name", ["f16", "f32"])
def test_strides_and_in_place(how, name):
    torch = _torch()
    for shape in ((45,), (2, 33)):
        rope = Rope(64, 48)
        q, k = _qk(shape, 6, 2, 64, name)
        pos = torch.randint(0, 9000, shape, device="cuda")
        want = rope.apply(q, k, positions=pos)
        a, b = _strided(q, how), _strided(k, how)
        got = rope.apply(a, b, positions=pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        rope.apply(a, b, positions=pos, out=(a, b))
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
        if how != "heads first":
            assert (a._base[..., 0] == 3).all() and (a._base[..., -1] == 3).all()


def test_views_of_one_fused_array_in_place():
    torch = _torch()
    rope = Rope(64)
    for shape in ((40,), (3, 20)):
        qkv = torch.randn((*shape, 8, 64), device="cuda", dtype=torch.float16)
        before = qkv.clone()
        q, k = qkv[..., :4, :], qkv[..., 4:6, :]
        want = rope.apply(q.clone(), k.clone())
        rope.apply(q, k, out=(q, k))
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(qkv[..., 6:, :], before[..., 6:, :])


def test_a_shared_head_may_be_read_many_times():
    torch = _torch()
    rope = Rope(32)
    q = torch.randn((20, 1, 32), device="cuda")
    y = rope.apply(q.expand(20, 5, 32), positions=torch.arange(20, device="cuda"))
    one = rope.apply(q, positions=torch.arange(20, device="cuda"))
    assert torch.equal(y, one.expand(20, 5, 32))


def test_no_tokens_and_no_heads():
    torch = _torch()
    rope = Rope(64)
    q, k = _qk((0,), 4, 2, 64, "f16")
    assert rope.apply(q, k)[0].shape == (0, 4, 64)
    g = torch.ones(64, device="cuda")
    assert rope.norm(q, k, g, g)[1].shape == (0, 2, 64)
    dq, dk, a, b = rope.norm_backward(q, k, q, k, g, g)
    assert not a.any() and not b.any()
    a.fill_(2.0)
    rope.norm_backward(q, k, q, k, g, g, dgain_q=a, dgain_k=b, accumulate=True)
    assert (a == 2).all()
    q, k = _qk((5,), 3, 0, 64, "f16")
    y, z = rope.apply(q, k)
    assert z.shape == (5, 0, 64) and torch.equal(y, rope.apply(q))


def test_far_strides():
    """Tokens 2^27 values apart: offsets past 2^32 bytes."""
    torch = _torch()
    rope = Rope(64)
    big = torch.empty((39 * (1 << 27) + 256,), dtype=torch.float16, device="cuda")
    far = torch.as_strided(big, (40, 4, 64), (1 << 27, 64, 1))
    q, k = _qk((40,), 4, 4, 64, "f16")
    far.copy_(q)
    want = rope.apply(q, k)
    assert torch.equal(rope.apply(far, k)[0], want[0])
    rope.apply(far, k, out=(far, k.clone()))
    assert torch.equal(far, want[0])


# ---- the norm -------------------------------------------------------------------

def _gains(d, name, seed=1):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(1 + 0.3 * torch.randn((d,), generator=g, device="cuda")).to(_dt(name))
            for _ in range(2)]


def _norm64(x, gain, turn):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    n = x * r * gain
    return turn(n), (x.shape[-1] / 2 + 18) * U * turn.size(n)


def _back64(dy, x, gain, turn, rows_axes):
    """(dx, its bound, dgain, its bound)."""
    d = x.shape[-1]
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    h = x * r
    dn, dn_size = turn(dy, True), turn.size(dy)
    w, w_size = dn * gain, dn_size * np.abs(gain)
    dx = r * (w - h * (w * h).mean(-1, keepdims=True))
    bound = (2 * d + 50) * U * r * (w_size + np.abs(h)
                                    * (w_size * np.abs(h)).mean(-1, keepdims=True))
    n = np.prod([x.shape[i] for i in rows_axes])
    size = (dn_size * np.abs(h)).sum(rows_axes)
    return dx, bound, (dn * h).sum(rows_axes), (n + d / 2 + 24) * U * size


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", HEADS)
@pytest.mark.parametrize("name", ["f16", "bf16", "f32"])
def test_norm_and_its_gradients(d, r, layout, name):
    torch = _torch()
    rope = Rope(d, r, layout=layout)
    for tokens, heads, kv in ((1, 2, 1), (33, 3, 1), (130, 6, 3)):
        q, k = _qk((tokens,), heads, kv, d, name, tokens)
        q[0] = 0.0                                  # a row of zeros: eps alone
        k *= 1e-3
        dq, dk = _qk((tokens,), heads, kv, d, name, tokens + 1)
        gains = _gains(d, name)
        pos = torch.randint(0, 5000, (tokens,), device="cuda")
        turn = Turn(pos.cpu().numpy(), d, r, layout)
        fwd = rope.norm(q, k, *gains, positions=pos, eps=EPS)
        back = rope.norm_backward(dq, dk, q, k, *gains, positions=pos, eps=EPS)
        for i, (x, dy, g) in enumerate(((q, dq, gains[0]), (k, dk, gains[1]))):
            _near(fwd[i], *_norm64(_f64(x), _f64(g), turn), name)
            dx, b, dg, gb = _back64(_f64(dy), _f64(x), _f64(g), turn, (0, 1))
            _near(back[i], dx, b, name)
            _near(back[2 + i], dg, gb)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", HEADS)
@pytest.mark.parametrize("name", ["f16", "bf16", "f32"])
def test_norm_keeping_8_bits(d, r, layout, name):
    """The forward pass writes what pack gives; the backward pass from it is
    the one from the values it stands for."""
    torch = _torch()
    rope = Rope(d, r, layout=layout)
    for shape, heads, kv in (((1,), 2, 1), ((31,), 3, 1), ((2, 33), 4, 2), ((256,), 12, 4)):
        q, k = _qk(shape, heads, kv, d, name, heads)
        dq, dk = _qk(shape, heads, kv, d, name, heads + 1)
        gains = _gains(d, name)
        pos = torch.randint(0, 5000, shape, device="cuda")
        turn = Turn(pos.cpu().numpy(), d, r, layout)
        yq, yk, aq, ak = rope.norm(q, k, *gains, positions=pos, eps=EPS, keep8=True)
        plain = rope.norm(q, k, *gains, positions=pos, eps=EPS)
        for y, x, g in ((yq, q, gains[0]), (yk, k, gains[1])):
            _near(y, *_norm64(_f64(x), _f64(g), turn), name)
        for a, x in ((aq, q), (ak, k)):
            assert torch.equal(a.data, act.pack(x.reshape(-1, a.columns)).data)
        back = rope.norm_backward(dq, dk, aq, ak, *gains, positions=pos, eps=EPS)
        axes = tuple(range(len(shape) + 1))
        for i, (a, dy, g) in enumerate(((aq, dq, gains[0]), (ak, dk, gains[1]))):
            x = _f64(act.unpack(a)).reshape(dy.shape)
            dx, b, dg, gb = _back64(_f64(dy), x, _f64(g), turn, axes)
            _near(back[i], dx, b, name)
            _near(back[2 + i], dg, gb)


@pytest.mark.parametrize("name", ["f16", "f32"])
@pytest.mark.parametrize("how", ["fused", "odd", "heads first"])
def test_norm_strides(how, name):
    torch = _torch()
    rope = Rope(64, 32)
    gains = _gains(64, "f32")
    for shape in ((45,), (2, 33)):
        q, k = _qk(shape, 6, 2, 64, name)
        dq, dk = _qk(shape, 6, 2, 64, name, 3)
        want = rope.norm(q, k, *gains)
        wback = rope.norm_backward(dq, dk, q, k, *gains)
        s = [_strided(x, how) for x in (q, k, dq, dk)]
        got = rope.norm(s[0], s[1], *gains)
        back = rope.norm_backward(s[2], s[3], s[0], s[1], *gains, out=(s[2], s[3]))
        assert back[0] is s[2]
        for a, b in zip((*got, *back[:2]), (*want, *wback[:2])):
            assert torch.equal(a, b)
        turn = Turn(np.broadcast_to(np.arange(shape[-1]), shape), 64, 32, "half")
        axes = tuple(range(len(shape) + 1))
        for i, (x, dy, g) in enumerate(((q, dq, gains[0]), (k, dk, gains[1]))):
            _, _, dg, gb = _back64(_f64(dy), _f64(x), _f64(g), turn, axes)
            _near(back[2 + i], dg, gb)


def test_norm_8_bits_of_fused_and_given_buffers():
    """q and k as slices of one projection, 8-bit forms into given buffers, the
    forward pass in place."""
    torch = _torch()
    rope = Rope(64)
    gains = _gains(64, "f16")
    for shape in ((70,), (2, 64)):
        qkv = torch.randn((*shape, 9, 64), device="cuda", dtype=torch.float16)
        q, k = qkv[..., :6, :], qkv[..., 6:8, :]
        want = rope.norm(q.clone(), k.clone(), *gains, keep8=True)
        rows = int(np.prod(shape))
        kept = (act.Act8(rows, 6 * 64, torch.float16), act.Act8(rows, 2 * 64, torch.float16))
        got = rope.norm(q, k, *gains, out=(q, k), keep8=kept)
        assert got[2] is kept[0]
        for a, b in zip(got[:2], want[:2]):
            assert torch.equal(a, b)
        for a, b in zip(got[2:], want[2:]):
            assert torch.equal(a.data, b.data)


def test_norm_8_bits_of_heads_that_are_not_side_by_side():
    torch = _torch()
    rope = Rope(32)
    gains = _gains(32, "f16")
    q, k = _qk((2, 40), 3, 2, 32, "f16")
    want = rope.norm(q, k, *gains, keep8=True)
    got = rope.norm(_strided(q, "heads first"), _strided(k, "heads first"), *gains, keep8=True)
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a, b)
    for a, b in zip(got[2:], want[2:]):
        assert torch.equal(a.data, b.data)


def test_non_finite_values_stay_in_their_rows():
    torch = _torch()
    rope = Rope(64)
    gains = _gains(64, "f16")
    q, k = _qk((40,), 3, 2, 64, "f16")
    q[5, 1, 7] = float("inf")
    k[39, 0, 0] = float("nan")
    yq, yk, aq, ak = rope.norm(q, k, *gains, keep8=True)
    assert torch.isnan(yq[5, 1]).any()
    yq[5, 1] = 0
    assert torch.isfinite(yq).all() and torch.isnan(yk[39, 0]).all()
    dq, dk = _qk((40,), 3, 2, 64, "f16", 2)
    gq = rope.norm_backward(dq, dk, aq, ak, *gains)
    assert torch.isnan(gq[0][:32, 1]).all() and torch.isfinite(gq[0][32:]).all()
    assert torch.isfinite(gq[0][:, 0]).all() and not torch.isfinite(gq[2]).all()


def test_gradients_by_differences():
    """dL of L = sum(dy * norm(x)), by central differences of the 64-bit
    definition, along random directions of x and of the gain."""
    torch = _torch()
    rng = np.random.default_rng(3)
    for d, r, layout in ((64, 64, "half"), (40, 24, "interleaved")):
        rope = Rope(d, r, layout=layout)
        q, k = _qk((20,), 3, 1, d, "f32")
        dq, dk = _qk((20,), 3, 1, d, "f32", 5)
        gains = _gains(d, "f32")
        turn = Turn(np.arange(20), d, r, layout)
        gq, gk, dgq, dgk = rope.norm_backward(dq, dk, q, k, *gains, eps=EPS)
        for x, dy, g, dx, dg in ((q, dq, gains[0], gq, dgq), (k, dk, gains[1], gk, dgk)):
            x, dy, g, dx, dg = (_f64(v) for v in (x, dy, g, dx, dg))
            loss = lambda x, g: (dy * _norm64(x, g, turn)[0]).sum()
            for _ in range(3):
                v, w = rng.standard_normal(x.shape), rng.standard_normal(g.shape)
                h = 1e-4
                # a central difference is off by h^2 of third derivatives (about
                # 1e-8 of these sums); the kernel's sums by 1e-5 of magnitudes
                fx = (loss(x + h * v, g) - loss(x - h * v, g)) / (2 * h)
                fg = (loss(x, g + h * w) - loss(x, g - h * w)) / (2 * h)
                assert abs(fx - (dx * v).sum()) <= 1e-5 * np.abs(dx * v).sum()
                assert abs(fg - (dg * w).sum()) <= 1e-5 * np.abs(dg * w).sum()


def test_rotating_back_is_the_transpose():
    torch = _torch()
    rope = Rope(96, 64, scaling={"kind": "yarn", "factor": 16, "original": 2048})
    q, k = _qk((50,), 3, 1, 96, "f32")
    dq, dk = _qk((50,), 3, 1, 96, "f32", 2)
    pos = torch.randint(0, 40000, (50,), device="cuda")
    y, b = rope.apply(q, k, positions=pos), rope.apply(dq, dk, positions=pos, inverse=True)
    for x, dy, yy, bb in zip((q, k), (dq, dk), y, b):
        x, dy, yy, bb = (_f64(v) for v in (x, dy, yy, bb))
        # each side's error is 8 u of magnitudes up to 2 m |x| |dy|
        assert abs((dy * yy).sum() - (bb * x).sum()) <= 64 * U * 2 * (np.abs(x) * np.abs(dy)).sum()


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("tokens", [3, 1000, 20000])
def test_gain_gradients_accumulate_and_repeat(tokens, keep8):
    torch = _torch()
    rope = Rope(64)
    q, k = _qk((tokens,), 4, 2, 64, "f16")
    dq, dk = _qk((tokens,), 4, 2, 64, "f16", 2)
    gains = _gains(64, "f32")
    kept = rope.norm(q, k, *gains, keep8=True)[2:] if keep8 else (q, k)
    first = rope.norm_backward(dq, dk, *kept, *gains)
    a, b = torch.full((64,), 3.0, device="cuda"), torch.full((64,), -2.0, device="cuda")
    again = rope.norm_backward(dq, dk, *kept, *gains, dgain_q=a, dgain_k=b, accumulate=True)
    assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    assert torch.equal(a, first[2] + 3.0) and torch.equal(b, first[3] - 2.0)


def test_on_another_stream_and_in_a_graph():
    torch = _torch()
    rope = Rope(128)
    gains = _gains(128, "bf16")
    q, k = _qk((500,), 8, 2, 128, "bf16")
    dq, dk = _qk((500,), 8, 2, 128, "bf16", 2)
    out = [torch.empty_like(x) for x in (q, k, dq, dk)]
    grads = [torch.empty(128, device="cuda") for _ in range(2)]
    kept = [act.Act8(500, x.shape[1] * 128, torch.bfloat16) for x in (q, k)]

    def go():
        rope.norm(q, k, *gains, out=out[:2], keep8=kept)
        rope.norm_backward(dq, dk, *kept, *gains, out=out[2:], dgain_q=grads[0],
                           dgain_k=grads[1])

    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        go()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        go()
    for i in range(4):
        for x in (q, k, dq, dk):
            x.normal_()
        go()
        torch.cuda.synchronize()
        want = [t.clone() for t in out + grads + [a.data for a in kept]]
        for t in out + grads:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in
                   zip(want, out + grads + [a.data for a in kept])), i


def test_refusals():
    torch = _torch()
    rope = Rope(64)
    q, k = _qk((10,), 4, 2, 64, "f16")
    g = torch.ones(64, device="cuda")
    with pytest.raises(ValueError):
        Rope(64, layout="other")
    with pytest.raises(ArkOptError, match="rotary_dim"):
        Rope(64, 66)
    with pytest.raises(ArkOptError, match="head_dim"):
        Rope(513, 4)
    for bad in (q[..., :32], q.cpu(), q.double(), q[0], q.transpose(-1, -2)):
        with pytest.raises(ValueError):
            rope.apply(bad, k)
    with pytest.raises(ValueError):
        rope.apply(q, k[:9])
    for pos in (torch.arange(9, device="cuda"), torch.arange(10), torch.ones(10, device="cuda"),
                torch.arange(10, device="cuda").short()):
        with pytest.raises(ValueError):
            rope.apply(q, k, positions=pos)
    with pytest.raises(ValueError):
        rope.norm(q, k, g[:63], g)
    with pytest.raises(ValueError):
        rope.norm(q, k, g, g, keep8=(act.Act8(10, 256, torch.float16),
                                     act.Act8(10, 64, torch.float16)))
    with pytest.raises(ValueError):
        rope.norm_backward(q, k, q, k, g, g, accumulate=True)
    with pytest.raises(ArkOptError, match="overlap"):
        rope.apply(q, k, out=(q, q[:, 2:]))
    with pytest.raises(ArkOptError, match="overlap"):
        rope.apply(q[:9], out=q[1:])
    with pytest.raises(ArkOptError, match="overlap each other"):
        rope.apply(q, out=q[:, :1].expand(10, 4, 64))
    with pytest.raises(ArkOptError, match="eps"):
        rope.norm(q, k, g, g, eps=-1.0)
