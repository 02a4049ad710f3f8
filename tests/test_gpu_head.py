"""The loss over a vocabulary, its gradients, and distillation
(include/ark_head.h), against their formulas in 64 bits.

Tolerances, from the arithmetic alone (u: half a step of the 16-bit type):
* A logit is a sum of d products in fp32: within bz = (d + 4) 2^-23 of the sum of
  magnitudes, and 2^-23 of itself for the scale.
* log(sum exp): every exponential's argument is off by bz and by 2^-22 of its
  distance from the row's largest, the exponential by 2^-21, a sum of V terms in
  stretches by (64 + V / 4096) 2^-24; weighted by the exponentials' shares q.
* dz = g (q - p): q is rounded twice, and an entry at a target once; in fp16, a
  q below 2^-14 of its span's largest loses up to 2^-25 of that, and dz 2^-38 of
  the largest gradient; in bf16 both vanish below fp32's smallest normal number,
  2^-126 (an exponential's result and a matrix instruction's factor there may be
  taken for 0), which is at most 2^-126 of a q and of the largest gradient.
* dx and dw: the products of what dz is off by, (terms + 4) 2^-23 of the sum of
  magnitudes (in which fp16 factors count as 2^-14 at least), and one rounding.
"""
import math

import pytest

from ark_amd import _abi, head
from ark_amd._lib import ArkOptError

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16"]
SIZES = [(1, 1, 1), (1, 64, 300), (3, 8, 5), (64, 64, 256), (65, 96, 257), (63, 129, 1000),
         (257, 72, 513), (300, 100, 33), (130, 256, 2049), (513, 65, 640), (16, 1030, 70)]

# whose logits and gradients are of the large tiles (checked without a GPU): rows of
# several tiles, a last one of few rows and of few columns, and steps that go through
# their buffers several times
LARGE = [(517, 768, 32308), (1100, 800, 20011), (1290, 160, 32001)]
LARGE_LOGITS = [(745, 134, 9082)]  # of the logits alone
LARGE_GRADS = [(259, 644, 15187)]  # of the gradients alone


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch


def _dt(name):
    torch = _torch()
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def _half(dtype):
    return _torch().finfo(dtype).eps / 2


def make(t, d, v, name, masked=0.2, seed=0):
    """x, w and targets, some of them without a token (outside the vocabulary)."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed + 1000 * t + v)
    w = torch.randn((v, d), generator=gen, device="cuda") * (2.0 / d ** 0.5)
    y = torch.randint(0, v, (t,), generator=gen, device="cuda")
    x = torch.randn((t, d), generator=gen, device="cuda")
    x += 3.0 * torch.rand((t, 1), generator=gen, device="cuda") * w[y]
    off = torch.rand((t,), generator=gen, device="cuda") < masked
    y = torch.where(off, torch.where(torch.rand((t,), generator=gen, device="cuda") < 0.5, -100,
                                     v + 7), y)
    return x.to(_dt(name)), w.to(_dt(name)), y


class Want:
    """Loss and gradients in 64 bits of a wanted distribution p (t x v; rows of
    zeros have no loss), and how far the kernels' may be off."""

    def __init__(self, x, w, p, live, scale, g, own=0.0):
        torch = _torch()
        f16 = x.dtype == torch.float16
        u = _half(x.dtype)
        x = torch.where(live[:, None], x.double(), 0.0)
        w = w.double()
        t, d = x.shape
        v = len(w)
        z = (x @ w.t()) * scale
        lse = torch.logsumexp(z, 1, keepdim=True)
        q = (z - lse).exp()
        self.loss = torch.where(live, own + (p * (lse - z)).sum(1), 0.0)
        bz = (d + 4) * 2.0 ** -23 * scale * (x.abs() @ w.abs().t()) + 2.0 ** -23 * z.abs()
        r = lse - z
        b_lse = (q * (bz + 2.0 ** -22 * r + 2.0 ** -21)).sum(1, keepdim=True)
        b_lse += (64 + v / 4096) * 2.0 ** -24 + 2.0 ** -23 * lse.abs()
        size = (p * (lse.abs() + z.abs() + r.abs())).sum(1)
        self.b_loss = live * (b_lse[:, 0] + (p * bz).sum(1)
                              + 2.0 ** -20 * (size + abs(own)) + 1e-30)
        gs = (live * g).double()[:, None] * scale
        most = gs.abs().max() if t else 0.0
        dz = gs * (q - p)
        delta = bz + b_lse + 2.0 ** -22 * r + 2.0 ** -21
        e = gs.abs() * (q * (2.1 * u + delta) + p * (1.05 * u + 2.0 ** -22))
        if f16:
            e = e + gs.abs() * 2.0 ** -24 + (gs != 0) * most * 2.0 ** -37
        else:
            e = e + (gs.abs() + (gs != 0) * most) * 2.0 ** -125
        least = 2.0 ** -14 if f16 else 0.0
        dz_size = dz.abs() + e + (2.0 ** -27 * most if f16 else 0.0)
        tiny = 2.0 ** -24 if f16 else 2.0 ** -133

        def out(value, err, sizes, n):
            b = err + (n + 4) * 2.0 ** -23 * sizes
            return b + u * (value.abs() + b) + tiny
        self.dx = dz @ w
        aw = w.abs().clamp_min(least)
        self.b_dx = out(self.dx, e @ w.abs(), dz_size @ aw, v)
        self.dw = dz.t() @ x
        ax = torch.where(live[:, None], x.abs().clamp_min(least), 0.0)
        self.b_dw = out(self.dw, e.t() @ x.abs(), dz_size.t() @ ax, t)

    def check(self, loss, dx, dw):
        for name, got in (("loss", loss), ("dx", dx), ("dw", dw)):
            if got is None:
                continue
            want, b = getattr(self, name), getattr(self, "b_" + name)
            off = (got.double() - want).abs()
            assert (off <= b).all(), (name, (off / b).max().item())


def one_hot(y, live, v):
    torch = _torch()
    p = torch.zeros((len(y), v), dtype=torch.float64, device="cuda")
    rows = live.nonzero()[:, 0]
    p[rows, y[rows].long()] = 1.0
    return p


def ce(x, w, y, scale=1.0, g=1.0, ignore=-100):
    torch = _torch()
    live = (y >= 0) & (y < len(w)) & (y != ignore)
    g = torch.as_tensor(g, device="cuda").double().expand(len(x))
    return Want(x, w, one_hot(y, live, len(w)), live, scale, g)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,d,v", SIZES)
def test_cross_entropy(t, d, v, name):
    torch = _torch()
    x, w, y = make(t, d, v, name)
    want = ce(x, w, y, g=8.0 / t)
    want.check(head.cross_entropy(x, w, y), None, None)
    loss, dx, dw = head.cross_entropy_grad(x, w, y, grad=8.0 / t)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and loss.dtype == torch.float32
    want.check(loss, dx, dw)
    live = (y >= 0) & (y < v)
    assert (dx[~live] == 0).all() and (loss[~live] == 0).all()
    # a number for each token, int32 targets, fp32 dw
    g = torch.rand(t, device="cuda") * torch.exp2(torch.randint(-12, 6, (t,), device="cuda"))
    loss, dx, dw = head.cross_entropy_grad(x, w, y.int(), grad=g,
                                           dw=torch.empty((v, d), device="cuda"))
    ce(x, w, y, g=g).check(loss, dx, dw)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("scale", [0.125, 30.0])
def test_scale(scale, name):
    x, w, y = make(100, 48, 301, name)
    want = ce(x, w, y, scale=scale, g=0.5)
    want.check(*head.cross_entropy_grad(x, w, y, grad=0.5, scale=scale))
    want.check(head.cross_entropy(x, w, y, scale=scale), None, None)


@pytest.mark.parametrize("name", TYPES)
def test_strides_and_what_lies_beside(name):
    """Rows of any stride and alignment; nothing beside a written row changes."""
    torch = _torch()
    t, d, v = 150, 40, 290
    x, w, y = make(t, d, v, name)
    want = ce(x, w, y, g=0.25)
    for off, wide in ((0, 64), (3, 47), (8, 56)):
        def beside(a, fill):
            b = torch.full((len(a), wide + d), fill, dtype=a.dtype, device="cuda")
            b[:, off:off + d] = a
            return b, b[:, off:off + d]
        bx, xs = beside(x, float("nan"))
        bw, ws = beside(w, float("nan"))
        bdx, dx = beside(torch.empty_like(x), 7.0)
        for dt in (w.dtype, torch.float32):
            bdw, dw = beside(torch.empty((v, d), dtype=dt, device="cuda"), 7.0)
            loss, a, b = head.cross_entropy_grad(xs, ws, y, grad=0.25, dx=dx, dw=dw)
            assert a is dx and b is dw
            want.check(loss, dx, dw)
            for full in (bdx, bdw):
                assert (full[:, :off] == 7).all() and (full[:, off + d:] == 7).all()
        want.check(head.cross_entropy(xs, ws, y), None, None)


@pytest.mark.parametrize("name", TYPES)
def test_accumulate_and_parts(name):
    torch = _torch()
    x, w, y = make(200, 64, 700, name)
    want = ce(x, w, y, g=0.1)
    before = torch.randn((700, 64), device="cuda")
    dw = before.clone()
    loss, dx, out = head.cross_entropy_grad(x, w, y, grad=0.1, dw=dw, accumulate=True)
    assert out is dw
    want.check(loss, dx, None)
    off = (dw.double() - before.double() - want.dw).abs()
    assert (off <= want.b_dw + 2.0 ** -23 * (before.abs().double() + want.dw.abs())).all()
    fresh = head.cross_entropy_grad(x, w, y, grad=0.1, dw=torch.empty_like(before))[2]
    assert torch.equal(dw, fresh + before)
    a = head.cross_entropy_grad(x, w, y, grad=0.1, dx=False)
    b = head.cross_entropy_grad(x, w, y, grad=0.1, dw=False)
    c = head.cross_entropy_grad(x, w, y, grad=0.1)
    assert a[1] is None and b[2] is None
    assert torch.equal(a[2], c[2]) and torch.equal(b[1], c[1]) and torch.equal(a[0], b[0])
    assert head.cross_entropy_grad(x, w, y, dx=False, dw=False)[1:] == (None, None)


@pytest.mark.parametrize("name", TYPES)
def test_tokens_without_a_loss_reach_nothing(name):
    """NaN and inf in their rows and numbers, whole blocks of them, and no others."""
    torch = _torch()
    t, d, v = 600, 32, 100
    x, w, y = make(t, d, v, name, masked=0.0)
    off = torch.zeros(t, dtype=torch.bool, device="cuda")
    off[:70] = off[200:300] = off[599] = True
    off[400::3] = True
    y[off] = -100
    clean = head.cross_entropy_grad(x, w, y, grad=0.5)
    ce(x, w, y, g=0.5).check(*clean)
    bad = x.clone()
    bad[off] = float("nan")
    bad[:35] = float("inf")
    for a, b in zip(clean, head.cross_entropy_grad(bad, w, y, grad=0.5)):
        assert torch.equal(a, b)
    g = torch.full((t,), 0.5, device="cuda")
    g[off] = float("nan")
    for a, b in zip(clean, head.cross_entropy_grad(bad, w, y, grad=g)):
        assert torch.equal(a, b)
    y[:] = -100
    loss, dx, dw = head.cross_entropy_grad(bad, w, y, grad=g)
    assert not loss.any() and not dx.any() and not dw.any()
    assert not head.cross_entropy(bad, w, y).any()
    dw = torch.ones((v, d), device="cuda")
    head.cross_entropy_grad(bad, w, y, grad=g, dw=dw, accumulate=True)
    assert (dw == 1).all()


def test_ignored_index_in_the_vocabulary():
    torch = _torch()
    x, w, y = make(90, 24, 12, "f16", masked=0.0)
    want = ce(x, w, y, ignore=3, g=1.0)
    want.check(*head.cross_entropy_grad(x, w, y, ignore=3))
    assert (head.cross_entropy(x, w, y, ignore=3)[y == 3] == 0).all()
    far = torch.where(y == 3, torch.tensor(2 ** 40 + 5, device="cuda"), y)
    assert torch.equal(head.cross_entropy(x, w, far), head.cross_entropy(x, w, y, ignore=3))


@pytest.mark.parametrize("name", TYPES)
def test_what_is_not_finite_shows(name):
    torch = _torch()
    x, w, y = make(120, 64, 500, name, masked=0.1)
    good = head.cross_entropy(x, w, y)
    live = ((y >= 0) & (y < 500)).nonzero()[:, 0]
    for value in (float("nan"), float("inf")):
        bad = x.clone()
        bad[live[5], 3] = value
        loss, dx, dw = head.cross_entropy_grad(bad, w, y)
        others = torch.arange(120, device="cuda") != live[5]
        assert not torch.isfinite(loss[live[5]]) and torch.equal(loss[others], good[others])
        assert not torch.isfinite(dx[live[5]]).any() and torch.isfinite(dx[others]).all()
        assert not torch.isfinite(dw).all(1).any()
    g = torch.ones(120, device="cuda")
    g[live[2]] = float("inf")
    loss, dx, dw = head.cross_entropy_grad(x, w, y, grad=g)
    assert torch.equal(loss, good) and not torch.isfinite(dw).all()
    assert not torch.isfinite(dx[live[2]]).all()


@pytest.mark.parametrize("name", TYPES)
def test_far_logits(name):
    """Logits in the thousands, rows that are sure of a token, rows without any
    difference."""
    torch = _torch()
    x, w, y = make(80, 64, 400, name, masked=0.0)
    x = x * 64
    x[10:20] = 0
    want = ce(x, w, y, scale=16.0)
    want.check(*head.cross_entropy_grad(x, w, y, scale=16.0))
    # all but one logit -inf
    w2 = torch.full((7, 8), -60000.0, device="cuda").to(_dt(name))
    w2[3] = 0
    x2 = torch.full((5, 8), 60000.0, device="cuda").to(_dt(name))
    y2 = torch.tensor([3, 3, 2, -1, 3], device="cuda")
    loss, dx, dw = head.cross_entropy_grad(x2, w2, y2, scale=3e38 / 2 ** 34)
    assert loss[0] == loss[1] == loss[3] == loss[4] == 0 and loss[2] > 1e30
    assert (dx[0] == 0).all() and (dx[4] == 0).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,v", [(9, 300), (300, 2100)])
def test_large_logits_close_together(t, v, name):
    """Whole numbers, whose logits (about 1500) are exact: what is left are an
    exponential's argument, of its distance r from the row's sum, by 2^-22, its value
    by 2^-21, the sum of them and the logarithm, in all 2^-18 and 2^-21 of r."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(v)
    base = torch.randint(-8, 9, (256,), generator=gen, device="cuda")
    w = base.repeat(v, 1)
    w.scatter_add_(1, torch.randint(0, 256, (v, 3), generator=gen, device="cuda"),
                   torch.randint(-1, 2, (v, 3), generator=gen, device="cuda"))
    x = base.repeat(t, 1)
    x.scatter_add_(1, torch.randint(0, 256, (t, 3), generator=gen, device="cuda"),
                   torch.randint(-1, 2, (t, 3), generator=gen, device="cuda"))
    y = torch.randint(0, v, (t,), generator=gen, device="cuda")
    z = (x.double() @ w.double().t()) * 0.25
    y[::2] = z[::2].argmax(1)
    x, w = x.to(_dt(name)), w.to(_dt(name))
    lse = torch.logsumexp(z, 1, keepdim=True)
    want = (lse - z.gather(1, y[:, None]))[:, 0]
    far = (torch.exp(z - lse) * (lse - z)).sum(1) + want
    limit = 2.0 ** -18 + 2.0 ** -21 * far
    loss, dx, dw = head.cross_entropy_grad(x, w, y, scale=0.25)
    assert ((loss.double() - want).abs() <= limit).all()
    assert torch.equal(head.cross_entropy(x, w, y, scale=0.25), loss)
    ce(x, w, y, scale=0.25).check(loss, dx, dw)
    index = torch.stack([y, (y + 1) % v, (y + 2) % v], 1)
    logits = torch.tensor([1.0, 0.5, 0.0], device="cuda").repeat(t, 1)
    p = torch.softmax(logits.double() / 4, 1)
    want = (p * (p.log() - (z.gather(1, index) - lse))).sum(1)
    far = far + (p * (lse - z.gather(1, index))).sum(1)
    got = head.distill(x, w, index, logits, temperature=4.0)
    assert ((got.double() - want).abs() <= 2.0 ** -17 + 2.0 ** -21 * far).all()


def test_pieces():
    """More tokens than a piece, by tokens and by the vocabulary's size."""
    torch = _torch()
    for t, d, v in ((16384 * 2 + 77, 8, 40), (700, 8, (1 << 20) + 3)):
        x, w, y = make(t, d, v, "bf16")
        g = torch.rand(t, device="cuda")
        for dt in (torch.bfloat16, torch.float32):
            got = head.cross_entropy_grad(x, w, y, grad=g, dw=torch.empty((v, d), dtype=dt,
                                                                          device="cuda"))
            ce(x, w, y, g=g).check(*got)
        ce(x, w, y).check(head.cross_entropy(x, w, y), None, None)


def test_no_tokens():
    torch = _torch()
    x, w, y = (torch.empty((0, 16), device="cuda").half(), torch.ones((9, 16), device="cuda").half(),
               torch.empty(0, dtype=torch.long, device="cuda"))
    assert head.cross_entropy(x, w, y).numel() == 0
    loss, dx, dw = head.cross_entropy_grad(x, w, y)
    assert loss.numel() == dx.numel() == 0 and (dw == 0).all() and dw.shape == (9, 16)
    g = torch.empty(0, device="cuda")
    dw = torch.ones((9, 16), device="cuda")
    head.cross_entropy_grad(x, w, y, grad=g, dw=dw, accumulate=True)
    assert (dw == 1).all()
    head.cross_entropy_grad(x, w, y, grad=g, dw=dw)
    assert (dw == 0).all()


@pytest.mark.parametrize("grad", [0.0, 1e-30, 3e30, -2.0])
def test_sizes_of_the_gradient(grad):
    """Gradients far from 1, in bf16, whose range holds them."""
    torch = _torch()
    x, w, y = make(70, 32, 90, "bf16")
    g = torch.full((70,), grad, device="cuda")
    want = ce(x, w, y, g=g)
    want.check(*head.cross_entropy_grad(x, w, y, grad=grad))
    want.check(*head.cross_entropy_grad(x, w, y, grad=g))


@pytest.mark.parametrize("grad", [1e36, 1e-37])
def test_sizes_of_the_gradient_of_fp16(grad):
    """dw in fp32 holds what the 16 bits of dz do not."""
    torch = _torch()
    x, w, y = make(70, 32, 90, "f16")
    got = head.cross_entropy_grad(x, w, y, grad=grad, dx=False, dw=torch.empty_like(w).float())
    ce(x, w, y, g=grad).check(*got)


@pytest.mark.parametrize("t", [70, 1500])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_token_of_no_finite_gradient_leaves_the_others(value, t):
    torch = _torch()
    x, w, y = make(t, 32, 90, "f16", masked=0.0)
    g = torch.full((t,), 1e-4, device="cuda")
    g[t // 2] = value
    loss, dx, _ = head.cross_entropy_grad(x, w, y, grad=g)
    assert not torch.isfinite(dx[t // 2]).any()
    g[t // 2], dx[t // 2] = 0.0, 0.0
    ce(x, w, y, g=g).check(loss, dx, None)


def test_loss_by_differences():
    """The sum of the losses along a line, by central differences of step h: off by
    h^2 / 6 of the third derivative, at most twice the cube of the largest range of
    a logit's slope, and by the losses' own tolerance over h."""
    torch = _torch()
    x, w, y = make(40, 32, 200, "f16")
    x = (x * 64).round() / 64
    x = x.clamp(-7, 7)
    gen = torch.Generator(device="cuda").manual_seed(5)
    line = torch.randint(-1, 2, x.shape, generator=gen, device="cuda").to(x.dtype)
    h = 2.0 ** -5
    want = ce(x, w, y)
    up, down = (head.cross_entropy(x + s * h * line, w, y).double().sum() for s in (1, -1))
    slope = line.double() @ w.double().t()
    reach = 2 * (slope.max(1).values - slope.min(1).values) ** 3
    limit = h * h / 6 * reach.sum() + 2.1 * want.b_loss.sum() / (2 * h)
    dx = head.cross_entropy_grad(x, w, y)[1].double()
    limit = limit + (want.b_dx * line.abs().double()).sum()
    assert ((up - down) / (2 * h) - (dx * line.double()).sum()).abs() <= limit
    # and along w
    line = torch.randint(-1, 2, w.shape, generator=gen, device="cuda").to(w.dtype)
    w = (w * 256).round() / 256
    want = ce(x, w, y)
    h = 2.0 ** -6
    up, down = (head.cross_entropy(x, w + s * h * line, y).double().sum() for s in (1, -1))
    slope = x.double() @ line.double().t()
    reach = 2 * (slope.max(1).values - slope.min(1).values) ** 3
    dw = head.cross_entropy_grad(x, w, y)[2].double()
    limit = (h * h / 6 * reach.sum() + 2.1 * want.b_loss.sum() / (2 * h)
             + (want.b_dw * line.abs().double()).sum())
    assert ((up - down) / (2 * h) - (dw * line.double()).sum()).abs() <= limit


# ---- distillation -----------------------------------------------------------------

def teacher(t, v, k, seed=0, dtype=None):
    """index (repeats and entries outside the vocabulary among them) and logits,
    garbage where left out, -inf here and there."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed + 31 * t + k)
    index = torch.randint(0, v, (t, k), generator=gen, device="cuda")
    logits = 4.0 * torch.randn((t, k), generator=gen, device="cuda")
    lot = torch.rand((t, k), generator=gen, device="cuda")
    logits = torch.where(lot < 0.1, -float("inf"), logits)
    index = torch.where(lot > 0.85, torch.where(lot > 0.93, -1, v), index)
    logits = torch.where(lot > 0.9, float("nan"), logits)
    index = torch.where((lot > 0.9) & (index < v), -1, index)
    index[0] = -1
    if t > 2:
        logits[1] = -float("inf")
    return index, logits.to(dtype or torch.float32)


def kl(x, w, index, logits, tau, g):
    torch = _torch()
    v = len(w)
    ok = (index >= 0) & (index < v) & (logits != -float("inf"))
    live = ok.any(1)
    a = torch.where(ok, logits.double() / tau, -float("inf"))
    a = torch.where(live[:, None], a, 0.0)
    log_p = torch.log_softmax(a, 1)
    p = torch.where(ok, log_p.exp(), 0.0)
    own = torch.where(ok, p * log_p, 0.0).sum(1)
    dense = torch.zeros((len(x), v), dtype=torch.float64, device="cuda")
    dense.scatter_add_(1, torch.where(ok, index, 0).long(), p)
    g = torch.as_tensor(g, device="cuda").double().expand(len(x))
    return Want(x, w, dense, live, 1.0 / tau, g, own)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,d,v,k", [(1, 8, 3, 1), (5, 64, 40, 256), (33, 72, 300, 7),
                                     (130, 40, 1000, 64), (300, 128, 513, 65), (64, 64, 256, 130)])
def test_distill(t, d, v, k, name):
    torch = _torch()
    x, w, _ = make(t, d, v, name)
    index, logits = teacher(t, v, k)
    for tau in (1.0, 2.5):
        want = kl(x, w, index, logits, tau, 4.0 / t)
        want.check(head.distill(x, w, index, logits, tau), None, None)
        want.check(*head.distill_grad(x, w, index, logits, grad=4.0 / t, temperature=tau))
    g = torch.rand(t, device="cuda")
    for dt in (torch.float16, torch.bfloat16):
        narrow = logits.to(dt)
        wide = torch.full((t, k + 5), 3, device="cuda", dtype=torch.int32)
        wide[:, 2:2 + k] = index
        want = kl(x, w, index, narrow, 1.0, g)
        want.check(*head.distill_grad(x, w, wide[:, 2:2 + k], narrow, grad=g,
                                      dw=torch.empty((v, d), device="cuda")))


def test_distill_without_entries():
    torch = _torch()
    x, w, _ = make(70, 16, 50, "f16")
    x[:] = float("nan")
    index = torch.full((70, 4), -1, device="cuda")
    logits = torch.full((70, 4), float("nan"), device="cuda")
    loss, dx, dw = head.distill_grad(x, w, index, logits)
    assert not loss.any() and not dx.any() and not dw.any()
    index[:] = 3
    logits[:] = -float("inf")
    assert not head.distill(x, w, index, logits).any()


def test_distill_of_one_certain_entry_is_cross_entropy():
    torch = _torch()
    x, w, y = make(99, 64, 333, "bf16")
    live = (y >= 0) & (y < 333)
    a = head.cross_entropy_grad(x, w, y, grad=0.5)
    b = head.distill_grad(x, w, y[:, None], torch.zeros((99, 1), device="cuda"), grad=0.5)
    for one, other in zip(a, b):
        assert torch.equal(one, other)
    # the same token three times over
    c = head.distill_grad(x, w, y[:, None].expand(99, 4).contiguous(),
                          torch.zeros((99, 4), device="cuda"), grad=0.5)
    want = Want(x, w, one_hot(y, live, 333), live, 1.0,
                torch.full((99,), 0.5, device="cuda"), torch.where(live, -math.log(4.0), 0.0))
    want.check(*c)  # four entries of 1/4 each: sum of p log p = -log 4


def test_distill_shows_what_is_not_finite():
    torch = _torch()
    x, w, _ = make(10, 16, 50, "f16")
    index = torch.arange(4, device="cuda").expand(10, 4).contiguous()
    logits = torch.zeros((10, 4), device="cuda")
    good = head.distill(x, w, index, logits)
    for value in (float("nan"), float("inf")):
        bad = logits.clone()
        bad[6, 2] = value
        loss, dx, dw = head.distill_grad(x, w, index, bad)
        keep = torch.arange(10, device="cuda") != 6
        assert torch.isnan(loss[6]) and torch.equal(loss[keep], good[keep])
        assert not torch.isfinite(dw).all()


# ---- how it runs --------------------------------------------------------------------

def _calls(x, w, y, index, logits):
    return [head.cross_entropy(x, w, y), *head.cross_entropy_grad(x, w, y, grad=0.5),
            head.distill(x, w, index, logits, 2.0),
            *head.distill_grad(x, w, index, logits, temperature=2.0)]


@pytest.mark.parametrize("t,d,v", [(40, 64, 700), (300, 72, 1500)])
def test_equal_calls_give_equal_bits_also_side_by_side(t, d, v):
    torch = _torch()
    x, w, y = make(t, d, v, "f16")
    index, logits = teacher(t, v, 9)
    first = _calls(x, w, y, index, logits)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_calls(x, w, y, index, logits))
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(first, g):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("t,d,v", [(8, 64, 500), (200, 100, 900)])
def test_in_a_graph(t, d, v):
    torch = _torch()
    x, w, y = make(t, d, v, "bf16")
    index, logits = teacher(t, v, 5)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _calls(x, w, y, index, logits)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = _calls(x, w, y, index, logits)
    for k in range(4):
        x.normal_()
        y.random_(-5, v)
        torch.cuda.synchronize()
        for o in out:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, _calls(x, w, y, index, logits)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), k


def test_a_training_loop_of_the_two_ends():
    """Lookup, loss and both gradients of a tied embedding into an optimizer's fp32
    gradients: the step sees their sum."""
    torch = _torch()
    from ark_amd import embed
    from ark_amd.eko import TensorSpec
    from ark_amd.optimizer import AdamConfig, AmpConfig, Optimizer, ParamSet
    t, d, v = 130, 64, 600
    ps = ParamSet([TensorSpec("embed", (v, d), True, False)], 0.0, grad_dtype=_abi.GRAD_F32)
    table = ps.w(0).view(v, d)
    table.normal_(0.0, 0.3)
    opt = Optimizer(AdamConfig(), ps, AmpConfig(loss_scale_init=1024.0))
    tokens = torch.randint(0, v, (t,), device="cuda")
    targets = torch.randint(0, v, (t,), device="cuda")
    x = embed.lookup(table, tokens, scale=4.0)
    grad = ps.g(0).view(v, d)
    g = opt.loss_scale / t
    loss, dx, _ = head.cross_entropy_grad(x, table, targets, grad=g, dw=grad)
    embed.lookup_grad(dx, tokens, v, scale=4.0, dw=grad, accumulate=True)
    want = ce(x, table, targets, g=g)
    want.check(loss, dx, None)
    both = want.dw.clone().index_add_(0, tokens, 4.0 * dx.double())
    size = torch.zeros_like(both).index_add_(0, tokens, 4.0 * dx.double().abs())
    assert ((grad.double() - both).abs() <= want.b_dw + t * 2.0 ** -23 * (size + both.abs())).all()
    info = opt.step_all(1e-3, info=True)[1]
    norm = grad.double().norm().item() / 1024.0
    assert info.applied == 1 and abs(info.grad_norm - norm) <= 1e-6 * norm
    opt.close()


def test_refusals():
    torch = _torch()
    x, w, y = make(20, 16, 30, "f16")
    index, logits = teacher(20, 30, 4)
    bad = pytest.raises(ValueError)
    with bad:
        head.cross_entropy(x.float(), w.float(), y)
    with bad:
        head.cross_entropy(x, w.bfloat16(), y)
    with bad:
        head.cross_entropy(x.t(), w, y)
    with bad:
        head.cross_entropy(x, w[:, :15], y)
    with bad:
        head.cross_entropy(x, w, y[:19])
    with bad:
        head.cross_entropy(x, w, y.float())
    with bad:
        head.cross_entropy(x, w, y, ignore=2 ** 31)
    with bad:
        head.cross_entropy(x.cpu(), w.cpu(), y.cpu())
    with bad:
        head.cross_entropy_grad(x, w, y, grad=torch.ones(19, device="cuda"))
    with bad:
        head.cross_entropy_grad(x, w, y, accumulate=True)
    with bad:
        head.cross_entropy_grad(x, w, y, dw=torch.empty((30, 16), device="cuda").bfloat16())
    with bad:
        head.cross_entropy_grad(x, w, y, dx=torch.empty((20, 16), device="cuda"))
    with bad:
        head.distill(x, w, index[:, :3], logits)
    with bad:
        head.distill(x, w, index.float(), logits)
    with pytest.raises(ArkOptError, match="fp32 dw"):
        head.cross_entropy_grad(x, w, y, dw=torch.empty_like(w), accumulate=True)
    with pytest.raises(ArkOptError, match="overlap"):
        head.cross_entropy_grad(x, w, y, dx=x)
    with pytest.raises(ArkOptError, match="overlap"):
        head.cross_entropy_grad(x, w, y, dw=w)
    with pytest.raises(ArkOptError, match="scale"):
        head.cross_entropy(x, w, y, scale=0.0)
    for tau in (0.0, -1.0, float("inf"), float("nan"), 1e-45):
        with pytest.raises(ArkOptError, match="temperature"):
            head.distill(x, w, index, logits, temperature=tau)
    with pytest.raises(ArkOptError, match="top"):
        many = torch.zeros((20, 257), device="cuda")
        head.distill(x, w, many.long(), many)
    for t in (x, w, logits):
        t.requires_grad_()
        with pytest.raises(ValueError, match="requires grad"):
            head.distill(x, w, index, logits)
        with torch.no_grad():
            head.distill(x, w, index, logits)
        head.distill_grad(x, w, index, logits)
        t.requires_grad_(False)


def test_threads_with_a_stream_each():
    """Calls from several host threads at once, sizes of their own: the bits of calls
    one after another."""
    import threading
    torch = _torch()
    sets = [make(t, d, v, name) for t, d, v, name in ((300, 64, 700, "f16"), (40, 100, 900, "bf16"),
                                                      (1100, 72, 300, "f16"))]
    want = [head.cross_entropy_grad(*s, grad=2.0) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = head.cross_entropy_grad(*sets[i], grad=2.0)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("t", [70, 1500])
@pytest.mark.parametrize("grad,scale", [(3e38, 2.0), (2.0 ** 127, 4.0)])
def test_a_token_whose_gradient_passes_fp32_leaves_the_others(grad, scale, t):
    """|grad| is finite and |grad * scale| is not: as an infinite one."""
    torch = _torch()
    x, w, y = make(t, 32, 90, "f16", masked=0.0)
    x = x / scale  # the logits as they were
    for others in (1e-4, 3e-9):
        g = torch.full((t,), others, device="cuda")
        g[t // 2] = grad
        loss, dx, _ = head.cross_entropy_grad(x, w, y, grad=g, scale=scale)
        assert not torch.isfinite(dx[t // 2]).any()
        g[t // 2], dx[t // 2] = 0.0, 0.0
        ce(x, w, y, scale=scale, g=g).check(loss, dx, None)
        index, logits = y[:, None], torch.zeros((t, 1), device="cuda")
        g[t // 2] = grad
        loss, dx, _ = head.distill_grad(x, w, index, logits, grad=g, temperature=1.0 / scale)
        assert not torch.isfinite(dx[t // 2]).any()
        g[t // 2], dx[t // 2] = 0.0, 0.0
        ce(x, w, y, scale=scale, g=g).check(loss, dx, None)


@pytest.mark.parametrize("t", [70, 1500])
def test_a_gradient_whose_product_with_scale_is_below_fp32(t):
    """grad * scale is 5.2 of the smallest fp32, or none of it, and dw, its product
    with large rows of x, is an ordinary number."""
    torch = _torch()
    x, w, y = make(t, 32, 90, "bf16")
    scale = 2.0 ** -43
    x, w = x * 2.0 ** 66, w * 2.0 ** -23
    for grad in (1.3 * 2.0 ** -104, 1.3 * 2.0 ** -109):
        g = torch.full((t,), grad, device="cuda")
        want = ce(x, w, y, scale=scale, g=g)
        for one in (grad, g):
            got = head.cross_entropy_grad(x, w, y, grad=one, scale=scale,
                                          dw=torch.empty((90, 32), device="cuda"))
            want.check(*got)


@pytest.mark.parametrize("name", TYPES)
def test_distill_from_logits_that_pass_fp32_over_the_temperature(name):
    """p is a softmax of differences: logits whose quotient is not finite still have
    one, and those below the largest by as much have a p of 0."""
    torch = _torch()
    x, w, _ = make(6, 32, 90, name)
    x[:] = 0  # student's logits of 0
    index = torch.tensor([[3, 80, 5]], device="cuda").repeat(6, 1)
    logits = torch.tensor([[100.0, 50.0, -100.0], [-100.0, -50.0, -200.0], [100.0, 100.0, 0.0],
                           [-100.0, -100.0, -100.0], [3e38, -3e38, 0.0], [-1e3, -1e3, -1e4]],
                          device="cuda")
    tau = 1e-37
    got = head.distill_grad(x, w, index, logits, grad=tau, temperature=tau)
    kl(x, w, index, logits, tau, tau).check(*got)
    assert torch.equal(head.distill(x, w, index, logits, temperature=tau), got[0])


def test_pieces_of_the_loss_alone_of_a_large_vocabulary():
    """4200 tokens over 2^21 are two pieces: rows of both against 64 bits."""
    torch = _torch()
    x, w, y = make(4200, 8, 1 << 21, "f16")
    loss = head.cross_entropy(x, w, y)
    assert torch.isfinite(loss).all()
    for lo in (0, 2070, 4180):
        part = slice(lo, lo + 20)
        ce(x[part], w, y[part]).check(loss[part], None, None)


# ---- large tiles --------------------------------------------------------------------

def _scattered(y, seed):
    """y with a third masked: some here and there, and whole stretches."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    y = torch.where(torch.rand(y.shape, generator=gen, device="cuda") < 0.2, -100, y)
    y[100:180] = y[255:258] = -100
    return y


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,d,v", LARGE + LARGE_LOGITS + LARGE_GRADS)
def test_large_tiles(t, d, v, name):
    torch = _torch()
    x, w, y = make(t, d, v, name)
    y = _scattered(y, t)
    y[::50], y[1::50] = v - 1, 0  # the last, ragged span, and the first
    live = (y >= 0) & (y < v)
    x[~live] = float("nan")
    g = torch.rand(t, device="cuda")
    want = ce(x, w, y, g=g)
    want.check(head.cross_entropy(x, w, y), None, None)
    first = head.cross_entropy_grad(x, w, y, grad=g)
    want.check(*first)
    assert (first[1][~live] == 0).all() and (first[0][~live] == 0).all()
    before = torch.randn((v, d), device="cuda")
    dw = before.clone()
    loss, dx, _ = head.cross_entropy_grad(x, w, y, grad=g, dw=dw, accumulate=True)
    assert torch.equal(loss, first[0]) and torch.equal(dx, first[1])
    off = (dw.double() - before.double() - want.dw).abs()
    assert (off <= want.b_dw + 2.0 ** -23 * (before.abs().double() + want.dw.abs())).all()
    again = head.cross_entropy_grad(x, w, y, grad=g)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,d,v", LARGE + LARGE_LOGITS + LARGE_GRADS)
@pytest.mark.parametrize("k", [1, 8, 65, 130, 256])
def test_distill_of_large_tiles(k, t, d, v, name):
    torch = _torch()
    x, w, _ = make(t, d, v, name)
    index, logits = teacher(t, v, k)
    index[100:180] = -1
    index[200:210, 0] = v - 1
    logits[200:210, 0] = 3.0
    index[210:230] = torch.arange(k, device="cuda") + 120  # neighbours, over spans' ends
    logits[210:230] = torch.randn((20, k), device="cuda")
    g = torch.rand(t, device="cuda")
    want = kl(x, w, index, logits, 2.0, g)
    want.check(head.distill(x, w, index, logits, 2.0), None, None)
    first = head.distill_grad(x, w, index, logits, grad=g, temperature=2.0)
    want.check(*first)
    again = head.distill_grad(x, w, index, logits, grad=g, temperature=2.0)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---- pieces, graphs and strides that the tests above leave out --------------------------

@pytest.mark.parametrize("t,d,v,k", [(16384 * 2 + 77, 8, 40, 5), (700, 8, (1 << 20) + 3, 9)])
def test_pieces_of_distillation(t, d, v, k):
    torch = _torch()
    x, w, _ = make(t, d, v, "f16")
    index, logits = teacher(t, v, k)
    wide = torch.full((t, k + 3), 1, device="cuda", dtype=torch.int32)
    wide[:, 2:2 + k] = index
    want = kl(x, w, index, logits.bfloat16(), 0.5, 0.25)
    want.check(head.distill(x, w, wide[:, 2:2 + k], logits.bfloat16(), 0.5), None, None)
    for dt in (torch.float16, torch.float32):
        dw = torch.full((v, d), 7.0, dtype=dt, device="cuda")
        want.check(*head.distill_grad(x, w, wide[:, 2:2 + k], logits.bfloat16(), grad=0.25,
                                      temperature=0.5, dw=dw))
    one = head.distill_grad(x, w, index, logits.bfloat16(), grad=0.25, temperature=0.5, dx=False)
    assert one[1] is None
    want.check(one[0], None, one[2])


def test_all_of_many_tokens_masked():
    torch = _torch()
    x, w, y = make(20000, 16, 90, "f16")
    y[:] = -100
    x[:] = float("nan")
    dw = torch.ones((90, 16), device="cuda")
    loss, dx, _ = head.cross_entropy_grad(x, w, y, dw=dw, accumulate=True)
    assert not loss.any() and not dx.any() and (dw == 1).all()
    assert not head.cross_entropy_grad(x, w, y)[2].any()
    assert not head.cross_entropy(x, w, y).any()


@pytest.mark.parametrize("t,d,v", [(1500, 40, 700), (1290, 160, 32001)])
def test_many_tokens_in_a_graph(t, d, v):
    """Replays over other masks: other numbers of live rows, parts and tiles than the
    captured call's."""
    torch = _torch()
    x, w, y = make(t, d, v, "f16")
    before = torch.randn((v, d), device="cuda")
    dw = before.clone()
    run = lambda o: (head.cross_entropy(x, w, y),
                     *head.cross_entropy_grad(x, w, y, grad=0.5, dw=o, accumulate=True),
                     *head.cross_entropy_grad(x, w, y, grad=0.5))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run(dw.clone())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = run(dw)
    for k, share in enumerate((0.0, 0.97, 1.0, 0.5, 0.0)):
        x.normal_()
        y.random_(0, v)
        y[torch.rand(t, device="cuda") < share] = -100
        dw.copy_(before)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, run(before.clone())):
            assert torch.equal(a, b), k


@pytest.mark.parametrize("t,d,v,stride", [(150, 64, 290, (1 << 22) - 8), (150, 64, 290, (1 << 22) - 1),
                                          (600, 60, 200, (1 << 21) + 4)])
def test_rows_of_w_far_apart(t, d, v, stride):
    torch = _torch()
    x, near, y = make(t, d, v, "bf16")
    far = torch.full(((v - 1) * stride + d,), float("nan"), device="cuda", dtype=near.dtype)
    w = far.as_strided((v, d), (stride, 1))
    w.copy_(near)
    for a, b in zip(head.cross_entropy_grad(x, w, y, grad=0.5), head.cross_entropy_grad(x, near, y, grad=0.5)):
        assert torch.equal(a, b)
    assert torch.equal(head.cross_entropy(x, w, y), head.cross_entropy(x, near, y))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,v", [(3, 10), (70, 300)])
def test_the_most_columns(t, v, name):
    x, w, y = make(t, 65536, v, name)
    want = ce(x, w, y, g=0.5)
    want.check(*head.cross_entropy_grad(x, w, y, grad=0.5))
    want.check(head.cross_entropy(x, w, y), None, None)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("scale", [2.0 ** 12, 2.0 ** 17 * 1.1, 2.0 ** 22 * 1.3, 2.0 ** 30 * 1.7, 1e33])
def test_logits_past_the_whole_numbers(scale, name):
    """Products are small whole numbers, of which equal ones have equal logits whatever
    the scale: a row is shared evenly by its largest, and every other token's q is 0
    (but for the first scale, e^-4096 at most)."""
    torch = _torch()
    t, d, v = 90, 32, 700
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.zeros((t, d), device="cuda")
    x[torch.arange(t), torch.arange(t) % d] = 1.0
    w = torch.randint(-40, 41, (v, d), generator=gen, device="cuda").float()
    w[:, 5] -= 200  # every logit far below 0
    z = x @ w.t()
    most = z.max(1, keepdim=True).values
    top = (z == most).double()
    y = torch.randint(0, v, (t,), generator=gen, device="cuda")
    y[::2] = z[::2].argmax(1)
    q = top / top.sum(1, keepdim=True)
    p = one_hot(y, y >= 0, v)
    gap = (most - z.gather(1, y[:, None]))[:, 0].double()
    s = torch.tensor(scale, dtype=torch.float32).double()
    want = top.sum(1).log() + gap * s
    # a logit that far is known to 2^-23 of itself, and so is the distance of another one
    slack = torch.where(gap > 0, 2.0 ** -22 * s * (most.abs()[:, 0].double() + gap), 0.0)
    xx, ww = x.to(_dt(name)), w.to(_dt(name))
    g = 1.0 / scale
    loss, dx, dw = head.cross_entropy_grad(xx, ww, y, grad=g, scale=scale,
                                           dw=torch.empty((v, d), device="cuda"))
    assert ((loss.double() - want).abs() <= slack + 2.0 ** -20 * (1 + want)).all()
    assert torch.equal(head.cross_entropy(xx, ww, y, scale=scale), loss)
    dz = s * torch.tensor(g, dtype=torch.float32).double() * (q - p)
    u = _half(xx.dtype)
    off = 2.2 * u * (q + p) + 2.0 ** -36
    assert ((dw.double() - dz.t() @ x.double()).abs() <= off.t() @ x.double() * 1.01).all()
    b = off @ w.double().abs()
    assert ((dx.double() - dz @ w.double()).abs() <= b + u * ((dz @ w.double()).abs() + b) + 2.0 ** -24).all()
    index = torch.stack([y, z.argmax(1)], 1)
    teacher_says = torch.tensor([[0.0, 0.0]], device="cuda").repeat(t, 1)
    got = head.distill(xx, ww, index, teacher_says, temperature=1.0 / scale)
    inv = (1.0 / torch.tensor(1.0 / scale, dtype=torch.float32)).double()
    want = top.sum(1).log() + 0.5 * gap * inv - math.log(2.0)
    assert ((got.double() - want).abs() <= slack + 2.0 ** -20 * (1 + want.abs())).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,d,v", [(1, 1, 300), (9, 32, 2500), (70, 80, 1000), (517, 768, 32308)])
def test_dz_is_rounded_once_to_its_type(t, d, v, name):
    """Rows of x that are 1 in one column make dw dz itself.  An exponential is kept to
    2^-13 or 2^-10 of itself (a quarter of the type's half step) until its row's sum is
    known, and dz then to half a step; of an exponential, its argument and the row's sum 2^-18 more."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(t)
    w = (3 * torch.randn((v, d), generator=gen, device="cuda")).to(_dt(name))
    x = torch.zeros((t, d), device="cuda", dtype=w.dtype)
    x[torch.arange(t), torch.arange(t)] = 1.0
    y = torch.randint(0, v, (t,), generator=gen, device="cuda")
    index = torch.stack([y, (y + 1) % v], 1)
    u = _half(w.dtype)
    q = torch.softmax(w[:, :t].t().double(), 1)
    for p, call in (
            (one_hot(y, y >= 0, v), lambda o: head.cross_entropy_grad(x, w, y, grad=0.75, dw=o)),
            (0.5 * one_hot(y, y >= 0, v) + 0.5 * one_hot(index[:, 1], y >= 0, v),
             lambda o: head.distill_grad(x, w, index, torch.zeros((t, 2), device="cuda"), grad=0.75,
                                         dw=o))):
        dw = call(torch.empty((v, d), device="cuda"))[2]
        off = (dw[:, :t].t().double() / 0.75 - (q - p)).abs()
        at = p > 0
        # an entry at a target is q - p in fp32, rounded once
        limit = torch.where(at, u * (q - p).abs() + 2.0 ** -18 * (q + p), q * (1.27 * u + 2.0 ** -18))
        if name == "f16":
            # an exponential below 2^-14 of 2^t, which its span's largest is to sqrt(2), is off
            # by 2^-27 of that, a dz below 2^-27 of the largest gradient by 2^-38
            limit = limit + 2.0 ** -26.5 + 2.0 ** -38
        assert (off <= limit * (1 + u)).all(), (off / limit).max().item()
        assert not dw[:, t:].any()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t", [40, 1100])
@pytest.mark.parametrize("grad", [1 / 3, 46.88, 1e-3 * 1.0078, -0.7])
def test_one_gradient_of_all_tokens_is_not_rounded(grad, t, name):
    """Tokens that are not expected (q of 1 / v) have -grad (1 - q) at their targets:
    with the one number in its place as a power of two, what is left of its rounding is q,
    the same direction for all tokens and so in every sum of them otherwise."""
    torch = _torch()
    d, v = 1100, 5000
    w = torch.zeros((v, d), device="cuda", dtype=_dt(name))
    x = torch.zeros((t, d), device="cuda", dtype=_dt(name))
    x[torch.arange(t), torch.arange(t) % d] = 1.0
    y = torch.randperm(v, device="cuda")[:t]
    dw = head.cross_entropy_grad(x, w, y, grad=grad, dw=torch.empty((v, d), device="cuda"))[2]
    at = dw[y, torch.arange(t, device="cuda") % d].double()
    exact = torch.tensor(grad, dtype=torch.float32).double()
    assert ((at / exact + 1 - 1 / v).abs() <= 1 / v + 2.0 ** -18).all()
    g = torch.full((t,), grad, device="cuda")
    again = head.cross_entropy_grad(x, w, y, grad=g, dw=torch.empty((v, d), device="cuda"))[2]
    assert torch.equal(dw, again)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,d,v", [(1, 40, 300), (7, 32, 2500), (32, 300, 700), (33, 90, 5000),
                                   (64, 256, 3000), (50, 768, 32000)])
def test_few_tokens_have_dz_in_two_parts(t, d, v, name):
    """dw is dz itself where rows of x are 1 in one column, and dx where rows of w are: of
    at most 64 tokens only the exponentials' 16 bits (a quarter of half a step) are left of
    dz's rounding, at targets none, and dx has its own.  A first part of half a step u leaves
    at most u of dz, which the second has to u of itself: u^2 of dz (2^-16 in bf16)."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(t + d)
    w = (3 * torch.randn((v, d), generator=gen, device="cuda")).to(_dt(name))
    x = torch.zeros((t, d), device="cuda", dtype=w.dtype)
    x[torch.arange(t), torch.arange(t) % d] = 1.0
    w[: d - 1] = 0
    w[torch.arange(d - 1), torch.arange(1, d)] = 1.0  # column c is one of row c - 1, and of others
    w[d - 1:, 1:] = 0  # whose only column is 0
    y = torch.randint(0, v, (t,), generator=gen, device="cuda")
    y[1::5] = -100
    live = y >= 0
    g = torch.rand(t, generator=gen, device="cuda") + 0.1
    g[2::7] *= -3e-3
    u = _half(w.dtype)
    q = torch.softmax(x.double() @ w.double().t(), 1)
    p = one_hot(y, live, v)
    scale = (g.double() * live)[:, None]
    dz = scale * (q - p)
    loss, dx, dw = head.cross_entropy_grad(x, w, y, grad=g, dw=torch.empty((v, d), device="cuda"))
    off = scale.abs() * torch.where(p > 0, 2.0 ** -18 * (q + p), q * (0.25 * u + 2.0 ** -18))
    off = off * (1 + u) + u * u * dz.abs()
    if name == "f16":  # a small exponential's 2^-27, and dz's 2^-39 of the largest gradient
        off = off + scale.abs() * 2.0 ** -26.5 + (scale != 0) * scale.abs().max() * 2.0 ** -38
    limit = off.t() @ x.double()
    assert ((dw.double() - dz.t() @ x.double()).abs() <= limit * 1.01 + 1e-30).all()
    want = dz[:, :d - 1]
    err = off[:, :d - 1] * 1.01
    tiny = 2.0 ** -25 if name == "f16" else 0.0
    assert ((dx[:, 1:].double() - want).abs() <= err + u * (want.abs() + err) + tiny).all()
    assert not dx[~live].any()
    # accumulated, and of a teacher's one entry
    before = torch.randn((v, d), device="cuda")
    both = head.cross_entropy_grad(x, w, y, grad=g, dw=before.clone(), accumulate=True)[2]
    assert torch.equal(both, before + dw)
    again = head.distill_grad(x, w, y[:, None], torch.zeros((t, 1), device="cuda"), grad=g,
                              dw=torch.empty((v, d), device="cuda"))
    assert torch.equal(again[1], dx) and torch.equal(again[2], dw)
    for dropped in ({"dx": False}, {"dw": False}):
        part = head.cross_entropy_grad(x, w, y, grad=g, **dropped)
        assert torch.equal(part[1], dx) if part[1] is not None else part[2] is not None
