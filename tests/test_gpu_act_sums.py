"""How exact the weight gradient's sums are (include/ark_act.h) where fp16
factors are subnormal.

Every product is exact in fp32, and stays so in a sum that fp32 holds exactly.
Elsewhere each of a sum's T additions may be off by 2^-23 of the largest number
it aligns to: the sum so far, or the product by its factors' exponent fields.  A
subnormal fp16's field is that of 2^-14, so a dy below 2^-14 counts as that, and
an activation more than 2^23 below its column's largest 2^e, which is subnormal
where that is brought near fp16's top, as 2^-23 of it; zeros count as nothing."""
import numpy as np
import pytest

from ark_amd import act
from tests.test_gpu_act import _f64, _torch, eight

pytestmark = pytest.mark.gpu


def _half(x):
    return _torch().from_numpy(np.ascontiguousarray(x)).half().cuda()


@pytest.mark.parametrize("layout", ["in_out", "out_in"])
@pytest.mark.parametrize("t,c,n", [(1, 16, 1023), (64, 64, 64), (100, 130, 257), (128, 500, 3)])
def test_subnormal_gradients_keep_all_their_bits(t, c, n, layout):
    """Odd multiples of 2^-24 up to 1023 of them: 128 x 127 x 1023 < 2^24."""
    rng = np.random.default_rng(t + c + n)
    x = rng.integers(-127, 128, (t, c)).astype(np.float64)
    x[::32] = 127.0
    dy = (rng.integers(0, 512, (t, n)) * 2 + 1) * rng.choice([-1.0, 1.0], (t, n)) * 2.0 ** -24
    for e in (0, -24, 9):          # the activations' exponent: fp16's smallest and largest
        dw = act.weight_grad(act.pack(_half(x * 2.0 ** e)), _half(dy), layout=layout)
        want = (x * 2.0 ** e).T @ dy
        np.testing.assert_array_equal(_f64(dw), want if layout == "in_out" else want.T)


def _bound(x, dy):
    """Of act's values x and dy: (T + 1) 2^-23 of the sum of what products count as."""
    m, e = np.frexp(np.abs(x).max(0))
    least = np.exp2(np.where(m > 127 / 128, e - 6, e - 7) - 23.0)
    a = np.where(x == 0, 0.0, np.maximum(np.abs(x), least))
    b = np.where(dy == 0, 0.0, np.maximum(np.abs(dy), 2.0 ** -14))
    return (len(x) + 1) * 2.0 ** -23 * (a.T @ b)


def _check(x, dy):
    x, dy = _half(x), _half(dy)
    a, b = eight(_f64(x), "f16"), _f64(dy)
    assert (np.abs(_f64(act.weight_grad(act.pack(x), dy)) - a.T @ b) <= _bound(a, b)).all()


@pytest.mark.parametrize("e", [-8, -12, -16, -20])
@pytest.mark.parametrize("small", [1, 1001])
def test_a_subnormal_gradient_beside_ordinary_ones(e, small):
    """A sum of small activations by ordinary gradients, then a large activation by a
    subnormal gradient."""
    rng = np.random.default_rng(small - e)
    x = np.full((64, 64), 127.0)
    x[:32] = rng.integers(-127, 128, (32, 64)) * 2.0 ** e
    dy = np.zeros((64, 64))
    dy[:32] = rng.integers(1024, 2048, (32, 64)) * rng.choice([-1, 1], (32, 64)) * 2.0 ** -23
    dy[37] = small * 2.0 ** -24
    _check(x, dy)


@pytest.mark.parametrize("e", [-10, -14, -20, -24])
def test_activations_far_below_their_column(e):
    """The column's largest activations have no gradient (a masked token)."""
    rng = np.random.default_rng(-e)
    x = rng.integers(-127, 128, (96, 64)) * 2.0 ** e
    x[:32] = 63 * 1024.0
    dy = rng.integers(1024, 2048, (96, 64)) * 2.0 ** (rng.integers(-13, 5, (96, 1)) - 10.0)
    dy[:32] = 0.0
    _check(x, dy)


@pytest.mark.parametrize("t", [33, 2048, 5000])
def test_gradients_of_a_low_loss_scale(t):
    """Gradients mostly below 2^-14, tokens and groups of many sizes."""
    rng = np.random.default_rng(t)
    x = rng.standard_normal((t, 70)) * np.exp2(rng.integers(-20, 4, (-(-t // 32), 1))).repeat(32, 0)[:t]
    dy = rng.standard_normal((t, 90)) * np.exp2(rng.integers(-24, -10, (t, 1)))
    _check(x, dy)
