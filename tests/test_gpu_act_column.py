"""The 8-bit form of a single column (include/ark_act.h) longer than a launch
has lanes."""
import numpy as np
import pytest

from ark_amd import act
from tests.test_gpu_act import _dt, _f64, _torch, eight

pytestmark = pytest.mark.gpu


def test_a_column_of_more_than_2_to_the_32_tokens():
    torch = _torch()
    t = (1 << 32) + 1000
    x = torch.zeros((t, 1), dtype=torch.float16, device="cuda")
    places = [(lo, lo + 320) for lo in (0, (1 << 28) - 160, (1 << 31), (1 << 32) - 160, t - 319)]
    for lo, hi in places:
        x[lo:hi] = torch.randn((min(hi, t) - lo, 1), device="cuda").half()
    kept = act.pack(x)
    back = act.unpack(kept, torch.full_like(x, 5.0))
    seen = torch.zeros((), dtype=torch.int64, device="cuda")
    for lo, hi in places:
        a, b = lo // 32 * 32, min(-(-hi // 32) * 32, t)
        np.testing.assert_array_equal(_f64(back[a:b]), eight(_f64(x[a:b]), "f16"))
        seen += torch.count_nonzero(back[a:b])
    total = sum(torch.count_nonzero(back[i:i + (1 << 28)]) for i in range(0, t, 1 << 28))
    assert int(total) == int(seen)          # and zeros everywhere else


@pytest.mark.parametrize("name", ["f16", "bf16", "f32"])
def test_a_column_of_another_stride(name):
    """Longer than one turn of the kernels' grids (2^20 blocks of 256 lanes)."""
    torch = _torch()
    t = (1 << 28) + 77
    wide = torch.zeros((t, 2), dtype=_dt(name), device="cuda")
    wide[:, 1] = 3.0
    wide[:1000, 0] = torch.randn(1000, device="cuda").to(_dt(name))
    wide[-1000:, 0] = torch.randn(1000, device="cuda").to(_dt(name))
    out = torch.full_like(wide, 7.0)
    act.unpack(act.pack(wide[:, :1]), out[:, :1])
    lo = (t - 1000) // 32 * 32
    for a, b in ((0, 1024), (lo, t)):
        np.testing.assert_array_equal(_f64(out[a:b, :1]), eight(_f64(wide[a:b, :1]), name))
    assert not out[1024:lo, 0].any() and (out[:, 1] == 7).all()
