"""Activations in 8 bits and the weight gradient from them
(include/ark_act.h), against their definition in 64 bits.

The 8-bit form is defined to the bit, so what is packed and read back must
equal the definition exactly.  The weight gradient's products are exact in
fp32, so whole-number inputs whose sums stay below 2^24 must give exact sums in
any order; elsewhere a sum of T terms may be off by (T + 1) 2^-23 of the sum of
magnitudes (one rounding, to nearest or toward zero, an addition)."""
import numpy as np
import pytest

from ark_amd import act
from ark_amd._lib import ArkOptError

pytestmark = pytest.mark.gpu

TYPES = ["f16", "bf16", "f32"]


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch


def _dt(name):
    torch = _torch()
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def eight(x, name):
    """The values the 8-bit form of x (float64 numpy, tokens x columns) stands for."""
    t, c = x.shape
    g = np.concatenate([x, np.zeros((-t % 32, c))]).reshape(-1, 32, c)
    a = np.abs(g).max(1, keepdims=True)
    bad = ~np.isfinite(g).all(1, keepdims=True)
    a = np.where(bad, 1.0, a)
    m, e = np.frexp(a)                      # a = m 2^e, m in [0.5, 1)
    e = np.where(m > 127 / 128, e - 6, e - 7)
    e = np.where(a == 0, -1000, e)
    e = np.clip(e, -24 if name == "f16" else -126, 121)
    top = np.where(e >= 10, 63.0, 127.0) if name == "f16" else 127.0
    with np.errstate(invalid="ignore"):
        q = np.clip(np.rint(np.ldexp(g, -e)), -top, top)
    return np.where(bad, np.nan, np.ldexp(q, e)).reshape(-1, c)[:t]


def _f64(t):
    return t.double().cpu().numpy()


def _values(rng, t, c, name):
    """Normal values over many binades, whole groups of zeros and tiny values."""
    x = rng.standard_normal((t, c)) * np.exp2(rng.integers(-30, 12, (1, c)))
    x[:, ::7] *= np.exp2(rng.integers(-10, 3, (t, 1)))
    if c > 3:
        x[:, 3] = 0.0
    return np.clip(x, -65504, 65504) if name == "f16" else x


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,c", [(1, 1), (1, 64), (31, 5), (32, 64), (33, 65), (100, 1),
                                 (257, 333), (64, 768), (1000, 129)])
def test_round_trip(t, c, name):
    torch = _torch()
    x = torch.from_numpy(_values(np.random.default_rng(t * 1000 + c), t, c, name)).to(_dt(name))
    x = x.cuda()
    kept = act.pack(x)
    assert kept.nbytes == -(-t // 32) * c * 33
    back = act.unpack(kept)
    np.testing.assert_array_equal(_f64(back), eight(_f64(x), name))
    wide = act.unpack(kept, torch.empty((t, c), dtype=torch.float32, device="cuda"))
    np.testing.assert_array_equal(_f64(wide), eight(_f64(x), name))


@pytest.mark.parametrize("name", TYPES)
def test_edges_of_the_exponent(name):
    """Largest magnitudes at, just below and just above 127 * 2^e, the type's
    largest and smallest numbers, and ties of the rounding."""
    torch = _torch()
    cols = []
    for e in (range(-24, 10) if name == "f16" else (-126, -125, -60, 0, 60, 119, 120)):
        for m in (127.0, 126.5, 127.5, 128.0, 64.0, 63.5):
            cols.append(np.ldexp(np.linspace(-m, m, 32), e))
            cols.append(np.ldexp(np.concatenate([[m], np.arange(31) + 0.5]), e))
    for v in {"f16": (65504.0, 65024.0, 64512.0, 2.0 ** -24, 2.0 ** -14),
              "bf16": (3.3895e38, 2.0 ** -133, 2.0 ** -126),
              "f32": (3.4028234663852886e38, 2.0 ** -149, 2.0 ** -126, 1.0 - 2.0 ** -24)}[name]:
        cols.append(np.linspace(-v, v, 32))
        cols.append(np.full(32, -v))
    x = torch.from_numpy(np.clip(np.stack(cols, 1), -3.4028234663852886e38, 3.4028234663852886e38))
    x = x.float().to(_dt(name)).cuda()
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    back = act.unpack(act.pack(x))
    assert torch.isfinite(back).all()
    np.testing.assert_array_equal(_f64(back), eight(_f64(x), name))


@pytest.mark.parametrize("name", TYPES)
def test_every_value_is_near(name):
    """A read-back value is within half a step, a step being at most 2 / 127 of
    the group's largest magnitude (a whole step where fp16's top binds)."""
    torch = _torch()
    x = torch.randn((4096, 96), device="cuda").to(_dt(name))
    d = (act.unpack(act.pack(x)).double() - x.double()).abs().view(-1, 32, 96)
    most = x.double().abs().view(-1, 32, 96).amax(1, keepdim=True)
    assert (d <= most / 127 * (1 + 1e-12)).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_non_finite_value_makes_its_group_nan(name, bad):
    torch = _torch()
    x = torch.randn((70, 40), device="cuda").to(_dt(name))
    x[33, 7] = bad
    x[69, 0] = bad
    back = act.unpack(act.pack(x))
    np.testing.assert_array_equal(_f64(back), eight(_f64(x), name))
    assert torch.isnan(back[32:64, 7]).all() and torch.isnan(back[64:, 0]).all()
    assert int(torch.isnan(back).sum()) == 32 + 6


def test_strided_rows_and_untouched_gaps():
    torch = _torch()
    big = torch.randn((100, 500), device="cuda", dtype=torch.float16)
    x = big[3:80, 7:130]          # odd offset: rows not aligned to 4 bytes
    kept = act.pack(x)
    want = eight(_f64(x), "f16")
    out = torch.full((77, 300), 5.0, device="cuda", dtype=torch.float16)
    act.unpack(kept, out[:, 11:134])
    np.testing.assert_array_equal(_f64(out[:, 11:134]), want)
    assert (out[:, :11] == 5).all() and (out[:, 134:] == 5).all()
    one = act.pack(big[:1, ::1].expand(40, 500))   # rows at stride 0
    np.testing.assert_array_equal(_f64(act.unpack(one)), eight(_f64(big[:1].expand(40, 500)),
                                                               "f16"))


def test_nothing_is_written_past_the_buffers():
    torch = _torch()
    for t, c in ((33, 5), (1, 1), (64, 130)):
        n = -(-t // 32) * c * 33
        raw = torch.full((n + 64,), 77, dtype=torch.uint8, device="cuda")
        x = torch.randn((t, c), device="cuda")
        kept = act.Act8(t, c, torch.float32, data=raw[:n])
        act.pack(x, kept)
        assert (raw[n:] == 77).all()
        out = torch.full((t + 1, c), 5.0, device="cuda")
        act.unpack(kept, out[:t])
        assert (out[t:] == 5).all()


def test_more_than_2_to_the_32_values():
    torch = _torch()
    t, c = 32 * 66000 + 5, 2048
    x = torch.zeros((t, c), dtype=torch.float16, device="cuda")
    tail = torch.randn((101, c), device="cuda").half()
    x[-101:] = tail
    x[:64] = tail[:64]
    kept = act.pack(x)
    back = act.unpack(kept)
    lo = t - t % 32 - 64
    np.testing.assert_array_equal(_f64(back[lo:]), eight(_f64(x[lo:]), "f16"))
    np.testing.assert_array_equal(_f64(back[:64]), eight(_f64(x[:64]), "f16"))
    assert not back[64:t - 101].any()
    del back
    dy = torch.zeros((t, 8), dtype=torch.float16, device="cuda")
    dy[-3:] = 1.0
    dw = act.weight_grad(kept, dy)
    want = eight(_f64(x[lo:]), "f16")[-3:].sum(0)
    bound = 4 * 2.0 ** -23 * np.abs(eight(_f64(x[lo:]), "f16")[-3:]).sum(0)
    assert (np.abs(_f64(dw) - want[:, None]) <= bound[:, None]).all()


# ---- the weight gradient ------------------------------------------------------

def _whole(rng, t, c, n):
    """Whole numbers with exponent 0 in every group (its first value is 127),
    few enough in size that sums stay exact."""
    x = rng.integers(-127, 128, (t, c)).astype(np.float64)
    x[::32] = 127.0
    dy = rng.integers(-3, 4, (t, n)).astype(np.float64)
    assert t * 127 * 3 < 2 ** 24
    return x, dy


SHAPES = [(1, 1, 1), (1, 64, 64), (5, 3, 7), (31, 16, 16), (32, 16, 16), (33, 17, 15),
          (64, 64, 64), (65, 130, 70), (127, 128, 128), (128, 129, 257), (300, 1, 300),
          (300, 300, 1), (333, 333, 901), (512, 256, 256), (1000, 100, 40), (2048, 768, 96),
          (4099, 96, 768), (8192, 64, 64), (16384, 33, 50), (40000, 8, 8), (4096, 520, 392)]


@pytest.mark.parametrize("t,c,n", SHAPES)
@pytest.mark.parametrize("name,layout", [("f16", "in_out"), ("f16", "out_in"),
                                         ("bf16", "in_out"), ("bf16", "out_in")])
def test_weight_grad_is_exact_on_whole_numbers(t, c, n, name, layout):
    torch = _torch()
    x, dy = _whole(np.random.default_rng(t + c + n), t, c, n)
    kept = act.pack(torch.from_numpy(x).to(_dt(name)).cuda())
    dw = act.weight_grad(kept, torch.from_numpy(dy).to(_dt(name)).cuda(), layout=layout)
    want = x.T @ dy
    np.testing.assert_array_equal(_f64(dw), want if layout == "in_out" else want.T)


@pytest.mark.parametrize("kept_type,dy_type", [("f16", "f16"), ("f16", "bf16"), ("bf16", "bf16"),
                                               ("f32", "bf16")])
@pytest.mark.parametrize("t,c,n", [(100, 64, 48), (777, 200, 130), (4000, 96, 64)])
def test_weight_grad_types(t, c, n, kept_type, dy_type):
    torch = _torch()
    rng = np.random.default_rng(t)
    x = torch.from_numpy(_values(rng, t, c, kept_type)).to(_dt(kept_type)).cuda()
    dy = torch.from_numpy(rng.standard_normal((t, n)) * 0.3).to(_dt(dy_type)).cuda()
    dw = act.weight_grad(act.pack(x), dy)
    a, b = eight(_f64(x), kept_type), _f64(dy)
    assert (np.abs(_f64(dw) - a.T @ b) <= (t + 1) * 2.0 ** -23 * (np.abs(a).T @ np.abs(b))).all()


def test_weight_grad_keeps_small_numbers():
    """fp16 values below 2^-14 on both sides, and exponents at both ends."""
    torch = _torch()
    rng = np.random.default_rng(5)
    x = rng.integers(-127, 128, (64, 40)) * 2.0 ** -24
    x[:, 20:] = rng.integers(-63, 64, (64, 20)) * 1024.0
    dy = rng.integers(-9, 10, (64, 24)) * 2.0 ** -24
    kept = act.pack(torch.from_numpy(x).half().cuda())
    dw = act.weight_grad(kept, torch.from_numpy(dy).half().cuda())
    np.testing.assert_array_equal(_f64(dw), eight(x, "f16").T @ dy)


@pytest.mark.parametrize("layout", ["in_out", "out_in"])
@pytest.mark.parametrize("t,c,n", [(70, 40, 24), (3000, 130, 260), (0, 40, 24)])
def test_weight_grad_accumulates_and_keeps_strides(t, c, n, layout):
    torch = _torch()
    x, dy = _whole(np.random.default_rng(9), max(t, 1), c, n)
    x, dy = x[:t], dy[:t]
    shape = (c, n) if layout == "in_out" else (n, c)
    big = torch.full((shape[0], shape[1] + 9), 7.0, device="cuda")
    dw = big[:, 5:5 + shape[1]]
    dyb = torch.zeros((t, n + 3), dtype=torch.float16, device="cuda")
    dyb[:, 1:n + 1] = torch.from_numpy(dy).half().cuda()
    kept = act.pack(torch.from_numpy(x).half().cuda())
    want = x.T @ dy if layout == "in_out" else (x.T @ dy).T
    act.weight_grad(kept, dyb[:, 1:n + 1], dw, accumulate=True, layout=layout)
    np.testing.assert_array_equal(_f64(dw), want + 7)
    act.weight_grad(kept, dyb[:, 1:n + 1], dw, layout=layout)
    np.testing.assert_array_equal(_f64(dw), want)
    act.weight_grad(kept, dyb[:, 1:n + 1], dw, accumulate=True, layout=layout)
    np.testing.assert_array_equal(_f64(dw), 2 * want)
    assert (big[:, :5] == 7).all() and (big[:, 5 + shape[1]:] == 7).all()


def test_weight_grad_passes_non_finite_values_on():
    torch = _torch()
    x = torch.randn((100, 40), device="cuda").half()
    dy = torch.randn((100, 24), device="cuda").half()
    x[50, 3] = float("inf")
    dy[99, 5] = float("nan")
    dw = act.weight_grad(act.pack(x), dy)
    bad = ~torch.isfinite(dw)
    assert bad[3].all() and bad[:, 5].all()
    assert int(bad.sum()) == 24 + 40 - 1


def test_weight_grad_ignores_what_lies_past_the_last_row():
    """Rows of dy after the last token, and past its outputs, hold NaN."""
    torch = _torch()
    for t in (1, 33, 63, 65, 100):
        x, dy = _whole(np.random.default_rng(t), t, 20, 24)
        big = torch.full((t + 64, 31), float("nan"), dtype=torch.float16, device="cuda")
        big[:t, :24] = torch.from_numpy(dy).half().cuda()
        dw = act.weight_grad(act.pack(torch.from_numpy(x).half().cuda()), big[:t, :24])
        np.testing.assert_array_equal(_f64(dw), x.T @ dy)


def test_weight_grad_far_strides():
    """Rows of dy 2^27 values apart: offsets past 2^32 bytes."""
    torch = _torch()
    x, dy = _whole(np.random.default_rng(2), 40, 24, 16)
    big = torch.empty(((40 - 1) * (1 << 27) + 16,), dtype=torch.float16, device="cuda")
    far = torch.as_strided(big, (40, 16), (1 << 27, 1))
    far.copy_(torch.from_numpy(dy).half().cuda())
    dw = act.weight_grad(act.pack(torch.from_numpy(x).half().cuda()), far)
    np.testing.assert_array_equal(_f64(dw), x.T @ dy)


def test_the_same_bits_every_time_on_any_stream():
    torch = _torch()
    x = torch.randn((5000, 200), device="cuda").half()
    dy = torch.randn((5000, 300), device="cuda").half()
    torch.cuda.synchronize()
    first = act.weight_grad(act.pack(x), dy)
    s = torch.cuda.Stream()
    got = []
    with torch.cuda.stream(s):
        for _ in range(4):
            got.append(act.weight_grad(act.pack(x), dy))
    torch.cuda.synchronize()
    assert all(torch.equal(first, g) for g in got)


def test_in_a_graph():
    """Captured, then replayed with other work between: every replay's results
    are the eager call's."""
    torch = _torch()
    x = torch.randn((3000, 96), device="cuda").half()
    dy = torch.randn((3000, 160), device="cuda").half()
    kept, dw = act.Act8(3000, 96, torch.float16), torch.empty((96, 160), device="cuda")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        act.pack(x, kept)
        act.weight_grad(kept, dy, dw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        act.pack(x, kept)
        act.weight_grad(kept, dy, dw)
    for k in range(4):
        x.normal_()
        dy.normal_()
        torch.cuda.synchronize()
        dw.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, act.weight_grad(act.pack(x), dy)), k


def test_gradient_by_differences():
    """L(w) = <x8 w, dy> is linear in w: a change of one weight by 1 changes L
    by its gradient, formed here in 64 bits."""
    torch = _torch()
    rng = np.random.default_rng(4)
    x = torch.from_numpy(rng.standard_normal((90, 12))).half().cuda()
    dy = torch.from_numpy(rng.standard_normal((90, 10))).half().cuda()
    kept = act.pack(x)
    dw, x8, d = _f64(act.weight_grad(kept, dy)), _f64(act.unpack(kept)), _f64(dy)
    w = rng.standard_normal((12, 10))
    base = ((x8 @ w) * d).sum()
    for c, o in ((0, 0), (11, 9), (5, 3)):
        w2 = w.copy()
        w2[c, o] += 1.0
        diff = ((x8 @ w2) * d).sum() - base
        assert abs(diff - dw[c, o]) <= 91 * 2.0 ** -23 * (np.abs(x8[:, c]) @ np.abs(d[:, o])) + 1e-9


def test_refusals():
    torch = _torch()
    x = torch.randn((64, 16), device="cuda").half()
    kept = act.pack(x)
    with pytest.raises(ValueError):
        act.pack(x.double())
    with pytest.raises(ValueError):
        act.pack(x.t())
    with pytest.raises(ValueError):
        act.pack(x.cpu())
    with pytest.raises(ValueError):
        act.pack(x, act.Act8(64, 17, torch.float16))
    with pytest.raises(ValueError):
        act.weight_grad(kept, x[:63])
    with pytest.raises(ValueError):
        act.weight_grad(kept, x, accumulate=True)
    with pytest.raises(ValueError):
        act.weight_grad(kept, x, layout="other")
    with pytest.raises(ArkOptError, match="dy is fp16 or bf16"):
        act.weight_grad(kept, x.float())
    with pytest.raises(ArkOptError, match="fp16 dy"):
        act.weight_grad(act.pack(x.float()), x)
    with pytest.raises(ArkOptError, match="exceeds its allocation"):
        torch.cuda.empty_cache()
        big = torch.empty(40 << 20, dtype=torch.uint8, device="cuda")
        from ark_amd import _abi
        from ark_amd._lib import check, lib
        check(lib().ark_act_unpack(big.data_ptr(), 1 << 20, 64, _abi.ACT_F16, x.data_ptr(), 64,
                                   None))


def test_a_gradient_of_an_optimizer_loses_its_units():
    """weight_grad writes gradients the optimizer's norm units may describe: a
    step after it reads the gradients, whatever the hand-off had written."""
    torch = _torch()
    from ark_amd import _abi
    from ark_amd.eko import TensorSpec
    from ark_amd.grad import GradPlan
    from ark_amd.optimizer import AdamConfig, AmpConfig, Optimizer, ParamSet
    spec = [TensorSpec("w", (64, 96), True, False)]
    infos = []
    for handoff in (False, True):
        ps = ParamSet(spec, 0.1, grad_dtype=_abi.GRAD_F32)
        ps.g(0).zero_()
        opt = Optimizer(AdamConfig(), ps, AmpConfig(loss_scale_init=1.0))
        x = torch.full((40, 64), 2.0, device="cuda").half()
        dy = torch.full((40, 96), 0.5, device="cuda").half()
        if handoff:
            plan = GradPlan([(ps.g(0), torch.ones(64 * 96, device="cuda"))])
            plan.run(final_for=opt)
            ps.g(0).zero_()
        act.weight_grad(act.pack(x), dy, ps.g(0).view(64, 96), accumulate=True)
        infos.append(opt.step_all(1e-3, info=True)[1])
        opt.close()
    assert infos[0].grad_norm == infos[1].grad_norm == np.sqrt(np.float32(1600.0 * 64 * 96))
