"""Rotary positions and head norms (include/ark_rope.h) where q and k differ: one of
zero heads beside one that has some, or both of none, or one kept in 8 bits and the
other a tensor.  A part without heads is no work, and its gain's gradient is zero
(or stays as it was, when it is added to)."""
import numpy as np
import pytest

from ark_amd import act
from ark_amd.rope import Rope
from tests.test_gpu_act import _f64, _torch
from tests.test_gpu_rope import Turn, _back64, _gains, _norm64, _qk, _round_to

pytestmark = pytest.mark.gpu


def _near(got, want, bound, name="f32"):
    """Within the bound; a NaN is not."""
    assert (np.abs(_f64(got) - want) <= _round_to(bound, want, name)).all()


@pytest.mark.parametrize("name,d,r", [("f16", 64, 64), ("bf16", 66, 66), ("f32", 256, 128),
                                      ("f16", 510, 38), ("f32", 5, 4)])
def test_q_of_no_heads(name, d, r):
    torch = _torch()
    rope = Rope(d, r)
    gains = _gains(d, "f32")
    for shape in ((1,), (40,), (2, 350)):
        q, k = _qk(shape, 0, 3, d, name)
        dq, dk = _qk(shape, 0, 3, d, name, 2)
        turn = Turn(np.broadcast_to(np.arange(shape[-1]), shape), d, r, "half")
        x, g = _f64(k), _f64(gains[1])
        y = rope.apply(q, k)
        assert y[0].shape == q.shape and torch.equal(y[1], rope.apply(k))
        assert torch.equal(rope.apply(dq, dk, inverse=True)[1], rope.apply(dk, inverse=True))
        yq, yk, aq, ak = rope.norm(q, k, *gains, keep8=True)
        assert aq.nbytes == 0
        _near(yk, *_norm64(x, g, turn), name)
        _near(rope.norm(q, k, *gains)[1], *_norm64(x, g, turn), name)
        for kept in ((q, k), (aq, ak)):
            if kept[1] is ak:
                x = _f64(act.unpack(ak)).reshape(k.shape)
            back = rope.norm_backward(dq, dk, *kept, *gains)
            dx, b, dg, gb = _back64(_f64(dk), x, g, turn, tuple(range(len(shape) + 1)))
            _near(back[1], dx, b, name)
            _near(back[3], dg, gb)
            assert not back[2].any()
            a, c = torch.full((d,), 5.0, device="cuda"), torch.zeros(d, device="cuda")
            rope.norm_backward(dq, dk, *kept, *gains, dgain_q=a, dgain_k=c, accumulate=True)
            assert (a == 5.0).all() and torch.equal(c, back[3])


def test_neither_has_heads():
    torch = _torch()
    rope = Rope(64)
    gains = _gains(64, "f32")
    for shape in ((1,), (3, 50)):
        q, k = _qk(shape, 0, 0, 64, "f16")
        assert rope.apply(q, k)[1].shape == k.shape
        for kept in ((q, k), rope.norm(q, k, *gains, keep8=True)[2:]):
            a, b = torch.full((64,), 5.0, device="cuda"), torch.full((64,), 5.0, device="cuda")
            rope.norm_backward(q, k, *kept, *gains, dgain_q=a, dgain_k=b)
            assert not a.any() and not b.any()
            a.fill_(3.0), b.fill_(3.0)
            rope.norm_backward(q, k, *kept, *gains, dgain_q=a, dgain_k=b, accumulate=True)
            assert (a == 3.0).all() and (b == 3.0).all()


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("d", [64, 66, 256])
@pytest.mark.parametrize("tokens", [1, 40, 700, 30000])
def test_k_of_no_heads_has_a_gradient_of_zeros(tokens, d, keep8):
    torch = _torch()
    rope = Rope(d)
    gains = _gains(d, "f32")
    # both parts first: memory used before holds what they left
    q, k = _qk((tokens,), 4, 2, d, "f16")
    dq, dk = _qk((tokens,), 4, 2, d, "f16", 2)
    want = rope.norm_backward(dq, dk, q, k, *gains)
    none, dnone = k[:, :0], dk[:, :0]
    kept = rope.norm(q, none, *gains, keep8=True)[2:] if keep8 else (q, none)
    a, b = (torch.full((d,), 5.0, device="cuda") for _ in range(2))
    got = rope.norm_backward(dq, dnone, *kept, *gains, dgain_q=a, dgain_k=b)
    assert got[1].shape == (tokens, 0, d) and not b.any()
    if not keep8:
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    b.fill_(5.0)
    first = a.clone()
    rope.norm_backward(dq, dnone, *kept, *gains, dgain_q=a, dgain_k=b, accumulate=True)
    assert (b == 5.0).all() and torch.equal(a, first + first)


@pytest.mark.parametrize("name,d", [("f16", 64), ("bf16", 128), ("f32", 66)])
@pytest.mark.parametrize("which", [0, 1])
def test_one_input_kept_and_the_other_a_tensor(name, d, which):
    torch = _torch()
    rope = Rope(d)
    gains = _gains(d, "f32")
    for shape in ((1,), (2, 70)):
        xs, dys = _qk(shape, 4, 2, d, name), _qk(shape, 4, 2, d, name, 2)
        kept = list(xs)
        kept[which] = rope.norm(*xs, *gains, keep8=True)[2 + which]
        back = rope.norm_backward(*dys, *kept, *gains)
        turn = Turn(np.broadcast_to(np.arange(shape[-1]), shape), d, d, "half")
        for i in range(2):
            x = _f64(act.unpack(kept[i])).reshape(xs[i].shape) if i == which else _f64(xs[i])
            dx, b, dg, gb = _back64(_f64(dys[i]), x, _f64(gains[i]), turn,
                                    tuple(range(len(shape) + 1)))
            _near(back[i], dx, b, name)
            _near(back[2 + i], dg, gb)


def test_one_input_kept_by_the_c_entry():
    """ark_rope_norm with a q_act or a k_act alone writes what pack gives."""
    torch = _torch()
    import ctypes as C
    from ark_amd import _abi, _lib
    rope = Rope(64)
    g = _gains(64, "f32")
    q, k = _qk((2, 45), 3, 2, 64, "f16")
    want = rope.norm(q, k, *g)
    lay = [(C.c_uint64 * 4)(x.shape[2], x.stride(0), x.stride(1), x.stride(2)) for x in (q, k)]
    for which in (0, 1):
        out = [torch.empty_like(x) for x in (q, k)]
        kept = act.Act8(90, 64 * (3, 2)[which], torch.float16)
        kept.data.fill_(1)
        acts = [kept.data.data_ptr() if i == which else None for i in range(2)]
        _lib.check(_lib.lib().ark_rope_norm(
            rope._h, _abi.ACT_F16, 2, 45, None, 0, 0, 1e-5, g[0].data_ptr(), g[1].data_ptr(),
            _abi.ACT_F32, q.data_ptr(), lay[0], out[0].data_ptr(), lay[0], acts[0], k.data_ptr(),
            lay[1], out[1].data_ptr(), lay[1], acts[1], _lib.current_stream(q)))
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert torch.equal(kept.data, act.pack((q, k)[which].reshape(90, -1)).data)
