"""The weight gradient at sizes that take each of its tiles, with one sum and
with the tokens' sum split (ark_act_weight_grad chooses by sizes), and in
workspace of the caller's.  Whole numbers whose sums stay below 2^24 have exact
sums in any order."""
import ctypes as C

import pytest

from ark_amd import _abi, _lib, act

pytestmark = pytest.mark.gpu

# tokens, columns, outputs, whether the call splits
CUTS = [(1, 1, 8, False), (4000, 500, 8, True),        # 64 x 64
        (40, 3000, 1025, False), (4100, 1153, 513, True),    # 128 x 64
        (33, 3000, 1500, False), (4100, 700, 1500, True),    # 192 x 128
        (65, 3000, 4000, False), (4100, 3000, 700, True),    # 192 x 256
        (3000, 130, 4, True),
        (3000, 130, 3, False), (70, 5, 1, False)]            # fewer than four outputs


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch


def _need(t, c, n, stride=None):
    need = C.c_uint64()
    assert _lib.lib().ark_act_weight_grad_workspace(t, c, stride or n, n, C.byref(need)) == _abi.OK
    return need.value


@pytest.mark.parametrize("t,c,n,split", CUTS)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["in_out", "out_in"])
def test_every_cut_is_exact(t, c, n, split, name, layout):
    torch = _torch()
    dt = {"f16": torch.float16, "bf16": torch.bfloat16}[name]
    assert (_need(t, c, n) > 0) == split
    g = torch.Generator(device="cuda").manual_seed(t * 7 + c)
    x = torch.randint(-5, 6, (t, c), device="cuda", generator=g).to(dt)
    dy = torch.randint(-4, 5, (t, n), device="cuda", generator=g).to(dt)
    start = torch.randint(-9, 10, (c, n) if layout == "in_out" else (n, c), device="cuda",
                          generator=g).float()
    want = x.double().t().contiguous() @ dy.double()
    if layout == "out_in":
        want = want.t()
    kept = act.pack(x)
    assert torch.equal(act.weight_grad(kept, dy, layout=layout).double(), want)
    dw = start.clone()
    act.weight_grad(kept, dy, dw, accumulate=True, layout=layout)
    assert torch.equal(dw.double(), want + start)


@pytest.mark.parametrize("t,c,n", [(4000, 500, 8), (4100, 700, 1500), (70, 64, 64)])
def test_own_workspace_gives_the_same_bits(t, c, n):
    torch = _torch()
    L = _lib.lib()
    x = torch.randn((t, c), device="cuda").half()
    dy = torch.randn((t, n), device="cuda").half()
    kept = act.pack(x)
    need = _need(t, c, n)
    outs = [torch.empty((c, n), device="cuda") for _ in range(2)]
    ws = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    args = lambda dw: (kept.data.data_ptr(), _abi.ACT_F16, t, c, dy.data_ptr(), n, _abi.ACT_F16, n,
                       dw.data_ptr(), n, 0)
    s = _lib.current_stream(x)
    assert L.ark_act_weight_grad(*args(outs[0]), s) == _abi.OK
    assert L.ark_act_weight_grad_noalloc(*args(outs[1]), ws.data_ptr() if need else None, need,
                                         s) == _abi.OK
    assert torch.equal(*outs)
    assert (ws[need:] == 0xA5).all()


def test_workspace_refusals():
    torch = _torch()
    L = _lib.lib()
    t, c, n = 4000, 500, 8
    kept = act.pack(torch.zeros((t, c), device="cuda").half())
    dy = torch.zeros((t, n), device="cuda").half()
    dw = torch.full((c, n), 3.0, device="cuda")
    need = _need(t, c, n)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")

    def call(p, size):
        return L.ark_act_weight_grad_noalloc(
            kept.data.data_ptr(), _abi.ACT_F16, t, c, dy.data_ptr(), n, _abi.ACT_F16, n,
            dw.data_ptr(), n, 0, p, size, _lib.current_stream(dw))

    for p, size, word in [(ws.data_ptr(), need - 1, "needed"), (None, 0, "needed"),
                          (ws.data_ptr() + 4, need, "16-byte"),
                          (None, need, "workspace"), (dw.data_ptr(), need, "overlaps"),
                          (kept.data.data_ptr(), need, "overlaps")]:
        assert call(p, size) == _abi.EINVAL
        assert word in L.ark_opt_last_error().decode(), L.ark_opt_last_error()
    torch.cuda.synchronize()
    assert (dw == 3.0).all()
    assert call(ws.data_ptr(), need) == _abi.OK
    assert (dw == 0.0).all()
