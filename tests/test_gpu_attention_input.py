"""The example that runs the rotation, the norms, the 8-bit activations and
their weight gradient with the optimizer (examples/attention_input.py): its
gradients are those of the same block in 64 bits, and it learns.

The 64-bit gradients are taken at the values the kernels read (the 8-bit forms,
the fp16 gradient of the rotated heads).  A head's gradient passes through the
norm in fp32 and is rounded once to fp16, 2^-11 of itself or half of fp16's
smallest step, 2^-25; the sum over T tokens adds (T + 2) 2^-23 of the sum of
magnitudes, in which the norm's own fp32 roundings (under 2^-18 of the magnitudes
it mixes, at most twice the row's largest) are counted by 2^-16 of the row's
norm."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                     "attention_input.py")


@pytest.fixture(scope="module")
def example():
    import torch
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    spec = importlib.util.spec_from_file_location("attention_input", _PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("tokens,heads,kv_heads,head", [(257, 4, 2, 32), (1, 3, 3, 64)])
def test_gradients(example, norm, tokens, heads, kv_heads, head):
    import torch
    from ark_amd import act
    torch.manual_seed(3)
    hidden = 48
    block = example.AttentionInput(hidden, heads, kv_heads, head, norm)
    if norm:
        for i in (2, 3):
            block.params.w(i).normal_(1.0, 0.2)
    x = torch.randn((tokens, hidden), device="cuda").half()
    q, k, kept = block.forward(x)
    x8 = act.unpack(kept[0]).double()
    angle = torch.arange(tokens, device="cuda").double()[:, None] * torch.tensor(
        block.rope.inv_freq, device="cuda", dtype=torch.float64)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    dq, dk = (torch.randn_like(t) for t in (q, k))
    given = dq.clone(), dk.clone()
    block.backward(dq, dk, kept, accumulate=False)
    for i, d in enumerate(given):
        n = heads if i == 0 else kv_heads
        u, v = d.double().split(head // 2, -1)
        back = torch.cat([u * c + v * s, v * c - u * s], -1)
        size = back.abs()
        if norm:
            h = act.unpack(kept[1 + i]).double().view(tokens, n, head)
            gain = block.params.w(2 + i).double()
            r = (h.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
            gains = (back * h * r).sum((0, 1))
            bound = (2.0 ** -16 + (tokens * n + 2) * 2.0 ** -23) * (
                back.norm(dim=-1, keepdim=True) * (h * r).norm(dim=-1, keepdim=True)).sum((0, 1))
            assert ((block.params.g(2 + i).double() - gains).abs() <= bound).all()
            back = r * (back * gain - h * (back * gain * h).mean(-1, keepdim=True) * r * r)
            size = r * ((back / r).norm(dim=-1, keepdim=True) + gain.abs().max() * size.norm(
                dim=-1, keepdim=True))
        bound = 2.0 ** -11 * back.abs() + 2.0 ** -25 + 2.0 ** -16 * size
        want = x8.t() @ back.reshape(tokens, -1)
        limit = x8.abs().t() @ (bound + (tokens + 2) * 2.0 ** -23 * (back.abs() + bound)).reshape(
            tokens, -1)
        got = block.params.g(i).view(hidden, -1).double()
        assert ((got - want).abs() <= limit).all()


@pytest.mark.parametrize("norm", [True, False])
def test_learns_and_repeats(example, norm):
    run = lambda: example.train(hidden=96, heads=3, kv_heads=1, head=32, tokens=300, steps=40,
                                norm=norm, lr=1e-2)
    losses = run()
    assert losses[-1] < 0.2 * losses[0], losses
    assert losses == run()
