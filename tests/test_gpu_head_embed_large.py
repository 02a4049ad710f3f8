"""The vocabulary loss and the embedding where offsets pass 32 bits: tables, rows
and gradients of over 4 GiB, of which only the far rows are looked at, and the
largest table.

Tolerances: a logit z of d products is within (d + 4) 2^-23 of its magnitudes, and
so are the loss and, relative, a probability; a gradient of bf16 has two roundings
of dz (2.3 2^-8 of the magnitudes), one of its own, and its sum's."""
import pytest

from ark_amd import embed, head

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    return torch


def test_a_table_of_over_4_gib():
    torch = _torch()
    v, d, t = 1 << 21, 1040, 40
    w = torch.empty((v, d), device="cuda", dtype=torch.bfloat16)
    for lo in range(0, v, 1 << 18):
        w[lo:lo + (1 << 18)].normal_(0.0, 0.02)
    x = torch.randn((t, d), device="cuda").bfloat16()
    y = torch.randint(v - 50, v, (t,), device="cuda")
    y[::7], y[5] = -100, 3
    live = y >= 0
    z = torch.empty((t, v), dtype=torch.float64, device="cuda")
    big = torch.empty_like(z)
    xd = x.double()
    for lo in range(0, v, 1 << 18):
        part = w[lo:lo + (1 << 18)].double().t().contiguous()
        z[:, lo:lo + (1 << 18)] = xd @ part
        big[:, lo:lo + (1 << 18)] = xd.abs() @ part.abs()
    bz = (d + 4) * 2.0 ** -23 * big.max().item()
    lse = torch.logsumexp(z, 1)
    at = torch.where(live, y, 0)[:, None]
    want = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    g = 8.0
    dw = torch.full((v, d), 7.0, device="cuda")
    loss, dx, out = head.cross_entropy_grad(x, w, y, grad=g, dw=dw)
    assert out is dw
    assert ((loss.double() - want).abs() <= 2 * bz + 2.0 ** -18 * lse.abs().max()).all()
    q = g * torch.exp(z - lse[:, None]) * live[:, None]
    dz = q.clone().scatter_add_(1, at, -g * live[:, None].double())
    size = q.scatter_add_(1, at, g * live[:, None].double())
    off = 2.3 * 2.0 ** -8 + bz + 2.0 ** -18
    for lo in (0, v - 64):  # rows of dw that have targets, and others
        rows = slice(lo, lo + 64)
        limit = off * size[:, rows].t() @ xd.abs() * (1 + 2.0 ** -8) + 1e-30
        assert ((dw[rows].double() - dz[:, rows].t() @ xd).abs() <= limit).all()
    assert torch.isfinite(dw[::4099]).all() and (dw[::4099] != 7).all()
    gx, sx = torch.zeros_like(xd), torch.zeros_like(xd)
    for lo in range(0, v, 1 << 18):
        part = w[lo:lo + (1 << 18)].double()
        gx += dz[:, lo:lo + (1 << 18)] @ part
        sx += size[:, lo:lo + (1 << 18)] @ part.abs()
    sums = 2.0 ** -23 * 2048  # an order of sums of 2^21 terms by parts and steps
    assert ((dx.double() - gx).abs() <= (off + sums) * sx + 2.0 ** -8 * gx.abs() + 1e-30).all()


def test_rows_of_x_and_dx_far_apart():
    torch = _torch()
    t, d, v, stride = 2100, 64, 90, 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(3)
    near = torch.randn((t, d), generator=gen, device="cuda").half()
    w = torch.randn((v, d), generator=gen, device="cuda").half()
    y = torch.randint(0, v, (t,), generator=gen, device="cuda")
    far = torch.empty(t * stride, device="cuda", dtype=torch.float16)  # 4.4 GB
    x, dx = far.as_strided((t, d), (stride, 1)), far.as_strided((t, d), (stride, 1), 128)
    assert (t - 1) * stride * 2 > 1 << 32
    x.copy_(near)
    dx_at = dx.data_ptr()
    want = head.cross_entropy_grad(near, w, y)
    # two views of one array interleave: their spans overlap, which a call refuses
    with pytest.raises(Exception, match="overlap"):
        head.cross_entropy_grad(x, w, y, dx=dx)
    assert dx_at == dx.data_ptr()
    got = head.cross_entropy_grad(x, w, y)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    far.fill_(7.0)
    got = head.cross_entropy_grad(near, w, y, dx=dx)
    assert got[1] is dx and torch.equal(dx, want[1]) and torch.equal(got[2], want[2])
    assert (far.view(t, stride)[:, :128] == 7).all() and (far.view(t, stride)[:, 192:256] == 7).all()


def test_lookup_and_gradient_of_over_4_gib():
    torch = _torch()
    v, d = 1 << 21, 1100
    table = torch.empty((v, d), device="cuda", dtype=torch.float16)
    table[-100:].normal_()
    table[:100].normal_()
    assert table.numel() * 2 > 1 << 32
    for n in (60, 900):
        tokens = torch.randint(v - 100, v, (n,), device="cuda")
        tokens[::3] -= v - 100
        assert torch.equal(embed.lookup(table, tokens), table[tokens])
        dy = torch.randint(-4, 5, (n, d), device="cuda").half()
        dw = embed.lookup_grad(dy, tokens, v)
        want = torch.zeros((200, d), device="cuda")
        want.index_add_(0, torch.where(tokens < 100, tokens, tokens - v + 200), dy.float())
        assert torch.equal(dw[:100], want[:100]) and torch.equal(dw[-100:], want[100:])
        assert not dw[100:-100:997].any()
        del dw


@pytest.mark.parametrize("n", [3, 700])
def test_the_largest_table(n):
    torch = _torch()
    v = 1 << 28
    tokens = torch.randint(0, v, (n,), device="cuda")
    tokens[0], tokens[1], tokens[2] = v - 1, 0, v  # the last is none
    dy = torch.ones((n, 1), device="cuda")
    dw = embed.lookup_grad(dy, tokens, v)
    assert dw[v - 1] >= 1 and dw[0] >= 1 and dw.sum(dtype=torch.float64) == n - 1
    assert torch.equal(embed.lookup(dw, tokens)[:2], dw[tokens[:2]])


@pytest.mark.parametrize("d", [1, 5])
@pytest.mark.parametrize("v", [7, (1 << 27) + 1, 1 << 28])
def test_no_tokens_and_the_largest_table(v, d):
    """An empty batch's gradient is zeros, in tables whose few tokens are sorted too."""
    torch = _torch()
    none = torch.empty(0, dtype=torch.long, device="cuda")
    dw = torch.full((v, d + 1), 7.0, device="cuda")
    embed.lookup_grad(torch.empty((0, d), device="cuda"), none, v, dw=dw[:, :d])
    assert not dw[:, :d].any() and (dw[:, d] == 7).all()
    dw.fill_(1.0)
    embed.lookup_grad(torch.empty((0, d), device="cuda"), none, v, dw=dw[:, :d], accumulate=True)
    assert (dw == 1).all()
