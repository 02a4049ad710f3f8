"""Token lookup and its gradient (include/ark_embed.h), against their formulas in
64 bits.

A row is one product and one rounding: within 2^-24 and half a step of the output's
type.  A gradient is a sum of n rows in fp32, by groups of 16: within
(min(n, 64) + n / 16 + 2) 2^-24 of the sum of their magnitudes, 2^-24 of it for the
scale and, accumulated, another of the result; whole numbers are exact."""
import pytest

from ark_amd import embed
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


def _tokens(n, v, kind, seed=0):
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(seed + n * 7 + v)
    if kind == "same":
        return torch.full((n,), v // 2, device="cuda")
    if kind == "text":
        u = torch.rand((n,), generator=gen, device="cuda")
        return torch.exp(u * torch.log(torch.tensor(float(v)))).long().clamp(0, v - 1)
    return torch.randint(-2, v + 2, (n,), generator=gen, device="cuda")  # some outside


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (5, 3, 8), (7, 1000, 768), (300, 40, 33),
                                   (1000, 128, 520)])
def test_lookup(n, v, d, name):
    torch = _torch()
    table = torch.randn((v, d), device="cuda").to(_dt(name))
    tokens = _tokens(n, v, "any")
    ok = (tokens >= 0) & (tokens < v)
    rows = torch.where(ok[:, None], table[tokens.clamp(0, v - 1)], 0)
    assert torch.equal(embed.lookup(table, tokens), rows)
    assert torch.equal(embed.lookup(table, tokens.int()), rows)
    for out in TYPES:
        u = torch.finfo(_dt(out)).eps / 2
        got = embed.lookup(table, tokens, scale=27.7, dtype=_dt(out))
        assert got.dtype == _dt(out)
        scale = torch.tensor(27.7, dtype=torch.float32).double().item()
        want = rows.double() * scale
        limit = want.abs() * (u + 2.0 ** -24) * 1.01 + (2.0 ** -25 if out == "f16" else 1e-38)
        assert ((got.double() - want).abs() <= limit).all()


def test_lookup_of_slices_and_shapes():
    torch = _torch()
    wide = torch.randn((50, 70), device="cuda").half()
    for lo, d in ((0, 64), (3, 40), (8, 16)):
        table = wide[:, lo:lo + d]
        tokens = torch.randint(0, 50, (4, 5), device="cuda")
        assert torch.equal(embed.lookup(table, tokens), table[tokens])
        beside = torch.full((20, 90), 7.0, device="cuda").half()
        out = embed.lookup(table, tokens.flatten(), out=beside[:, 5:5 + d])
        assert torch.equal(out, table[tokens.flatten()])
        assert (beside[:, :5] == 7).all() and (beside[:, 5 + d:] == 7).all()
    assert embed.lookup(wide, torch.empty((0, 3), dtype=torch.int, device="cuda")).shape == (0, 3, 70)


def _check(dw, dy, tokens, v, scale=1.0, before=None):
    torch = _torch()
    ok = (tokens >= 0) & (tokens < v)
    at, rows = tokens[ok].long(), dy[ok].double()
    want = torch.zeros((v, dy.shape[1]), dtype=torch.float64, device="cuda")
    size, n = torch.zeros_like(want), torch.zeros(v, dtype=torch.float64, device="cuda")
    want.index_add_(0, at, rows)
    size.index_add_(0, at, rows.abs())
    n.index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    s = torch.tensor(scale, dtype=torch.float32).double().item()
    limit = ((n.clamp_max(64) + n / 16 + 3) * 2.0 ** -24)[:, None] * size * abs(s)
    want = want * s
    if before is not None:
        want = want + before.double()
        limit = limit + 2.0 ** -24 * (want.abs() + limit)
    assert ((dw.double() - want).abs() <= limit + 1e-37).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kind", ["any", "text", "same"])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (63, 5, 8), (64, 128, 24), (65, 129, 513),
                                   (1000, 256, 520), (5000, 300, 33), (4096, 1000, 768)])
def test_gradient(n, v, d, kind, name):
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    tokens = _tokens(n, v, kind)
    dy = torch.randn((n, d), generator=gen, device="cuda").to(_dt(name))
    _check(embed.lookup_grad(dy, tokens, v), dy, tokens, v)
    before = torch.randn((v, d), generator=gen, device="cuda")
    dw = before.clone()
    assert embed.lookup_grad(dy, tokens.int(), v, scale=3.3, dw=dw, accumulate=True) is dw
    _check(dw, dy, tokens, v, 3.3, before)
    absent = torch.ones(v, dtype=torch.bool, device="cuda")
    absent[tokens[(tokens >= 0) & (tokens < v)].long()] = False
    assert torch.equal(dw[absent], before[absent])
    whole = torch.randint(-4, 5, (n, d), generator=gen, device="cuda").to(_dt(name))
    ok = (tokens >= 0) & (tokens < v)
    want = torch.zeros((v, d), device="cuda").double().index_add_(0, tokens[ok].long(),
                                                                  whole[ok].double())
    assert torch.equal(embed.lookup_grad(whole, tokens, v).double(), want)


@pytest.mark.parametrize("kind", ["any", "text", "same"])
@pytest.mark.parametrize("n,v,d", [(511, 1000, 1100), (512, 17, 3), (512, 33, 2053), (513, 17, 3),
                                   (513, 33, 1029), (16384, 129, 8), (16385, 129, 8)])
def test_gradient_on_both_sides_of_its_kernels_sizes(n, v, d, kind):
    test_gradient(n, v, d, kind, "bf16")


@pytest.mark.parametrize("n", [30, 600])
def test_few_and_many_tokens_of_slices(n):
    torch = _torch()
    tokens = _tokens(n, 90, "text")
    base = torch.randn((n, 61), device="cuda").half()
    for off, d in ((3, 40), (1, 3), (60, 1)):
        dy = base[:, off:off + d]
        big = torch.full((90, 61), 7.0, device="cuda")
        embed.lookup_grad(dy, tokens, 90, dw=big[:, off:off + d])
        _check(big[:, off:off + d], dy, tokens, 90)
        embed.lookup_grad(dy, tokens, 90, dw=big[:, off:off + d], accumulate=True)
        assert (big[:, :off] == 7).all() and (big[:, off + d:] == 7).all()
    clean = embed.lookup_grad(base, tokens, 90)
    base[tokens == -1] = float("nan")
    tokens[:n // 2] = 90
    base[:n // 2] = float("nan")
    got = embed.lookup_grad(base, tokens, 90)
    assert torch.isfinite(got).all() and got.shape == clean.shape
    _check(got, base, tokens, 90)


def test_rows_without_a_token_are_not_read():
    torch = _torch()
    tokens = _tokens(500, 64, "text")
    dy = torch.randn((500, 40), device="cuda").half()
    tokens[100:300] = -1
    clean = embed.lookup_grad(dy, tokens, 64)
    dy[100:300] = float("nan")
    assert torch.equal(embed.lookup_grad(dy, tokens, 64), clean)
    tokens[:] = 64
    assert not embed.lookup_grad(dy, tokens, 64).any()
    assert embed.lookup(torch.full((64, 8), float("nan"), device="cuda"), tokens).abs().max() == 0


def test_strides_and_what_lies_beside():
    torch = _torch()
    tokens = _tokens(400, 90, "text")
    for off, d, wide in ((0, 64, 96), (3, 40, 61), (4, 8, 20)):
        base = torch.randn((400, wide), device="cuda").half()
        dy = base[:, off:off + d]
        big = torch.full((90, wide), 7.0, device="cuda")
        embed.lookup_grad(dy, tokens, 90, dw=big[:, off:off + d])
        assert torch.equal(big[:, off:off + d], embed.lookup_grad(dy.contiguous(), tokens, 90))
        assert (big[:, :off] == 7).all() and (big[:, off + d:] == 7).all()
    one = embed.lookup_grad(torch.randn((4, 5, 16), device="cuda"), tokens[:20].view(4, 5), 90)
    assert one.shape == (90, 16)
    row = torch.randn((1, 16), device="cuda").expand(400, 16)  # one row for all
    _check(embed.lookup_grad(row, tokens, 90), row, tokens, 90)


def test_no_tokens():
    torch = _torch()
    none = torch.empty(0, dtype=torch.long, device="cuda")
    dy = torch.empty((0, 12), device="cuda")
    assert not embed.lookup_grad(dy, none, 7).any()
    dw = torch.ones((7, 12), device="cuda")
    embed.lookup_grad(dy, none, 7, dw=dw, accumulate=True)
    assert (dw == 1).all()


def test_equal_bits_on_streams_and_in_a_graph():
    torch = _torch()
    tokens = _tokens(3000, 500, "text")
    dy = torch.randn((3000, 136), device="cuda").bfloat16()
    table = torch.randn((500, 136), device="cuda").bfloat16()
    run = lambda: (embed.lookup(table, tokens, 2.0), embed.lookup_grad(dy, tokens, 500, 2.0))
    first = run()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(first, g))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=streams[0]):
        out = run()
    for k in range(4):
        dy.normal_()
        tokens.random_(-3, 500)
        torch.cuda.synchronize()
        for o in out:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run())), k


def test_gradient_by_differences():
    """<lookup(table), dy> is linear in the table: a change of one value by 1 changes
    it by the gradient (whole numbers, exact)."""
    torch = _torch()
    table = torch.randint(-5, 6, (9, 6), device="cuda").float()
    tokens = _tokens(50, 9, "any")
    dy = torch.randint(-5, 6, (50, 6), device="cuda").float()
    dw = embed.lookup_grad(dy, tokens, 9, scale=2.0)
    value = lambda t: (embed.lookup(t, tokens, 2.0).double() * dy.double()).sum()
    base = value(table)
    for v, c in ((0, 0), (8, 5), (4, 2)):
        t2 = table.clone()
        t2[v, c] += 1
        assert value(t2) - base == dw[v, c]


def test_refusals():
    torch = _torch()
    table = torch.randn((10, 8), device="cuda")
    tokens = torch.arange(4, device="cuda")
    bad = pytest.raises(ValueError)
    with bad:
        embed.lookup(table.double(), tokens)
    with bad:
        embed.lookup(table, tokens.float())
    with bad:
        embed.lookup(table, tokens.cpu())
    with bad:
        embed.lookup(table, tokens, out=torch.empty((3, 8), device="cuda"))
    with bad:
        embed.lookup(table, tokens, out=torch.empty((4, 7), device="cuda"))
    with bad:
        embed.lookup_grad(table[:3], tokens, 10)
    with bad:
        embed.lookup_grad(table[:4], tokens, 10, accumulate=True)
    with bad:
        embed.lookup_grad(table[:4], tokens, 10, dw=torch.empty((10, 7), device="cuda"))
    with pytest.raises(ArkOptError, match="overlap"):
        embed.lookup(table, tokens, out=table[:4])
    with pytest.raises(ArkOptError, match="vocab"):
        embed.lookup_grad(table[:4], tokens, 0)
    table.requires_grad_()
    with pytest.raises(ValueError, match="requires grad"):
        embed.lookup(table, tokens)
    with torch.no_grad():
        embed.lookup(table, tokens)


@pytest.mark.parametrize("n,v", [(40, 300), (700, 300), (16384, 1000), (20000, 1000)])
def test_tokens_of_32_and_64_bits_give_equal_bits(n, v):
    torch = _torch()
    tokens = _tokens(n, v, "any")
    tokens[::9] = -2 ** 31  # a 32-bit token's sign is its own
    dy = torch.randn((n, 40), device="cuda").half()
    table = torch.randn((v, 40), device="cuda")
    assert torch.equal(embed.lookup_grad(dy, tokens.int(), v), embed.lookup_grad(dy, tokens, v))
    assert torch.equal(embed.lookup(table, tokens.int()), embed.lookup(table, tokens))
    tokens[::9] = 2 ** 32 + 1  # and a 64-bit one's upper half counts
    _check(embed.lookup_grad(dy, tokens, v), dy, tokens, v)


@pytest.mark.parametrize("n", [7, 700])
def test_the_most_columns(n):
    torch = _torch()
    v, d = 50, 65536
    tokens = _tokens(n, v, "any")
    dy = torch.randn((n, d), device="cuda").half()
    _check(embed.lookup_grad(dy, tokens, v), dy, tokens, v)
    table = torch.randn((v, d), device="cuda").bfloat16()
    ok = (tokens >= 0) & (tokens < v)
    assert torch.equal(embed.lookup(table, tokens),
                       torch.where(ok[:, None], table[tokens.clamp(0, v - 1)], 0))


@pytest.mark.parametrize("n", [8, 300, 700])
def test_few_and_many_tokens_in_a_graph(n):
    torch = _torch()
    v, d = 900, 72
    tokens = _tokens(n, v, "text")
    dy = torch.randn((n, d), device="cuda").half()
    before = torch.randn((v, d), device="cuda")
    dw = before.clone()
    run = lambda o: (embed.lookup_grad(dy, tokens, v, dw=o, accumulate=True),
                     embed.lookup_grad(dy, tokens, v, 3.0))
    first = run(dw.clone())
    assert all(torch.isfinite(o).all() for o in first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(dw)
    for k in range(4):
        dy.normal_()
        tokens.random_(-3, (v, 5, 900, 1)[k])
        dw.copy_(before)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run(before.clone()))), k
