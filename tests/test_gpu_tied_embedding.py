"""The example that trains a tied embedding with the lookup, the losses and their
gradients (examples/tied_embedding.py): it runs, repeats its bits, and its
gradients are those of the same model in 64 bits.

The 64-bit gradients are taken at the fp16 values that the kernels read (the rows
h, their gradient dh, the gradient of the embedded rows): the embedding's is the
loss's, checked by its own tests' tolerance of two roundings of dz (2.2 2^-11 of
the magnitudes, and what fp32 sums lose), plus a sum of rows in fp32."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                     "tied_embedding.py")


@pytest.fixture(scope="module")
def example():
    import torch
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    spec = importlib.util.spec_from_file_location("tied_embedding", _PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("distill", [False, True])
def test_runs_and_repeats(example, distill):
    run = lambda: example.train(vocab=300, columns=64, tokens=200, steps=6, distill=distill)
    losses = run()
    assert len(losses) == 6 and all(0 < x < 20 for x in losses)
    assert losses == run()


@pytest.mark.parametrize("tokens,vocab,columns", [(1, 9, 16), (150, 333, 48)])
def test_gradients(example, tokens, vocab, columns):
    import torch
    from ark_amd import head
    torch.manual_seed(1)
    model = example.Bigram(vocab, columns)
    now = torch.randint(0, vocab, (tokens,), device="cuda")
    nxt = torch.randint(0, vocab, (tokens,), device="cuda")
    seen = []

    def loss_grad(h, table, dw, accumulate):
        out = head.cross_entropy_grad(h, table, nxt, grad=4.0, dw=dw, accumulate=accumulate)
        seen.extend((h.clone(), out[1].clone(), dw.clone()))
        return out
    model.params.g(0).fill_(7.0)  # overwritten, not added to
    loss = model.step(now, loss_grad, False)
    h, dh, from_loss = (t.double() for t in seen)
    w = model.table.double()
    z = h @ w.t()
    q = torch.softmax(z, 1)
    assert ((loss.double() - torch.nn.functional.cross_entropy(z, nxt, reduction="none")).abs()
            <= 2.0 ** -18 * (1 + z.abs().max())).all()
    p = torch.zeros_like(q).scatter_(1, nxt[:, None], 1.0)
    dz = 4.0 * (q - p)
    off = 4.0 * (q + p) * (2.3 * 2.0 ** -11) + 2.0 ** -22
    dw = dz.t() @ h
    limit = off.t() @ h.abs() + (tokens + 4) * 2.0 ** -22 * (dz.abs() + off).t() @ h.abs() + 1e-6
    assert ((from_loss - dw).abs() <= limit).all()
    limit = off @ w.abs()
    assert ((dh - dz @ w).abs() <= limit + 2.0 ** -10 * (dz @ w).abs() + 1e-5).all()
    # the lookup's gradient, added
    rows = (seen[1] @ model.layer.t()).double() * model.scale
    both = from_loss.clone().index_add_(0, now, rows)
    size = from_loss.abs().index_add_(0, now, rows.abs())
    got = model.params.g(0).view(vocab, columns).double()
    assert ((got - both).abs() <= (tokens + 4) * 2.0 ** -23 * size + 1e-12).all()


@pytest.mark.parametrize("distill", [False, True])
def test_two_micro_batches_add_up(example, distill):
    """The head's gradient of a second micro-batch is added to what the first left of
    both ends, and so is the layer's."""
    import torch
    from ark_amd import head
    torch.manual_seed(2)
    vocab, columns, tokens = 200, 64, 90
    model = example.Bigram(vocab, columns)
    want = torch.zeros((vocab, columns), dtype=torch.float64, device="cuda")
    limit, size = torch.zeros_like(want), torch.zeros_like(want)
    layer = torch.zeros((columns, columns), dtype=torch.float64, device="cuda")
    layer_size, loose = torch.zeros_like(layer), 0.0
    model.params.g(0).fill_(7.0)  # overwritten, not added to
    model.params.g(1).fill_(7.0)
    w = model.table.double()
    for half in range(2):
        now = torch.randint(0, vocab, (tokens,), device="cuda")
        nxt = torch.randint(0, vocab, (tokens, 3), device="cuda")
        seen = []

        def loss_grad(h, table, dw, accumulate):
            if distill:
                out = head.distill_grad(h, table, nxt, torch.zeros_like(nxt).half(), grad=4.0, dw=dw,
                                        accumulate=accumulate)
            else:
                out = head.cross_entropy_grad(h, table, nxt[:, 0].contiguous(), grad=4.0, dw=dw,
                                              accumulate=accumulate)
            seen.extend((h.double(), out[1].clone()))
            return out
        model.step(now, loss_grad, half > 0)
        h, dh = seen
        q = torch.softmax(h @ w.t(), 1)
        at = nxt if distill else nxt[:, :1]
        p = torch.zeros_like(q).scatter_add_(1, at, torch.full(at.shape, 1.0 / at.shape[1],
                                                               dtype=q.dtype, device="cuda"))
        dz = 4.0 * (q - p)
        off = 4.0 * (q + p) * (2.3 * 2.0 ** -11) + 2.0 ** -22
        want += dz.t() @ h
        limit += off.t() @ h.abs()
        size += (dz.abs() + off).t() @ h.abs()
        rows = (dh @ model.layer.t()).double() * model.scale
        want.index_add_(0, now, rows)
        size.index_add_(0, now, rows.abs())
        x = model.table[now].double() * model.scale
        layer += x.t() @ dh.double()
        layer_size += x.abs().t() @ dh.double().abs()
        # x in 8 bits: half a step of a group's largest, 1/127 of it, for every value
        loose += x.abs().max() / 126 * tokens * dh.double().abs().max()
    got = model.params.g(0).view(vocab, columns).double()
    assert ((got - want).abs() <= limit + (2 * tokens + 8) * 2.0 ** -22 * size + 1e-6).all()
    dlayer = model.params.g(1).view(columns, columns).double()
    assert ((dlayer - layer).abs() <= loose + 2.0 ** -10 * layer_size).all()


def test_every_step_moves_the_weights_against_their_gradients(example, monkeypatch):
    """Adam's first step is lr against the gradient's sign, whatever its size."""
    import torch
    seen = []

    class Seen(example.Optimizer):
        def __init__(self, cfg, params, amp):
            super().__init__(cfg, params, amp)
            self.seen_params = params

        def step_all(self, *args, **kw):
            p = self.seen_params
            w, g = ([f(i).clone().view(-1).float() for i in (0, 1)] for f in (p.w, p.g))
            out = super().step_all(*args, **kw)
            torch.cuda.synchronize()
            seen.append((w, g, [p.w(i).clone().view(-1).float() for i in (0, 1)]))
            return out
    monkeypatch.setattr(example, "Optimizer", Seen)
    example.train(vocab=300, columns=64, tokens=200, steps=3, lr=0.0625)
    assert len(seen) == 3
    w, g, after = seen[0]
    for i in (0, 1):
        far = g[i].abs() > 1e-3 * g[i].abs().max()
        moved = after[i] - w[i]
        assert far.sum() > 1000 and (torch.sign(moved) == -torch.sign(g[i]))[far].all()
        # sqrt(v) + eps over the sign: lr to what fp16 keeps of a weight, and eps takes
        assert ((moved.abs() - 0.0625).abs()[far] <= 0.0625 * 0.01 + 2.0 ** -10 * w[i][far].abs()
                + 2.0 ** -10).all()
    assert all((a != b).any() for w, _, after in seen for a, b in zip(w, after))
