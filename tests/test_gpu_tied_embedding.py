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
