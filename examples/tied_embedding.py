"""A model of the next token whose embedding is also its output layer, trained
from data or from a teacher's best logits: lookup, one layer, loss, and both
gradients of the embedding in the fp32 gradients that the optimizer steps on.

    python examples/tied_embedding.py [--steps N] [--tokens T] [--distill] ...

The text is a Markov chain; the layer is a product with its input kept in 8 bits
for the weight gradient.  No logits are in memory at any time.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ark_amd import _abi, act, embed, head  # noqa: E402
from ark_amd.eko import TensorSpec  # noqa: E402
from ark_amd.optimizer import AdamConfig, AmpConfig, Optimizer, ParamSet  # noqa: E402


class Bigram:
    """An embedding (vocab x columns) and a layer (columns x columns), fp16."""

    def __init__(self, vocab, columns):
        self.vocab, self.columns = vocab, columns
        self.params = ParamSet([TensorSpec("embed", (vocab, columns), True, False),
                                TensorSpec("layer", (columns, columns), True, False)], 0.0,
                               grad_dtype=_abi.GRAD_F32)
        self.params.w(0).normal_(0.0, columns ** -0.5)
        self.params.w(1).normal_(0.0, columns ** -0.5)
        self.scale = columns ** 0.5  # rows of the embedding come in at size 1

    @property
    def table(self):
        return self.params.w(0).view(self.vocab, self.columns)

    @property
    def layer(self):
        return self.params.w(1).view(self.columns, self.columns)

    def forward(self, tokens):
        """The rows that the loss takes, and what backward does."""
        x = embed.lookup(self.table, tokens, scale=self.scale)
        return x @ self.layer, act.pack(x)

    def step(self, tokens, loss_grad, accumulate):
        """The tokens' losses, every gradient in the ParamSet.  loss_grad(h, table,
        dw): the loss and gradients of rows h against the table."""
        p = self.params
        shape = (self.vocab, self.columns)
        h, kept = self.forward(tokens)
        loss, dh, _ = loss_grad(h, self.table, p.g(0).view(shape), accumulate)
        act.weight_grad(kept, dh, p.g(1).view(self.columns, self.columns), accumulate=accumulate)
        embed.lookup_grad(dh @ self.layer.t(), tokens, self.vocab, scale=self.scale,
                          dw=p.g(0).view(shape), accumulate=True)
        return loss


def _text(vocab, n, gen):
    """n tokens, each one of four that its predecessor allows."""
    follow = torch.randint(0, vocab, (vocab, 4), generator=gen)
    pick = torch.randint(0, 4, (n,), generator=gen)
    out = [0]
    for k in pick.tolist():
        out.append(int(follow[out[-1], k]))
    return torch.tensor(out[1:]), follow


def train(vocab=1000, columns=128, tokens=512, steps=100, distill=False, top=8, lr=5e-3, seed=0,
          report=None):
    """The mean loss of every step."""
    torch.manual_seed(seed)
    gen = torch.Generator().manual_seed(seed)
    text, follow = _text(vocab, 8 * tokens + 1, gen)
    text, follow = text.cuda(), follow.cuda()
    model = Bigram(vocab, columns)
    opt = Optimizer(AdamConfig(lr=lr, grad_clip=1.0), model.params,
                    AmpConfig(loss_scale_init=1024.0))
    losses = []
    for n in range(steps):
        grad = opt.loss_scale / (2 * tokens)
        total = 0.0
        for half in range(2):  # two micro-batches a step
            at = (2 * n + half) % 8 * tokens
            now, nxt = text[at:at + tokens], text[at + 1:at + tokens + 1].contiguous()

            def loss_grad(h, table, dw, accumulate):
                if distill:  # a teacher that knows the four, in a list padded with -1
                    index = torch.full((tokens, top), -1, device="cuda")
                    index[:, :4] = follow[now]
                    return head.distill_grad(h, table, index, torch.zeros_like(index).half(),
                                             grad=grad, dw=dw, accumulate=accumulate)
                return head.cross_entropy_grad(h, table, nxt, grad=grad, dw=dw,
                                               accumulate=accumulate)
            total = total + model.step(now, loss_grad, half > 0).mean()
        opt.step_all(lr=lr)
        losses.append(float(total) / 2)
        if report:
            report(n, losses[-1])
    return losses


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("vocab", 1000), ("columns", 128), ("tokens", 512), ("steps", 100),
                        ("top", 8)):
        p.add_argument(f"--{name}", type=int, default=value)
    p.add_argument("--distill", action="store_true", help="from a teacher's logits")
    a = p.parse_args(argv)
    train(a.vocab, a.columns, a.tokens, a.steps, a.distill, a.top,
          report=lambda n, loss: print(f"step {n:3d}  loss {loss:.4f}", flush=True))


if __name__ == "__main__":
    main()
