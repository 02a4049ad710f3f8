"""The input side of an attention layer, trained: queries and keys projected
from x, normed by head and rotated, with what the backward pass needs kept in 8
bits, and the weight gradients formed from that into an optimizer's fp32
gradients.

    python examples/attention_input.py [--steps N] [--tokens T] [--no-norm] ...

Kept from the forward pass are x in 8 bits, once for both projections, and the
projected heads in 8 bits (without the norm, nothing of them).  The task is a
teacher's rotated queries and keys, with targets of the same form; a step sums
the gradients of two micro-batches.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ark_amd import _abi, act  # noqa: E402
from ark_amd.eko import TensorSpec  # noqa: E402
from ark_amd.optimizer import AdamConfig, AmpConfig, Optimizer, ParamSet  # noqa: E402
from ark_amd.rope import Rope  # noqa: E402


class AttentionInput:
    """Weights (hidden x heads * head_dim, fp16) and gains in a ParamSet."""

    def __init__(self, hidden, heads, kv_heads, head, norm=True):
        self.hidden, self.heads, self.kv_heads, self.head, self.norm = (hidden, heads, kv_heads,
                                                                       head, norm)
        specs = [TensorSpec("wq", (hidden, heads * head), True, False),
                 TensorSpec("wk", (hidden, kv_heads * head), True, False)]
        if norm:
            specs += [TensorSpec("gain_" + part, (head,), False, True) for part in "qk"]
        self.params = ParamSet(specs, 0.0, grad_dtype=_abi.GRAD_F32)
        self.rope = Rope(head)
        for i in range(2):
            self.params.w(i).normal_(0.0, hidden ** -0.5)
        for i in range(2, len(specs)):
            self.params.w(i).fill_(1.0)

    def weight(self, i):
        return self.params.w(i).view(self.hidden, -1)

    def forward(self, x):
        """q and k (tokens, heads, head_dim) of x (tokens, hidden), and what
        backward takes."""
        q = (x @ self.weight(0)).view(-1, self.heads, self.head)
        k = (x @ self.weight(1)).view(-1, self.kv_heads, self.head)
        kept = act.pack(x)
        if not self.norm:
            return *self.rope.apply(q, k, out=(q, k)), (kept,)
        q, k, q8, k8 = self.rope.norm(q, k, self.params.w(2), self.params.w(3), out=(q, k),
                                      keep8=True)
        return q, k, (kept, q8, k8)

    def backward(self, dq, dk, kept, accumulate):
        """From the gradients of q and k (overwritten): the parameters' into the
        ParamSet, the gradient of x returned."""
        p = self.params
        if self.norm:
            self.rope.norm_backward(dq, dk, kept[1], kept[2], p.w(2), p.w(3), out=(dq, dk),
                                    dgain_q=p.g(2), dgain_k=p.g(3), accumulate=accumulate)
        else:
            self.rope.apply(dq, dk, inverse=True, out=(dq, dk))
        dq, dk = dq.flatten(1), dk.flatten(1)
        for i, d in enumerate((dq, dk)):
            act.weight_grad(kept[0], d, p.g(i).view(self.hidden, -1), accumulate=accumulate)
        return dq @ self.weight(0).t() + dk @ self.weight(1).t()


def train(hidden=768, heads=12, kv_heads=12, head=64, tokens=2048, steps=60, norm=True, lr=2e-3,
          seed=0, report=None):
    """The loss of every step."""
    torch.manual_seed(seed)
    teacher = AttentionInput(hidden, heads, kv_heads, head, norm)
    student = AttentionInput(hidden, heads, kv_heads, head, norm)
    opt = Optimizer(AdamConfig(lr=lr, grad_clip=1.0), student.params,
                    AmpConfig(loss_scale_init=256.0))
    batches = [torch.randn((tokens, hidden), device="cuda").half() for _ in range(2)]
    targets = [teacher.forward(x)[:2] for x in batches]
    losses = []
    for step in range(steps):
        scale = opt.loss_scale
        loss = 0.0
        for n, (x, (tq, tk)) in enumerate(zip(batches, targets)):
            q, k, kept = student.forward(x)
            eq, ek = q.float() - tq.float(), k.float() - tk.float()
            loss = loss + (eq.square().sum() + ek.square().sum()) / (2 * tokens)
            student.backward((eq * (scale / tokens)).half(), (ek * (scale / tokens)).half(), kept,
                             accumulate=n > 0)
        opt.step_all(lr=lr)
        losses.append(float(loss) / len(batches))
        if report:
            report(step, losses[-1])
    return losses


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("hidden", 768), ("heads", 12), ("kv-heads", 12), ("head", 64),
                        ("tokens", 2048), ("steps", 60)):
        p.add_argument(f"--{name}", type=int, default=value)
    p.add_argument("--no-norm", action="store_true", help="rotation alone")
    a = p.parse_args(argv)
    train(a.hidden, a.heads, a.kv_heads, a.head, a.tokens, a.steps, not a.no_norm,
          report=lambda step, loss: print(f"step {step:3d}  loss {loss:.4f}", flush=True))


if __name__ == "__main__":
    main()
