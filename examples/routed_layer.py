"""A one-layer next-token model with routed experts, trained and then decoded.

    python examples/routed_layer.py [--steps 60] [--dtype bf16|f16|f32]

tokens -> flagsparse_embedding -> a router's best experts per token ->
prepare_expert_route -> flagsparse_expert_dispatch -> flagsparse_expert_product,
activation, flagsparse_expert_product -> flagsparse_expert_combine with the
router's weights -> logits against the same table.  Gradients come from the
operators' own backward passes.  The data is synthetic: each token is followed
by a fixed other one, with some noise.
"""

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import flagsparse_amd as fs  # noqa: E402

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class RoutedLayer:
    """Parameters of the model and its forward pass."""

    def __init__(self, vocab=1024, width=256, hidden=512, experts=8, slots=2, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def randn(*shape, scale):
            return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype).requires_grad_()

        self.experts, self.slots, self.scale = experts, slots, math.sqrt(width)
        self.table = randn(vocab, width, scale=width**-0.5)
        self.router = randn(width, experts, scale=width**-0.5)
        self.into = randn(experts, hidden, width, scale=width**-0.5)  # (outputs, inputs) an expert
        self.back = randn(experts, width, hidden, scale=hidden**-0.5)

    def parameters(self):
        return [self.table, self.router, self.into, self.back]

    def route(self, x):
        """The slots' experts and weights, and the route of one batch of tokens."""
        scores = torch.softmax((x @ self.router).float(), dim=1)
        weights, experts = torch.topk(scores, self.slots, dim=1)
        weights = weights / weights.sum(dim=1, keepdim=True)
        return weights, fs.prepare_expert_route(experts, self.experts)

    def __call__(self, tokens):
        """Logits, (tokens, vocab), in float32."""
        x = fs.flagsparse_embedding(self.table, tokens, scale=self.scale)
        weights, route = self.route(x)
        rows = fs.flagsparse_expert_dispatch(x, route)
        rows = torch.nn.functional.silu(fs.flagsparse_expert_product(rows, self.into, route, op="trans"))
        rows = fs.flagsparse_expert_product(rows, self.back, route, op="trans")
        x = x + fs.flagsparse_expert_combine(rows, route, weights)
        return (x @ self.table.t()).float()


def batch(successor, n, seed):
    """n tokens and their successors, one in ten replaced at random."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    vocab = successor.numel()
    tokens = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    noise = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    keep = torch.rand(n, device="cuda", generator=g) < 0.9
    return tokens, torch.where(keep, successor[tokens], noise)


def train(model, successor, steps, tokens_a_step=2048, rate=3e-3, report=None):
    """Adam on float32 copies of the parameters; the loss of each step."""
    masters = [p.detach().float().clone() for p in model.parameters()]
    optimizer = torch.optim.Adam([m.requires_grad_() for m in masters], lr=rate)
    losses = []
    for step in range(steps):
        tokens, targets = batch(successor, tokens_a_step, step)
        loss = torch.nn.functional.cross_entropy(model(tokens), targets)
        grads = torch.autograd.grad(loss, model.parameters())
        for m, grad in zip(masters, grads):
            m.grad = grad.float()
        optimizer.step()
        with torch.no_grad():
            for p, m in zip(model.parameters(), masters):
                p.copy_(m)
        losses.append(loss.detach())
        if report and step % report == 0:
            print(f"step {step}: loss {float(losses[-1]):.3f}", flush=True)
    return [float(v) for v in losses]


@torch.no_grad()
def decode(model, first, count):
    """Greedy next tokens, one at a time."""
    token, out = first.reshape(1), []
    for _ in range(count):
        token = model(token).argmax(dim=1)
        out.append(token)
    return torch.cat(out)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    args = ap.parse_args()
    model = RoutedLayer(dtype=DTYPES[args.dtype])
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    successor = torch.randperm(model.table.shape[0], device="cuda", generator=g)
    losses = train(model, successor, args.steps, report=10)
    print(f"last loss {losses[-1]:.3f}")
    first = torch.tensor(3, device="cuda")
    got, want, token = decode(model, first, 12).tolist(), [], 3
    for _ in range(12):
        token = int(successor[token])
        want.append(token)
    print("decoded ", got)
    print("expected", want)


if __name__ == "__main__":
    main()
