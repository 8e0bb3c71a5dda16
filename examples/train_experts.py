"""A small model with layers of experts, trained with CRESSO5 under a clipped norm.

    python examples/train_experts.py [--steps 60]

    tokens -> embedding -> [norm -> router -> rows to the experts -> up -> silu -> down -> back -> seam] x layers -> head
    backward -> CRESSO5.clip_gradients -> CRESSO5.step()

Each token goes to two of eight experts; a bias that takes no gradient is moved
against the load, so that no expert runs idle.  Some tokens are padding: their
logits are masked, they go to no expert and have no label.  The task is a fixed
table of the next word of each word.
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import cresso_amd

VOCAB, WIDTH, HIDDEN, EXPERTS, TOP, LAYERS = 500, 128, 192, 8, 2, 2
PAD = -1


class Model:
    def __init__(self, seed: int = 0):
        gen = torch.Generator().manual_seed(seed)
        make = lambda *shape, std: torch.nn.Parameter((std * torch.randn(*shape, generator=gen)).cuda().bfloat16())   # noqa: E731
        self.table = make(VOCAB, WIDTH, std=0.02)
        self.gate = [make(EXPERTS, WIDTH, std=WIDTH ** -0.5) for _ in range(LAYERS)]
        self.up = [make(EXPERTS, HIDDEN, WIDTH, std=WIDTH ** -0.5) for _ in range(LAYERS)]
        self.down = [make(EXPERTS, WIDTH, HIDDEN, std=HIDDEN ** -0.5) for _ in range(LAYERS)]
        self.pre = [torch.nn.Parameter(torch.ones(WIDTH, device="cuda")) for _ in range(LAYERS + 1)]
        self.head = make(VOCAB, WIDTH, std=WIDTH ** -0.5)
        self.bias = [torch.zeros(EXPERTS, device="cuda") for _ in range(LAYERS)]

    def parameters(self):
        return [self.table, *self.gate, *self.up, *self.down, *self.pre, self.head]

    def __call__(self, tokens: torch.Tensor) -> torch.Tensor:
        hidden = torch.where(tokens == PAD, -math.inf, 0.0).unsqueeze(1)
        h = cresso_amd.embedding(tokens, self.table, scale=math.sqrt(WIDTH))
        h, x = cresso_amd.residual_norm(h, pre_weight=self.pre[0])
        for i in range(LAYERS):
            weights, routing = cresso_amd.route_experts((x @ self.gate[i].t()).float() + hidden, TOP, bias=self.bias[i])
            rows = cresso_amd.dispatch_rows(x, routing)
            rows = torch.nn.functional.silu(cresso_amd.expert_product(rows, self.up[i], routing.offsets))
            rows = cresso_amd.expert_product(rows, self.down[i], routing.offsets)
            y = cresso_amd.combine_rows(rows, routing, weights)
            h, x = cresso_amd.residual_norm(h, y, pre_weight=self.pre[i + 1])
            load = routing.offsets.diff().float()
            self.bias[i] += 1e-2 * torch.sign(load.mean() - load)
        return x @ self.head.t()


def train(steps: int = 60, size: int = 512, lr: float = 4e-3, max_norm: float = 1.0, seed: int = 0):
    """-> (the loss, the gradients' norm before clipping) of each step."""
    model = Model(seed)
    follows = torch.randperm(VOCAB, generator=torch.Generator().manual_seed(seed + 1)).cuda()
    none = torch.full((size, 1), -1, dtype=torch.int32, device="cuda")   # no teacher: the labels alone
    opt = cresso_amd.CRESSO5(model.parameters(), lr=lr, rank=4, hash_bins=64, cuda_ops="required")
    losses, norms = [], []
    for step in range(steps):
        gen = torch.Generator(device="cuda").manual_seed(1000 + step)
        tokens = torch.randint(0, VOCAB, (size,), generator=gen, device="cuda")
        tokens[torch.rand(size, generator=gen, device="cuda") < 0.1] = PAD
        labels = torch.where(tokens == PAD, -100, follows[tokens.clamp(min=0)])
        logits = model(tokens)
        loss = cresso_amd.distill_loss(logits, none, none.float(), labels=labels, mix=0.0)
        opt.zero_grad()
        loss.backward()
        norms.append(opt.clip_gradients(max_norm))
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist(), torch.stack(norms).tolist()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--lr", type=float, default=4e-3)
    ap.add_argument("--max-norm", type=float, default=1.0)
    args = ap.parse_args()
    for step, (loss, norm) in enumerate(zip(*train(args.steps, lr=args.lr, max_norm=args.max_norm))):
        if step % 10 == 0 or step == args.steps - 1:
            print(f"step {step:4d}  loss {loss:.4f}  norm {norm:.3f}", flush=True)


if __name__ == "__main__":
    main()
