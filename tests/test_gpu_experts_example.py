"""The example of layers of experts runs, repeats bit by bit, and its gradients
are those of the same model in 64 bits."""

import importlib.util
import math
from pathlib import Path

import pytest
import torch

from gpu_util import announce, needs_gpu

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "train_experts.py"
    spec = importlib.util.spec_from_file_location("train_experts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_runs_and_repeats(example):
    announce("example train_experts")
    losses, norms = example.train(steps=6)
    assert all(math.isfinite(v) for v in losses + norms)
    assert example.train(steps=6) == (losses, norms)


def test_gradients(example):
    """Of the first layer's experts: the model in 64 bits from the same parameters, with the experts that the model chose."""
    announce("gradients of the example")
    chosen = []
    route = example.cresso_amd.route_experts

    def watched(*args, **kw):
        weights, routing = route(*args, **kw)
        chosen.append(routing.experts.cpu().long())
        return weights, routing

    model = example.Model()
    tokens = torch.randint(0, example.VOCAB, (200,), generator=torch.Generator().manual_seed(5))
    tokens[::9] = example.PAD
    labels = torch.where(tokens == example.PAD, -100, (tokens * 7) % example.VOCAB)
    example.cresso_amd.route_experts = watched
    try:
        logits = model(tokens.cuda())
    finally:
        example.cresso_amd.route_experts = route
    none = torch.full((200, 1), -1, dtype=torch.int32, device="cuda")
    example.cresso_amd.distill_loss(logits, none, none.float(), labels=labels.cuda(), mix=0.0).backward()

    table, head = (p.detach().double().cpu() for p in (model.table, model.head))
    gate = [p.detach().double().cpu() for p in model.gate]
    up, down = ([p.detach().double().cpu().requires_grad_(True) for p in ps] for ps in (model.up, model.down))
    rms = lambda v: v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)   # noqa: E731
    there = (tokens != example.PAD).unsqueeze(1)
    h = torch.where(there, table[tokens.clamp(min=0)] * math.sqrt(example.WIDTH), 0.0)
    x = rms(h)
    for i in range(example.LAYERS):
        e = chosen[i]
        z = (x @ gate[i].t()).gather(1, e.clamp(min=0))
        w = torch.where(e >= 0, torch.softmax(z, 1), 0.0)
        y = torch.zeros_like(x)
        for k in range(example.TOP):
            for j in range(example.EXPERTS):
                t = (e[:, k] == j).nonzero().squeeze(1)
                y = y.index_add(0, t, w[t, k, None] * (torch.nn.functional.silu(x[t] @ up[i][j].t()) @ down[i][j].t()))
        h = h + y
        x = rms(h)
    loss = -torch.log_softmax(x @ head.t(), 1)[there.squeeze(1), labels[there.squeeze(1)]].sum() / 200
    want = torch.autograd.grad(loss, [*up, *down])
    # bf16 rounds at a dozen places in each layer, forward and back: 2^-8 each, some 2 x 12 x 2 of them, as independent errors
    room = math.sqrt(2 * 12 * 2) * 2.0 ** -8
    for p, g in zip([*model.up, *model.down], want):
        got = p.grad.double().cpu()
        assert float((got - g).norm()) <= room * float(g.norm())
