"""The operators in captured graphs, replayed with new inputs, and on tensors of
more than 2^31 elements."""

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]


def norm_step(h, y, g, w):
    leaves = [t.detach().requires_grad_(True) for t in (h, y, w)]
    out, normed = cresso_amd.residual_norm(leaves[0], leaves[1], gate=leaves[2], post_weight=leaves[2], pre_weight=leaves[2])
    return [out, normed, *torch.autograd.grad((out, normed), leaves, (g, g))]


def make(kind):
    if kind == "norm":
        return [rand((300, 513), torch.bfloat16, k) for k in range(3)] + [rand((513,), torch.bfloat16, 5, 0.1, 1.0)], norm_step
    if kind == "embedding":
        ids = torch.randint(-1, 900, (3000,)).cuda()
        return [rand((900, 72), torch.float32, 1), rand((3000, 72), torch.float32, 2)], \
            lambda w, g: [cresso_amd.embedding(ids, w, scale=2.0), cresso_amd.embedding_grad(ids, g, 900, 2.0)]
    if kind == "distill":
        index, labels = torch.randint(-1, 5000, (40, 9)).cuda(), torch.randint(0, 5000, (40,)).cuda()
        return [rand((40, 5000), torch.bfloat16, 1), rand((40, 9), torch.float32, 2)], \
            lambda z, a: list(cresso_amd.distill_loss_and_grad(z, index, a, labels=labels, temperature=2.0, mix=0.5))
    rows = int(kind[7:])
    values, scales = cresso_amd.quantize_blocks(rand((700, 390)))

    def product_step(x, d):
        leaf = x.detach().requires_grad_(True)
        y = cresso_amd.block_product(leaf, values, scales)
        return [y, torch.autograd.grad(y, leaf, d)[0]]
    return [rand((rows, 390), torch.bfloat16, 1), rand((rows, 700), torch.bfloat16, 2)], product_step


@pytest.mark.parametrize("kind", ["norm", "embedding", "distill", "product5", "product300"])
def test_graphs(kind):
    announce(f"graph of {kind}")
    inputs, step = make(kind)
    step(*inputs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*inputs)   # the autograd threads' and streams' first use is not captured
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*inputs)
    for k in range(3):
        for j, t in enumerate(inputs):
            t.copy_(rand(tuple(t.shape), t.dtype, 20 + 5 * k + j))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step(*inputs)):
            assert torch.equal(a, b)


def test_tables_and_rows_past_32_bits():
    announce("more than 2^31 elements")
    rows, width = 70000, 32768
    table = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    marks = torch.tensor([0, 1, 40000, 65535, 65537, 69999]).cuda()
    table[marks] = rand((6, width), torch.bfloat16, 1)
    assert torch.equal(cresso_amd.embedding(marks, table), table[marks])
    grad = rand((6, width), torch.bfloat16, 2)
    g = cresso_amd.embedding_grad(marks, grad, rows)
    assert torch.equal(g[marks], grad)
    g[marks] = 0
    assert not g.any()
    del table, g
    h = torch.zeros(150000, 16384, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 131071, 131073, 149999]).cuda()
    h[at] = rand((4, 16384), torch.bfloat16, 3)
    w = torch.ones(16384, device="cuda")
    out, normed = cresso_amd.residual_norm(h, h, post_weight=w, pre_weight=w)
    want = cresso_amd.residual_norm(h[at], h[at], post_weight=w, pre_weight=w)
    assert torch.equal(out[at], want[0]) and torch.equal(normed[at], want[1])
    assert not out[1:131071].any()


def test_logits_and_outputs_past_32_bits():
    z = torch.zeros(20000, 131072, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 16383, 16385, 19999]).cuda()
    z[at] = rand((4, 131072), torch.bfloat16, 4)
    index, a = torch.randint(0, 131072, (20000, 4)).cuda(), rand((20000, 4), seed=5)
    weights = torch.ones(20000, device="cuda")
    _, g = cresso_amd.distill_loss_and_grad(z, index, a, row_weights=weights)
    rows = cresso_amd.distill_loss(z, index, a, row_weights=weights, reduction="none")
    want = cresso_amd.distill_loss(z[at], index[at], a[at], row_weights=weights[:4], reduction="none")
    torch.testing.assert_close(rows[at], want, rtol=1e-5, atol=0)   # other workgroups' sizes: another order of sums
    _, want = cresso_amd.distill_loss_and_grad(z[at], index[at], a[at], row_weights=weights[:4])
    torch.testing.assert_close(g[at].float(), want.float(), rtol=2.0 ** -7, atol=0)
    del z, g
    values, scales = cresso_amd.quantize_blocks(rand((65536, 128), torch.bfloat16, 6))
    x = torch.zeros(40000, 128, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 32767, 32769, 39999]).cuda()
    x[at] = torch.randint(-4, 5, (4, 128)).cuda().to(torch.bfloat16)
    y = cresso_amd.block_product(x, values, scales)
    w = values.float().double() * scales.double().repeat_interleave(128, 0)
    want = x[at].double() @ w.t()
    close(y[at], want, x[at].double().abs() @ w.abs().t(), 160)
    assert not y[1:32767].any()
