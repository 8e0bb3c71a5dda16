"""The router against a 64-bit evaluation: scores, ties, masked experts, tokens
without any, biases, infinities and NaN, the order of the slots, gradients."""

import math

import numpy as np
import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, differences, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def choose(z, bias, top):
    """-> (experts [tokens, top] with -1 for absent ones) of CPU logits, keys in fp32 as they are defined."""
    key = z.float() if bias is None else z.float() + bias
    best = torch.sort(key, dim=1, descending=True, stable=True)
    return torch.where(best.values[:, :top] == -math.inf, -1, best.indices[:, :top])


def weights64(z, experts, score, normalize, scale):
    """The weights as a function of fp64 logits, for autograd too."""
    there = experts >= 0
    zc = z.gather(1, experts.clamp(min=0))
    if score == "softmax":
        over = zc.masked_fill(~there, -math.inf) if normalize else z
        m = over.amax(1, keepdim=True).detach()
        m = torch.where(m == -math.inf, 0.0, m)
        e = torch.where(there, torch.exp(torch.where(there, zc, 0.0) - m), 0.0)
        total = (e if normalize else torch.where(z == -math.inf, 0.0, torch.exp(torch.where(z == -math.inf, 0.0, z) - m))).sum(1, keepdim=True)
    else:
        e = torch.where(there, torch.sigmoid(torch.where(there, zc, 0.0)), 0.0)
        total = e.sum(1, keepdim=True) if normalize else torch.ones_like(zc[:, :1])
    total = torch.where(there.any(1, keepdim=True), total, 1.0)
    return scale * e / total


def check_order(routing, experts, n):
    flat = torch.where(experts < 0, n, experts).flatten().numpy()
    order = np.argsort(flat, kind="stable")
    places = np.empty_like(order)
    places[order] = np.arange(flat.size)
    offsets = np.searchsorted(flat[order], np.arange(n + 1))
    assert torch.equal(routing.experts.cpu(), experts.int())
    assert np.array_equal(routing.order.cpu().numpy(), order)
    assert np.array_equal(routing.places.cpu().numpy().ravel(), places) and routing.places.shape == experts.shape
    assert np.array_equal(routing.offsets.cpu().numpy(), offsets)
    assert all(t.dtype == torch.int32 for t in routing)


def check(z, top, score="softmax", normalize=True, scale=1.0, bias=None):
    n = z.shape[1]
    leaf = z.detach().requires_grad_(True)
    weights, routing = cresso_amd.route_experts(leaf, top, score=score, normalize=normalize, scale=scale, bias=bias)
    assert weights.dtype == torch.float32 and not any(t.requires_grad for t in routing)
    z64 = z.detach().cpu().double().requires_grad_(True)
    experts = choose(z.detach().cpu(), None if bias is None else bias.cpu(), top)
    check_order(routing, experts, n)
    want = weights64(z64, experts, score, normalize, scale)
    # an exponent's difference is off by 2^-24 of its size, which is that much of the exponential; exponentials and
    # quotients by 2 units each, sums by an addition for each of a lane's experts and 6 for the wave
    fine = torch.where(torch.isfinite(z64), z64, 0.0).detach()
    size = 1 + (fine.amax(1, keepdim=True) - fine.amin(1, keepdim=True)).clamp(max=200.0) + fine.abs().amax(1, keepdim=True).clamp(max=200.0)
    chain = 16 + n // 64
    close(weights, want.detach(), want.detach().abs() * size, chain, "weights")
    d = rand(tuple(weights.shape), torch.float32, 9)
    weights.backward(d)
    d64 = d.double().cpu()
    grad = torch.autograd.grad(want, z64, d64)[0]
    assert leaf.grad.dtype == z.dtype and leaf.grad.shape == z.shape
    p = (want / scale).detach()
    room = torch.zeros_like(grad).scatter_add_(1, experts.clamp(min=0), want.detach().abs() * (d64.abs() + (p.abs() * d64.abs()).sum(1, keepdim=True)))
    if score == "softmax" and not normalize:
        every = torch.softmax(torch.where(torch.isfinite(z64).any(1, keepdim=True), z64, 0.0), 1).detach()
        room += abs(scale) * every * (p.abs() * d64.abs()).sum(1, keepdim=True)
    close(leaf.grad, grad, room * size, 2 * chain + 8, "gradient")
    # without a gradient the same answer
    again, same = cresso_amd.route_experts(z.detach(), top, score=score, normalize=normalize, scale=scale, bias=bias)
    assert torch.equal(again, weights.detach()) and all(torch.equal(a, b) for a, b in zip(same, routing))
    return weights, routing


FORMS = [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)]


@pytest.mark.parametrize("score,normalize", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,n,top", [(1, 1, 1), (1, 2, 2), (3, 5, 2), (8, 64, 8), (16, 63, 32), (64, 8, 2), (65, 8, 2), (64, 64, 8),
                                          (17, 65, 31), (100, 128, 6), (333, 129, 4), (1000, 256, 8), (50, 300, 5), (40, 513, 7), (33, 1024, 32),
                                          (2777, 37, 3)])
def test_sizes(tokens, n, top, dtype, score, normalize):
    announce(f"route {tokens} x {n} top {top} {dtype} {score} {normalize}")
    check(rand((tokens, n), dtype, 3, 2.0), top, score, normalize, 1.5)


@pytest.mark.parametrize("score,normalize", FORMS)
def test_biases_and_hidden_experts(score, normalize):
    announce(f"route bias {score} {normalize}")
    for tokens, n, top in ((9, 12, 5), (500, 40, 6), (300, 200, 8)):
        z, bias = rand((tokens, n), torch.float32, 5), rand((n,), torch.float32, 6)
        z[torch.rand((tokens, n), generator=torch.Generator().manual_seed(1)) < 0.6] = -math.inf
        z[::3] = -math.inf                    # nothing left
        z[1::5, : n - 2] = -math.inf          # fewer than top
        check(z, top, score, normalize, 0.7, bias)
        bias[3], bias[5] = -math.inf, 40.0    # an expert out of use, one that everybody takes
        check(z, top, score, normalize, 0.7, bias)
        check(z.bfloat16(), top, score, normalize, -2.0)


def test_ties():
    announce("route ties")
    for n in (7, 64, 200):
        z = torch.zeros(70, n).cuda()
        _, r = check(z, min(n, 5))
        assert torch.equal(r.experts.cpu(), torch.arange(min(n, 5)).expand(70, -1).int())
        z = torch.randint(-2, 3, (300, n), generator=torch.Generator().manual_seed(2)).float().cuda()
        z[z == 0] *= torch.where(torch.rand(int((z == 0).sum()), generator=torch.Generator().manual_seed(3)) < 0.5, -1.0, 1.0).cuda()   # zeros of both signs
        check(z, min(n, 6))


def test_large_and_small_logits():
    announce("route extremes")
    z = rand((40, 30), torch.float32, 7, 30.0)
    for score, normalize in FORMS:
        check(z, 4, score, normalize)
        check(z - 150.0, 4, score, normalize)    # sigmoids below fp32's range
        check(z + 100.0, 4, score, normalize)
    low = torch.full((5, 9), torch.finfo(torch.float32).min).cuda()   # masked by the lowest number: equal, and there
    low[0, 4] = 1.0
    w, r = cresso_amd.route_experts(low, 3)
    assert torch.equal(r.experts.cpu()[0], torch.tensor([4, 0, 1]).int()) and w[0].tolist() == [1.0, 0.0, 0.0]
    assert torch.equal(r.experts.cpu()[1], torch.tensor([0, 1, 2]).int()) and torch.allclose(w[1], torch.full((3,), 1 / 3).cuda())


@pytest.mark.parametrize("score,normalize", FORMS)
def test_nan_stays_in_its_row(score, normalize):
    announce(f"route nan {score} {normalize}")
    z = rand((70, 20), torch.float32, 8)
    z[3, 7], z[5, 2], z[5, 9] = math.nan, math.nan, math.nan
    w, r = cresso_amd.route_experts(z, 3, score=score, normalize=normalize)
    check_order(r, choose(z.cpu(), None, 3), 20)
    assert r.experts[3, 0] == 7 and r.experts[5, :2].tolist() == [2, 9]
    assert torch.isnan(w[3, 0]) and torch.isnan(w[5, :2]).all()
    keep = torch.ones(70, dtype=torch.bool)
    keep[[3, 5]] = False
    assert torch.isfinite(w[keep.cuda()]).all()


def test_no_tokens():
    announce("route no tokens")
    w, r = cresso_amd.route_experts(torch.empty(0, 6).cuda(), 2)
    assert w.shape == (0, 2) and r.order.shape == (0,) and r.places.shape == (0, 2) and r.offsets.tolist() == [0] * 7
    leaf = torch.empty(0, 6).cuda().requires_grad_(True)
    cresso_amd.route_experts(leaf, 2)[0].sum().backward()
    assert leaf.grad.shape == (0, 6)


def test_strides():
    announce("route strides")
    wide = rand((200, 50), torch.float32, 4)
    check(wide[:, 3:40], 4)
    check(wide.t(), 4)
    check(wide[::2, :33], 3, "sigmoid")


def test_many_tokens():
    announce("route 50000 tokens")
    check(rand((50001, 16), torch.bfloat16, 4), 2)
    check(rand((20000, 100), torch.float32, 4), 8, "softmax", False)


def test_gradient_against_differences():
    announce("route differences")
    z = rand((6, 9), torch.float32, 11)
    d, along = rand((6, 3), torch.float32, 12), rand((6, 9), torch.float32, 13)
    for score, normalize in FORMS:
        leaf = z.clone().requires_grad_(True)
        w, r = cresso_amd.route_experts(leaf, 3, score=score, normalize=normalize, scale=1.3)
        got = float((torch.autograd.grad(w, leaf, d)[0].double() * along.double()).sum())
        experts = r.experts.cpu().long()
        f = lambda x: float((weights64(torch.from_numpy(x), experts, score, normalize, 1.3) * d.double().cpu()).sum())   # noqa: E731
        want = differences(f, z.double().cpu().numpy(), along.double().cpu().numpy(), 1e-5)
        assert abs(got - want) <= 1e-5 * (1 + abs(want))


def test_arriving_gradient_layouts():
    announce("route gradient layouts")
    z = rand((90, 12), torch.float32, 1).requires_grad_(True)
    d = rand((3, 90), torch.float32, 2)
    w, _ = cresso_amd.route_experts(z, 3)
    a = torch.autograd.grad(w, z, d.t(), retain_graph=True)[0]
    b = torch.autograd.grad(w, z, d.t().contiguous())[0]
    assert torch.equal(a, b)
    w, _ = cresso_amd.route_experts(z, 3)
    assert torch.autograd.grad(w.sum(), z)[0].shape == z.shape   # an expanded gradient


def test_refusals():
    announce("route refusals")
    z = rand((4, 6), torch.float32, 1)
    for bad, text in (((z, 0), "top 0"), ((z, 7), "top 7"), ((z.view(-1), 1), "tokens, experts"), ((z.int(), 1), "fp32, bf16 or fp16"),
                      ((z.double(), 1), "fp32, bf16 or fp16"), ((torch.zeros(2, 1025).cuda(), 1), "1025 experts"),
                      ((torch.zeros(2, 100).cuda(), 33), "top 33"), ((torch.zeros(2, 0).cuda(), 1), "0 experts")):
        with pytest.raises(ValueError, match=text):
            cresso_amd.route_experts(*bad)
    for bias in (torch.zeros(5).cuda(), torch.zeros(6).cuda().half(), torch.zeros(1, 6).cuda()):
        with pytest.raises(ValueError, match="bias must be"):
            cresso_amd.route_experts(z, 2, bias=bias)
    with pytest.raises(ValueError, match="score must be"):
        cresso_amd.route_experts(z, 2, score="relu")
    with pytest.raises(ValueError, match="scale"):
        cresso_amd.route_experts(z, 2, scale=math.inf)
    with pytest.raises(RuntimeError, match="GPU only"):
        cresso_amd.route_experts(z, 2, bias=torch.zeros(6))
