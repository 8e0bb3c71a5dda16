"""Rows to the experts and back against a 64-bit evaluation, with gradients."""

import math

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make_routing(tokens, n, top, absent=0.0, seed=1):
    gen = torch.Generator().manual_seed(seed)
    experts = torch.rand((tokens, n), generator=gen).argsort(1)[:, :top]
    experts[torch.rand((tokens, top), generator=gen) < absent] = -1
    flat = torch.where(experts < 0, n, experts).flatten()
    order = torch.sort(flat, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(tokens * top)
    offsets = torch.searchsorted(flat[order], torch.arange(n + 1))
    return cresso_amd.Routing(*(t.int().cuda() for t in (experts, order, places.view(tokens, top), offsets)))


def check(tokens, width, top, dtype, absent=0.0, weighted=True, n=None):
    announce(f"rows {tokens} x {width} top {top} {dtype} absent {absent}")
    r = make_routing(tokens, n or top + 3, top, absent)
    there, places = (r.experts >= 0).cpu(), r.places.cpu().long()
    x = rand((tokens, width), dtype, 1).requires_grad_(True)
    rows = cresso_amd.dispatch_rows(x, r)
    assert rows.shape == (tokens * top, width) and rows.dtype == dtype
    want = torch.zeros(tokens * top, width).double()
    want[places[there]] = x.detach().double().cpu()[there.nonzero()[:, 0]]
    assert torch.equal(rows.detach().double().cpu(), want)
    d = rand((tokens * top, width), dtype, 2)
    with torch.no_grad():
        d[r.places[~r.experts.ge(0)].long()] = math.nan   # gradients of rows that are nobody's
    got = torch.autograd.grad(rows, x, d)[0]
    d64 = torch.where(there.unsqueeze(2), d.double().cpu()[places], 0.0)
    close(got, d64.sum(1), d64.abs().sum(1), top, "gradient of dispatch")

    y = rand((tokens * top, width), dtype, 3)
    with torch.no_grad():
        y[r.places[~r.experts.ge(0)].long()] = math.nan
    y.requires_grad_(True)
    weights = rand((tokens, top), torch.float32, 4).requires_grad_(True) if weighted else None
    out = cresso_amd.combine_rows(y, r, weights)
    w64 = (weights.detach().double().cpu() if weighted else torch.ones(tokens, top).double()) * there
    y64 = torch.where(there.unsqueeze(2), y.detach().double().cpu()[places], 0.0)
    terms = w64.unsqueeze(2) * y64
    close(out, terms.sum(1), terms.abs().sum(1), top, "combine")
    d = rand((tokens, width), dtype, 5)
    grads = torch.autograd.grad(out, [y, weights] if weighted else [y], d)
    d64 = d.double().cpu()
    want = torch.zeros(tokens * top, width).double()
    want[places.flatten()] = (w64.unsqueeze(2) * d64.unsqueeze(1)).view(tokens * top, width)
    close(grads[0], want, want.abs(), 1, "gradient of the rows")
    if weighted:
        dots = d64.unsqueeze(1) * y64
        close(grads[1], dots.sum(2), dots.abs().sum(2), width // 8 + 16, "gradient of the weights")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,width,top", [(1, 1, 1), (1, 8, 2), (2, 7, 3), (8, 2048, 8), (33, 64, 2), (5, 65, 32), (333, 1001, 3),
                                              (100, 512, 6), (64, 4096, 2), (3, 20000, 2), (1000, 33, 4)])
def test_sizes(tokens, width, top, dtype):
    check(tokens, width, top, dtype)
    check(tokens, width, top, dtype, absent=0.4)


def test_without_weights():
    check(50, 130, 3, torch.bfloat16, 0.2, weighted=False)


def test_many_rows():
    check(20000, 24, 4, torch.bfloat16, 0.1)


def test_all_absent():
    check(10, 40, 2, torch.float32, absent=1.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    announce(f"rows strides {dtype}")
    r = make_routing(40, 6, 2, 0.2)
    wide = rand((40, 100), dtype, 1)
    assert torch.equal(cresso_amd.dispatch_rows(wide[:, 5:70], r), cresso_amd.dispatch_rows(wide[:, 5:70].contiguous(), r))
    assert torch.equal(cresso_amd.dispatch_rows(wide[:, ::2], r), cresso_amd.dispatch_rows(wide[:, ::2].contiguous(), r))
    one = rand((1, 65), dtype, 2).expand(40, 65)
    assert torch.equal(cresso_amd.dispatch_rows(one, r), cresso_amd.dispatch_rows(one.contiguous(), r))
    rows, w = rand((80, 100), dtype, 3), rand((2, 40), torch.float32, 4).t()
    assert torch.equal(cresso_amd.combine_rows(rows[:, 5:70], r, w), cresso_amd.combine_rows(rows[:, 5:70].contiguous(), r, w.contiguous()))
    leaf = rows[:, 5:70].detach().requires_grad_(True)
    weights = w.detach().requires_grad_(True)
    out = cresso_amd.combine_rows(leaf, r, weights)
    a = torch.autograd.grad(out, (leaf, weights), wide[:, 5:70], retain_graph=True)
    b = torch.autograd.grad(out, (leaf, weights), wide[:, 5:70].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    turned = cresso_amd.Routing(r.experts.t().contiguous().t(), r.order, r.places.t().contiguous().t(), r.offsets)
    assert torch.equal(cresso_amd.dispatch_rows(wide, turned), cresso_amd.dispatch_rows(wide, r))


def test_only_wanted_gradients():
    announce("rows wanted gradients")
    r = make_routing(30, 6, 2)
    rows, w, d = rand((60, 50), torch.float32, 1), rand((30, 2), torch.float32, 2), rand((30, 50), torch.float32, 3)
    both = [rows.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    want = torch.autograd.grad(cresso_amd.combine_rows(both[0], r, both[1]), both, d)
    assert torch.equal(torch.autograd.grad(cresso_amd.combine_rows(both[0], r, w), both[0], d)[0], want[0])
    assert torch.equal(torch.autograd.grad(cresso_amd.combine_rows(rows, r, both[1]), both[1], d)[0], want[1])


def test_places_outside_are_not_touched():
    """Places are read from the GPU: a bad one is neither read nor written."""
    announce("rows bad places")
    r = make_routing(20, 5, 2)
    bad = r.places.clone()
    bad[3, 0], bad[4, 1], bad[5, 0] = 40, -1, 2 ** 31 - 1
    x = rand((20, 30), torch.float32, 1)
    good = torch.ones(20, 2, dtype=torch.bool)
    good[3, 0] = good[4, 1] = good[5, 0] = False
    rows = cresso_amd.dispatch_rows(x, r._replace(places=bad))
    keep = r.places.cpu()[good].long()
    assert torch.equal(rows.cpu()[keep], cresso_amd.dispatch_rows(x, r).cpu()[keep])
    y = rand((40, 30), torch.float32, 2)
    w = torch.ones(20, 2).cuda() * good.cuda()
    assert torch.equal(cresso_amd.combine_rows(y, r._replace(places=bad)), cresso_amd.combine_rows(y, r, w))


def test_nothing():
    announce("rows nothing")
    r = make_routing(0, 4, 2)
    assert cresso_amd.dispatch_rows(torch.empty(0, 5).cuda(), r).shape == (0, 5)
    assert cresso_amd.combine_rows(torch.empty(0, 5).cuda(), r).shape == (0, 5)
    r = make_routing(3, 4, 2)
    leaf, w = torch.empty(6, 0).cuda().requires_grad_(True), torch.ones(3, 2).cuda().requires_grad_(True)
    out = cresso_amd.combine_rows(leaf, r, w)
    out.sum().backward()
    assert out.shape == (3, 0) and leaf.grad.shape == (6, 0) and not w.grad.any()


def test_refusals():
    announce("rows refusals")
    r = make_routing(4, 5, 2)
    x, rows = rand((4, 6), torch.float32, 1), rand((8, 6), torch.float32, 2)
    for bad in (rand((5, 6)), rand((4,)), rand((4, 6, 1))):
        with pytest.raises(ValueError, match="x must be"):
            cresso_amd.dispatch_rows(bad, r)
        with pytest.raises(ValueError, match="rows must be"):
            cresso_amd.combine_rows(bad, r)
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        cresso_amd.dispatch_rows(x.double(), r)
    with pytest.raises(ValueError, match="experts and places"):
        cresso_amd.dispatch_rows(x, r._replace(experts=r.experts.long()))
    with pytest.raises(ValueError, match="experts and places"):
        cresso_amd.dispatch_rows(x, r._replace(places=r.places.flatten()))
    for bad in (torch.ones(4, 3), torch.ones(8), torch.ones(4, 2).double()):
        with pytest.raises(ValueError, match="weights must be"):
            cresso_amd.combine_rows(rows, r, bad.cuda())
    with pytest.raises(ValueError, match="route_experts returns"):
        cresso_amd.dispatch_rows(x, (r.experts, r.order))
    with pytest.raises(RuntimeError, match="GPU only"):
        cresso_amd.dispatch_rows(x, r._replace(places=r.places.cpu()))
