"""The router and the rows' kernels on as many tokens as one call takes."""

import pytest
import torch

from gpu_util import announce, needs_gpu

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

MOST = (1 << 26) - 16


def test_most_tokens():
    announce("router and rows, most tokens")
    logits = torch.zeros((MOST, 1), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    weights, r = cresso_amd.route_experts(logits, 1)
    every = torch.arange(MOST, dtype=torch.int32, device="cuda")
    assert (weights.detach() == 1.0).all() and not r.experts.any() and r.offsets.tolist() == [0, MOST]
    assert torch.equal(r.order, every) and torch.equal(r.places.view(-1), every)
    (d,) = torch.autograd.grad(weights, logits, torch.ones_like(weights))
    assert d.shape == logits.shape and not d.any()
    x = (every.view(-1, 1) % 251).half().requires_grad_(True)
    rows = cresso_amd.dispatch_rows(x, r)
    assert torch.equal(rows, x)
    y = cresso_amd.combine_rows(rows, r, weights.detach().requires_grad_(True))
    assert torch.equal(y, x)
    assert torch.equal(torch.autograd.grad(y, x, x.detach())[0], x)


def test_more_tokens_are_refused():
    announce("router and rows, too many tokens")
    logits = torch.zeros((1, 1), dtype=torch.bfloat16, device="cuda").expand(MOST + 1, 1)
    places = torch.zeros((1, 1), dtype=torch.int32, device="cuda").expand(MOST + 1, 1)
    r = cresso_amd.Routing(places, places, places, places)
    for call in (lambda: cresso_amd.route_experts(logits, 1), lambda: cresso_amd.dispatch_rows(logits, r),
                 lambda: cresso_amd.combine_rows(logits, r)):
        with pytest.raises(ValueError, match="more than one call takes"):
            call()
