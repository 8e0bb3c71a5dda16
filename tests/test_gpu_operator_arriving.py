"""The gradient that arrives at an operator's backward pass: views that stand for
the negative of their memory (autograd makes them where complex numbers are
conjugated) count as what they are, dual tensors are refused."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from gpu_util import announce, needs_gpu
from operator_util import rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]


def calls():
    """name -> (the operator of one fp32 leaf, that leaf)"""
    ids, index, teacher = torch.tensor([1, 2, 2]).cuda(), torch.tensor([[1], [2], [0]]).cuda(), rand((3, 1), seed=2)
    values, scales = cresso_amd.quantize_blocks(rand((20, 12)))
    logits = rand((9, 5), seed=3)
    weights, routing = cresso_amd.route_experts(logits, 2)
    matrices = rand((5, 7, 12), seed=5)
    rows = rand((18, 12), seed=6)
    return {
        "embedding": (lambda t: cresso_amd.embedding(ids, t), rand((5, 12))),
        "seam": (lambda t: cresso_amd.residual_norm(t, rand((3, 12), seed=7))[0], rand((3, 12))),
        "seam norm": (lambda t: cresso_amd.residual_norm(t, pre_weight=rand((12,), seed=8))[1], rand((3, 12))),
        "block product": (lambda t: cresso_amd.block_product(t, values, scales), rand((3, 12))),
        "distill": (lambda t: cresso_amd.distill_loss(t, index, teacher), rand((3, 12))),
        "distill rows": (lambda t: cresso_amd.distill_loss(t, index, teacher, reduction="none"), rand((3, 12))),
        "route": (lambda t: cresso_amd.route_experts(t, 2, normalize=False)[0], logits),
        "dispatch": (lambda t: cresso_amd.dispatch_rows(t, routing), rand((9, 12))),
        "combine": (lambda t: cresso_amd.combine_rows(t, routing, weights), rows),
        "combine weights": (lambda t: cresso_amd.combine_rows(rows, routing, t), weights),
        "product": (lambda t: cresso_amd.expert_product(t, matrices, routing.offsets), rows),
        "product weight": (lambda t: cresso_amd.expert_product(rows, t, routing.offsets), matrices),
    }


NAMES = ["embedding", "seam", "seam norm", "block product", "distill", "distill rows", "route", "dispatch", "combine", "combine weights",
         "product", "product weight"]


@pytest.mark.parametrize("name", NAMES)
def test_negative_views_arrive(name):
    announce(f"negative view arrives: {name}")
    call, x = calls()[name]
    x = x.detach().requires_grad_(True)
    y = call(x)
    d = rand(tuple(y.shape), seed=11)
    (want,) = torch.autograd.grad(y, x, d)
    (got,) = torch.autograd.grad(call(x), x, torch._neg_view(-d))
    assert want.any() and not got.is_neg() and torch.equal(got, want)
    # as autograd makes one: the gradient of the imaginary part of what is conjugated afterwards
    y = call(x)
    (got,) = torch.autograd.grad(torch.complex(torch.zeros_like(y), y).conj(), x, torch.complex(torch.zeros_like(d), -d))
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", NAMES)
def test_dual_tensors_that_arrive_are_refused(name):
    """An answer without a tangent would say that the gradient does not change with what arrives."""
    announce(f"dual tensor arrives: {name}")
    call, x = calls()[name]
    x = x.detach().requires_grad_(True)
    y = call(x)
    d = rand(tuple(y.shape), seed=11)
    (want,) = torch.autograd.grad(y, x, d, retain_graph=True)
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, fwad.make_dual(d, torch.ones_like(d)), retain_graph=True)
        assert torch.equal(torch.autograd.grad(y, x, d)[0], want)
