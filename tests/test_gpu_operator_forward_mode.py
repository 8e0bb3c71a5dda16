"""The operators have no forward-mode derivatives: a dual tensor is refused, not
answered without its tangent."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from gpu_util import needs_gpu
from operator_util import rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]


def calls():
    ids = torch.tensor([1, 2, 2]).cuda()
    values, scales = cresso_amd.quantize_blocks(rand((20, 12)))
    index, a = torch.tensor([[1], [2], [0]]).cuda(), rand((3, 1), seed=2)
    v = rand((12,), seed=4)
    return {   # name -> (the call of one tensor, that tensor)
        "embedding": (lambda t: cresso_amd.embedding(ids, t), rand((5, 12))),
        "embedding_grad": (lambda t: cresso_amd.embedding_grad(ids, t, 5), rand((3, 12))),
        "residual": (lambda t: cresso_amd.residual_norm(t)[0], rand((3, 12))),
        "update": (lambda t: cresso_amd.residual_norm(rand((3, 12)), t)[0], rand((3, 12))),
        "gate": (lambda t: cresso_amd.residual_norm(rand((3, 12)), rand((3, 12)), gate=t)[0], v),
        "post": (lambda t: cresso_amd.residual_norm(rand((3, 12)), rand((3, 12)), post_weight=t)[0], v),
        "pre": (lambda t: cresso_amd.residual_norm(rand((3, 12)), pre_weight=t)[1], v),
        "scale": (lambda t: cresso_amd.residual_norm(rand((3, 12)), residual_scale=t)[0], v),
        "product": (lambda t: cresso_amd.block_product(t, values, scales), rand((3, 12))),
        "product scales": (lambda t: cresso_amd.block_product(rand((3, 12)), values, t), scales),
        "quantize": (lambda t: cresso_amd.quantize_blocks(t)[1], rand((20, 12))),
        "distill": (lambda t: cresso_amd.distill_loss(t, index, a), rand((3, 12))),
        "teacher": (lambda t: cresso_amd.distill_loss(rand((3, 12)), index, t), a),
        "weights": (lambda t: cresso_amd.distill_loss(rand((3, 12)), index, a, row_weights=t), torch.ones(3).cuda()),
        "distill and grad": (lambda t: cresso_amd.distill_loss_and_grad(t, index, a)[0], rand((3, 12))),
    }


NAMES = ["embedding", "embedding_grad", "residual", "update", "gate", "post", "pre", "scale", "product", "product scales", "quantize",
         "distill", "teacher", "weights", "distill and grad"]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_dual_tensors_are_refused(name, grad):
    call, x = calls()[name]
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(fwad.make_dual(x.detach().requires_grad_(grad), torch.ones_like(x)))
        call(x)   # without a tangent, inside a level, as ever
    call(x)
