"""Grouped products in forms that small cases do not reach: no expert at all."""

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 6, 100])
@pytest.mark.parametrize("inner,outer", [(4096, 5), (5, 4096), (4096, 4096), (1001, 3001)])
def test_no_expert(rows, inner, outer, dtype):
    """No row has an expert: zeros, however long a sum would be."""
    announce(f"expert_product without experts, {rows} rows {inner} -> {outer} {dtype}")
    x = rand((rows, inner), dtype, 1).requires_grad_(True)
    w = torch.zeros((0, outer, inner), dtype=dtype, device="cuda", requires_grad=True)
    for first in (0, 3):
        y = cresso_amd.expert_product(x, w, torch.tensor([first], dtype=torch.int32).cuda())
        assert y.shape == (rows, outer) and not y.detach().any()
        dx, dw = torch.autograd.grad(y, (x, w), rand((rows, outer), dtype, 2))
        assert dx.shape == x.shape and dw.shape == w.shape and not dx.any()
