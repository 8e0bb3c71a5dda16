"""A weight block whose scale is 0 counts as zeros whatever its values are, by
every number of rows; and rows that round to zero give exact zeros."""

import math

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import rand
from test_gpu_block_product import check, make_weight

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("zero", [0.0, -0.0])
@pytest.mark.parametrize("rows", [1, 4, 16, 17, 200, 700])
def test_nan_under_a_scale_of_zero(rows, zero):
    announce(f"block_product NaN under scale 0, {rows} rows")
    values, scales = make_weight(640, 512)
    scales[1, 2] = zero
    plain = values.clone()
    plain.view(torch.uint8)[128:256, 256:384] = 0      # what the block counts as
    for held in (0x7F, 0xFF, 0x7E):                    # NaN of both signs, the largest number
        values.view(torch.uint8)[128:256, 256:384] = held
        x = rand((rows, 512), torch.bfloat16, 3)
        d = rand((rows, 640), torch.bfloat16, 4)
        out = []
        for w in (plain, values):
            leaf = x.detach().requires_grad_(True)
            y = cresso_amd.block_product(leaf, w, scales)
            out.append((y, torch.autograd.grad(y, leaf, d)[0]))
        for a, b in zip(*out):
            assert torch.isfinite(b).all() and torch.equal(a, b)
    check(rand((rows, 512), torch.float32, 5), plain, scales)


@pytest.mark.parametrize("rows", [4, 200])
def test_what_is_not_finite_in_x_meets_a_scale_of_zero(rows):
    values, scales = make_weight(160, 300)
    scales[:, 1] = 0.0
    x = rand((rows, 300), torch.float32, 8)
    x[1, 130], x[2, 255] = math.inf, math.nan
    y = cresso_amd.block_product(x, values, scales)
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[3:]).all()


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_what_rounds_to_nothing_gives_exact_zeros(rows):
    """1e-44 over the smallest power of two, 2^-117, is far below half of e4m3's smallest step."""
    values = torch.eye(256).cuda().to(torch.float8_e4m3fn)
    x = torch.full((rows, 256), 1e-44).cuda()
    y = cresso_amd.block_product(x, values, torch.ones(2, 2).cuda())
    assert not y.any()
