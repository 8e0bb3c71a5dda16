"""Grouped products in forms that small cases do not reach: no expert at all,
sums over k that are cut into parts for few rows by many experts, rows that lie
far apart or begin at odd addresses."""

import math

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import rand
from test_gpu_expert_product import check

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


def spread(rows, experts):
    """`rows` rows of as many experts, or fewer: no two of one expert's lie in neighbouring ones."""
    counts = [0] * experts
    for i in range(rows):
        counts[i * 7 % experts] += 1
    return counts


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,experts,inner,outer,turned", [
    (8, 64, 4096, 256, False),     # along k in parts, results in pieces of 8
    (8, 64, 256, 4096, False),     # the gradient of x, across k
    (8, 64, 4096, 256, True),      # across k
    (1, 130, 2048, 200, False),
    (1, 1, 7168, 8, False),
    (17, 33, 2056, 72, False),     # the last part is no whole stage
    (8, 24, 4097, 255, False),     # through registers
    (8, 24, 255, 4097, False),
    (8, 24, 2049, 250, True),
    (300, 3, 2048, 136, False),    # parts of several tiles
])
def test_parts_of_k(rows, experts, inner, outer, turned, dtype):
    check(rows, spread(rows, experts), inner, outer, dtype, turned=turned)


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_of_k_beside_rows_without_an_expert(dtype):
    """They hold NaN, and have no sums that could be joined: zeros."""
    for inner, outer in ((4096, 200), (200, 4096), (2049, 77)):
        check(60, spread(9, 20), inner, outer, dtype, first=13)
        check(60, [0] * 5, inner, outer, dtype, first=13)


def far_rows(rows, width, dtype, seed, begin=1, apart=(1 << 21) + 1):
    """Rows 2^21 + 1 elements apart, NaN around them."""
    flat = torch.empty(rows * apart + width + begin, dtype=dtype, device="cuda")
    view = flat.as_strided((rows, width), (apart, 1), begin)
    for lo, hi in ((-begin, 0), (width, width + 24)):
        flat.as_strided((rows, hi - lo), (apart, 1), begin + lo).fill_(math.nan)
    view.copy_(rand((rows, width), dtype, seed))
    return view


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner,outer", [(33, 70), (64, 128), (1030, 31), (31, 1030)])
def test_rows_far_apart(inner, outer, dtype):
    counts = [17, 0, 20, 1]
    check(40, counts, inner, outer, dtype, x=far_rows(40, inner, dtype, 1), d=far_rows(40, outer, dtype, 2, begin=3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("turned", [False, True])
def test_matrices_of_rows_far_apart(turned, dtype):
    inner, outer = (37, 20) if not turned else (20, 37)
    flat = far_rows(40, 37, dtype, 3)
    weight = flat.unflatten(0, (2, 20))
    if turned:
        weight = weight.transpose(1, 2)
    check(50, [30, 20], inner, outer, dtype, x=rand((50, inner), dtype, 1), d=rand((50, outer), dtype, 2), weight=weight)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,counts,inner,outer", [(100, [30, 0, 70], 128, 64), (8, [3, 5], 2048, 64), (1500, [700, 800], 256, 512)])
def test_whole_sizes_at_odd_addresses(rows, counts, inner, outer, dtype):
    """Sizes that are whole pieces, in rows that begin between them."""
    wide, dwide, big = rand((rows, inner + 11), dtype, 1), rand((rows, outer + 9), dtype, 2), rand((len(counts), outer, inner + 3), dtype, 3, 0.5)
    check(rows, counts, inner, outer, dtype, x=wide[:, 3:3 + inner], d=dwide[:, 1:1 + outer], weight=big[:, :, 1:1 + inner])
