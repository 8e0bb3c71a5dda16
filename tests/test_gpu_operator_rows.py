"""Rows of more than two dimensions at one common stride are taken where they
lie; other layouts are copied.  Both give what a contiguous copy gives."""

import pytest
import torch

from gpu_util import needs_gpu
from operator_util import rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]


def slices():
    """(what, x of shape (2, 3, 5, 264) in some layout, whether its rows lie at one stride)"""
    base = rand((2, 3, 5, 264), torch.bfloat16, 1)
    wide = torch.zeros(2, 3, 5, 400, dtype=torch.bfloat16).cuda()
    wide[..., 7:271] = base
    yield "slice of the last dimension", wide[..., 7:271], True
    long = torch.zeros(2, 3, 9, 264, dtype=torch.bfloat16).cuda()
    long[:, :, 2:7] = base
    yield "slice of an inner dimension", long[:, :, 2:7], False
    yield "turned dimensions", base.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3), False
    yield "broadcast", base[:1].expand(2, 3, 5, 264), False
    yield "last dimension at a stride", base.transpose(2, 3).contiguous().transpose(2, 3), False


def peak(fn):
    """Bytes that a call allocates at most beyond what was held before."""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = fn()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


def test_values_do_not_depend_on_the_layout():
    w, pre = rand((264,), torch.bfloat16, 2), rand((264,), torch.bfloat16, 3)
    values, scales = cresso_amd.quantize_blocks(rand((70, 264), torch.bfloat16, 4))
    ids = torch.randint(0, 9, (2, 3, 5)).cuda()

    def seam(x, y, d):
        a, b = x.detach().requires_grad_(True), y.detach().requires_grad_(True)
        out, normed = cresso_amd.residual_norm(a, b, post_weight=w, pre_weight=pre)
        return [out, normed, *torch.autograd.grad((out, normed), (a, b), (d, d))]

    for what, x, _ in slices():
        dense = x.contiguous()
        for a, b in zip(seam(x, x, x), seam(dense, dense, dense)):
            assert torch.equal(a, b), what
        assert torch.equal(cresso_amd.block_product(x, values, scales), cresso_amd.block_product(dense, values, scales)), what
        assert torch.equal(cresso_amd.embedding_grad(ids, x, 9), cresso_amd.embedding_grad(ids, dense, 9)), what


def test_dimensions_of_one():
    wide = rand((1, 4, 1, 300), torch.bfloat16, 5)
    for x in (wide[..., 3:67], wide[:, 1:2, :, 3:67], wide.permute(2, 1, 0, 3)[..., 3:67], wide[0, 0, 0, 3:67],
              wide.as_strided((1, 4, 64), (7, 300, 1), 3), wide.as_strided((4, 1, 64), (300, 1, 1), 3)):
        out, _ = cresso_amd.residual_norm(x, residual_scale=2.0)
        assert out.shape == x.shape and torch.equal(out, 2 * x.contiguous())


def test_rows_at_one_stride_are_not_copied():
    wide = torch.zeros(4, 64, 8, 600, dtype=torch.bfloat16).cuda()
    x = wide[..., 8:520]
    size = x.numel() * 2
    for fn, outputs in ((lambda: cresso_amd.residual_norm(x, x), 1),
                        (lambda: cresso_amd.embedding_grad(torch.zeros(4, 64, 8, dtype=torch.int64).cuda(), x, 3), 0)):
        fn()
        _, held = peak(fn)
        dense = x.contiguous()
        x_dense, x = x, dense
        _, held_dense = peak(fn)
        x = x_dense
        assert held <= held_dense + size // 2, (held, held_dense, outputs)
