"""Logits and teachers of any finite size against the 64-bit evaluation: masks
of large finite numbers and of the type's lowest, in whole rows, in whole
units of a row (a thread then sees nothing else) and between other logits."""

import pytest
import torch

from gpu_util import announce, needs_gpu
from test_gpu_distill import check, make

pytestmark = [pytest.mark.gpu, needs_gpu]

LOWEST = "lowest"


def mask_of(low, dtype):
    return torch.finfo(dtype).min if low == LOWEST else low


def within(z, index, lab, dtype):
    """The teacher's entries and the labels get logits of an ordinary size."""
    z.scatter_(1, index.clamp(min=0), torch.linspace(-3, 3, index.shape[1], device="cuda").to(dtype).expand(index.shape).contiguous())
    z.scatter_(1, lab.clamp(min=0).unsqueeze(1), 0.5)


@pytest.mark.parametrize("t", [1.0, 1.5, 2.0, 3.0])
@pytest.mark.parametrize("dtype,low", [(torch.float32, -1e10), (torch.float32, -1e30), (torch.float32, LOWEST), (torch.bfloat16, -1e10),
                                       (torch.bfloat16, -1e30), (torch.bfloat16, LOWEST), (torch.float16, LOWEST)])
def test_masks_of_any_size(dtype, low, t):
    announce(f"distill masks {low} {dtype} t {t}")
    for vocab in (200, 5000, 40001):
        z, index, a, lab = make(5, vocab, 6, dtype, seed=21)
        keep = torch.zeros(vocab, dtype=torch.bool)
        keep[::7] = True
        keep[vocab // 4:vocab // 2] = False        # whole units, and whole threads, of masks
        z[:, ~keep.cuda()] = mask_of(low, dtype)
        within(z, index, lab, dtype)
        check(z, index, a, lab, None, t, 0.5, "with labels")
        check(z, index, a, None, None, t, 1.0, "without labels")


@pytest.mark.parametrize("t", [1.0, 1.5, 2.0, 3.0])
@pytest.mark.parametrize("dtype,low", [(torch.float32, -1e10), (torch.float32, LOWEST), (torch.bfloat16, LOWEST), (torch.float16, LOWEST)])
def test_rows_of_nothing_but_masks(dtype, low, t):
    """Equal logits, whatever their size: every word is as likely."""
    announce(f"distill rows of masks {low} {dtype} t {t}")
    for vocab in (9, 3000):
        z, index, a, lab = make(4, vocab, 4, dtype, seed=22)
        z[1:3] = mask_of(low, dtype)
        z[3] = -mask_of(low, dtype)
        rows, g = check(z, index, a, lab, None, t, 0.5)
        assert torch.isfinite(rows).all() and torch.isfinite(g).all()


@pytest.mark.parametrize("t", [1.0, 1.5, 2.0])
def test_rows_of_large_logits(t):
    """fp32 numbers around 1e10 lie 1024 apart: one word is certain, or two that are equal share the row."""
    z, index, a, lab = make(4, 1000, 5, torch.float32, seed=23)
    z[0] += 1e10
    z[1] = z[1] * 1e9 - 3e10
    z[2] = 1e10 + 1024.0 * torch.randint(-3, 4, (1000,)).cuda()
    z[3, 500:] = -1e20
    at = z.argmax(1)                               # the teacher wants what is possible
    index[:, 1:] = -1
    index[:, 0] = at
    lab[:] = at
    check(z, index, a, lab, None, t, 0.5)


@pytest.mark.parametrize("t", [1.0, 1.5, 2.0])
@pytest.mark.parametrize("dtype,low", [(torch.float32, -1e10), (torch.float32, LOWEST), (torch.bfloat16, LOWEST)])
def test_masked_teachers(dtype, low, t):
    z, index, a, lab = make(5, 300, 8, dtype, seed=24)
    a[0, 3:] = mask_of(low, dtype)
    a[1] = mask_of(low, dtype)                     # eight entries that are equally likely
    a[2] = -mask_of(low, dtype)
    check(z, index, a, lab, None, t, 0.5)
