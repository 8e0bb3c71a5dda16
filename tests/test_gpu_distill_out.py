"""Where distill_loss_and_grad writes: in the logits' place, beside them in one
buffer, and never over what it has yet to read."""

import pytest
import torch

from gpu_util import needs_gpu
from test_gpu_distill import make

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

ROWS, VOCAB = 40, 3001


@pytest.fixture(scope="module")
def case():
    z, index, a, lab = make(ROWS, VOCAB, 6, torch.bfloat16, seed=31)
    kw = dict(labels=lab, row_weights=torch.full((ROWS,), 0.5).cuda(), temperature=2.0, mix=0.5)
    return z, index, a, kw, cresso_amd.distill_loss_and_grad(z, index, a, **kw)


def test_places_that_are_taken(case):
    z, index, a, kw, (want, g) = case
    wide = torch.zeros(ROWS, 2 * VOCAB + 9, dtype=torch.bfloat16).cuda()
    logits, beside = wide[:, 3:3 + VOCAB], wide[:, 3 + VOCAB:3 + 2 * VOCAB]
    for out in (logits, beside, wide[:, 6 + VOCAB:6 + 2 * VOCAB]):   # in place, right beside the rows, a little further
        wide.zero_()
        logits.copy_(z)
        loss, got = cresso_amd.distill_loss_and_grad(logits, index, a, out=out, **kw)
        assert got is out and torch.equal(loss, want) and torch.equal(out, g)
    both = torch.zeros(2 * ROWS, VOCAB, dtype=torch.bfloat16).cuda()
    both[:ROWS] = z
    loss, _ = cresso_amd.distill_loss_and_grad(both[:ROWS], index, a, out=both[ROWS:], **kw)
    assert torch.equal(loss, want) and torch.equal(both[ROWS:], g) and torch.equal(both[:ROWS], z)
    one = z[:1].clone()   # one row has no stride
    loss, got = cresso_amd.distill_loss_and_grad(one, index[:1], a[:1], out=one.as_strided((1, VOCAB), (VOCAB + 5, 1)))
    assert torch.equal(got, cresso_amd.distill_loss_and_grad(z[:1], index[:1], a[:1])[1])
    turned = z.t().contiguous().t()   # columns at a stride are copied, and the copy is read
    place = torch.as_strided(turned, (ROWS, VOCAB), (VOCAB, 1))
    loss, got = cresso_amd.distill_loss_and_grad(turned, index, a, out=place, **kw)
    assert torch.equal(loss, want) and torch.equal(got, g)


def test_places_that_are_refused(case):
    z, index, a, kw, _ = case
    room = torch.zeros(ROWS + 2, VOCAB + 5, dtype=torch.bfloat16).cuda()
    logits = room[:ROWS, :VOCAB]
    logits.copy_(z)
    held = room.clone()
    flat = room.view(-1)
    for out in (room[1:ROWS + 1, :VOCAB], room[:ROWS, 1:VOCAB + 1], room[:ROWS, 5:],
                flat[:ROWS * VOCAB].view(ROWS, VOCAB), flat[VOCAB + 5:].as_strided((ROWS, VOCAB), (VOCAB, 1))):
        with pytest.raises(ValueError, match="shares memory with the logits"):
            cresso_amd.distill_loss_and_grad(logits, index, a, out=out, **kw)
    mem = torch.zeros(ROWS * VOCAB, dtype=torch.bfloat16).cuda()
    out = mem.view(ROWS, VOCAB)
    inside = {
        "teacher's logits": ((z, index, mem[:ROWS * 6].view(ROWS, 6)), kw),
        "teacher's indexes": ((z, mem[:ROWS * 24].view(torch.int64).view(ROWS, 6), a), kw),
        "labels": ((z, index, a), {**kw, "labels": mem[-ROWS * 4:].view(torch.int64)}),
        "row weights": ((z, index, a), {**kw, "row_weights": mem[VOCAB + 1:VOCAB + 1 + 2 * ROWS].view(torch.float32)}),
    }
    for what, (args, k) in inside.items():
        with pytest.raises(ValueError, match=what):
            cresso_amd.distill_loss_and_grad(*args, out=out, **k)
    assert torch.equal(room, held) and not mem.any()
