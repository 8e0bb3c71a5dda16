"""The distillation loss and its gradient against 64-bit evaluations: teachers
of no, one and many entries, absent and repeated indexes, labels that are
ignored or also the teacher's, masked logits and rows, temperatures, types,
strides, the gradient in the logits' place, refusals."""

import math

import numpy as np
import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(z, index, a, labels, weights, t, mix, ignore=-100):
    """Rows' losses and the gradient of their sum, with the magnitudes they are sums of; numpy in 64 bits."""
    z, index, a = z.double().cpu().numpy(), index.cpu().numpy(), a.double().cpu().numpy()
    rows, vocab = z.shape
    labels = None if labels is None else labels.cpu().numpy()
    w = np.full(rows, 1.0 / max(rows, 1)) if weights is None else weights.double().cpu().numpy()
    loss, loss_m = np.zeros(rows), np.zeros(rows)
    grad, grad_m = np.zeros((rows, vocab)), np.zeros((rows, vocab))
    with np.errstate(all="ignore"):
        for r in range(rows):
            on = (index[r] >= 0) & (index[r] < vocab)
            idx, ar = index[r][on], a[r][on] / t
            label = -1 if labels is None or labels[r] == ignore or not 0 <= labels[r] < vocab else labels[r]
            if w[r] == 0 or (not on.any() and label < 0):
                continue
            m = z[r].max()
            m = 0.0 if m == -np.inf else m
            soft = on.any() and not np.all(ar == -np.inf)
            if soft:
                x = (z[r] - m) / t
                log_s = np.log(np.exp(x).sum())
                at = ar.max()
                p = np.exp(ar - at)
                total = p.sum()
                p = p / total
                use = ~(p == 0)
                parts = p[use] * ((ar[use] - at - np.log(total)) - (x[idx[use]] - log_s))
                size = np.abs(ar[use] - at) + np.abs(np.log(total)) + np.abs(x[idx[use]]) + np.abs(log_s) + 1
                loss[r] += mix * t * t * parts.sum()
                loss_m[r] += mix * t * t * (p[use] * size).sum()
                q = np.exp(x - log_s)
                grad[r] += mix * t * q
                # an exponent is off by its own size times 2^-24
                grad_m[r] += mix * t * q * (2 + np.abs(np.where(np.isfinite(x), x, 0)) + np.abs(log_s))
                np.subtract.at(grad[r], idx, mix * t * p)
                np.add.at(grad_m[r], idx, mix * t * p * (2 + np.abs(np.where(np.isfinite(ar), ar - at, 0))))
            if label >= 0:
                x = z[r] - m
                log_s = np.log(np.exp(x).sum())
                loss[r] += (1 - mix) * (log_s - x[label])
                loss_m[r] += (1 - mix) * (np.abs(log_s) + np.abs(x[label]) + 1)
                q = np.exp(x - log_s)
                grad[r] += (1 - mix) * q
                grad_m[r] += (1 - mix) * q * (2 + np.abs(np.where(np.isfinite(x), x, 0)) + np.abs(log_s))
                grad[r, label] -= 1 - mix
                grad_m[r, label] += 1 - mix
    w1 = w[:, None]
    back = torch.from_numpy
    return back(loss * w), back(np.nan_to_num(np.abs(loss_m * w), posinf=0.0)), back(grad * w1), back(np.nan_to_num(np.abs(grad_m * w1)))


def chain(vocab):
    """A lane's additions (a wave-wide row of 512 lanes), the merge of lanes and waves, and the rounding of each
    exponential, quotient and product."""
    return vocab // 512 + 16 + 6 + 8 + 16


def check(z, index, a, labels=None, weights=None, t=1.0, mix=1.0, what=""):
    loss, loss_m, grad, grad_m = reference(z, index, a, labels, weights, t, mix)
    n = chain(z.shape[1])
    kw = dict(labels=labels, row_weights=weights, temperature=t, mix=mix)
    rows = cresso_amd.distill_loss(z, index, a, reduction="none", **kw)
    close(rows, loss, loss_m, n, what + " rows")
    total = cresso_amd.distill_loss(z, index, a, **kw)
    close(total, loss.sum(), loss_m.sum(), n + 2, what + " total")
    leaf = z.detach().requires_grad_(True)
    cresso_amd.distill_loss(leaf, index, a, **kw).backward()
    close(leaf.grad, grad, grad_m, n, what + " gradient")
    both, g = cresso_amd.distill_loss_and_grad(z, index, a, **kw)
    close(both, loss.sum(), loss_m.sum(), n + 2, what + " loss of both")
    close(g, grad, grad_m, n, what + " gradient of both")
    place = z.contiguous().clone()
    again, g2 = cresso_amd.distill_loss_and_grad(place, index, a, out=place, **kw)
    assert g2 is place and torch.equal(torch.nan_to_num(g2.float()), torch.nan_to_num(g.float()))
    assert torch.equal(again.nan_to_num(), both.nan_to_num())
    return rows, g


def make(rows, vocab, top, dtype=torch.float32, seed=0, absent=0.0, labels=True, wide=True):
    gen = torch.Generator().manual_seed(seed)
    z = rand((rows, vocab), dtype, seed + 1, 2.0)
    index = torch.stack([torch.randperm(vocab, generator=gen)[:top] for _ in range(rows)]) if rows else torch.zeros(0, top)
    index = index.long()
    if absent:
        index[torch.rand(index.shape, generator=gen) < absent] = -1
    a = rand((rows, top), dtype, seed + 2, 2.0, 5.0)
    lab = None
    if labels:
        lab = torch.randint(0, vocab, (rows,), generator=gen)
        lab[::3] = -100
        if top and rows > 1:
            lab[1] = index[1, 0].clamp(min=0)
        lab = lab.cuda() if wide else lab.int().cuda()
    return z, (index if wide else index.int()).cuda(), a, lab


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (4, 7, 7), (3, 511, 1), (5, 1000, 64), (2, 4097, 300), (3, 40001, 33),
                                            (2, 1024, 1024), (2, 131072, 16)])
def test_sizes(rows, vocab, top, dtype):
    announce(f"distill {rows} x {vocab} top {top} {dtype}")
    for mix, t in ((1.0, 1.0), (0.6, 2.0), (0.3, 1.7)):
        z, index, a, lab = make(rows, vocab, top, dtype, seed=rows, wide=top % 2 == 0)
        check(z, index, a, lab, None, t, mix, f"mix {mix}")
    check(z, index, a, None, None, 4.0, 0.9, "no labels")


def test_absent_entries_and_rows():
    z, index, a, lab = make(12, 300, 9, seed=3, absent=0.5)
    index[2], index[3] = -1, 300          # no teacher; label 3 is ignored
    index[5], lab[5] = -1, -100           # neither
    a[7] = -math.inf                      # a teacher of nothing
    a[8, 1:] = -math.inf
    index[8, 0] = 17
    weights = torch.full((12,), 0.25).cuda()
    weights[9], z[9] = 0.0, math.nan      # a masked row may hold anything
    z[5] = math.nan
    rows, g = check(z, index, a, lab, weights, 2.0, 0.5)
    for r in (5, 9):
        assert rows[r] == 0 and not g[r].any()


def test_no_entries_at_all():
    z, _, _, lab = make(6, 90, 3)
    none = torch.zeros(6, 0, dtype=torch.int32).cuda()
    check(z, none, torch.zeros(6, 0).cuda(), lab, None, 1.0, 0.25)
    rows, g = check(z, none, torch.zeros(6, 0).cuda(), None, None, 1.0, 0.25)
    assert not rows.any() and not g.any()


def test_an_index_given_twice_counts_twice():
    z, index, a, lab = make(4, 50, 6, seed=5)
    index[0] = 7
    index[1, 3] = index[1, 0]
    lab[0], lab[1] = 7, int(index[1, 0])
    check(z, index, a, lab, None, 1.5, 0.5)


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_masked_logits(low):
    z, index, a, lab = make(6, 200, 5, seed=8)
    keep = torch.zeros(200, dtype=torch.bool)
    keep[::7] = True
    z[:, ~keep.cuda()] = low
    index[:] = torch.arange(0, 200, 7)[torch.stack([torch.randperm(29)[:5] for _ in range(6)])].cuda()
    lab[:] = 14
    check(z, index, a, lab, None, 2.0, 0.5)
    if low == -math.inf:
        index[0, 0] = 1                   # the teacher wants what the student cannot say
        lab[1] = 2
        rows, g = check(z, index, a, lab, None, 2.0, 0.5)
        assert rows[0] == math.inf and rows[1] == math.inf and torch.isfinite(g).all()


def test_rows_that_are_not_numbers():
    z, index, a, lab = make(5, 64, 4, seed=9)
    z[0], z[1, 3], z[2, 5] = -math.inf, math.nan, math.inf
    lab[:] = 1
    index[:, 0] = 1
    rows, g = check(z, index, a, lab, None, 1.0, 0.5)
    assert torch.isnan(rows[:3]).all() and torch.isfinite(rows[3:]).all() and torch.isfinite(g[3:]).all()


def test_large_and_shifted_logits():
    for shift in (-3e4, 0.0, 3e4):
        z, index, a, lab = make(4, 700, 8, seed=11)
        z = z * 8 + shift
        check(z, index, a + shift, lab, None, 1.0, 0.5, f"shift {shift}")


def test_strides_and_types():
    z, index, a, lab = make(7, 333, 6, torch.bfloat16, seed=12)
    wide = torch.full((7, 400), math.nan, dtype=torch.bfloat16).cuda()
    wide[:, 5:338] = z
    idx, teach = torch.zeros(7, 20, dtype=torch.int64).cuda() - 1, torch.zeros(7, 20).cuda()
    idx[:, 3:9], teach[:, 3:9] = index, a.float()
    kw = dict(labels=lab, temperature=2.0, mix=0.5)
    want, g = cresso_amd.distill_loss_and_grad(z, index, a.float(), **kw)
    got, g2 = cresso_amd.distill_loss_and_grad(wide[:, 5:338], idx[:, 3:9], teach[:, 3:9], out=wide[:, 5:338], **kw)
    assert torch.equal(want, got) and torch.equal(g, wide[:, 5:338])
    assert torch.isnan(wide[:, :5]).all() and torch.isnan(wide[:, 338:]).all()
    check(z.t().contiguous().t(), index, a.half(), lab, None, 2.0, 0.5)


def test_what_arrives_at_the_loss():
    z, index, a, lab = make(6, 100, 5, seed=13)
    _, _, grad, grad_m = reference(z, index, a, lab, None, 2.0, 0.5)
    kw = dict(labels=lab, temperature=2.0, mix=0.5)
    leaf = z.detach().requires_grad_(True)
    (cresso_amd.distill_loss(leaf, index, a, **kw) * -3.0).backward()
    close(leaf.grad, grad * -3, grad_m * 3, chain(100) + 2)
    leaf = z.detach().requires_grad_(True)
    by = rand((6,), seed=14)
    cresso_amd.distill_loss(leaf, index, a, reduction="none", **kw).backward(by)
    s = by.double().cpu().unsqueeze(1)
    close(leaf.grad, grad * s, grad_m * s.abs(), chain(100) + 2)
    leaf = z.detach().requires_grad_(True)
    cresso_amd.distill_loss(leaf, index, a, reduction="none", **kw).sum().backward()   # one number for every row
    close(leaf.grad, grad, grad_m, chain(100) + 2)


def test_gradient_against_differences():
    z, index, a, lab = make(3, 60, 5, seed=15)
    _, g = cresso_amd.distill_loss_and_grad(z, index, a, labels=lab, temperature=1.5, mix=0.4)
    direction = torch.from_numpy(np.random.RandomState(1).randn(3, 60))
    step = 1e-5
    base = z.double().cpu()
    value = lambda x: float(reference(x, index, a, lab, None, 1.5, 0.4)[0].sum())   # noqa: E731
    slope = (value(base + step * direction) - value(base - step * direction)) / (2 * step)
    got = float((g.double().cpu() * direction).sum())
    assert abs(got - slope) <= 2e-5 * float((g.double().cpu() * direction).abs().sum())


def test_logits_that_were_overwritten_are_noticed():
    z = rand((4, 30), seed=17).requires_grad_(True)
    y = torch.sigmoid(z)   # keeps its output for its own gradient
    index, a = torch.zeros(4, 1, dtype=torch.int64).cuda(), torch.zeros(4, 1).cuda()
    _, g = cresso_amd.distill_loss_and_grad(y, index, a, out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(g)


def test_without_rows():
    z, index, a = torch.zeros(0, 10).cuda(), torch.zeros(0, 3, dtype=torch.int64).cuda(), torch.zeros(0, 3).cuda()
    assert cresso_amd.distill_loss(z, index, a).item() == 0.0
    loss, g = cresso_amd.distill_loss_and_grad(z, index, a)
    assert loss.item() == 0.0 and g.shape == (0, 10)
    leaf = z.requires_grad_(True)
    cresso_amd.distill_loss(leaf, index, a).backward()
    assert leaf.grad.shape == (0, 10)


def test_same_bits_on_another_stream():
    z, index, a, lab = make(40, 5000, 16, torch.bfloat16, seed=16)
    want = cresso_amd.distill_loss_and_grad(z, index, a, labels=lab, temperature=2.0, mix=0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cresso_amd.distill_loss_and_grad(z, index, a, labels=lab, temperature=2.0, mix=0.5)
    side.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_refusals():
    z, index, a, lab = make(4, 30, 3)
    cases = [
        ((z[0], index, a), {}, "logits must be"), ((z, index[:3], a), {}, "must both be"), ((z, index, a[:, :2]), {}, "must both be"),
        ((z.double(), index, a), {}, "fp32, bf16 or fp16"), ((z, index.float(), a), {}, "int32 or int64"),
        ((z, index, a), dict(labels=lab[:2]), r"labels must be \[4\]"), ((z, index, a), dict(labels=lab.float()), "int32 or int64"),
        ((z, index, a), dict(row_weights=torch.ones(4).cuda().half()), "row_weights"), ((z, index, a), dict(temperature=0.0), "temperature"),
        ((z, index, a), dict(mix=1.5), "mix"), ((z, torch.zeros(4, 1025, dtype=torch.int32).cuda(), torch.zeros(4, 1025).cuda()), {}, "at most 1024"),
    ]
    for args, kw, msg in cases:
        for fn in (cresso_amd.distill_loss, cresso_amd.distill_loss_and_grad):
            with pytest.raises(ValueError, match=msg):
                fn(*args, **kw)
    with pytest.raises(ValueError, match="reduction"):
        cresso_amd.distill_loss(z, index, a, reduction="mean")
    with pytest.raises(ValueError, match="out is"):
        cresso_amd.distill_loss_and_grad(z, index, a, out=z.half())
    with pytest.raises(ValueError, match="one piece"):
        cresso_amd.distill_loss_and_grad(z, index, a, out=torch.zeros(30, 4).cuda().t())
    with pytest.raises(RuntimeError, match="GPU only"):
        cresso_amd.distill_loss(z, index.cpu(), a)


@pytest.mark.parametrize("mix", [0.0, 1.0])
def test_a_factor_of_zero_leaves_its_term_out(mix):
    """An infinite term must not come through a factor of 0 as NaN: as if what makes the term were not given."""
    z, index, a, _ = make(6, 700, 5, seed=11, labels=False)
    index[index == 0] = 699
    lab = torch.zeros(6, dtype=torch.int64, device="cuda")
    lab[4] = -100
    gone = lab.clamp(min=0) if mix == 1.0 else index[:, 1]
    z[torch.arange(6, device="cuda"), gone] = -math.inf
    kw = dict(temperature=1.5, mix=mix)
    want = cresso_amd.distill_loss_and_grad(z, index if mix == 1.0 else torch.full_like(index, -1), a,
                                            labels=None if mix == 1.0 else lab, **kw)
    got = cresso_amd.distill_loss_and_grad(z, index, a, labels=lab, **kw)
    assert torch.isfinite(got[0]) and torch.isfinite(got[1]).all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    zr = z.clone().requires_grad_(True)
    loss = cresso_amd.distill_loss(zr, index, a, labels=lab, **kw)
    (grad,) = torch.autograd.grad(loss, zr)
    assert torch.equal(loss.detach(), want[0]) and torch.isfinite(grad).all()
    assert torch.equal(got[1] == 0, grad == 0)
    if mix == 1.0:   # a row with nothing but a label has no term left
        alone = cresso_amd.distill_loss(z, torch.full_like(index, -1), a, labels=lab, reduction="none", **kw)
        assert torch.equal(alone, torch.zeros_like(alone))
