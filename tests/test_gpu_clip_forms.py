"""Gradient norm and clipping in forms that the general tests do not reach: fp64
gradients whose squares leave fp64's range, slices that interleave, parameters
in their gradients' stead."""

import math

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import EPS32, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]


def times(t, e):
    """t * 2^e by two factors that are numbers."""
    return t * 2.0 ** (e // 2) * 2.0 ** (e - e // 2)


def norm_of(grads):
    """m, e: the 2-norm is m * 2^e, m from 1/2 to the root of the number of elements."""
    flat = torch.cat([g.double().cpu().reshape(-1) for g in grads])
    e = math.frexp(float(flat.abs().max()))[1]
    return float(times(flat, -e).norm()), e


def wide(n, exponent, seed, spread=0):
    """Normal numbers times 2^exponent, and each times 2 to up to +-spread more."""
    more = torch.randint(-spread, spread + 1, (n,), generator=torch.Generator().manual_seed(seed + 50)).double().cuda()
    return times(rand((n,), seed=seed).double() * 2.0 ** more, exponent)


CASES = {
    "above": [(5000, 700, 0)],                  # squares above fp64's range
    "below": [(5000, -700, 0)],                 # squares below it
    "denormal": [(3000, -1062, 0)],
    "high": [(20000, 1000, 0), (7, 3, 0)],
    "around the upper border": [(9000, 480, 6), (70000, 478, 0)],
    "around the lower border": [(9000, -480, 6), (70000, -482, 0)],
    "all": [(9000, -900, 0), (33, 0, 0), (20000, 900, 0)],
    "low and middle": [(9000, -900, 0), (20000, 0, 0)],
    "low and less": [(9000, -600, 300)],
}


@pytest.mark.parametrize("others", [False, True])
@pytest.mark.parametrize("name", list(CASES))
def test_fp64_of_any_size(name, others):
    announce(f"clip fp64 {name} {others}")
    make = lambda: [wide(n, e, i, s) for i, (n, e, s) in enumerate(CASES[name])] + (   # noqa: E731
        [rand((10000,), torch.float32, 7), rand((333,), torch.bfloat16, 8)] if others else [])
    grads = make()
    m, e = norm_of(grads)
    try:
        exact = math.ldexp(m, e)
    except OverflowError:
        exact = math.inf
    got = cresso_amd.gradient_norm(grads)
    if exact > 3.5e38:
        assert float(got) == math.inf    # above fp32
    else:
        assert abs(float(got.double()) - exact) <= (EPS32 + 2.0 ** -40) * exact + 2.0 ** -150
    for low in (2, 1000):         # limits of a quarter of the norm and of 2^-1000 of it
        max_norm = math.ldexp(m, e - low)
        if not 0.0 < max_norm < math.inf or exact == math.inf or max_norm < 2.0 ** -1022:
            continue
        grads = make()
        cresso_amd.clip_gradients(grads, max_norm)
        for g, b in zip(grads, make()):
            if g.dtype != torch.float64:
                continue
            want = times(b, -low)
            # sums and their root as 1e-11 covers any number of terms; numbers below 2^-1022 are rounded to multiples of 2^-1074
            assert torch.allclose(g, want, rtol=1e-11, atol=2.0 ** -1073), (name, low)


def test_fp64_largest_of_any_size():
    announce("clip fp64 by the largest")
    for exponent in (-1000, -600, 600, 1000):
        g = wide(5000, exponent, 1)
        before, top = g.clone(), float(g.abs().max())
        cresso_amd.clip_gradients(g, math.ldexp(top, -2), norm_type=math.inf)
        assert torch.allclose(g, before / 4, rtol=1e-15, atol=0.0)
    g = torch.full((1000,), 2.0 ** 1000, dtype=torch.float64, device="cuda")
    cresso_amd.clip_gradients(g, 2.0 ** -60, norm_type=math.inf)
    assert torch.equal(g, torch.full_like(g, 2.0 ** -60))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_fp64_norms_that_are_not_finite(bad):
    announce(f"clip fp64 large numbers with {bad}")
    for where in (0, 1):
        grads = [wide(5000, 700, 1), rand((10000,), torch.float32, 2)]
        grads[where][77] = bad
        want = [g.clone() for g in grads]
        norm = cresso_amd.clip_gradients(grads, 0.5)
        assert math.isnan(norm) if math.isnan(bad) else float(norm) == math.inf
        for g, w in zip(grads, want):
            assert torch.equal(torch.nan_to_num(g, nan=3.0), torch.nan_to_num(w, nan=3.0))


def slices(buffer, kind):
    if kind == "columns":
        return [buffer[:, :30], buffer[:, 30:31], buffer[:, 31:]]
    if kind == "columns that begin within":
        return [buffer.view(-1)[50:50 + 37 * 64].view(37, 64)[:, :20], buffer[:, 6:50]]   # columns 50 to 63 and 0 to 5
    if kind == "middle":
        return list(buffer.view(10, 4, 64).split([1, 3], 1))
    if kind == "every other":
        return [buffer[:, ::2], buffer[:, 1::2]]
    raise ValueError(kind)


KINDS = ["columns", "columns that begin within", "middle", "every other"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("kind", KINDS)
def test_slices_that_interleave(kind, dtype):
    """They share no memory: clipped in place, and to slices of another buffer, with nothing beside them changed."""
    announce(f"clip {kind} {dtype}")
    for elsewhere in (False, True):
        buffer, other = rand((40, 64), dtype, 1), torch.full((40, 64), 7.0, dtype=dtype, device="cuda")
        norm = float(torch.cat([t.double().flatten() for t in slices(buffer, kind)]).norm())
        want, to = buffer.clone(), other if elsewhere else buffer
        marks = torch.zeros_like(buffer, dtype=torch.bool)
        for t in slices(marks, kind):
            assert not t.any()
            t.fill_(True)
        got = cresso_amd.clip_gradients(slices(buffer, kind), 0.5, out=slices(other, kind) if elsewhere else None)
        assert abs(float(got) - norm) <= 2.0 ** -23 * norm
        assert torch.equal(to[~marks], (torch.full_like(want, 7.0) if elsewhere else want)[~marks])
        exact = want.double() * (0.5 / norm)
        # half a step of the type, and what fp32 adds in front of a rounding to 16 bits
        assert ((to.double() - exact).abs() <= exact.abs() * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + 2.0 ** -40))[marks].all()


def test_gradients_of_a_concatenation():
    """Autograd hands out the columns of one tensor."""
    announce("clip gradients of a concatenation")
    leaves = [rand((30, n), seed=n).requires_grad_(True) for n in (7, 20, 1)]
    d = rand((30, 28), seed=4)
    y = torch.cat(leaves, 1)
    grads = torch.autograd.grad(y, leaves, d)
    want, norm = [g.clone() for g in grads], float(d.double().norm())
    cresso_amd.clip_gradients(grads, 0.5)
    for g, w in zip(grads, want):
        assert torch.allclose(g, w * (0.5 / norm), rtol=2.0 ** -22, atol=0.0)


def test_slices_that_share_are_refused():
    announce("clip slices that share")
    b = rand((40, 64))
    flat = b.view(-1)
    for grads in ([b[:, :30], b[:, 29:]], [b[:, :30], b[:, :30]], [b[:, :30], b[:, 40:], b[3, 20:45]],
                  [flat[50:50 + 37 * 64].view(37, 64)[:, :20], b[:, :10]], [flat[50:50 + 37 * 64].view(37, 64)[:, :20], b[:, 55:]],
                  [b[:, ::2], b[:, 2:4]], [b.t()[:30], b[:, 29:]], [b[:, :30], flat[:2000].view(40, 50)[:, 45:]]):
        with pytest.raises(ValueError, match="belongs to two"):
            cresso_amd.clip_gradients(grads, 0.5)
        cresso_amd.gradient_norm(grads)
    with pytest.raises(ValueError, match="belongs to two"):   # an input's columns are another's output
        cresso_amd.clip_gradients([b[:, :30], b[:, 30:]], 0.5, out=[b[:, 20:50], rand((40, 34))])
    cresso_amd.clip_gradients([b[:, :30], b[:, :30]], 0.5, out=[b[:, 30:60], rand((40, 30))])   # inputs may share


def test_parameters_are_not_taken_for_gradients():
    announce("clip parameters")
    p, q = (torch.nn.Parameter(rand((20, 8), seed=i)) for i in (1, 2))
    want = p.detach().clone()
    for call in (lambda: cresso_amd.clip_gradients([p, q], 0.1), lambda: cresso_amd.clip_gradients(p.view(-1), 0.1),
                 lambda: cresso_amd.clip_gradients([want], 0.1, out=[p])):
        with pytest.raises(RuntimeError, match="leaf that requires a gradient"):
            call()
        assert torch.equal(p, want)
    assert abs(float(cresso_amd.gradient_norm([p])) / float(want.norm()) - 1.0) < 1e-6   # reading is fine
    cresso_amd.clip_gradients([p], 0.1, out=[torch.empty_like(want)])
    (g,) = torch.autograd.grad((p * p).sum(), p, create_graph=True)
    cresso_amd.clip_gradients([g], 0.1)   # a gradient with a history of its own is no leaf
    assert abs(float(g.detach().norm()) - 0.1) < 1e-6
    opt = cresso_amd.CRESSO5([p, q])
    p.grad = torch.ones_like(p).requires_grad_(True)
    assert abs(float(opt.clip_gradients(0.5)) / 160 ** 0.5 - 1.0) < 1e-6
    assert abs(float(p.grad.detach().norm()) - 0.5) < 1e-6
