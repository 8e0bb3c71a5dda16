"""Gradients of the seam where a row holds an infinite element and the formula
has no norm that would spread it: terms that are left out, not multiplied by 0."""

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, rand
from test_gpu_residual_norm import EPS, NAMES, chain_of, magnitudes, reduce_to, seam64

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]


def run(shape, dtype, parts, where, gate_shape=None, only_out=True):
    """Gradients against the 64-bit formula with one element of `where` infinite; what is not finite there has to be
    the same, everything else close."""
    width = shape[-1]
    t = {k: None for k in NAMES}
    t["residual"] = rand(shape, dtype, 1, 2.0)
    if "u" in parts:
        t["update"] = rand(shape, dtype, 2, 0.7)
    if "g" in parts:
        t["gate"] = rand(gate_shape or (width,), dtype, 3, 0.5, 0.3)
    for i, (k, letter) in enumerate((("post", "1"), ("pre", "2"), ("scale", "s"))):
        if letter in parts:
            t[k] = rand((width,), dtype, 4 + i, 0.2, 1.0)
    clean = {k: None if v is None else v.double().cpu() for k, v in t.items()}
    t[where].view(-1, width)[1, width // 2] = float("inf")
    leaves = {k: None if v is None else v.detach().requires_grad_(True) for k, v in t.items()}
    out, normed = cresso_amd.residual_norm(leaves["residual"], leaves["update"], gate=leaves["gate"], post_weight=leaves["post"],
                                           pre_weight=leaves["pre"], residual_scale=1.0 if t["scale"] is None else leaves["scale"], eps=EPS)
    d_out = rand(shape, dtype, 8)
    names = [k for k in NAMES if t[k] is not None and k != "pre"]
    got = torch.autograd.grad(out, [leaves[k] for k in names], d_out)
    t64 = {k: None if v is None else v.detach().double().cpu().requires_grad_(True) for k, v in t.items()}
    want = torch.autograd.grad(seam64(t64, 1.0, "none")[0], [t64[k] for k in names], d_out.double().cpu())
    with torch.no_grad():   # the magnitudes of what is finite are those of the rows without the infinity
        m = magnitudes(clean, 1.0, "none", d_out.double().cpu(), None)[2]
    chain, column = chain_of(width, out.numel() // width)
    for k, a, b in zip(names, got, want):
        terms = reduce_to(m[k], t[k].shape) + torch.zeros_like(t64[k])
        close(a, b, terms, chain + (0 if t[k].shape == shape else column), "d_" + k)
    return dict(zip(names, got))


WIDTHS = [(6, 130), (4, 1000), (5, 4096), (5, 4100), (3, 9000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", WIDTHS)
@pytest.mark.parametrize("parts", ["", "s", "2", "us", "u1s", "ug1s", "ug12s"])
def test_an_infinite_residual(parts, shape, dtype):
    """Nothing but `out` arrives: an infinite element has no part in the other columns."""
    announce(f"seam gradient, infinite residual, parts {parts!r} {shape} {dtype}")
    g = run(shape, dtype, parts, "residual")
    assert torch.isfinite(g["residual"]).all()
    if "1" in parts:
        assert torch.isfinite(g["update"]).all() and torch.isfinite(g["post"]).all()
    if "s" in parts:
        assert int((~torch.isfinite(g["scale"])).sum()) == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", WIDTHS)
@pytest.mark.parametrize("parts", ["u", "ug", "ugs", "ug2"])
def test_an_infinite_update_without_its_norm(parts, shape, dtype):
    announce(f"seam gradient, infinite update, parts {parts!r} {shape} {dtype}")
    g = run(shape, dtype, parts, "update")
    assert torch.isfinite(g["update"]).all() and torch.isfinite(g["residual"]).all()
    if "g" in parts:
        assert int((~torch.isfinite(g["gate"])).sum()) == 1


@pytest.mark.parametrize("width", [72, 5000])
def test_gates_of_other_rows_keep_their_gradients(width):
    g = run((3, 4, width), torch.bfloat16, "ug1s", "residual", gate_shape=(3, 1, width))
    assert torch.isfinite(g["gate"]).all() and torch.isfinite(g["post"]).all()


@pytest.mark.parametrize("width", [130, 5000])
def test_an_update_without_its_norm_beside_the_next(width):
    """Both outputs arrive and the norm spreads the infinity over its row, but no further."""
    h, y, w = rand((6, width)), rand((6, width), seed=1), rand((width,), seed=2, std=0.1, mean=1.0)
    y[2, 5] = float("inf")
    leaves = [v.requires_grad_(True) for v in (h, y, w)]
    out, normed = cresso_amd.residual_norm(leaves[0], leaves[1], pre_weight=leaves[2])
    dh, dy = torch.autograd.grad((out, normed), leaves[:2], (rand((6, width), seed=3), rand((6, width), seed=4)))
    for r in (0, 1, 3, 4, 5):
        assert torch.isfinite(dh[r]).all() and torch.isfinite(dy[r]).all()
    assert torch.isnan(dh[2]).all()
