"""Error bounds of the operators' tests: every result is compared with a plain
64-bit evaluation of the operator's formula on the same inputs."""

from __future__ import annotations

import numpy as np
import torch

# unit roundoff and half the spacing of the smallest numbers
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
EPS32 = 2.0 ** -24


def close(got, want, terms, chain, what=""):
    """|got - want| <= chain * 2^-24 * terms + the rounding of want to got's type.

    want: the 64-bit result; terms: the same formula over the magnitudes of
    what it adds; chain: how many fp32 operations an input passes through on
    its way to the result (each may be off by 2^-24 of the magnitudes).
    NaN and infinities must be the same ones.
    """
    assert got.shape == want.shape, (what, got.shape, want.shape)
    got_type = got.dtype
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    t = torch.broadcast_to(torch.as_tensor(terms, dtype=torch.float64).cpu(), w.shape)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what
    inf = torch.isinf(w)
    assert torch.equal(g[inf], w[inf]), what
    fine = torch.isfinite(w)
    assert torch.isfinite(g[fine]).all(), what
    g, w, t = g[fine], w[fine], t[fine]
    room = chain * EPS32 * t * (1 + ROUND[got_type]) + ROUND[got_type] * w.abs() * (1 + chain * EPS32) + TINY[got_type]
    over = (g - w).abs() - room
    if over.numel() and float(over.max()) > 0:
        i = int(over.argmax())
        raise AssertionError(f"{what}: {float(g[i])!r} for {float(w[i])!r}, room {float(room[i])!r} "
                             f"({int((over > 0).sum())} of {over.numel()} are off)")


def rand(shape, dtype=torch.float32, seed=0, std=1.0, mean=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * std + mean).to(dtype).cuda()


def differences(f, x, direction, step):
    """Central difference of the scalar f along `direction` (numpy, fp64)."""
    x = np.asarray(x, dtype=np.float64)
    return (f(x + step * direction) - f(x - step * direction)) / (2 * step)
