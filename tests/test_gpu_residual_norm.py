"""The seam between blocks and its gradient against 64-bit evaluations: every
combination of its parts, gates per channel, sequence and element, odd and
large widths, strides, mixed types, rows of zeros, refusals."""

import itertools

import numpy as np
import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

EPS = 1e-6
NAMES = ("residual", "update", "gate", "post", "pre", "scale")


def act64(kind, g):
    return torch.sigmoid(g) if kind == "sigmoid" else torch.tanh(g) if kind == "tanh" else g


def seam64(t, scale, kind, eps=EPS):
    """The formula in 64 bits; t: name -> fp64 tensor or None."""
    h, y, g, w1, w2 = (t[k] for k in NAMES[:5])
    s = t["scale"] if t["scale"] is not None else scale
    out = s * h
    if y is not None:
        if w1 is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w1
        out = out + (act64(kind, g) * y if g is not None else y)
    normed = None
    if w2 is not None:
        normed = out / torch.sqrt((out * out).mean(-1, keepdim=True) + eps) * w2
    return out, normed


def magnitudes(t, scale, kind, d_out, d_normed, eps=EPS):
    """What the results are sums of, as magnitudes: outputs, then gradients by name."""
    a = {k: None if v is None else v.detach().abs() for k, v in t.items()}
    h, y, w1, w2 = a["residual"], a["update"], a["post"], a["pre"]
    s = a["scale"] if a["scale"] is not None else abs(scale)
    one = torch.ones((), dtype=torch.float64)
    ga = act64(kind, t["gate"].detach()).abs() if t["gate"] is not None else one
    ry = one
    yn = torch.zeros_like(h)
    if y is not None:
        if w1 is not None:
            ry = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        yn = y * ry
    w1 = one if w1 is None else w1
    out = s * h + ga * yn * w1
    exact, _ = seam64({k: None if v is None else v.detach() for k, v in t.items()}, scale, kind, eps)
    rh = 1 / torch.sqrt((exact * exact).mean(-1, keepdim=True) + eps)
    w2 = torch.zeros((), dtype=torch.float64) if w2 is None else w2
    hn = out * rh
    e = (d_normed.abs() if d_normed is not None else 0.0) * w2
    d = (d_out.abs() if d_out is not None else 0.0) + rh * (e + hn * (e * hn).mean(-1, keepdim=True))
    d = d + torch.zeros_like(h)
    f = d * ga * w1
    grads = dict(residual=s * d, update=ry * (f + yn * (f * yn).mean(-1, keepdim=True)), gate=d * yn * w1,
                 post=d * ga * yn, pre=(d_normed.abs() if d_normed is not None else 0.0) * hn, scale=d * h)
    return out, hn * w2, grads


def reduce_to(x, shape):
    x = x + torch.zeros(())
    while x.ndim > len(shape):
        x = x.sum(0)
    for i, n in enumerate(shape):
        if n == 1 and x.shape[i] != 1:
            x = x.sum(i, keepdim=True)
    return x


def chain_of(width, rows):
    """Additions on the way: a row sum (16 elements in a lane, six lane steps, 16 waves) passes through a norm
    twice and more in the gradient; sums over rows add a worker's rows and then its share of the workers."""
    row = 16 + 6 + 16
    return 4 * row + 32, rows // 512 + 129 + 8


def run(shape, dtype, parts, kind="none", gate_shape=None, scale=1.0, vec_dtype=None, seed=0, outs="both", stride=0):
    vec = vec_dtype or dtype
    width = shape[-1]
    t = {k: None for k in NAMES}
    wide = rand((*shape[:-1], width + stride), dtype, seed, 2.0)
    t["residual"] = wide[..., stride:]
    if "u" in parts:
        t["update"] = rand(shape, dtype, seed + 1, 0.7)
    if "g" in parts:
        t["gate"] = rand(gate_shape or (width,), vec, seed + 2, 0.5, 0.3)
    if "1" in parts:
        t["post"] = rand((width,), vec, seed + 3, 0.2, 1.0)
    if "2" in parts:
        t["pre"] = rand((width,), vec, seed + 4, 0.2, 1.0)
    if "s" in parts:
        t["scale"] = rand((width,), vec, seed + 5, 0.1, 0.9)
    leaves = {k: v.detach().requires_grad_(True) if v is not None else None for k, v in t.items()}
    out, normed = cresso_amd.residual_norm(
        leaves["residual"], leaves["update"], gate=leaves["gate"], gate_act=kind, post_weight=leaves["post"],
        pre_weight=leaves["pre"], residual_scale=scale if t["scale"] is None else leaves["scale"], eps=EPS)
    assert (normed is None) == (t["pre"] is None)
    t64 = {k: None if v is None else v.detach().double().cpu().requires_grad_(True) for k, v in t.items()}
    want_out, want_normed = seam64(t64, scale, kind)
    d_out = rand(shape, dtype, seed + 6) if outs in ("both", "out") or normed is None else None
    d_normed = rand(shape, dtype, seed + 7) if normed is not None and outs in ("both", "normed") else None
    used = [(o, w, g) for o, w, g in ((out, want_out, d_out), (normed, want_normed, d_normed)) if g is not None]
    names = [k for k in NAMES if t[k] is not None]
    with torch.no_grad():
        m_out, m_normed, m = magnitudes(t64, scale, kind, None if d_out is None else d_out.double().cpu(),
                                        None if d_normed is None else d_normed.double().cpu())
    chain, column = chain_of(width, out.numel() // width)
    close(out, want_out, m_out, chain, "out")
    if normed is not None:
        close(normed, want_normed, m_normed, chain, "normed")
    got = torch.autograd.grad([o for o, _, _ in used], [leaves[k] for k in names], [g for _, _, g in used])
    want = torch.autograd.grad([w for _, w, _ in used], [t64[k] for k in names], [g.double().cpu() for _, _, g in used],
                               allow_unused=True)
    for k, a, b in zip(names, got, want):
        assert a.dtype == t[k].dtype
        b = torch.zeros_like(t64[k]) if b is None else b
        terms = reduce_to(m[k], t[k].shape)
        if k == "gate":   # the slope of the activation, at most 1
            terms = terms + b.detach().abs()
        close(a, b, terms, chain + (column if t[k].ndim < len(shape) or t[k].shape != shape else 0), "d_" + k)
    return out, normed


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("parts", ["", "2", "s2", "u", "u1", "ug", "ug1", "u12", "ug12s", "us2", "ug2"])
def test_every_combination_of_parts(parts):
    announce(f"residual_norm parts {parts!r}")
    for dtype, outs in itertools.product((torch.float32, torch.bfloat16), ("both", "out", "normed")):
        run((9, 130), dtype, parts, scale=0.75, outs=outs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (1, 4096), (5, 512), (4, 513), (600, 1000), (2, 1024), (33, 2047),
                                        (3, 4097), (7, 8192), (2, 16384), (2, 16383), (1500, 64)])
def test_sizes(rows, width, dtype):
    announce(f"residual_norm {rows} x {width} {dtype}")
    run((rows, width), dtype, "ug12s", kind="sigmoid", seed=rows)


@pytest.mark.parametrize("kind", ["none", "sigmoid", "tanh"])
@pytest.mark.parametrize("shape,gate", [((4, 300, 72), (4, 1, 72)), ((700, 2, 40), (700, 1, 40)), ((3, 5, 33), (3, 5, 33)),
                                        ((2, 900, 36), (2, 900, 36)), ((1, 1, 50), (1, 1, 50)), ((6, 7, 40), (40,)),
                                        ((2, 3, 1111, 24), (2, 3, 1, 24)), ((2, 600, 3, 24), (2, 1, 1, 24))])
def test_gates(shape, gate, kind):
    announce(f"residual_norm gate {gate} of {shape} {kind}")
    for dtype in (torch.float32, torch.bfloat16):
        run(shape, dtype, "ug12s", kind=kind, gate_shape=gate)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_vectors_in_fp32(dtype):
    announce(f"residual_norm fp32 vectors {dtype}")
    run((50, 515), dtype, "ug12s", kind="tanh", vec_dtype=torch.float32)
    run((10, 4, 515), dtype, "ug12s", gate_shape=(10, 1, 515), vec_dtype=torch.float32)


def test_rows_at_a_stride():
    for stride in (1, 3, 8):
        run((20, 200), torch.bfloat16, "ug12s", stride=stride)


def test_rows_of_zeros_and_large_numbers():
    h, y = torch.zeros(4, 100).cuda(), torch.zeros(4, 100).cuda()
    h[1], y[1] = 1e15, 1e15
    h[2], y[2] = 1e-20, 1e-20
    w = torch.ones(100).cuda()
    out, normed = cresso_amd.residual_norm(h, y, post_weight=w, pre_weight=w, eps=EPS)
    want_out, want = seam64(dict(residual=h.double().cpu(), update=y.double().cpu(), gate=None, post=w.double().cpu(),
                                 pre=w.double().cpu(), scale=None), 1.0, "none")
    close(out, want_out, want_out.abs(), 200)
    close(normed, want, want.abs(), 200)


def test_a_bad_row_spoils_no_other():
    h, y = rand((6, 300)), rand((6, 300), seed=1)
    h[2, 5], y[4, 7] = float("inf"), float("nan")
    w = torch.ones(300).cuda()
    out, normed = cresso_amd.residual_norm(h, y, post_weight=w, pre_weight=w)
    for r in (0, 1, 3, 5):
        assert torch.isfinite(out[r]).all() and torch.isfinite(normed[r]).all()
    assert torch.isnan(normed[2, 5]) and torch.isnan(out[4]).all()


def test_shapes_without_elements():
    h = torch.zeros(0, 64).cuda().requires_grad_(True)
    w = torch.ones(64).cuda().requires_grad_(True)
    out, normed = cresso_amd.residual_norm(h, pre_weight=w)
    assert out.shape == normed.shape == (0, 64)
    (out.sum() + normed.sum()).backward()
    assert w.grad.shape == (64,) and not w.grad.any()


def test_same_bits_again_and_on_another_stream():
    args = [rand((1000, 700), torch.bfloat16, k) for k in range(2)]
    vecs = [rand((700,), torch.bfloat16, 5 + k, 0.1, 1.0) for k in range(4)]

    def once():
        leaves = [t.detach().requires_grad_(True) for t in args + vecs]
        h, y, g, w1, w2, s = leaves
        out, normed = cresso_amd.residual_norm(h, y, gate=g, post_weight=w1, pre_weight=w2, residual_scale=s)
        return [out, normed, *torch.autograd.grad((out, normed), leaves, (args[1], args[0]))]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_gradient_against_differences():
    """The gradient of a scalar of both outputs along random directions, by central differences in 64 bits."""
    shape, kind = (3, 4, 40), "sigmoid"
    t = dict(residual=rand(shape, seed=1), update=rand(shape, seed=2), gate=rand((3, 1, 40), seed=3),
             post=rand((40,), seed=4, mean=1.0), pre=rand((40,), seed=5, mean=1.0), scale=rand((40,), seed=6, mean=1.0))
    a, b = rand(shape, seed=7), rand(shape, seed=8)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    out, normed = cresso_amd.residual_norm(leaves["residual"], leaves["update"], gate=leaves["gate"], gate_act=kind,
                                           post_weight=leaves["post"], pre_weight=leaves["pre"],
                                           residual_scale=leaves["scale"], eps=EPS)
    grads = torch.autograd.grad((out, normed), list(leaves.values()), (a, b))
    base = {k: v.detach().double().cpu() for k, v in t.items()}

    def value(k, x):
        o, n = seam64({**base, k: x}, 1.0, kind)
        return float((o * a.double().cpu()).sum() + (n * b.double().cpu()).sum())

    for k, g in zip(leaves, grads):
        direction = torch.from_numpy(np.random.RandomState(3).randn(*base[k].shape))
        step = 1e-5
        slope = (value(k, base[k] + step * direction) - value(k, base[k] - step * direction)) / (2 * step)
        got = float((g.double().cpu() * direction).sum())
        scale = float((g.double().cpu() * direction).abs().sum())
        # fp32 results, 1e-5 steps whose second-order term is 1e-10 of the third derivatives
        assert abs(got - slope) <= 2e-5 * scale, (k, got, slope)


def test_refusals():
    h, y, w = rand((4, 8)), rand((4, 8)), rand((8,))
    cases = [
        (dict(update=rand((4, 9))), "update is"), (dict(update=y.bfloat16()), "update is"), (dict(gate=w), "needs an update"),
        (dict(update=y, gate=rand((3, 8))), "gate of shape"), (dict(update=y, gate=rand((1, 1, 8))), "gate of shape"),
        (dict(update=y, gate=rand((4, 1))), "gate of shape"), (dict(update=y, gate_act="relu"), "gate_act"),
        (dict(pre_weight=rand((7,))), "pre_weight of shape"), (dict(pre_weight=w.half()), "must be fp32"),
        (dict(eps=0.0), "eps must be positive"), (dict(residual_scale=rand((1,))), "residual_scale of shape"),
    ]
    for kw, msg in cases:
        with pytest.raises(ValueError, match=msg):
            cresso_amd.residual_norm(h, **kw)
    with pytest.raises(ValueError, match="above 16384"):
        cresso_amd.residual_norm(torch.zeros(1, 16385).cuda())
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        cresso_amd.residual_norm(h.double())
    with pytest.raises(RuntimeError, match="GPU only"):
        cresso_amd.residual_norm(h, pre_weight=w.cpu())
