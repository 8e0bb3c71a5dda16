"""Gradient norm and clipping against a 64-bit evaluation: types and mixtures of
them, odd sizes and addresses, more tensors than one launch describes, norms
that are not finite, outputs elsewhere, layouts, refusals, the optimizer's method."""

import math

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import EPS32, close, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def norm64(grads, norm_type=2.0):
    flat = torch.cat([g.detach().double().cpu().reshape(-1) for g in grads]) if grads else torch.zeros(1).double()
    if not flat.numel():
        return 0.0
    return float(flat.abs().max()) if math.isinf(norm_type) else float(flat.norm())


def check_norm(got, want):
    """fp64 sums (2^-40 covers any number of terms here), rounded to fp32 once."""
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got.double()) - want) <= (EPS32 + 2.0 ** -40) * want + 2.0 ** -150


def check_scaled(got, want, what):
    if got.dtype == torch.float64:
        assert torch.allclose(got.cpu(), want, rtol=1e-11, atol=0.0), what
    else:
        close(got, want, want.abs(), 1, what)   # fp32 once, then the type


def make(sizes, dtypes, seed=1, std=1.0):
    flat = [rand((n,), torch.float32, seed + i, std * 4.0 ** -(i % 5)) for i, n in enumerate(sizes)]
    return [t.to(dtypes[i % len(dtypes)]) for i, t in enumerate(flat)]


def check(grads, max_norm, norm_type=2.0, grad_scale=1.0, out_dtype=None):
    before = [g.double().cpu() for g in grads]
    norm = abs(grad_scale) * norm64(grads, norm_type)
    factor = grad_scale * (max_norm / norm if norm > max_norm and math.isfinite(norm) else 1.0)
    if out_dtype is None:
        version = [g._version for g in grads]
        got = cresso_amd.clip_gradients(grads, max_norm, norm_type=norm_type, grad_scale=grad_scale)
        to = grads
        assert all(g._version > v for g, v in zip(grads, version))
    else:
        to = [torch.full(g.shape, 7.0, dtype=g.dtype if out_dtype == "same" else out_dtype, device="cuda") for g in grads]
        got = cresso_amd.clip_gradients(grads, max_norm, norm_type=norm_type, grad_scale=grad_scale, out=to)
        assert all(torch.equal(g.double().cpu(), b) for g, b in zip(grads, before))
    check_norm(got, norm)
    for i, (t, b) in enumerate(zip(to, before)):
        check_scaled(t, b * factor, f"gradient {i} of {tuple(b.shape)}")
    return got


SIZES = [1, 3, 7, 8, 9, 255, 4095, 4096, 4097, 8191, 8192, 8193, 16383, 16384, 16385, 50001, 100000]


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
def test_types_and_sizes(dtype, norm_type):
    announce(f"clip {dtype} norm {norm_type}")
    for max_norm in (0.37, 1e9, 0.0):
        check(make(SIZES, [dtype]), max_norm, norm_type)
    check_norm(cresso_amd.gradient_norm(make(SIZES, [dtype]), norm_type), norm64(make(SIZES, [dtype]), norm_type))


@pytest.mark.parametrize("n", [1, 2, 159, 160, 161, 320, 500, 1000])
def test_numbers_of_tensors(n):
    announce(f"clip {n} tensors")
    sizes = [(i * 37) % 301 if i % 7 else 20000 + i for i in range(n)]   # some are empty
    check(make(sizes, DTYPES), 0.5)
    check([g for g in make(sizes, DTYPES[:3])], 0.5, grad_scale=-0.25, out_dtype=torch.float32)


def test_outputs():
    announce("clip outputs")
    check(make(SIZES, DTYPES), 0.2, out_dtype="same")
    check(make(SIZES, DTYPES), 1e9, out_dtype="same", grad_scale=2.0 ** -10)
    check(make(SIZES, [torch.bfloat16, torch.float16, torch.float32]), 0.2, out_dtype=torch.float32)
    grads = make([1000, 3000], [torch.float32])
    own = [grads[0], torch.empty_like(grads[1])]   # one in place, one elsewhere
    before, norm = [g.double().cpu() for g in grads], norm64(grads)
    check_norm(cresso_amd.clip_gradients(grads, 0.1, out=own), norm)
    assert torch.equal(grads[1].double().cpu(), before[1])
    for t, b in zip(own, before):
        check_scaled(t, b * (0.1 / norm), "mixed outputs")


def test_addresses():
    """Gradients packed one behind another, at every alignment of their element."""
    announce("clip packed gradients")
    for dtype in DTYPES:
        flat = rand((60000,), torch.float32, 3).to(dtype)
        grads = list(flat.split([1, 2, 3, 5, 17, 9000, 8192, 16384, 20000, 6396]))
        check(grads, 0.5)
        check(grads, 0.01, out_dtype="same")


def test_below_the_limit_nothing_is_written():
    announce("clip below the limit")
    g = rand((30000,), torch.float32, 2)
    g[5] = float.fromhex("0x1.fffffep-1")
    want = g.clone()
    norm = float(cresso_amd.clip_gradients(g, 1e4))
    assert torch.equal(g, want)
    for max_norm in (norm * 1.000001, math.inf):
        cresso_amd.clip_gradients(g, max_norm)
        assert torch.equal(g, want)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norms_that_are_not_finite(dtype, bad):
    announce(f"clip {dtype} with {bad}")
    for norm_type in (2.0, math.inf):
        grads = make([5000, 20000], [dtype])
        grads[1][12345] = bad
        want = [g.clone() for g in grads]
        norm = cresso_amd.clip_gradients(grads, 0.5, norm_type=norm_type)
        assert math.isnan(norm) if math.isnan(bad) else float(norm) == math.inf
        for g, w in zip(grads, want):
            assert torch.equal(torch.nan_to_num(g, nan=3.0), torch.nan_to_num(w, nan=3.0))


def test_extreme_numbers():
    """Squares that leave fp32's range do not leave fp64's."""
    announce("clip extreme numbers")
    for value in (1e-30, 1e-42, 3e38):
        grads = [torch.full((n,), value, device="cuda") for n in (1000, 3)]
        norm, max_norm = norm64(grads), value / 4
        check_norm(cresso_amd.gradient_norm(grads), min(norm, math.inf)) if norm < 3e38 else None
        want = [g.double().cpu() * (max_norm / norm) for g in grads]
        cresso_amd.clip_gradients(grads, max_norm)
        for g, w in zip(grads, want):
            close(g, w, w.abs(), 1, f"{value}")
    assert float(cresso_amd.gradient_norm(torch.full((1000,), 3e38, device="cuda"))) == math.inf   # above fp32


def test_layouts():
    announce("clip layouts")
    conv = rand((8, 6, 5, 3), torch.float32, 4).to(memory_format=torch.channels_last)
    turned = rand((300, 40), torch.bfloat16, 5).t()
    gaps = rand((50, 64), torch.float32, 6)[:, 3:50]
    grads = [conv, turned, gaps]
    check(grads, 0.25)
    check(grads, 0.05, out_dtype="same")   # row-major outputs of other strides
    whole = rand((50, 64), torch.float32, 6)
    cresso_amd.clip_gradients([whole[:, 3:50]], 0.25)
    assert torch.equal(whole[:, :3], rand((50, 64), torch.float32, 6)[:, :3])
    scalar = torch.tensor(3.0, device="cuda")
    check([scalar, rand((1, 1, 1), torch.float32, 1)], 0.5)


def test_nothing_to_clip():
    announce("clip nothing")
    assert float(cresso_amd.clip_gradients([], 1.0)) == 0.0
    assert float(cresso_amd.gradient_norm([None, torch.empty(0, device="cuda")])) == 0.0
    g = torch.zeros(100, device="cuda")
    assert float(cresso_amd.clip_gradients([g, None], 1.0)) == 0.0 and not g.any()


def test_same_result_on_every_run():
    announce("clip determinism")
    grads = make([300000] * 20, DTYPES)
    first = cresso_amd.gradient_norm(grads)
    for _ in range(5):
        assert torch.equal(cresso_amd.gradient_norm(grads), first)


def test_refusals():
    announce("clip refusals")
    g = rand((64,), torch.float32, 1)
    for grads in ([g, g], [g, g[8:]], [g[:33], g[32:]]):
        with pytest.raises(ValueError, match="belongs to two"):
            cresso_amd.clip_gradients(grads, 1.0)
        cresso_amd.gradient_norm(grads)   # reading is fine
    with pytest.raises(ValueError, match="belongs to two"):
        cresso_amd.clip_gradients([g[:32], g[32:]], 1.0, out=[g[32:], torch.empty(32, device="cuda")])
    with pytest.raises(ValueError, match="several elements"):
        cresso_amd.clip_gradients([torch.ones(1, device="cuda").expand(5)], 1.0)
    with pytest.raises(ValueError, match="its own type or"):
        cresso_amd.clip_gradients([g], 1.0, out=[g.double()])
    with pytest.raises(ValueError, match="outputs for"):
        cresso_amd.clip_gradients([g], 1.0, out=[])
    with pytest.raises(ValueError, match="no output"):
        cresso_amd.clip_gradients([g], 1.0, out=[None])
    with pytest.raises(ValueError, match="must be fp32"):
        cresso_amd.gradient_norm([torch.ones(3, dtype=torch.int32, device="cuda")])
    with pytest.raises(ValueError, match="sparse"):
        cresso_amd.gradient_norm([torch.eye(3, device="cuda").to_sparse()])
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            cresso_amd.clip_gradients([g], bad)
    for bad in (math.inf, math.nan):
        with pytest.raises(ValueError, match="grad_scale"):
            cresso_amd.clip_gradients([g], 1.0, grad_scale=bad)
    with pytest.raises(RuntimeError, match="GPU only"):
        cresso_amd.clip_gradients([g, torch.zeros(3)], 1.0)


def test_optimizer_clips_its_gradients():
    announce("CRESSO5.clip_gradients")
    params = [torch.nn.Parameter(rand(s, torch.float32, i, 0.05)) for i, s in enumerate([(256, 192), (4096, 16), (100,), (7,)])]
    opt = cresso_amd.CRESSO5([dict(params=params[:2]), dict(params=params[2:], lr=1e-3)], rank=4, hash_bins=64, cuda_ops="required")
    for step in range(3):
        for i, p in enumerate(params[:3]):   # one has no gradient
            p.grad = rand(tuple(p.shape), torch.float32, 10 * step + i)
        before = [p.grad.double().cpu() for p in params[:3]]
        norm = norm64([p.grad for p in params[:3]])
        check_norm(opt.clip_gradients(0.5), norm)
        for p, b in zip(params, before):
            check_scaled(p.grad, b * (0.5 / norm), "optimizer")
        opt.step()
    assert all(torch.isfinite(p).all() for p in params)


def test_graph():
    announce("clip in a graph")
    grads = make([100, 70000, 33], DTYPES)
    out = [torch.empty_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cresso_amd.clip_gradients(grads, 0.5, out=out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = cresso_amd.clip_gradients(grads, 0.5, out=out)
    for k in range(4):
        for j, g in enumerate(grads):
            g.copy_(rand((g.numel(),), torch.float32, 50 + 3 * k + j, 10.0 ** (k - 3)))
        graph.replay()
        torch.cuda.synchronize()
        other = [torch.empty_like(g) for g in grads]
        want = cresso_amd.clip_gradients(grads, 0.5, out=other)   # eager work between replays
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(out, other))
        check_norm(norm, norm64(grads))
