"""Products with an 8-bit weight against 64-bit evaluations of the same rounded
numbers: the rounding itself bit for bit, sizes that are multiples of nothing,
few and many rows, types, strides, what is not finite, the gradient, refusals."""

import math

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
BLOCK = 128


def e4m3_64(q):
    """|q| <= 448 rounded to four significant bits (steps of 2^-9 below 2^-6), halves to even, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(q / step) * step


def rounded(x):
    """What the product multiplies in x's place, in 64 bits."""
    x = x.detach().double().cpu().clone()
    for k in range(0, x.shape[1], BLOCK):
        part = x[:, k:k + BLOCK]
        top = torch.where(torch.isfinite(part), part, torch.zeros_like(part)).abs().amax(1, keepdim=True)
        m, e = torch.frexp(top / 448.0)
        e = torch.where(m == 0.5, e - 1, e)   # the smallest e with top/448 <= 2^e
        unit = torch.where(top > 0, torch.exp2(e.double().clamp(min=-117.0)), 1.0)
        q = e4m3_64(part / unit)
        q = torch.where(unit == 2.0 ** 120, q.clamp(-240.0, 240.0), q)   # 256 * 2^120 is no fp32 number
        x[:, k:k + BLOCK] = torch.where(torch.isfinite(part), q * unit, torch.full_like(part, math.nan))
    return x


def weight64(values, scales):
    w = values.float().double().cpu()
    s = scales.double().cpu().repeat_interleave(BLOCK, 0)[:w.shape[0]].repeat_interleave(BLOCK, 1)[:, :w.shape[1]]
    return w * s


def make_weight(outer, inner, seed=1):
    w = rand((outer, inner), torch.float32, seed, 0.05) * torch.exp(rand((outer, 1), seed=seed + 1))
    return cresso_amd.quantize_blocks(w)


def chain(depth):
    """128 products in the matrix unit, a scale and an addition for each block of the depth, joins of a split depth."""
    return 128 + 2 * (depth // BLOCK + 1) + 16


def check(x, values, scales, grad=True):
    w = weight64(values, scales)
    leaf = x.detach().requires_grad_(grad)
    y = cresso_amd.block_product(leaf, values, scales)
    flat = x.reshape(-1, x.shape[-1])
    q = rounded(flat)
    close(y.reshape(-1, w.shape[0]), q @ w.t(), q.abs() @ w.t().abs(), chain(w.shape[1]), "product")
    if grad:
        d = rand(tuple(y.shape), x.dtype, 9)
        y.backward(d)
        assert leaf.grad.shape == x.shape and leaf.grad.dtype == x.dtype
        q = rounded(d.reshape(-1, w.shape[0]))
        close(leaf.grad.reshape(-1, w.shape[1]), q @ w, q.abs() @ w.abs(), chain(w.shape[0]), "gradient")
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,inner,outer", [
    (1, 1, 1), (1, 128, 128), (2, 16, 5), (3, 129, 127), (5, 1000, 300), (8, 2048, 640), (16, 512, 130), (17, 640, 256),
    (31, 257, 1025), (32, 384, 96), (33, 1001, 333), (64, 4096, 64), (65, 100, 4096), (127, 256, 256), (128, 128, 384),
    (129, 250, 515), (300, 384, 640), (513, 640, 1153),
])
def test_sizes(rows, inner, outer, dtype):
    announce(f"block_product {rows} x {inner} x {outer} {dtype}")
    values, scales = make_weight(outer, inner)
    check(rand((rows, inner), dtype, 4), values, scales)


def test_larger_products():
    announce("block_product larger")
    for rows, inner, outer in ((1000, 1024, 1536), (2048, 512, 2048), (20, 8192, 1024), (4, 1024, 16384)):
        values, scales = make_weight(outer, inner)
        check(rand((rows, inner), torch.bfloat16, 4), values, scales)


def test_rounding_is_exact():
    """One input at a time through a weight of ones and scales of powers of two: the rounded numbers themselves."""
    inner = 640
    values = torch.eye(inner).cuda().to(torch.float8_e4m3fn)
    blocks = -(-inner // BLOCK)
    scales = torch.ones(blocks, blocks).cuda()
    x = rand((200, inner), torch.float32, 5)
    x *= torch.exp2(torch.randint(-60, 60, (200, blocks)).repeat_interleave(BLOCK, 1)[:, :inner].float()).cuda()
    x[0], x[1, :128], x[2, :128] = 0.0, 448.0, 448.0001
    x[3, :128] = 1e-44
    x[4, :128] = torch.arange(128).cuda() * 2.0 ** -10   # ties and subnormals
    x[4, 0] = 448.0
    x[5, :128] = torch.finfo(torch.float32).max
    y = cresso_amd.block_product(x, values, scales)
    want = rounded(x)
    want[3] = torch.where(want[3].abs() < 2.0 ** -126, y[3].double().cpu(), want[3])   # results below the normal numbers
    assert torch.equal(y.double().cpu(), want)
    for dtype in (torch.bfloat16, torch.float16):
        xs = x[6:].clamp(-6e4, 6e4).to(dtype)
        assert torch.equal(cresso_amd.block_product(xs, values, scales).double().cpu(), rounded(xs).to(dtype).double())


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_to_blocks(dtype):
    for rows, cols in ((1, 1), (130, 257), (128, 256), (300, 100)):
        w = rand((rows, cols), dtype, 6)
        if cols > 200:
            w[:128, 128:256] = 0.0
        values, scales = cresso_amd.quantize_blocks(w)
        w64 = w.double().cpu()
        for i in range(scales.shape[0]):
            for j in range(scales.shape[1]):
                part = w.float().cpu()[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK]
                top = part.abs().max()
                s = top / 448.0 if top > 0 else torch.tensor(1.0)
                assert scales[i, j].cpu() == s
                want = (part / s).clamp(-448, 448).to(torch.float8_e4m3fn)
                got = values[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK].cpu()
                assert torch.equal(got.float(), want.float())
        # a value is off by a sixteenth of itself, or half of the smallest step of its block's scale
        assert ((weight64(values, scales) - w64).abs() <= w64.abs() / 16 * (1 + 1e-6) + float(scales.max()) * 2.0 ** -10).all()
    bad = rand((4, 4))
    bad[1, 2], bad[2, 3] = math.inf, math.nan
    values, scales = cresso_amd.quantize_blocks(bad)
    assert torch.equal(torch.isnan(values.float()), ~torch.isfinite(bad)) and torch.isfinite(scales).all()
    wide = rand((50, 300), dtype, 7)
    a, b = cresso_amd.quantize_blocks(wide[:, 17:217]), cresso_amd.quantize_blocks(wide[:, 17:217].contiguous())
    assert torch.equal(a[0].float(), b[0].float()) and torch.equal(a[1], b[1])


def test_any_scales():
    values, scales = make_weight(300, 400)
    scales.copy_(torch.randn(scales.shape) * 10.0 ** torch.randint(-6, 6, scales.shape))   # of both signs
    scales[1, 2] = 0.0
    check(rand((40, 400), torch.float32, 8), values, scales)
    check(rand((3, 400), torch.float32, 8), values, scales)


@pytest.mark.parametrize("rows", [4, 200])
def test_what_is_not_finite(rows):
    values, scales = make_weight(160, 300)
    x = rand((rows, 300), torch.float32, 8)
    x[1, 7], x[2, 290], x[3] = math.inf, math.nan, 0.0
    y = check(x, values, scales, grad=False)
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[0]).all() and not y[3].any()
    values.view(torch.uint8)[5, 9] = 0x7F   # NaN
    y = cresso_amd.block_product(torch.ones(rows, 300).cuda(), values, scales)
    assert torch.isnan(y[:, 5]).all() and torch.isfinite(y[:, torch.arange(160) != 5]).all()


@pytest.mark.parametrize("rows", [3, 150])
def test_strides_and_shapes(rows):
    values, scales = make_weight(257, 333)
    x = rand((rows, 400), torch.bfloat16, 3)[:, 11:344]
    want = cresso_amd.block_product(x.contiguous(), values, scales)
    assert torch.equal(cresso_amd.block_product(x, values, scales), want)
    wide = torch.zeros(257, 400, dtype=torch.float8_e4m3fn).cuda()
    wide.view(torch.uint8)[:] = 0x7F
    wide.view(torch.uint8)[:, 16:349] = values.view(torch.uint8)
    assert torch.equal(cresso_amd.block_product(x, wide[:, 16:349], scales), want)
    wide.view(torch.uint8)[:, 3:336] = values.view(torch.uint8)
    assert torch.equal(cresso_amd.block_product(x, wide[:, 3:336], scales), want)
    check(rand((rows, 2, 333), torch.float16, 3), values, scales)
    check(rand((333,), torch.float32, 3), values, scales)
    assert torch.equal(cresso_amd.block_product(x, values, scales.t().contiguous().t()), want)
    assert torch.equal(cresso_amd.block_product(x, values.t().contiguous().t(), scales), want)


def test_weights_whose_rows_end_inside_a_block():
    """Past the end of a row lies the next one's memory, which may hold NaN."""
    for inner in (16, 112, 144, 1000, 1008):
        held = torch.zeros(140, 1024, dtype=torch.float8_e4m3fn).cuda()
        held.view(torch.uint8)[:] = 0x7F
        values, scales = make_weight(140, inner)
        held.view(torch.uint8)[:, :inner] = values.view(torch.uint8)
        for rows in (2, 140):
            check(rand((rows, inner), torch.float32, 2), held[:, :inner], scales)


def test_shapes_without_elements():
    values, scales = make_weight(20, 30)
    assert cresso_amd.block_product(torch.zeros(0, 30).cuda(), values, scales).shape == (0, 20)
    none = torch.zeros(20, 0, dtype=torch.float8_e4m3fn).cuda()
    y = cresso_amd.block_product(torch.zeros(5, 0).cuda(), none, torch.zeros(1, 0).cuda())
    assert y.shape == (5, 20) and not y.any()
    assert cresso_amd.quantize_blocks(torch.zeros(0, 7).cuda())[1].shape == (0, 1)


def test_same_bits_on_another_stream():
    values, scales = make_weight(700, 900)
    for rows in (5, 400):
        x = rand((rows, 900), torch.bfloat16, 3)
        want = cresso_amd.block_product(x, values, scales)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = cresso_amd.block_product(x, values, scales)
        side.synchronize()
        assert torch.equal(want, got)


def test_gradient_against_differences():
    """The gradient is that of the product with x unrounded: along a direction, up to the rounding of what arrives."""
    values, scales = make_weight(200, 150)
    w = weight64(values, scales)
    d = torch.exp2(torch.randint(-2, 2, (6, 200)).float()).cuda()   # powers of two: rounded to themselves
    leaf = rand((6, 150), torch.float32, 3).requires_grad_(True)
    cresso_amd.block_product(leaf, values, scales).backward(d)
    direction = torch.randn(6, 150, dtype=torch.float64)
    base = leaf.detach().double().cpu()
    value = lambda x: float(((x @ w.t()) * d.double().cpu()).sum())   # noqa: E731
    slope = (value(base + direction) - value(base - direction)) / 2
    got = float((leaf.grad.double().cpu() * direction).sum())
    assert abs(got - slope) <= chain(200) * 2.0 ** -24 * float((d.double().cpu() @ w.abs() * direction.abs()).sum())


def test_refusals():
    values, scales = make_weight(20, 30)
    x = rand((4, 30))
    cases = [
        ((x, values.float(), scales), "float8_e4m3fn"), ((x, values, scales.half()), "scales must be"),
        ((x, values, torch.ones(1, 2).cuda()), "scales must be"), ((x.double(), values, scales), "fp32, bf16 or fp16"),
        ((rand((4, 31)), values, scales), "30 inputs"), ((x, values[0], scales), r"\[outputs, inputs\]"),
    ]
    for args, msg in cases:
        with pytest.raises(ValueError, match=msg):
            cresso_amd.block_product(*args)
    with pytest.raises(ValueError, match=r"\[outputs, inputs\]"):
        cresso_amd.quantize_blocks(x[0])
    with pytest.raises(RuntimeError, match="GPU only"):
        cresso_amd.block_product(x, values.cpu(), scales)
