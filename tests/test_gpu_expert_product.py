"""Grouped products and their gradients against 64-bit products: types, sizes
that are no multiples of a tile, groups of any size, rows without an expert,
layouts of the weight, strides, numbers that are not finite, refusals."""

import math

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, differences, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def offsets_of(counts, first=0):
    return torch.tensor([first] + [first + sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32).cuda()


def check(rows, counts, inner, outer, dtype, first=0, turned=False, x=None, d=None, weight=None):
    """x W^T and both gradients; rows outside the groups hold NaN."""
    announce(f"expert_product {rows} rows {counts if len(counts) < 12 else len(counts)} {inner} -> {outer} {dtype}")
    offsets = offsets_of(counts, first)
    at = offsets.tolist()
    if x is None:
        x, d = rand((rows, inner), dtype, 1), rand((rows, outer), dtype, 2)
        for t in (x, d):
            t[:at[0]], t[at[-1]:] = math.nan, math.nan
    if weight is None:
        weight = rand((len(counts), outer, inner), dtype, 3, 0.5)
        if turned:
            weight = weight.transpose(1, 2).contiguous().transpose(1, 2)
    x, weight = x.detach().requires_grad_(True), weight.detach().requires_grad_(True)
    y = cresso_amd.expert_product(x, weight, offsets)
    assert y.shape == (rows, outer) and y.dtype == dtype
    dx, dw = torch.autograd.grad(y, (x, weight), d)
    assert dx.shape == x.shape and dw.shape == weight.shape and dx.dtype == dw.dtype == dtype
    want, want_dx, terms, terms_dx = (torch.zeros(rows, n, dtype=torch.float64, device="cuda") for n in (outer, inner, outer, inner))
    x64, w64, d64 = x.detach().double(), weight.detach().double(), d.double()
    for e in range(len(counts)):
        a, b = at[e], at[e + 1]
        want[a:b], terms[a:b] = x64[a:b] @ w64[e].t(), x64[a:b].abs() @ w64[e].abs().t()
        want_dx[a:b], terms_dx[a:b] = d64[a:b] @ w64[e], d64[a:b].abs() @ w64[e].abs()
        close(dw[e], d64[a:b].t() @ x64[a:b], d64[a:b].abs().t() @ x64[a:b].abs(), b - a + 16, f"weight gradient {e}")
    # an addition for each product, and joins where a sum is split
    close(y, want, terms, inner + 16, "product")
    close(dx, want_dx, terms_dx, outer + 16, "gradient")
    with torch.no_grad():
        assert torch.equal(cresso_amd.expert_product(x, weight, offsets), y)
    return y, dx, dw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,inner,outer", [
    ([1], 1, 1), ([1], 64, 64), ([3, 0, 2], 7, 5), ([0, 0, 1, 0], 33, 31), ([16], 128, 128), ([2, 2, 1, 3, 0, 4], 256, 96),
    ([15, 17, 16], 100, 130), ([64, 64], 64, 64), ([65, 63, 1], 128, 192), ([100, 5, 30], 1001, 257), ([130, 0, 128], 192, 320),
    ([300, 200], 72, 520), ([33] * 9, 129, 127), ([1] * 70, 40, 48), ([0] * 65 + [5] + [0] * 64, 24, 16), ([700, 1, 299], 384, 256),
])
def test_sizes(counts, inner, outer, dtype):
    check(sum(counts), counts, inner, outer, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_an_expert(dtype):
    check(100, [20, 0, 30], 72, 40, dtype, first=11)
    check(100, [0, 0], 64, 128, dtype, first=100)
    check(40, [0, 0, 0], 33, 17, dtype, first=0)
    check(300, [100, 50], 512, 256, dtype, first=0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_held_the_other_way_round(dtype):
    for counts, inner, outer in (([3, 5], 16, 24), ([70, 0, 130], 130, 72), ([300], 257, 129), ([200, 312], 256, 384)):
        weight = rand((len(counts), outer, inner), dtype, 3, 0.5)
        got = check(sum(counts), counts, inner, outer, dtype, turned=True)
        assert got[2].stride(1) == 1
        same = check(sum(counts), counts, inner, outer, dtype, weight=weight)
        assert same[2].is_contiguous()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_tiles(dtype):
    if dtype == torch.float32:
        check(1500, [700, 800], 520, 776, dtype)
        return
    check(5000, [2500, 100, 2400], 520, 1032, dtype)
    check(3000, [1000, 1, 1999], 1024, 512, dtype, turned=True)
    check(4100, [4100], 512, 1280, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,inner,outer,turned", [
    ([16640], 200, 1288, False),             # 330 tiles of 256: more than one to a workgroup, the rest in quarters
    ([8000, 0, 1, 9000, 3000], 136, 1544, True),
    ([130 + 3 * (e % 7) for e in range(48)], 1024, 1040, False),   # weight gradients of several tiles to a workgroup
    ([300, 0, 5, 700, 120, 260] * 9, 1032, 800, True),
])
def test_many_large_tiles(counts, inner, outer, turned, dtype):
    check(sum(counts) + 17, counts, inner, outer, dtype, first=5, turned=turned)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("inner", [64, 128, 192, 576])
def test_large_tiles_of_whole_pairs_of_stages(inner, dtype):
    """Depths of 64, of fewer stages than are on their way, and of an odd number of pairs; rows that begin within a cache line."""
    counts = [9000, 0, 300, 7300]
    check(16640, counts, inner, 1288, dtype, first=11)
    wide = rand((16640, inner + 24), dtype, 1)
    check(16640, counts, inner, 1288, dtype, first=11, x=wide[:, 8:8 + inner], d=rand((16640, 1288), dtype, 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,inner,outer,turned", [
    ([9000, 0, 300, 7300], 333, 1283, False),    # operands laid out anew, results in rows of any alignment
    ([9000, 0, 300, 7300], 1283, 333, False),
    ([9000, 0, 300, 7300], 1283, 333, True),
    ([9000, 0, 300, 7300], 336, 1283, True),     # one of the two sides is whole pieces
    ([130 + 3 * (e % 7) for e in range(48)], 1001, 1037, False),   # weight gradients of several large tiles to a workgroup
])
def test_large_products_of_odd_rows(counts, inner, outer, turned, dtype):
    check(sum(counts) + 17, counts, inner, outer, dtype, first=5, turned=turned)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_odd_rows_at_a_stride(dtype):
    """Slices of wider rows and of larger matrices: what lies beside them (NaN) is neither read nor written."""
    counts, inner, outer = [9000, 0, 300, 7300], 333, 1283
    offsets = offsets_of(counts)
    x, w, d = rand((16600, inner), dtype, 1), rand((4, outer, inner), dtype, 2, 0.5), rand((16600, outer), dtype, 3)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = cresso_amd.expert_product(a, b, offsets)
    want = [y, *torch.autograd.grad(y, (a, b), d)]
    wide, big, dwide = (torch.full(n, math.nan, dtype=dtype, device="cuda") for n in ((16600, inner + 9), (4, outer + 3, inner + 5), (16600, outer + 4)))
    wide[:, 3:3 + inner], big[:, 1:1 + outer, 2:2 + inner], dwide[:, 1:1 + outer] = x, w, d
    a, b = wide[:, 3:3 + inner].detach().requires_grad_(True), big[:, 1:1 + outer, 2:2 + inner].detach().requires_grad_(True)
    y = cresso_amd.expert_product(a, b, offsets)
    for got, exact in zip([y, *torch.autograd.grad(y, (a, b), dwide[:, 1:1 + outer])], want):
        assert torch.equal(got, exact)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_long_group(dtype):
    """A weight gradient whose sum is long and whose matrix is small."""
    check(9000, [4000, 5000], 64, 72, dtype)
    check(3000, [3000], 33, 20, dtype)


def test_strides():
    announce("expert_product strides")
    for dtype in DTYPES:
        offsets = offsets_of([30, 0, 34])
        wide, weight = rand((64, 200), dtype, 1), rand((3, 60, 130), dtype, 2)
        want = cresso_amd.expert_product(wide[:, 3:133].contiguous(), weight, offsets)
        assert torch.equal(cresso_amd.expert_product(wide[:, 3:133], weight, offsets), want)
        big = torch.full((3, 70, 140), math.nan, dtype=dtype, device="cuda")
        big[:, 4:64, 5:135] = weight
        assert torch.equal(cresso_amd.expert_product(wide[:, 3:133], big[:, 4:64, 5:135], offsets), want)
        odd = torch.full((3, 60, 260), math.nan, dtype=dtype, device="cuda")
        odd[:, :, ::2] = weight
        assert torch.equal(cresso_amd.expert_product(wide[:, 3:133], odd[:, :, ::2], offsets), want)
        shared = weight[:1].expand(3, 60, 130)   # one matrix for all experts
        assert torch.equal(cresso_amd.expert_product(wide[:, 3:133], shared, offsets),
                           cresso_amd.expert_product(wide[:, 3:133], shared.contiguous(), offsets))
        every = torch.zeros(8, dtype=torch.int32, device="cuda")
        every[::2] = offsets
        assert torch.equal(cresso_amd.expert_product(wide[:, 3:133], weight, every[::2]), want)
        x, w = wide[:, 3:133].detach().requires_grad_(True), big[:, 4:64, 5:135].detach().requires_grad_(True)
        d = rand((64, 100), dtype, 4)[:, 7:67]
        got = torch.autograd.grad(cresso_amd.expert_product(x, w, offsets), (x, w), d)
        x2, w2 = x.detach().contiguous().requires_grad_(True), weight.detach().requires_grad_(True)
        want = torch.autograd.grad(cresso_amd.expert_product(x2, w2, offsets), (x2, w2), d.contiguous())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner,outer", [(64, 64), (72, 100), (256, 320)])
def test_what_is_not_finite_stays_in_its_expert(inner, outer, dtype):
    announce(f"expert_product nan {inner} {outer} {dtype}")
    counts = [37, 70, 5]
    offsets = offsets_of(counts)
    x, weight, d = rand((112, inner), dtype, 1), rand((3, outer, inner), dtype, 2), rand((112, outer), dtype, 3)
    clean = [x.clone().requires_grad_(True), weight.clone().requires_grad_(True)]
    y0 = cresso_amd.expert_product(*clean, offsets)
    want = torch.autograd.grad(y0, clean, d)
    x[37:107], d[37:107], weight[1] = math.nan, math.inf, math.inf
    bad = [x.requires_grad_(True), weight.requires_grad_(True)]
    y = cresso_amd.expert_product(*bad, offsets)
    got = torch.autograd.grad(y, bad, d)
    keep = torch.ones(112, dtype=torch.bool)
    keep[37:107] = False
    assert torch.equal(y[keep.cuda()], y0[keep.cuda()]) and torch.isnan(y[37:107]).all()
    assert torch.equal(got[0][keep.cuda()], want[0][keep.cuda()])
    assert torch.equal(got[1][[0, 2]], want[1][[0, 2]]) and torch.isnan(got[1][1]).all()


def test_offsets_that_are_wrong_stay_within_the_rows():
    """Offsets are read from the GPU: whatever they hold, nothing outside the tensors is read or written."""
    announce("expert_product wrong offsets")
    x, w = rand((50, 64), torch.bfloat16, 1).requires_grad_(True), rand((3, 72, 64), torch.bfloat16, 2).requires_grad_(True)
    for bad in ([0, 20, 10, 50], [-5, 10, 70, 2 ** 31 - 1], [60, 40, 20, 0], [-2 ** 31, -7, -7, -1]):
        y = cresso_amd.expert_product(x, w, torch.tensor(bad, dtype=torch.int32).cuda())
        got = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert got[0].shape == x.shape and got[1].shape == w.shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("inner,outer", [(64, 2048), (2048, 64)])
def test_falling_offsets_take_no_more_tiles_than_others(inner, outer):
    """Groups that overlap would be ten times the work; the tiles are as many as of groups that do not, the largest ones too."""
    announce(f"expert_product falling offsets {inner} {outer}")
    x, w = rand((20000, inner), torch.bfloat16, 1).requires_grad_(True), rand((20, outer, inner), torch.bfloat16, 2, 0.1).requires_grad_(True)
    for bad in ([0, 20000] * 10 + [0], [20000] + [0, 2 ** 31 - 1] * 10, [*range(18000, -2000, -1000), 20000]):
        y = cresso_amd.expert_product(x, w, torch.tensor(bad, dtype=torch.int32).cuda())
        got = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert got[0].shape == x.shape and got[1].shape == w.shape
    torch.cuda.synchronize()


def test_one_matrix_for_all_experts():
    """A view that repeats one matrix takes the sum of the experts' gradients, as any view does."""
    announce("expert_product shared matrix")
    offsets = offsets_of([30, 0, 34])
    x, w, d = rand((64, 72), torch.float32, 1), rand((40, 72), torch.float32, 2), rand((64, 40), torch.float32, 3)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = cresso_amd.expert_product(a, b.expand(3, 40, 72), offsets)
    dx, dw = torch.autograd.grad(y, (a, b), d)
    x64, w64, d64 = x.double(), w.double(), d.double()
    close(y, x64 @ w64.t(), x64.abs() @ w64.abs().t(), 72 + 16, "product")
    close(dx, d64 @ w64, d64.abs() @ w64.abs(), 40 + 16, "gradient")
    close(dw, d64.t() @ x64, d64.abs().t() @ x64.abs(), 64 + 16 + 3, "weight gradient")


def test_nothing():
    announce("expert_product nothing")
    for rows, experts, outer, inner in ((0, 3, 5, 4), (6, 0, 5, 4), (6, 2, 0, 4), (6, 2, 5, 0)):
        x = rand((rows, inner), torch.bfloat16, 1).requires_grad_(True)
        w = rand((experts, outer, inner), torch.bfloat16, 2).requires_grad_(True)
        y = cresso_amd.expert_product(x, w, torch.linspace(0, rows, experts + 1).int().cuda())
        assert y.shape == (rows, outer) and not y.detach().any()
        y.sum().backward()
        assert x.grad.shape == x.shape and w.grad.shape == w.shape and not x.grad.any() and not w.grad.any()


def test_only_wanted_gradients():
    announce("expert_product wanted gradients")
    offsets = offsets_of([20, 13])
    x, w, d = rand((33, 48), torch.float32, 1), rand((2, 40, 48), torch.float32, 2), rand((33, 40), torch.float32, 3)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = torch.autograd.grad(cresso_amd.expert_product(a, b, offsets), (a, b), d)
    assert torch.equal(torch.autograd.grad(cresso_amd.expert_product(a, w, offsets), a, d)[0], want[0])
    assert torch.equal(torch.autograd.grad(cresso_amd.expert_product(x, b, offsets), b, d)[0], want[1])
    y = cresso_amd.expert_product(a, b, offsets)
    (again,) = torch.autograd.grad(y, a, d, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        again.sum().backward()


def test_gradient_against_differences():
    announce("expert_product differences")
    x, w, d = rand((9, 5), torch.float32, 1), rand((2, 4, 5), torch.float32, 2), rand((9, 4), torch.float32, 3)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(cresso_amd.expert_product(a, b, offsets_of([6, 2])), (a, b), d)
    d64 = d.double().cpu().numpy()
    x64, w64 = x.double().cpu().numpy(), w.double().cpu().numpy()
    f = lambda x, w: float(((x[:6] @ w[0].T) * d64[:6]).sum() + ((x[6:8] @ w[1].T) * d64[6:8]).sum())   # noqa: E731
    along_x, along_w = rand((9, 5), torch.float32, 5).double().cpu().numpy(), rand((2, 4, 5), torch.float32, 6).double().cpu().numpy()
    assert abs(float((dx.double().cpu().numpy() * along_x).sum()) - differences(lambda v: f(v, w64), x64, along_x, 1e-4)) <= 1e-4
    assert abs(float((dw.double().cpu().numpy() * along_w).sum()) - differences(lambda v: f(x64, v), w64, along_w, 1e-4)) <= 1e-4


def test_refusals():
    announce("expert_product refusals")
    x, w, o = rand((6, 4), torch.bfloat16, 1), rand((2, 3, 4), torch.bfloat16, 2), offsets_of([2, 4])
    for args, text in (((x, w[0], o), "weight must be"), ((x[:, :3], w, o), "x must be"), ((x.view(2, 3, 4), w, o), "x must be"),
                       ((x, w.float(), o), "weight is"), ((x, w, o.long()), "offsets must be"), ((x, w, o[:2]), "offsets must be"),
                       ((x.double(), w.double(), o), "fp32, bf16 or fp16")):
        with pytest.raises(ValueError, match=text):
            cresso_amd.expert_product(*args)
    with pytest.raises(RuntimeError, match="GPU only"):
        cresso_amd.expert_product(x, w, o.cpu())
