"""Embedding lookup and its gradient against a 64-bit evaluation: types, id
types, odd widths, ids outside the table, words that fill most of the text,
more tokens than one tile of the sort holds, strides, refusals."""

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, rand

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make_ids(tokens, rows, kind, seed=1):
    gen = torch.Generator().manual_seed(seed)
    if kind == "same":
        return torch.full((tokens,), rows // 2)
    ids = torch.randint(0, max(rows, 1), (tokens,), generator=gen)
    if kind == "skewed":
        ids[torch.rand(tokens, generator=gen) < 0.6] = rows // 3
    if kind == "outside":
        ids[torch.rand(tokens, generator=gen) < 0.4] = -1
        ids[torch.rand(tokens, generator=gen) < 0.2] = rows
        ids[torch.rand(tokens, generator=gen) < 0.1] = -(2 ** 31)
    return ids


def chain(ids):
    """Additions on a gradient's way: within a chunk of 32, then over the chunks' sums by four waves."""
    most = int(torch.bincount(ids.clamp(min=0)).max()) if ids.numel() else 0
    return min(most, 32) + most // 128 + 8


def reference_grad(ids, grad, rows, scale):
    there = (ids >= 0) & (ids < rows)
    g = grad.double().cpu().reshape(-1, grad.shape[-1])[there]
    total = torch.zeros(rows, g.shape[1], dtype=torch.float64).index_add_(0, ids[there], g)
    terms = torch.zeros(rows, g.shape[1], dtype=torch.float64).index_add_(0, ids[there], g.abs())
    return total * scale, terms * abs(scale)


CASES = [  # tokens, rows, width, kind
    (1, 1, 1, "plain"), (1, 50, 8, "plain"), (7, 3, 5, "plain"), (33, 100, 64, "plain"), (64, 100, 65, "skewed"),
    (257, 1000, 1001, "outside"), (300, 17, 4096, "same"), (1500, 40000, 24, "skewed"), (5000, 700, 130, "outside"),
    (16384, 512, 36, "plain"), (16385, 513, 36, "skewed"), (40000, 300000, 12, "outside"), (50001, 3, 9, "same"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,rows,width,kind", CASES)
def test_lookup_and_gradient(tokens, rows, width, kind, dtype):
    announce(f"embedding {tokens} tokens of {rows} x {width} {kind} {dtype}")
    ids = make_ids(tokens, rows, kind)
    table, grad = rand((rows, width), dtype, 2), rand((tokens, width), dtype, 3)
    scale = 3.7
    gpu_ids = (ids if tokens % 2 else ids.clamp(min=-2).int()).cuda()
    w = table.clone().requires_grad_(True)
    out = cresso_amd.embedding(gpu_ids, w, scale=scale)
    there = ((ids >= 0) & (ids < rows)).unsqueeze(1)
    want = table.double().cpu()[ids.clamp(0, rows - 1)] * there * scale
    close(out, want, want.abs(), 2, "rows")
    out.backward(grad)
    want, terms = reference_grad(ids, grad, rows, scale)
    close(w.grad, want, terms, chain(ids[there.squeeze(1)]), "gradient")
    again = cresso_amd.embedding_grad(gpu_ids, grad, rows, scale)
    assert torch.equal(again, w.grad)   # the order of the sums is fixed


def test_shapes_without_elements():
    table = rand((10, 6))
    assert cresso_amd.embedding(torch.zeros(0, dtype=torch.int64).cuda(), table).shape == (0, 6)
    assert cresso_amd.embedding(torch.zeros(4, 0, dtype=torch.int32).cuda(), table).shape == (4, 0, 6)
    assert cresso_amd.embedding(torch.zeros(3, dtype=torch.int32).cuda(), rand((10, 0))).shape == (3, 0)
    none = cresso_amd.embedding(torch.tensor([0, 5]).cuda(), rand((0, 6)))   # every id is outside
    assert none.shape == (2, 6) and not none.any()
    g = cresso_amd.embedding_grad(torch.zeros(0, dtype=torch.int64).cuda(), rand((0, 6)), 10)
    assert g.shape == (10, 6) and not g.any()
    assert cresso_amd.embedding_grad(torch.tensor([0, 1]).cuda(), rand((2, 6)), 0).shape == (0, 6)


def test_outputs_are_written_whole():
    """No row is left as the allocator found it."""
    for rows, width in ((100, 7), (1000, 64), (33, 4100)):
        torch.full((rows, width), float("nan"), device="cuda")
        g = cresso_amd.embedding_grad(torch.tensor([1, 1, 30]).cuda(), torch.ones(3, width).cuda(), rows)
        assert torch.equal(g.sum(1).nonzero().flatten().cpu(), torch.tensor([1, 30]))


def test_strides_and_shapes():
    wide = rand((40, 100), torch.bfloat16, 4)
    table = wide[:, 3:60]   # rows at a stride, at an address that is no multiple of 16
    ids = make_ids(24, 40, "plain").reshape(4, 6)
    strided = ids.t().contiguous().t().cuda()
    out = cresso_amd.embedding(strided, table, scale=0.5)
    want = table.double().cpu()[ids] * 0.5
    close(out, want, want.abs(), 2)
    grad = rand((4, 6, 200), torch.bfloat16, 5)[..., 50:107]
    got = cresso_amd.embedding_grad(strided, grad, 40, 0.5)
    want, terms = reference_grad(ids.flatten(), grad.reshape(24, 57), 40, 0.5)
    close(got, want, terms, 32)
    flat = rand((24, 200), torch.bfloat16, 5)[:, 50:107]
    assert torch.equal(cresso_amd.embedding_grad(strided.reshape(24), flat, 40, 0.5),
                       cresso_amd.embedding_grad(strided.reshape(24), flat.contiguous(), 40, 0.5))
    t = rand((57, 40)).t()   # columns at a stride: copied
    want = t.double().cpu()[ids]
    close(cresso_amd.embedding(strided, t), want, want.abs(), 2)


def test_infinities_stay_in_their_rows():
    table = rand((9, 20))
    table[4] = float("inf")
    table[5] = float("nan")
    out = cresso_amd.embedding(torch.tensor([3, 4, 5, -1, 6]).cuda(), table)
    assert torch.isinf(out[1]).all() and torch.isnan(out[2]).all()
    assert torch.isfinite(out[[0, 3, 4]]).all()
    grad = torch.ones(5, 20).cuda()
    grad[3] = float("nan")   # a token outside the table
    grad[1] = float("inf")
    g = cresso_amd.embedding_grad(torch.tensor([3, 4, 5, -1, 6]).cuda(), grad, 9)
    assert torch.isinf(g[4]).all() and torch.isfinite(g[[0, 1, 2, 3, 5, 6, 7, 8]]).all()


def test_no_second_derivative():
    ids, table = torch.tensor([1, 2, 2]).cuda(), rand((5, 4)).requires_grad_(True)
    by = rand((3, 4)).requires_grad_(True)
    g, = torch.autograd.grad(cresso_amd.embedding(ids, table), table, by, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        g.sum().backward()


def test_another_stream():
    ids, table, grad = make_ids(5000, 300, "skewed").cuda(), rand((300, 256)), rand((5000, 256), seed=6)
    want_out, want = cresso_amd.embedding(ids, table), cresso_amd.embedding_grad(ids, grad, 300)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, g = cresso_amd.embedding(ids, table), cresso_amd.embedding_grad(ids, grad, 300)
    side.synchronize()
    assert torch.equal(out, want_out) and torch.equal(g, want)


def test_captured_in_a_graph():
    ids, grad = make_ids(20000, 300, "skewed").cuda(), rand((20000, 40), seed=6)
    cresso_amd.embedding_grad(ids, grad, 300)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = cresso_amd.embedding_grad(ids, grad, 300)
    for k in range(3):
        grad.copy_(rand((20000, 40), seed=7 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, cresso_amd.embedding_grad(ids, grad, 300))


def test_refusals():
    ids, table = torch.tensor([1, 2]).cuda(), rand((5, 4))
    with pytest.raises(ValueError, match="int32 or int64"):
        cresso_amd.embedding(ids.float(), table)
    with pytest.raises(ValueError, match=r"\[rows, width\]"):
        cresso_amd.embedding(ids, table[0])
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        cresso_amd.embedding(ids, table.double())
    with pytest.raises(RuntimeError, match="GPU only"):
        cresso_amd.embedding(ids.cpu(), table)
    with pytest.raises(ValueError, match="for ids of shape"):
        cresso_amd.embedding_grad(ids, rand((3, 4)), 5)
    with pytest.raises(ValueError, match="negative"):
        cresso_amd.embedding_grad(ids, rand((2, 4)), -1)
