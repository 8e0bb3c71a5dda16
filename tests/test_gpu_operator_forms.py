"""The operators at sizes that reach forms which small cases do not: large tiles
of a product with several blocks and ragged ends, more than 64 blocks of scales,
rows of 257 units and more in batches of 512 and more, lookups of four units a
thread, wide seams with several rows to a worker."""

import pytest
import torch

from gpu_util import announce, needs_gpu
from operator_util import close, rand
from test_gpu_block_product import BLOCK, chain, make_weight, rounded
from test_gpu_distill import check as check_distill, make as make_distill
from test_gpu_embedding import make_ids
from test_gpu_residual_norm import run as run_seam

import cresso_amd

pytestmark = [pytest.mark.gpu, needs_gpu]

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def check_product(rows, inner, outer, dtype, any_scales=False):
    """Product and gradient against 64-bit products (on the GPU, of the numbers rounded on the CPU)."""
    announce(f"block_product {rows} x {inner} x {outer} {dtype}")
    values, scales = make_weight(outer, inner)
    if any_scales:
        gen = torch.Generator().manual_seed(4)
        factor = 2.0 ** torch.randint(-8, 9, scales.shape, generator=gen).double() * (1 + torch.rand(scales.shape, generator=gen))
        factor *= torch.where(torch.rand(scales.shape, generator=gen) < 0.5, -1.0, 1.0)
        factor[torch.rand(scales.shape, generator=gen) < 0.05] = 0.0
        scales = (scales.double().cpu() * factor).float().cuda()
    w = values.float().double() * scales.double().repeat_interleave(BLOCK, 0)[:outer].repeat_interleave(BLOCK, 1)[:, :inner]
    x, d = rand((rows, inner), dtype, 3), rand((rows, outer), dtype, 9)
    leaf = x.detach().requires_grad_(True)
    y = cresso_amd.block_product(leaf, values, scales)
    q = rounded(x).cuda()
    close(y, q @ w.t(), q.abs() @ w.abs().t(), chain(inner), "product")
    y.backward(d)
    q = rounded(d).cuda()
    close(leaf.grad, q @ w, q.abs() @ w.abs(), chain(outer), "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,inner,outer", [(3900, 700, 4000), (3900, 4000, 700), (3841, 512, 3968), (4096, 4096, 256)])
def test_large_tiles(rows, inner, outer, dtype):
    """256 x 256 tiles of several blocks of k, forward or turned, the last tiles cut in m and n."""
    check_product(rows, inner, outer, dtype, any_scales=dtype == torch.float32)


@pytest.mark.parametrize("rows,inner,outer", [(5, 8400, 300), (5, 300, 16500), (40, 8400, 200), (40, 200, 16500), (1000, 8320, 1100),
                                              (1000, 1100, 8320), (2000, 8320, 1500), (2000, 1500, 8320), (3900, 8320, 4000),
                                              (3900, 4000, 8320)])
def test_more_blocks_than_a_wave_holds_scales(rows, inner, outer):
    check_product(rows, inner, outer, torch.bfloat16, any_scales=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(511, 2300), (512, 2300), (513, 4000), (1100, 4001), (1030, 600), (2050, 129)])
def test_batches_of_rows(rows, vocab, dtype):
    announce(f"distill {rows} x {vocab} {dtype}")
    z, index, a, lab = make_distill(rows, vocab, 5, dtype, seed=rows, absent=0.2)
    weights = torch.full((rows,), 0.25).cuda()
    weights[::11] = 0.0
    check_distill(z, index, a, lab, weights, 2.0, 0.6)
    check_distill(z, index, a, None, None, 1.3, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,width", [(16384, 523), (20001, 520), (300001, 33)])
def test_long_lookups(tokens, width, dtype):
    announce(f"embedding {tokens} x {width} {dtype}")
    ids = make_ids(tokens, 700, "outside")
    table = rand((700, width), dtype, 2)
    out = cresso_amd.embedding(ids.cuda(), table, scale=0.3)
    there = ((ids >= 0) & (ids < 700)).unsqueeze(1)
    want = table.double().cpu()[ids.clamp(0, 699)] * there * 0.3
    close(out, want, want.abs(), 2, "rows")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,gate", [((700, 5000), None), ((550, 2, 5000), (550, 1, 5000)), ((5, 140, 4101), (5, 1, 4101)),
                                        ((300, 2, 9001), (300, 1, 9001)), ((520, 8192), None), ((2, 260, 16384), (2, 1, 16384))])
def test_wide_seams_of_many_rows(shape, gate, dtype):
    announce(f"seam {shape} gate {gate} {dtype}")
    run_seam(shape, dtype, "ug12s", kind="sigmoid", gate_shape=gate)


@pytest.mark.parametrize("shape,gate", [((2100, 2, 96), (2100, 1, 96)), ((2600, 3, 2048), (2600, 1, 2048)), ((1300, 4096), (1300, 4096))])
def test_narrow_seams_of_several_gates_to_a_worker(shape, gate):
    announce(f"seam {shape} gate {gate}")
    run_seam(shape, torch.bfloat16, "ug12s", kind="tanh", gate_shape=gate)
