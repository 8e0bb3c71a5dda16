"""CPU tests of the operators' contract: public names, refusals on the CPU, the
library's own checks of its arguments (all made before any launch)."""

import ctypes

import pytest
import torch

import cresso_amd
from cresso_amd import _native

NULL = None


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.skip("library not built (python -m cresso_amd.build)")
    return _native.load()


def test_public_names():
    for name in ("embedding", "embedding_grad", "residual_norm", "block_product", "quantize_blocks", "distill_loss",
                 "distill_loss_and_grad"):
        assert name in cresso_amd.__all__ and callable(getattr(cresso_amd, name)) and getattr(cresso_amd, name).__doc__


def test_no_cpu_path():
    x, ids = torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64)
    for fn, args in ((cresso_amd.embedding, (ids, x)), (cresso_amd.embedding_grad, (ids, x, 3)), (cresso_amd.residual_norm, (x,)),
                     (cresso_amd.distill_loss, (x, ids.view(2, 1), x[:, :1])),
                     (cresso_amd.distill_loss_and_grad, (x, ids.view(2, 1), x[:, :1])), (cresso_amd.quantize_blocks, (x,)),
                     (cresso_amd.block_product, (x, x.to(torch.float8_e4m3fn), torch.ones(1, 1)))):
        with pytest.raises(RuntimeError, match="GPU only"):
            fn(*args)
        with pytest.raises(ValueError, match="must be a tensor"):
            fn([1.0], *args[1:])


def refused(lib, rc, code, text):
    assert rc == code
    assert text in lib.cresso_hip_last_error().decode()


def test_embedding_arguments(lib):
    p, bf = ctypes.c_void_p(256), _native.BF16   # never read: the checks come first
    fwd = lambda **k: lib.cresso_embedding_forward(*{**dict(  # noqa: E731
        ids=p, size=8, tokens=4, table=p, rows=9, width=16, stride=16, dtype=bf, scale=1.0, out=p, stream=NULL), **k}.values())
    refused(lib, fwd(size=2), -1, "ids of 2 bytes")
    refused(lib, fwd(dtype=_native.F64), -3, "dtype 1")
    refused(lib, fwd(tokens=-1), -1, "negative")
    refused(lib, fwd(ids=NULL), -1, "null")
    refused(lib, fwd(out=NULL), -1, "null")
    refused(lib, fwd(stride=8), -1, "row stride")
    refused(lib, fwd(tokens=2 ** 40), -3, "more than one call takes")
    assert fwd(tokens=0) == 0 and fwd(width=0) == 0
    bwd = lambda **k: lib.cresso_embedding_backward(*{**dict(  # noqa: E731
        ids=p, size=8, tokens=4, grad=p, stride=16, rows=9, width=16, dtype=bf, scale=1.0, table=p, ws=p, nbytes=0,
        stream=NULL), **k}.values())
    need = lib.cresso_embedding_backward_workspace_bytes(4, 16, bf)
    assert need > 0 and lib.cresso_embedding_backward_workspace_bytes(4, 16, _native.F64) == 0
    refused(lib, bwd(nbytes=need - 1), -1, "workspace")
    refused(lib, bwd(nbytes=need, ws=NULL), -1, "workspace")
    refused(lib, bwd(nbytes=need, grad=NULL), -1, "null")
    assert bwd(rows=0) == 0


def test_residual_norm_arguments(lib):
    def desc(**k):
        d = _native.ResidualNormDesc()
        for name, v in {**dict(residual=256, update=256, out=256, rows=4, width=8, rows_per_gate=4, eps=1e-6, scale=1.0), **k}.items():
            setattr(d, name, v)
        return ctypes.byref(d)

    fwd, bwd = lib.cresso_residual_norm_forward, lib.cresso_residual_norm_backward
    refused(lib, fwd(NULL, NULL), -1, "null")
    refused(lib, fwd(desc(dtype=1), NULL), -3, "dtype 1")
    refused(lib, fwd(desc(width=0), NULL), -1, "width 0")
    refused(lib, fwd(desc(width=16385), NULL), -3, "above 16384")
    refused(lib, fwd(desc(residual=None), NULL), -1, "null")
    refused(lib, fwd(desc(out=None), NULL), -1, "null output")
    refused(lib, fwd(desc(pre=256), NULL), -1, "null output")
    refused(lib, fwd(desc(update=None, gate=256), NULL), -1, "not there")
    refused(lib, fwd(desc(gate=256, rows_per_gate=3), NULL), -1, "no multiple")
    refused(lib, fwd(desc(gate=256, act=7), NULL), -1, "unknown gate activation")
    refused(lib, fwd(desc(gate=256, gate_dtype=_native.BF16), NULL), -3, "gate of dtype")
    refused(lib, fwd(desc(eps=0.0), NULL), -1, "eps")
    assert fwd(desc(rows=0), NULL) == 0
    refused(lib, bwd(desc(post=256), NULL, 0, NULL), -1, "no stats")
    refused(lib, bwd(desc(stats=256, d_normed=256), NULL, 0, NULL), -1, "a gradient of a norm")
    refused(lib, bwd(desc(stats=256, d_gate=256), NULL, 0, NULL), -1, "an output for an input")
    need = lib.cresso_residual_norm_backward_workspace_bytes(desc())
    refused(lib, bwd(desc(stats=256), ctypes.c_void_p(256), need - 1, NULL), -1, "workspace")
    assert lib.cresso_residual_norm_backward_workspace_bytes(desc(width=0)) == 0


def test_distill_arguments(lib):
    def desc(**k):
        d = _native.DistillDesc()
        for name, v in {**dict(logits=256, index=256, teacher=256, loss=256, rows=2, vocab=9, top=3, index_bytes=4,
                               temperature=1.0, mix=1.0), **k}.items():
            setattr(d, name, v)
        return ctypes.byref(d)

    for fn in (lib.cresso_distill_loss, lib.cresso_distill_backward):
        refused(lib, fn(NULL, NULL), -1, "null")
        refused(lib, fn(desc(dtype=1), NULL), -3, "dtypes")
        refused(lib, fn(desc(vocab=0), NULL), -3, "logits")
        refused(lib, fn(desc(top=1025), NULL), -3, "at most 1024")
        refused(lib, fn(desc(index_bytes=2), NULL), -1, "4 or 8 bytes")
        refused(lib, fn(desc(labels=256), NULL), -1, "4 or 8 bytes")
        refused(lib, fn(desc(temperature=0.0), NULL), -1, "temperature")
        refused(lib, fn(desc(mix=-0.5), NULL), -1, "mix")
        refused(lib, fn(desc(teacher=None), NULL), -1, "null")
        assert fn(desc(rows=0), NULL) == 0
    refused(lib, lib.cresso_distill_loss(desc(loss=None), NULL), -1, "null")
    refused(lib, lib.cresso_distill_backward(desc(), NULL), -1, "null")


def test_block_product_arguments(lib):
    p = ctypes.c_void_p(256)
    call = lambda **k: lib.cresso_block_product(*{**dict(  # noqa: E731
        x=p, x_stride=32, dtype=_native.BF16, rows=4, cols=16, depth=32, w=p, w_stride=32, scales=p, scale_stride=1, turned=0,
        out=p, ws=p, nbytes=0, stream=NULL), **k}.values())
    need = lib.cresso_block_product_workspace_bytes(4, 16, 32, p, 32, 0)
    refused(lib, call(nbytes=need - 1), -1, "workspace")
    refused(lib, call(nbytes=need, out=NULL), -1, "null")
    refused(lib, call(nbytes=need, scales=NULL), -1, "null")
    refused(lib, call(dtype=1), -3, "dtype 1")
    refused(lib, call(rows=-1), -1, "negative")
    refused(lib, call(depth=2 ** 30), -3, "more than one call takes")
    assert call(rows=0) == 0 and call(cols=0) == 0
    refused(lib, lib.cresso_block_quantize(NULL, 4, 0, 4, 4, p, p, NULL), -1, "null")
    assert lib.cresso_block_quantize(NULL, 4, 0, 0, 4, p, p, NULL) == 0
