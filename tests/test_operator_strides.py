"""Strides that would lead outside the memory a caller names are refused by the
library's entry points (before any launch; the addresses are never read)."""

import ctypes

import pytest

from cresso_amd import _native

P = ctypes.c_void_p(256)
BF16, F32 = _native.BF16, _native.F32


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.skip("library not built (python -m cresso_amd.build)")
    return _native.load()


def refused(lib, rc, text):
    message = lib.cresso_hip_last_error().decode()
    assert rc == -1 and "stride" in message and text in message, (rc, message)


@pytest.mark.parametrize("turned", [0, 1])
@pytest.mark.parametrize("rows", [4, 200])
def test_block_product(lib, rows, turned):
    cols, depth = (300, 500) if not turned else (500, 300)

    def call(**k):
        a = dict(x=P, x_stride=depth, dtype=BF16, rows=rows, cols=cols, depth=depth, w=P, w_stride=500, scales=P, scale_stride=4,
                 turned=turned, out=P, ws=P, nbytes=0, stream=None)
        return lib.cresso_block_product(*{**a, **k}.values())

    for stride in (-1, 1, depth - 1, -depth):
        refused(lib, call(x_stride=stride), "of x below the depth")
    for stride in (-500, 0, 16, 499):
        refused(lib, call(w_stride=stride), "of a weight of 500 columns")
    for stride in (-4, 0, 3):
        refused(lib, call(scale_stride=stride), "of the scales of 500 columns")
    assert call() == -1 and "workspace" in lib.cresso_hip_last_error().decode()       # what is left to refuse
    assert call(x_stride=0) == -1 and "workspace" in lib.cresso_hip_last_error().decode()


def test_block_quantize(lib):
    for stride in (-30, 1, 29):
        refused(lib, lib.cresso_block_quantize(P, stride, F32, 4, 30, P, P, None), "below the width")


def test_embedding_gradient(lib):
    for stride in (-16, 1, 15):
        rc = lib.cresso_embedding_backward(P, 8, 4, P, stride, 9, 16, BF16, 1.0, P, P, 1 << 20, None)
        refused(lib, rc, "below the width")


@pytest.mark.parametrize("field,pointer,name", [("residual_stride", "residual", "residual"), ("update_stride", "update", "update"),
                                                ("gate_stride", "gate", "gate"), ("d_out_stride", "d_out", "gradient of out"),
                                                ("d_normed_stride", "d_normed", "gradient of normed")])
def test_residual_norm(lib, field, pointer, name):
    d = _native.ResidualNormDesc()
    given = dict(residual=256, update=256, pre=256, out=256, normed=256, stats=256, rows=4, width=8, rows_per_gate=2, eps=1e-6, scale=1.0,
                 residual_stride=8, update_stride=8, gate_stride=8, d_out_stride=8, d_normed_stride=8)
    for k, v in {**given, pointer: 256}.items():
        setattr(d, k, v)
    for stride in (-8, 1, 7):
        setattr(d, field, stride)
        refused(lib, lib.cresso_residual_norm_forward(ctypes.byref(d), None), f"of the {name} below the width")
        refused(lib, lib.cresso_residual_norm_backward(ctypes.byref(d), P, 1 << 20, None), f"of the {name} below the width")
        assert lib.cresso_residual_norm_backward_workspace_bytes(ctypes.byref(d)) == 0


@pytest.mark.parametrize("field,name", [("logits_stride", "logits"), ("index_stride", "teacher's indexes"),
                                        ("teacher_stride", "teacher's logits"), ("d_loss_stride", "gradient that arrives"),
                                        ("grad_stride", "gradient")])
def test_distill(lib, field, name):
    d = _native.DistillDesc()
    for k, v in dict(logits=256, index=1 << 20, teacher=1 << 21, loss=1 << 22, stats=1 << 23, d_loss=1 << 24, grad=1 << 25, rows=3, vocab=90,
                     top=5, index_bytes=4, temperature=1.0, mix=1.0, logits_stride=90, index_stride=5, teacher_stride=5, d_loss_stride=1,
                     grad_stride=90).items():
        setattr(d, k, v)
    for stride in (-90, -1) + (() if field == "d_loss_stride" else (1, 4)) + ((0, 89) if field == "grad_stride" else ()):
        setattr(d, field, stride)
        for fn in (lib.cresso_distill_loss, lib.cresso_distill_backward):
            refused(lib, fn(ctypes.byref(d), None), f"of the {name} below the width")
