"""CPU tests of the contract of the experts' operators and of clipping: public
names, no CPU path, the library's own checks of its arguments (all made before
any launch)."""

import ctypes
import math

import pytest
import torch

import cresso_amd
from cresso_amd import _native

NULL = None
P = ctypes.c_void_p(256)   # never read: the checks come first
BF16, F32, F64 = _native.BF16, _native.F32, _native.F64


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.skip("library not built (python -m cresso_amd.build)")
    return _native.load()


def refused(lib, rc, code, text):
    assert rc == code
    assert text in lib.cresso_hip_last_error().decode()


def test_public_names():
    for name in ("route_experts", "dispatch_rows", "combine_rows", "expert_product", "gradient_norm", "clip_gradients"):
        assert name in cresso_amd.__all__ and callable(getattr(cresso_amd, name)) and getattr(cresso_amd, name).__doc__
    assert "Routing" in cresso_amd.__all__ and cresso_amd.Routing._fields == ("experts", "order", "places", "offsets")
    assert cresso_amd.CRESSO5.clip_gradients.__doc__


def test_no_cpu_path():
    if not _native.library_path().exists():
        pytest.skip("library not built")
    x, i = torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int32)
    r = cresso_amd.Routing(i, i.flatten(), i, i.flatten())
    for fn, args in ((cresso_amd.route_experts, (x, 2)), (cresso_amd.dispatch_rows, (x, r)), (cresso_amd.combine_rows, (x, r)),
                     (cresso_amd.expert_product, (x, torch.zeros(1, 3, 4), i.flatten())), (cresso_amd.gradient_norm, ([x],)),
                     (cresso_amd.clip_gradients, ([x], 1.0))):
        with pytest.raises(RuntimeError, match="GPU only"):
            fn(*args)
        with pytest.raises(ValueError, match="must be a tensor"):
            fn([1.0], *args[1:])


def test_python_refusals():
    for bad in (1.0, 3.0, "2", 0.5):
        with pytest.raises(ValueError, match="norm_type"):
            cresso_amd.gradient_norm([], bad)
    with pytest.raises(ValueError, match="score"):
        cresso_amd.route_experts(torch.zeros(2, 4), 1, score="tanh")


def grads(*entries):
    arr = (_native.GradDesc * len(entries))()
    for d, e in zip(arr, entries):
        for k, v in {**dict(grad=256, out=None, numel=10, dtype=F32, out_dtype=F32), **e}.items():
            setattr(d, k, v)
    return arr


def test_clip_arguments(lib):
    def clip(arr, count=None, kind=2, max_norm=1.0, scale=1.0, norm=P, ws=P, nbytes=1 << 20):
        return lib.cresso_clip_gradients(arr, len(arr) if count is None else count, kind, max_norm, scale, norm, ws, nbytes, NULL)

    one = grads({})
    refused(lib, clip(one, kind=1), -1, "unknown norm")
    refused(lib, clip(one, max_norm=-1.0), -1, "max_norm")
    refused(lib, clip(one, max_norm=math.nan), -1, "max_norm")
    refused(lib, clip(one, scale=math.inf), -1, "grad_scale")
    refused(lib, clip(one, norm=NULL), -1, "null norm")
    refused(lib, clip(one, count=-1), -1, "negative count")
    refused(lib, clip(None, count=2), -1, "null")
    refused(lib, clip(grads(dict(dtype=7))), -3, "dtype 7")
    refused(lib, clip(grads(dict(numel=-1))), -1, "negative size")
    refused(lib, clip(grads(dict(grad=None))), -1, "is null")
    refused(lib, clip(grads(dict(out=512, out_dtype=BF16))), -3, "to dtype")
    refused(lib, clip(grads(dict(out=512, dtype=F64, out_dtype=F32))), -3, "to dtype")
    refused(lib, clip(grads(dict(numel=1 << 50))), -3, "more elements")
    need = lib.cresso_clip_workspace_bytes(one, 1)
    assert need > 0 and lib.cresso_clip_workspace_bytes(grads(dict(dtype=9)), 1) == 0
    refused(lib, clip(one, nbytes=need - 1), -1, "workspace")
    refused(lib, clip(one, ws=NULL), -1, "workspace")
    refused(lib, clip(one, ws=ctypes.c_void_p(260)), -1, "workspace")


def route(**k):
    d = _native.RouteDesc()
    for name, v in {**dict(logits=256, weights=256, experts=256, order=256, places=256, offsets=256, logits_stride=8, tokens=100,
                           num_experts=8, top=2, scale=1.0), **k}.items():
        setattr(d, name, v)
    return ctypes.byref(d)


def test_route_arguments(lib):
    fwd = lambda d, ws=P, nbytes=1 << 20: lib.cresso_route_forward(d, ws, nbytes, NULL)   # noqa: E731
    bwd = lambda d, dw=P, dz=P: lib.cresso_route_backward(d, dw, dz, NULL)   # noqa: E731
    for fn in (fwd, bwd):
        refused(lib, fn(NULL), -1, "null")
        refused(lib, fn(route(dtype=F64)), -3, "dtype 1")
        refused(lib, fn(route(tokens=-1)), -1, "negative")
        refused(lib, fn(route(num_experts=0)), -3, "0 experts")
        refused(lib, fn(route(num_experts=1025)), -3, "1025 experts")
        refused(lib, fn(route(top=0)), -3, "top 0")
        refused(lib, fn(route(top=9)), -3, "top 9")
        refused(lib, fn(route(num_experts=64, top=33)), -3, "top 33")
        refused(lib, fn(route(tokens=1 << 30)), -3, "more than one call takes")
        refused(lib, fn(route(tokens=1 << 26, top=1)), -3, "more than one call takes")   # a launch has fewer than 2^32 threads
        refused(lib, fn(route(score=2)), -1, "unknown score")
        refused(lib, fn(route(scale=math.nan)), -1, "scale")
        refused(lib, fn(route(logits=None)), -1, "null")
        refused(lib, fn(route(logits_stride=7)), -1, "row stride")
    for field in ("weights", "experts", "order", "places", "offsets"):
        refused(lib, fwd(route(**{field: None})), -1, "null")
    need = lib.cresso_route_workspace_bytes(route())
    assert need > 0 and lib.cresso_route_workspace_bytes(route(top=0)) == 0
    refused(lib, fwd(route(), nbytes=need - 1), -1, "workspace")
    refused(lib, fwd(route(), ws=NULL), -1, "workspace")
    refused(lib, bwd(route(), dw=NULL), -1, "null")
    refused(lib, bwd(route(), dz=NULL), -1, "null")
    assert bwd(route(tokens=0)) == 0


def test_rows_arguments(lib):
    def dispatch(**k):
        a = {**dict(x=P, stride=16, dtype=BF16, tokens=4, top=2, width=16, experts=P, places=P, rows=P, stream=NULL), **k}
        return lib.cresso_dispatch_rows(*a.values())

    def combine(**k):
        a = {**dict(rows=P, stride=16, dtype=BF16, tokens=4, top=2, width=16, experts=P, places=P, weights=NULL, out=P, stream=NULL), **k}
        return lib.cresso_combine_rows(*a.values())

    def back(**k):
        a = {**dict(rows=P, stride=16, by=P, by_stride=16, dtype=BF16, tokens=4, top=2, width=16, experts=P, places=P, weights=NULL,
                    d_rows=P, d_weights=P, stream=NULL), **k}
        return lib.cresso_combine_backward(*a.values())

    for fn in (dispatch, combine, back):
        refused(lib, fn(dtype=F64), -3, "dtype 1")
        refused(lib, fn(tokens=-1), -1, "negative")
        refused(lib, fn(width=-1), -1, "negative")
        refused(lib, fn(top=0), -3, "0 experts")
        refused(lib, fn(top=33), -3, "33 experts")
        refused(lib, fn(tokens=1 << 30), -3, "more than one call takes")
        refused(lib, fn(tokens=1 << 26, top=1), -3, "more than one call takes")
        refused(lib, fn(experts=NULL), -1, "null")
        refused(lib, fn(places=NULL), -1, "null")
        refused(lib, fn(stride=15), -1, "row stride")
        assert fn(tokens=0) == 0
    refused(lib, dispatch(x=NULL), -1, "null")
    refused(lib, dispatch(rows=NULL), -1, "null")
    refused(lib, combine(rows=NULL), -1, "null")
    refused(lib, combine(out=NULL), -1, "null")
    refused(lib, back(by=NULL), -1, "null")
    refused(lib, back(rows=NULL), -1, "null")
    refused(lib, back(by_stride=3), -1, "row strides")
    assert back(d_rows=NULL, d_weights=NULL) == 0


def test_product_arguments(lib):
    def product(**k):
        a = {**dict(x=P, stride=32, dtype=BF16, rows=40, cols=16, depth=32, w=P, expert=512, w_stride=32, turned=0, experts=3, offsets=P,
                    out=P, ws=P, nbytes=1 << 24, stream=NULL), **k}
        return lib.cresso_expert_product(*a.values())

    def weight(**k):
        a = {**dict(p=P, p_stride=32, pw=32, q=P, q_stride=16, qw=16, dtype=BF16, rows=40, experts=3, offsets=P, out=P, ws=P,
                    nbytes=1 << 24, stream=NULL), **k}
        return lib.cresso_expert_product_weight(*a.values())

    for fn in (product, weight):
        refused(lib, fn(dtype=F64), -3, "dtype 1")
        refused(lib, fn(rows=-1), -1, "negative")
        refused(lib, fn(experts=-1), -1, "negative")
        refused(lib, fn(rows=1 << 31), -3, "more than one call takes")
        refused(lib, fn(experts=70000), -3, "more than one call takes")
        refused(lib, fn(offsets=NULL), -1, "null")
        refused(lib, fn(out=NULL), -1, "null")
        refused(lib, fn(ws=NULL), -1, "workspace")
        refused(lib, fn(ws=ctypes.c_void_p(264)), -1, "workspace")
        refused(lib, fn(nbytes=0), -1, "workspace")
    refused(lib, product(x=NULL), -1, "null")
    refused(lib, product(w=NULL), -1, "null")
    refused(lib, product(stride=31), -1, "row stride")
    refused(lib, product(w_stride=31), -1, "row stride")
    refused(lib, product(turned=1, w_stride=15), -1, "row stride")
    refused(lib, product(expert=-1), -1, "stride between experts")
    refused(lib, product(depth=1 << 23), -3, "more than one call takes")
    refused(lib, product(rows=1 << 30, cols=64, dtype=F32), -3, "more than one call takes")   # 2^25 tiles of 32 x 64
    refused(lib, product(rows=1 << 21, cols=1 << 15), -3, "more than one call takes")
    refused(lib, weight(experts=1 << 16, pw=1024, qw=1024, p_stride=1024, q_stride=1024), -3, "more than one call takes")
    refused(lib, weight(p=NULL), -1, "null")
    refused(lib, weight(q_stride=15), -1, "row strides")
    assert product(rows=0) == 0 and product(cols=0) == 0 and weight(experts=0) == 0 and weight(pw=0) == 0
    assert lib.cresso_expert_product_workspace_bytes(4, 4, 4, 2, F64) == 0
    assert lib.cresso_expert_product_weight_workspace_bytes(4, 4, 4, -1, BF16) == 0
