"""The most tokens that the router and the rows' kernels take in one call: a
launch has 64 threads a token and fewer than 2^32 in all, workgroups that are
partly empty among them (CPU; the checks come before any launch)."""

import ctypes

import pytest

from cresso_amd import _native

MOST = (1 << 26) - 16
P = ctypes.c_void_p(256)   # never read


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.skip("library not built (python -m cresso_amd.build)")
    return _native.load()


def calls(lib):
    def route(tokens):
        d = _native.RouteDesc()
        for k, v in dict(weights=256, experts=256, order=256, places=256, offsets=256, logits_stride=1, tokens=tokens, num_experts=1,
                         top=1, scale=1.0).items():
            setattr(d, k, v)   # the logits are missing, which is found behind the sizes
        return ctypes.byref(d)

    return {
        "route": lambda t: lib.cresso_route_forward(route(t), P, 1 << 30, None),
        "route gradient": lambda t: lib.cresso_route_backward(route(t), P, P, None),
        "dispatch": lambda t: lib.cresso_dispatch_rows(None, 1, _native.F32, t, 1, 1, P, P, P, None),
        "combine": lambda t: lib.cresso_combine_rows(None, 1, _native.F32, t, 1, 1, P, P, None, P, None),
        "combine gradient": lambda t: lib.cresso_combine_backward(None, 1, None, 1, _native.F32, t, 1, 1, P, P, None, P, P, None),
    }


@pytest.mark.parametrize("name", ["route", "route gradient", "dispatch", "combine", "combine gradient"])
def test_most_tokens(lib, name):
    assert -(-MOST // 4) * 256 < 1 << 32 and -(-MOST // 16) * 1024 < 1 << 32 <= -(-(MOST + 1) // 16) * 1024
    call = calls(lib)[name]
    assert call(MOST) == -1 and "null" in lib.cresso_hip_last_error().decode()
    for tokens in (MOST + 1, MOST + 15, MOST + 16):
        assert call(tokens) == -3 and "more than one call takes" in lib.cresso_hip_last_error().decode()
