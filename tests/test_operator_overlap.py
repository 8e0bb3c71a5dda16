"""Where the gradient of the distillation loss may lie: in the logits' place or
apart from everything that is read.  The library's own check, on addresses
that are never read (every call is refused before a launch)."""

import ctypes

import pytest

from cresso_amd import _native

ROWS, VOCAB = 4, 32
ROW = 2 * VOCAB          # bytes of a bf16 row
AT = 1 << 20


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.skip("library not built (python -m cresso_amd.build)")
    return _native.load()


def desc(**k):
    d = _native.DistillDesc()
    given = dict(logits=AT, index=1 << 24, teacher=1 << 25, loss=1 << 26, stats=1 << 27, rows=ROWS, vocab=VOCAB, top=3, index_bytes=8,
                 temperature=1.0, mix=0.5, dtype=_native.BF16, teacher_dtype=_native.F32, logits_stride=VOCAB, index_stride=3,
                 teacher_stride=3, grad_stride=VOCAB)
    for name, v in {**given, **k}.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("what,k", [
    ("logits", dict(grad=AT + ROW)), ("logits", dict(grad=AT - ROW)), ("logits", dict(grad=AT + 2)), ("logits", dict(grad=AT - 2)),
    ("logits", dict(grad=AT, grad_stride=VOCAB + 8)), ("logits", dict(grad=AT, logits_stride=VOCAB + 8)),
    ("logits", dict(grad=AT + ROW * ROWS - 2)), ("logits", dict(grad=AT + ROW, grad_stride=3 * VOCAB, logits_stride=3 * VOCAB + 1)),
    ("logits", dict(grad=AT + ROW - 2, grad_stride=3 * VOCAB, logits_stride=3 * VOCAB)),
    ("logits", dict(grad=AT + 2 * ROW + 2, grad_stride=3 * VOCAB, logits_stride=3 * VOCAB)),
    ("teacher's indexes", dict(grad=(1 << 24) + 8)), ("teacher's logits", dict(grad=(1 << 25) - ROW)),
    ("labels", dict(grad=1 << 28, labels=(1 << 28) + 2 * ROW, label_bytes=4)), ("row weights", dict(grad=1 << 28, weights=(1 << 28) + 3 * ROW)),
    ("stats", dict(grad=1 << 27)),
])
def test_shared_memory_is_refused(lib, what, k):
    assert lib.cresso_distill_loss(ctypes.byref(desc(**k)), None) == -1
    text = lib.cresso_hip_last_error().decode()
    assert "overlaps" in text and what in text, text


def test_what_arrives_is_not_overwritten(lib):
    d = desc(grad=1 << 28, d_loss=(1 << 28) + 4, d_loss_stride=0)
    assert lib.cresso_distill_backward(ctypes.byref(d), None) == -1
    assert "gradient that arrives" in lib.cresso_hip_last_error().decode()
