"""The operators on packed weights refuse what they cannot compute, before any
device work (no GPU needed): the C ABI's checks and the Python ones."""

from __future__ import annotations

import ctypes

import pytest
import torch

P = ctypes.c_void_p


def norm(L, src=30, x=64, rows=2, k=64, stride=128, residual=None, rstride=0, weight=None, total=None, q=64, s=64):
    return L.qs_rms_norm_q8(src, P(x), rows, k, stride, P(residual), rstride, P(weight), 1e-6, P(total), P(q), P(s), None)


@pytest.mark.parametrize("bad,word", [
    (dict(src=5), b"source type"), (dict(rows=-1), b"rows"), (dict(k=48), b"multiple of 32"), (dict(k=0), b"multiple of 32"),
    (dict(k=1 << 18, stride=1 << 19), b"multiple of 32"), (dict(rows=1 << 40), b"2^34"), (dict(x=None), b"null"),
    (dict(q=None), b"null"), (dict(s=None), b"null"), (dict(total=64), b"needs a residual"), (dict(stride=120), b"row stride"),
    (dict(stride=64), b"row stride"), (dict(residual=64, rstride=100), b"row stride"), (dict(x=72), b"aligned"),
    (dict(weight=68), b"aligned"), (dict(q=68), b"aligned"), (dict(s=66), b"aligned"),
    (dict(rows=1 << 20, stride=1 << 50), b"2^62-byte span")])
def test_norm_refuses(qs, bad, word):
    L = qs.library()
    assert norm(L, **bad) == -22 and word in L.qs_last_error(), L.qs_last_error()


def test_norm_of_no_rows_is_no_work(qs):
    assert norm(qs.library(), rows=0, x=None, q=None, s=None) == 0


def test_values_refuses(qs):
    L = qs.library()
    assert L.qs_q8_values(P(64), P(64), 2, 64, 5, P(64), None) == -22 and b"destination type" in L.qs_last_error()
    assert L.qs_q8_values(P(64), P(64), 2, 40, 0, P(64), None) == -22
    assert L.qs_q8_values(P(64), P(64), -1, 64, 0, P(64), None) == -22
    assert L.qs_q8_values(P(None), P(64), 2, 64, 0, P(64), None) == -22
    assert L.qs_q8_values(P(64), P(64), 2, 64, 0, P(72), None) == -22
    assert L.qs_q8_values(P(64), P(64), 1 << 40, 64, 0, P(64), None) == -22
    assert L.qs_q8_values(P(None), P(None), 0, 64, 0, P(None), None) == 0


def linear(L, t=12, w=64, n=4, k=256, q=64, s=64, rows=2, dst=30, out=64, size=1 << 20, bank=None, ids=None, work=None, wsize=0):
    return L.qs_packed_linear(t, P(w), n, k, P(q), P(s), rows, dst, P(out), size, bank, P(ids), P(work), wsize, None)


@pytest.mark.parametrize("bad,word,code", [
    (dict(t=99), b"unknown ggml type", -95), (dict(dst=5), b"destination type", -22), (dict(n=-1), b"negative", -22),
    (dict(rows=-1), b"negative", -22), (dict(rows=(1 << 24) + 1), b"2^24", -22), (dict(k=255), b"row length", -22),
    (dict(k=0), b"row length", -22), (dict(k=128), b"row length", -22), (dict(n=1 << 40), b"2^34", -22),
    (dict(rows=1 << 23, k=1 << 20), b"2^34", -22), (dict(rows=1 << 23, n=1 << 12), b"2^34", -22),
    (dict(w=None), b"null", -22), (dict(out=None), b"null", -22), (dict(q=72), b"aligned", -22), (dict(w=65), b"aligned", -22),
    (dict(out=65), b"aligned", -22), (dict(size=15), b"dst holds", -22), (dict(ids=64), b"go together", -22)])
def test_linear_refuses(qs, bad, word, code):
    L = qs.library()
    assert linear(L, **bad) == code and word in L.qs_last_error(), L.qs_last_error()


def test_linear_of_nothing_is_no_work(qs):
    L = qs.library()
    assert linear(L, n=0, w=None, out=None) == 0 and linear(L, rows=0, q=None, s=None, out=None) == 0


def test_linear_refuses_adapters(qs):
    from importlib import import_module
    A = import_module("quant-studio_amd.packed")._Adapters
    L = qs.library()
    call = lambda ids=64, work=64, wsize=1 << 20, **f: linear(  # noqa: E731
        L, bank=ctypes.byref(A(*{**dict(count=2, type=30, max_rank=16, a=64, b=64, offsets=64, scales=64), **f}.values())),
        ids=ids, work=work, wsize=wsize)
    for bad, word in ((dict(ids=None), b"go together"), (dict(type=0), b"adapter type"), (dict(max_rank=12), b"multiple of 8"),
                      (dict(max_rank=8192), b"multiple of 8"), (dict(a=None), b"null adapter"), (dict(b=72), b"aligned"),
                      (dict(offsets=None), b"null adapter"), (dict(work=None), b"workspace"), (dict(wsize=100), b"workspace")):
        assert call(**bad) == -22 and word in L.qs_last_error(), (bad, L.qs_last_error())
    size = L.qs_packed_linear_workspace
    assert size(12, 4, 256, 10, 30, 16) >= 640 and size(12, 4, 256, 1, 30, 0) == 0 and size(12, 0, 256, 10, 30, 16) == 0
    assert size(12, 4, 256, -1, 30, 16) == -22 and size(12, 4, 256, 1, 30, 3) == -22 and size(12, 4, 256, 1, 5, 0) == -22
    assert size(99, 4, 256, 1, 30, 0) == -95 and size(12, 4, 100, 1, 30, 0) == -22


def test_python_refuses_what_it_can_see(qs):
    """Shapes and types; tensors that are not on a ROCm device."""
    x = torch.zeros((2, 64))
    with pytest.raises(ValueError, match="ROCm device"):
        qs.rms_norm_q8(x, torch.ones(64))
    with pytest.raises(ValueError, match="2-D"):
        qs.rms_norm_q8(x[0], torch.ones(64))
    with pytest.raises(ValueError, match="dtype"):
        qs.q8_rows(x.double())
    with pytest.raises(ValueError, match="int8"):
        qs.Q8Rows(x, x)
    with pytest.raises(ValueError, match="scale must be"):
        qs.Q8Rows(x.to(torch.int8), torch.ones((2, 3)))
    with pytest.raises(ValueError, match="ROCm device"):
        qs.Q8Rows(x.to(torch.int8), torch.ones((2, 2)))
    with pytest.raises(ValueError, match="unknown type"):
        qs.PackedWeight("q9_k", torch.zeros((2, 34), dtype=torch.uint8))
    with pytest.raises(ValueError, match="uint8"):
        qs.PackedWeight("q8_0", torch.zeros((2, 34)))
    with pytest.raises(ValueError, match="ROCm device"):
        qs.PackedWeight("q8_0", torch.zeros((2, 34), dtype=torch.uint8))
    with pytest.raises(ValueError, match="no adapters"):
        qs.AdapterBank([])
    with pytest.raises(ValueError, match="unsupported dtype"):
        qs.AdapterBank([(torch.zeros((8, 64)), torch.zeros((4, 8)), 1.0)])
