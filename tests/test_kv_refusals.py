"""The key-value cache refuses what it cannot hold or compute, before any device
work (no GPU needed): the C ABI's checks and the Python ones."""

from __future__ import annotations

import ctypes
from importlib import import_module

import pytest
import torch

P = ctypes.c_void_p


def cache(**f):
    C = import_module("quant-studio_amd.kv_cache")._Cache
    return ctypes.byref(C(*{**dict(k_type=8, v_type=2, heads=2, head_dim=64, page_size=16, pages=4, data=4096), **f}.values()))


BAD_CACHES = [(dict(k_type=12), b"cache types", -95), (dict(v_type=0), b"cache types", -95), (dict(heads=0), b"heads", -22),
              (dict(heads=1025), b"heads", -22), (dict(head_dim=96), b"head size", -22), (dict(head_dim=320), b"head size", -22),
              (dict(head_dim=0), b"head size", -22), (dict(page_size=8), b"power of two", -22), (dict(page_size=48), b"power of two", -22),
              (dict(page_size=2048), b"power of two", -22), (dict(pages=0), b"pages", -22), (dict(pages=-1), b"pages", -22),
              (dict(pages=1 << 27), b"2^31", -22), (dict(data=None), b"null", -22), (dict(data=4100), b"aligned", -22)]


def write(L, c, src=30, k=64, ks=256, v=64, vs=256, slots=64, rows=2):
    return L.qs_kv_write(c, src, P(k), ks, P(v), vs, P(slots), rows, None)


def read(L, c, slots=64, rows=2, dst=30, k=64, v=64):
    return L.qs_kv_read(c, P(slots), rows, dst, P(k), P(v), None)


def attention(L, c, t=30, q=64, qs=512, b=2, n=1, hq=4, tables=64, m=3, ts=3, lengths=64, window=0, out=64, size=1 << 20,
              work=1 << 20, wsize=1 << 40):
    return L.qs_kv_attention(c, t, P(q), qs, b, n, hq, P(tables), m, ts, P(lengths), 0.1, window, P(out), size, P(work), wsize, None)


@pytest.mark.parametrize("bad,word,code", BAD_CACHES)
def test_caches_that_cannot_be(qs, bad, word, code):
    L = qs.library()
    for call in (write, read, attention):
        assert call(L, cache(**bad)) == code and word in L.qs_last_error(), L.qs_last_error()
    assert L.qs_kv_attention_workspace(cache(**bad), 1, 1, 4, 1) == code
    for call in (write, read, attention):
        assert call(L, None) == -22 and b"null cache" in L.qs_last_error()


def test_page_bytes(qs):
    size = qs.library().qs_kv_page_bytes
    assert size(8, 8, 8, 128, 64) == 64 * 8 * 2 * (128 + 8) and size(8, 2, 1, 64, 16) == 16 * (64 + 32 + 8)
    assert size(8, 12, 1, 64, 16) == -95 and size(8, 8, 1, 80, 16) == -22 and size(8, 8, 0, 64, 16) == -22


@pytest.mark.parametrize("bad,word", [
    (dict(src=5), b"source type"), (dict(rows=-1), b"rows"), (dict(rows=(1 << 24) + 1), b"2^24"), (dict(k=None), b"null"),
    (dict(v=None), b"null"), (dict(slots=None), b"null"), (dict(k=72), b"aligned"), (dict(v=72), b"aligned"), (dict(slots=66), b"aligned"),
    (dict(ks=240), b"row stride"), (dict(vs=264), b"row stride"), (dict(vs=-256, rows=1), b"row stride"),
    (dict(ks=1 << 62), b"2^62-byte span")])
def test_write_refuses(qs, bad, word):
    L = qs.library()
    assert write(L, cache(), **bad) == -22 and word in L.qs_last_error(), L.qs_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(dst=5), b"destination type"), (dict(rows=-1), b"rows"), (dict(rows=(1 << 24) + 1), b"2^24"), (dict(k=None), b"null"),
    (dict(v=None), b"null"), (dict(slots=None), b"null"), (dict(k=72), b"aligned"), (dict(slots=66), b"aligned")])
def test_read_refuses(qs, bad, word):
    L = qs.library()
    assert read(L, cache(), **bad) == -22 and word in L.qs_last_error(), L.qs_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(t=5), b"query type"), (dict(b=-1), b"sequences"), (dict(b=(1 << 14) + 1), b"sequences"), (dict(n=17), b"new tokens"),
    (dict(n=-1), b"new tokens"), (dict(hq=3), b"query heads"), (dict(hq=0), b"query heads"), (dict(hq=258), b"query heads"),
    (dict(m=-1), b"tables"), (dict(m=1 << 27, ts=1 << 27), b"2^30"), (dict(b=1 << 12, m=1 << 20, ts=1 << 20), b"2^34"), (dict(window=-1), b"window"), (dict(q=None), b"null"),
    (dict(tables=None), b"null"), (dict(lengths=None), b"null"), (dict(out=None), b"null"), (dict(q=72), b"aligned"),
    (dict(out=72), b"aligned"), (dict(tables=66), b"aligned"), (dict(qs=496), b"token stride"), (dict(qs=520), b"token stride"),
    (dict(qs=1 << 62), b"2^62-byte span"), (dict(ts=2), b"table stride"), (dict(ts=1 << 60), b"2^62-byte span"), (dict(size=1023), b"out holds")])
def test_attention_refuses(qs, bad, word):
    L = qs.library()
    assert attention(L, cache(), **bad) == -22 and word in L.qs_last_error(), L.qs_last_error()


def test_attention_refuses_more_workgroups_than_a_launch_has(qs):
    L = qs.library()
    c = cache(heads=1024)
    assert attention(L, c, hq=4096, b=1 << 14, n=16, qs=1 << 20) == -22 and b"2^25" in L.qs_last_error()
    assert L.qs_kv_attention_workspace(c, 1 << 14, 16, 4096, 3) == -22
    assert L.qs_kv_attention_workspace(c, 1 << 14, 2, 4096, 3) == 0


def test_attention_refuses_workspaces(qs):
    L = qs.library()
    need = L.qs_kv_attention_workspace
    assert need(cache(), 2, 1, 4, 3) == 0 and need(cache(), 0, 1, 4, 300) == 0
    size = need(cache(), 2, 1, 4, 300)
    assert size > 0
    for bad in (dict(work=None), dict(work=(1 << 20) + 16), dict(wsize=size - 1)):
        assert attention(L, cache(), m=300, ts=300, **bad) == -22 and b"workspace" in L.qs_last_error()
    # a part of every workgroup's two segments and eight queries: not a multiple of the lengths
    assert need(cache(), 2, 1, 4, 1 << 20) == need(cache(), 2, 1, 4, 1 << 18) <= 1024 * 2 * 8 * (64 * 4 + 8) + 1024 * 16 + 1024


def test_nothing_is_no_work(qs):
    L, c = qs.library(), cache()
    assert write(L, c, rows=0, k=None, v=None, slots=None) == 0 and read(L, c, rows=0, k=None, v=None, slots=None) == 0
    assert attention(L, c, b=0, q=None, out=None, lengths=None) == 0 and attention(L, c, n=0, q=None, out=None, lengths=None) == 0


def test_python_refuses_what_it_can_see(qs):
    with pytest.raises(ValueError, match="unsupported type"):
        qs.KVCache(1, 16, 1, 64, "q4_k")
    for bad, word in (((1, 16, 1, 80), "head size"), ((1, 24, 1, 64), "power of two"), ((1, 16, 2000, 64), "heads")):
        with pytest.raises(qs.QuantSpecError, match=word):
            qs.KVCache(*bad)
    for bad in ((0, 16, 1, 64), (1, -16, 1, 64), (1 << 31, 16, 1, 64), (1 << 27, 16, 1, 64)):
        with pytest.raises(ValueError, match="2\\^31"):
            qs.KVCache(*bad)
    with pytest.raises(ValueError, match="contiguous uint8"):
        qs.KVCache(1, 16, 1, 64, data=torch.zeros((1, 100), dtype=torch.uint8))
    size = qs.library().qs_kv_page_bytes(8, 8, 1, 64, 16)
    with pytest.raises(ValueError, match="ROCm device"):
        qs.KVCache(1, 16, 1, 64, data=torch.zeros((1, size), dtype=torch.uint8))
