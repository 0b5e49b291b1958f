"""A bank of negative counts or ranks is no bank: refused, not left out (no GPU needed)."""

from __future__ import annotations

import ctypes
from importlib import import_module

import pytest

from test_packed_refusals import linear


@pytest.mark.parametrize("bad,word", [(dict(count=-1), b"count"), (dict(max_rank=-8), b"max_rank"),
                                      (dict(count=-1, max_rank=-8), b"count"), (dict(count=0, max_rank=-8), b"max_rank")])
def test_negative(qs, bad, word):
    A = import_module("quant-studio_amd.packed")._Adapters
    L = qs.library()
    bank = A(*{**dict(count=2, type=30, max_rank=16, a=64, b=64, offsets=64, scales=64), **bad}.values())
    # a workspace is needed and none given: were the bank left out, that would be refused, and nothing launched
    assert linear(L, bank=ctypes.byref(bank), ids=64, n=64, rows=40, k=2560) == -22
    assert word in L.qs_last_error(), L.qs_last_error()
