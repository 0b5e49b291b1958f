"""Which batches of attention over the key-value cache are split: what a call's workspace shows (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest


class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("k_type", "v_type", "heads", "head_dim", "page_size", "pages")] + [("data", ctypes.c_void_p)]


@pytest.mark.parametrize("batch,slots,split", [(40, 704, False), (190, 704, False), (40, 896, False), (100, 1472, False),
                                               (40, 1600, True), (120, 2176, True), (300, 2944, True), (1000, 12800, True)])
def test_a_long_sequence_among_short_ones_is_split(qs, batch, slots, split):
    """Lengths are on the device: tables may be wide for one sequence of many. Such batches are whole segments, one to a
    workgroup and without a workspace, only where the longest is no great part of all."""
    cache = Cache(8, 8, 8, 128, 64, 1000, 256)      # nothing is read there
    need = qs.library().qs_kv_attention_workspace(ctypes.byref(cache), batch, 1, 32, slots // 64)
    assert need >= 0 and (need > 0) == split
