"""The exact form in the C ABI: a bit beside the destination type (no GPU needed)."""

from __future__ import annotations

import ctypes

from test_packed_refusals import linear

EXACT = 0x100


def test_exact_is_a_bit_of_the_destination_type(qs):
    L = qs.library()
    size = L.qs_packed_linear_workspace
    for dst in (0, 1, 30):
        assert size(12, 64, 256, 4, dst | EXACT, 0) == size(12, 64, 256, 4, dst, 0) >= 0
    # a large product with a bf16 result: the exact form's workspace is an f32 result's
    big = (12, 9728, 2560, 4096)
    assert size(*big, 30 | EXACT, 16) == size(*big, 0, 16) != size(*big, 30, 16)
    for bad in (5, 5 | EXACT, 0x200, 30 | 0x200, EXACT << 1, -1, -1 & ~EXACT):
        assert size(12, 64, 256, 4, bad, 0) == -22 and b"destination type" in L.qs_last_error(), bad
        assert linear(L, dst=bad) == -22 and b"destination type" in L.qs_last_error(), bad
    assert linear(L, dst=30 | EXACT, n=0, w=None, out=None) == 0
    assert linear(L, dst=30 | EXACT, size=15) == -22 and b"dst holds" in L.qs_last_error()
    assert linear(L, dst=0 | EXACT, out=66) == -22 and b"aligned" in L.qs_last_error()
    assert ctypes.c_int(30 | EXACT).value == 286
