"""What a packed weight keeps between calls is bounded (no GPU needed)."""

from __future__ import annotations

import importlib


def weight_without_device(qs, name="q4_k", n=64, k=256):
    packed = importlib.import_module("quant-studio_amd.packed")
    packed._lib()
    w = object.__new__(qs.PackedWeight)
    w.name, w.ggml_type, w.n, w.k, w._work = name, int(qs.QUANT_TYPES[name].ggml_type), n, k, {}
    return packed, w


def test_workspace_sizes_of_many_row_counts(qs):
    """Prompts of every length: the sizes that a weight remembers stay few, and
    are the C ABI's."""
    packed, w = weight_without_device(qs)
    size = qs.library().qs_packed_linear_workspace
    for t in list(range(3000)) + [5, 2999, 5]:
        for rank in (0, 16):
            assert packed._workspace(w, t, 30, rank) == size(w.ggml_type, w.n, w.k, t, 30, rank)
    assert 0 < len(w._work) <= 256


def test_a_size_that_is_refused_is_not_remembered(qs):
    import pytest
    packed, w = weight_without_device(qs)
    with pytest.raises(qs.QuantSpecError, match="2\\^24"):
        packed._workspace(w, (1 << 24) + 1, 30, 0)
    assert not w._work
