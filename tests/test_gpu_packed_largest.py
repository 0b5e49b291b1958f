"""Sizes at which one launch would have 2^32 threads or more."""

from __future__ import annotations

import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, check, rows_on

pytestmark = pytest.mark.gpu


def test_norm_of_2_26_short_rows(qs):
    """A wave to a row: 2^32 threads for 2^26 rows. Blocks of 2^20 rows repeat, so
    their results do."""
    base, k, times = 1 << 20, 32, 64
    x = torch.randn((base, k), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    weight = torch.linspace(0.5, 1.5, k, device=DEV)
    want, total = qs.rms_norm_q8(x, weight, residual=x)
    big = torch.cat([x.repeat(times, 1), x[:5]])
    print(tuple(big.shape), flush=True)
    rows, h = qs.rms_norm_q8(big, weight, residual=big)
    for i in range(times):
        at = slice(i * base, (i + 1) * base)
        assert torch.equal(rows.q[at], want.q) and torch.equal(rows.scale[at], want.scale) and torch.equal(h[at], total), i
    assert torch.equal(rows.q[times * base:], want.q[:5]) and torch.equal(h[times * base:], total[:5])
    assert torch.equal(rows.scale[times * base:], want.scale[:5])

@pytest.mark.parametrize("t", [9, 32])
def test_product_with_2_29_short_weight_rows(qs, t):
    """256 threads to 32 of them: 2^32 threads. Runs of 2^15 weight rows repeat."""
    base, k, times = 1 << 15, 32, 1 << 14
    part = ref.random_packed("q4_0", base, k, 3)
    q, s = ref.random_rows(t, k, t)
    rows, small = rows_on(qs, q, s), torch.from_numpy(part).to(DEV)
    want = qs.packed_linear(rows, qs.PackedWeight("q4_0", small))
    check(want, *ref.linear64("q4_0", part, q, s, "bf16"), "one run")
    print(t, base * times, flush=True)
    y = qs.packed_linear(rows, qs.PackedWeight("q4_0", small.repeat(times, 1))).view(t, times, base)
    for i in range(0, times, 1024):
        assert torch.equal(y[:, i:i + 1024], want[:, None].expand(t, 1024, base)), i
