"""What the attention over the key-value cache keeps of its factors: results against 64
bits, 16-bit ones to their own rounding and no more than f32 sums beside it."""

from __future__ import annotations

import math

import pytest
import torch

import kv_ref as ref
from kv_ref import DEV

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DIGITS = {torch.bfloat16: 8, torch.float16: 11, torch.float32: 24}


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def half_spacing(x, dtype):
    """Half the distance between neighbours of dtype at |x|: what its rounding may take, at most half of what eps says."""
    low = -14 if dtype == torch.float16 else -126
    return torch.exp2((torch.frexp(x.abs().clamp_min(2.0 ** low))[1] - DIGITS[dtype] - 1).double())


def bound(q, rows, scale=None, window=0, offset=0.0):
    """(y, how far off a result may be) as in ref.attention64 for f32 sums, and the type's own rounding."""
    want, far = ref.attention64(q.float(), rows, scale, window, offset, q.dtype == torch.float32)
    return want, far + half_spacing(want.abs() + far, q.dtype)


def held(qs, cache, k, v, dtype=torch.float32):
    """Writes rows to the cache's first slots: what it holds of them, f64, and the table of its pages."""
    qs.kv_write(cache, k.to(DEV, dtype), v.to(DEV, dtype), torch.arange(len(k), dtype=torch.int32, device=DEV))
    rows = ref.values64(qs, cache.k_type, k.to(DEV, dtype)), ref.values64(qs, cache.v_type, v.to(DEV, dtype))
    return [rows], torch.arange(cache.pages, dtype=torch.int32, device=DEV)[None]


U = 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,below", [("q8_0", 9), ("q4_0", 11)])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_small_terms_of_values_beside_large_ones(qs, dtype, kind, below, d):
    """Eight slots of each 32 have codes of +-1 whose steps are powers of two and cancel; the others' steps are 2^below
    smaller, of eleven bits. All scores are 0 and every sum, in any order, is a whole number of the smallest
    step under 2^24 of them, so that f32 sums are exact: what is left are four roundings of f32, and the type's own."""
    g = torch.Generator().manual_seed(d)
    heads, n, top = 8, 64, 127.0 if kind == "q8_0" else -8.0
    step = (1024 + torch.randint(0, 1024, (n, heads, 1, 1), generator=g)).float() / 1024 * 2.0 ** -below
    codes = torch.randint(-7, 8, (n, heads, d // 32, 32), generator=g).float()
    for i in range(0, n, 32):
        large = i + torch.randperm(32, generator=g)[:8]
        step[large] = 1.0
        codes[large] = torch.tensor([1.0, -1.0] * 4).view(8, 1, 1, 1)
    codes[..., 0] = top
    v = (codes * step).view(n, heads, d)
    cache = qs.KVCache(4, 16, heads, d, "q8_0", kind)
    rows, table = held(qs, cache, torch.zeros_like(v), v)
    assert torch.equal(rows[0][1], v.double())
    y = qs.kv_attention(torch.ones((1, 1, heads, d), dtype=dtype, device=DEV), cache, table, ints(n))
    want = v.double().mean(0)[None, None]
    ref.check(y, want, 4 * U * want.abs() + half_spacing(want, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,below", [("q8_0", 11), ("q4_0", 13)])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_small_terms_of_scores_beside_large_ones(qs, dtype, kind, below, d):
    """Eight values of a query are 1 and meet codes of +-1 that cancel, the others are 2^-below and of eight bits, which
    every type has: each block's sum is a whole number of the smallest under 2^24 of them, exact in f32. Then a
    score is off by its blocks' sum and three roundings, (d / 32 + 4) u of the sum of their magnitudes, and the
    rest is as in ref.attention64."""
    g = torch.Generator().manual_seed(d)
    heads, group, n = 4, 4, 45
    codes = torch.randint(-7, 8, (n, heads, d // 32, 32), generator=g).float()
    codes[..., 1:9] = torch.tensor([1.0, -1.0] * 4)
    codes[..., 0] = 127.0 if kind == "q8_0" else -8.0
    k = (codes * (1024 + torch.randint(0, 1024, (n, heads, d // 32, 1), generator=g)).float() / 1024).view(n, heads, d)
    q = (128 + torch.randint(0, 128, (heads * group, d // 32, 32), generator=g)).float() / 128 * 2.0 ** -below
    q[..., 1:9] = 1.0
    q[..., 0] = 0.0
    q = q.view(1, 1, heads * group, d)
    cache = qs.KVCache(3, 16, heads, d, kind, "q8_0")
    rows, table = held(qs, cache, k, torch.randn((n, heads, d), generator=g))
    assert torch.equal(rows[0][0], k.double())
    scale = 2.0 ** below / (4 * math.sqrt(d))
    y = qs.kv_attention(q.to(DEV, dtype), cache, table, ints(n), scale=scale)
    blocks = (rows[0][0].repeat_interleave(group, 1) * q[0].double()).view(n, heads * group, d // 32, 32).sum(3) * scale
    s, a, v = blocks.sum(2), blocks.abs().sum(2), rows[0][1].repeat_interleave(group, 1)
    e_s = (d // 32 + 4) * U * a.amax(0) + 4 * U * s.abs().amax(0)
    p = torch.softmax(s, 0)[..., None]
    want, size = (p * v).sum(0), (p * v.abs()).sum(0)
    far = (2 * (2 * e_s + 4 * U)[:, None] + 2.0 ** -21 + 2 * (2 + 96) * U) * size
    ref.check(y[0, 0], want, far + half_spacing(want.abs() + far, dtype))
