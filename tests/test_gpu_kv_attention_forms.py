"""Attention over the key-value cache in the forms that large batches and extreme scores take, against 64 bits:
workgroups of one wave with every type, head size and number of queries, and scores of which one takes all."""

from __future__ import annotations

import pytest
import torch

import kv_ref as ref
from kv_ref import DEV

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
TYPES = ["q8_0", "q4_0"]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def workspace(qs, cache, b, n, heads, m):
    return qs.library().qs_kv_attention_workspace(cache._ref, b, n, heads, m)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k_type", TYPES)
@pytest.mark.parametrize("v_type", TYPES)
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_a_wave_to_a_segment(qs, dtype, k_type, v_type, d):
    """4,800 heads of sequences are more than all waves that any form has at a time: a wave takes one after another,
    whole ones where tables are narrow, runs of all steps where they are wide. One query of a head and more than 8,
    more than 16 in columns of 8 or 16, several new tokens, and a window."""
    batch, heads, page = 100, 48, 32
    g = torch.Generator().manual_seed(d)
    lengths = torch.randint(0, 40, (batch,), generator=g).tolist()
    lengths[3], lengths[50], lengths[-1] = 200, 97, 0
    cache = qs.KVCache(sum(-(-n // page) for n in lengths) + 1, page, heads, d, k_type, v_type)
    tables, rows = ref.fill(qs, cache, lengths, dtype, d, poison=True)
    wide = torch.full((batch, 400), -1, dtype=torch.int32, device=DEV)
    wide[:, :tables.shape[1]] = tables
    for group, n, window in ((1, 1, 0), (2, 5, 7), (17, 1, 30)):
        q = torch.randn((batch, n, heads * group, d), generator=g).to(DEV, dtype)
        print(group, n, window, flush=True)
        want, far = ref.attention64(q, rows, None, window, 0.0, dtype == torch.float32)
        ys = []
        for table in (tables, wide):
            assert (workspace(qs, cache, batch, n, heads * group, table.shape[1]) > 0) == (table is wide)
            ys.append(qs.kv_attention(q, cache, table, ints(lengths), window=window))
            ref.check(ys[-1], want, far)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", [None, -0.02])
def test_a_score_that_takes_all(qs, dtype, kind, scale):
    """Queries so large that the best score is over 100 above the next, more than both can be off by: the result is
    that position's value, to the 21 bits of P, four roundings of f32 and the type's own."""
    cache = qs.KVCache(20, 16, 2, 128, kind, kind)
    tables, rows = ref.fill(qs, cache, [200, 50], dtype, 6, poison=True)
    g = torch.Generator().manual_seed(6)
    q = (torch.randn((2, 1, 12, 128), generator=g).clamp(-3, 3) * 2e4).to(DEV, dtype)
    y = qs.kv_attention(q, cache, tables, ints([200, 50]), scale=scale).cpu().double()
    checked = 0
    for i, (k, v) in enumerate(rows):
        for h in range(12):
            x = (128 ** -0.5 if scale is None else scale) * q[i, 0, h].cpu().double()
            s, a = k[:, h // 6] @ x, k[:, h // 6].abs() @ x.abs()
            off = 2 * (((128 + 8) * 2.0 ** -24 + 2.0 ** -22) * a.max() + 4 * 2.0 ** -24 * s.abs().max())
            best = s.argmax()
            if s[best] - s[s.topk(2).indices[1]] < 100 + off:
                continue
            want = v[best, h // 6]
            ref.check(y[i, 0, h], want, (2.0 ** -21 + 4 * 2.0 ** -24 + ref.HALF_STEP[dtype]) * 1.001 * want.abs() + 1e-30)
            checked += 1
    print(checked, "of 24 queries")
    assert checked >= 12


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("length", [131071, 500000])
def test_averages_of_long_sequences(qs, dtype, kind, length):
    """Scores that are nearly equal over a whole sequence; what is allowed is a small part of the result."""
    cache = qs.KVCache(-(-length // 1024), 1024, 1, 64, kind)
    g = torch.Generator().manual_seed(length)
    k, v = torch.randn((2, length, 1, 64), generator=g)
    v = (v.abs() + 0.1).to(DEV)
    k = (k * 1e-2).to(DEV)
    qs.kv_write(cache, k, v, torch.arange(length, dtype=torch.int32, device=DEV))
    rows = [(ref.values64(qs, kind, k), ref.values64(qs, kind, v))]
    q = torch.randn((1, 1, 3, 64), generator=g).to(DEV, dtype)
    y = qs.kv_attention(q, cache, torch.arange(cache.pages, dtype=torch.int32, device=DEV)[None], ints([length]))
    want, far = ref.attention64(q, rows, wide=dtype == torch.float32)
    assert (far < 4e-3 * want.abs()).all()
    ref.check(y, want, far)
