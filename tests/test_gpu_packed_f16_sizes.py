"""Products with a bf16 result from 3 * 2^31 multiplications up, which take f16
factors: every format, tiles and parts of the groups, adapters, rows of any size,
with the bounds of the other products of f16 factors."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref
from test_gpu_packed_f16 import bounds, check
from test_gpu_packed_linear import DEV, TORCH, make_adapters, rows_on

pytestmark = pytest.mark.gpu


def case(qs, qtype, t, n, k):
    packed = ref.random_packed(qtype, n, k, t)
    q, s = ref.random_rows(t, k, n)
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64(qtype, packed))
    weight = qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV))
    return q, s, weight, bounds(torch.from_numpy(ref.rows64(q, s)).to(DEV), w, wa, k // 32)


SHAPES = [(1900, 3500), (140, 44100), (6400, 1030), (131, 48100), (900, 7010), (300, 21500)]


@pytest.mark.parametrize("i,qtype", list(enumerate(sorted(ref.BYTES))))
def test_every_format(qs, i, qtype):
    t, n = SHAPES[i % len(SHAPES)]
    k = 1056 if ref.BLOCK[qtype] == 32 else 1024
    print(qtype, t, n, k, flush=True)
    q, s, w, want = case(qs, qtype, t, n, k)
    check(qs.packed_linear(rows_on(qs, q, s), w), *want, f"{qtype} {t}x{n}x{k}")


@pytest.mark.parametrize("t,n,k", [(509, 2560, 9728), (300, 2050, 10752), (1000, 1030, 7680), (250, 10000, 2560), (2049, 1281, 2816),
                                   (2329, 2497, 1280), (1054, 957, 6656)])
def test_tiles_and_parts(qs, t, n, k):
    """Long rows, whose groups are split over workgroups, in parts with a shorter last one."""
    print(t, n, k, flush=True)
    q, s, w, want = case(qs, "q3_k", t, n, k)
    rows = rows_on(qs, q, s)
    y = qs.packed_linear(rows, w)
    check(y, *want, f"{t}x{n}x{k}")
    assert torch.equal(qs.packed_linear(rows, w), y)


@pytest.mark.parametrize("dtype,t,n,k", [("bf16", 2000, 3300, 1024), ("f16", 700, 9300, 1024), ("bf16", 509, 2560, 9728),
                                         ("f16", 300, 2050, 10752), ("f16", 2049, 2560, 1280), ("bf16", 140, 4437, 14592)])
def test_adapters(qs, dtype, t, n, k):
    """Packed sequences and mixed rows; ranks from 1 to 128; a NaN stays in its adapter's rows."""
    q, s, w, (want, bound) = case(qs, "q4_k", t, n, k)
    made = make_adapters([128, 8, 40, 16, 64, 3, 1], n, k, TORCH[dtype], 3)
    rng = np.random.default_rng(t)
    ids = (np.searchsorted(np.sort(rng.integers(0, t, 9)), np.arange(t), side="right") % 8 - 1).astype(np.int32)
    ids[t // 2:t // 2 + 70] = rng.integers(-1, 9, 70)
    ids[7] = 7          # the bank's last adapter, of NaN
    poison = (torch.full((8, k), float("nan"), dtype=TORCH[dtype]), torch.zeros((n, 8), dtype=TORCH[dtype]), 1.0)
    bank = qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in made + [poison]])
    ids[(ids == 7) & (np.arange(t) != 7)] = -1
    print(dtype, t, n, k, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), w, adapters=bank, ids=torch.from_numpy(ids).to(DEV))
    delta, more = ref.adapters64(ref.rows64(q, s), [(a.double().numpy(), b.double().numpy(), c) for a, b, c in made], ids, n)
    delta, more = torch.from_numpy(delta).to(DEV), torch.from_numpy(more).to(DEV)
    assert torch.isnan(y[7]).all()
    keep = [i for i in range(t) if i != 7]
    check(y[keep], (want + delta)[keep], (bound + more + ref.ROUND["bf16"] * delta.abs())[keep], f"{dtype} {t}x{n}x{k}")


def test_rows_of_any_size(qs):
    """Rows and weight rows from the smallest values to the largest the formats
    hold keep their own scale; zeros, NaN and infinities stay in their rows."""
    t, n, k = 1900, 3600, 1024
    packed = ref.random_packed("q8_0", n, k, 7)
    blocks = packed.reshape(n, -1, 34)
    blocks[0, :, 0:2] = np.full((1,), 65504.0, np.float16).view(np.uint8)       # the largest d
    blocks[1, :, 0:2] = np.full((1,), 6e-8, np.float16).view(np.uint8)          # the smallest
    blocks[2, :, 0:2] = 0
    q, s = ref.random_rows(t, k, 8)
    s[0] *= np.float32(1e28)
    s[1] *= np.float32(1e-28)
    q[2] = 0
    s[3, 5] = np.nan
    s[4, 6] = np.inf
    s[5] = 0
    print(t, n, k, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight("q8_0", torch.from_numpy(packed).to(DEV)))
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[4]).any()
    assert (y[2] == 0).all() and (y[5] == 0).all() and (y[6:, 2] == 0).all()
    keep = [0, 1] + list(range(6, t))
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64("q8_0", packed))
    want, bound = bounds(torch.from_numpy(ref.rows64(q[keep], s[keep])).to(DEV), w, wa, k // 32)
    assert ((y[keep].double() - want).abs() <= bound).all()
