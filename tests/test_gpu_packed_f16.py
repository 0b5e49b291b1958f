"""Large products with a bf16 result, which take factors rounded to f16, against
a 64-bit computation."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, TORCH, make_adapters, rows_on

pytestmark = pytest.mark.gpu

F16 = 2.0 ** -11        # rounding of a factor


def bounds(x, w, wa, groups):
    """The product in 64 bits and how far a bf16 result may be off: both factors
    rounded to f16 (2^-11 each of the value), the f32 arithmetic as in linear64
    with every product added singly, the result's rounding. Values under 2^-39
    of their row's largest possible one (a row's power of two takes that to 2^15,
    f16 ends at 2^-24) round to a multiple of that."""
    y = x @ w.T
    size = x.abs() @ w.abs().T
    low = 2.0 ** -38 * (x.abs().amax(1, keepdim=True) * wa.sum(1)[None] + x.abs().sum(1, keepdim=True) * wa.amax(1)[None])
    return y, 2.01 * F16 * size + (32 * groups + 14) * ref.U * (x.abs() @ wa.T) + 64 * low + ref.ROUND["bf16"] * y.abs() + 1e-30


def check(got, y, bound, what):
    g = got.double()
    worst = ((g - y).abs() / bound).max().item()
    # as a whole: f16 adds (1/8)^2 twice to the square of the bf16 rounding's
    off, least = (g - y).norm().item(), (y.to(torch.bfloat16).double() - y).norm().item()
    print(f"{what}: worst error {worst:.3f} of its bound, {off / least:.3f} of the rounding's", flush=True)
    assert torch.isfinite(g).all() and worst <= 1.0 and off <= 1.1 * least, what


SHAPES = [(600, 3500), (140, 15100), (2100, 1030), (4200, 515), (131, 16400), (1000, 2300), (300, 7001)]


@pytest.mark.parametrize("i,qtype", list(enumerate(sorted(ref.BYTES))))
def test_every_format(qs, i, qtype):
    t, n = SHAPES[i % len(SHAPES)]
    k = 1056 if ref.BLOCK[qtype] == 32 else 1024
    print(qtype, t, n, k, flush=True)
    packed = ref.random_packed(qtype, n, k, i)
    q, s = ref.random_rows(t, k, i)
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64(qtype, packed))
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)))
    check(y, *bounds(torch.from_numpy(ref.rows64(q, s)).to(DEV), w, wa, k // 32), f"{qtype} {t}x{n}x{k}")


@pytest.mark.parametrize("t,n,k", [(4096, 2560, 1024), (2049, 2561, 2560), (509, 2560, 2816), (1537, 9728, 1024), (250, 9728, 2560)])
def test_tiles(qs, t, n, k):
    """Sizes at which different tiles cost least, with columns and rows over."""
    print(t, n, k, flush=True)
    packed = ref.random_packed("q6_k", n, k, t)
    q, s = ref.random_rows(t, k, n)
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64("q6_k", packed))
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight("q6_k", torch.from_numpy(packed).to(DEV)))
    check(y, *bounds(torch.from_numpy(ref.rows64(q, s)).to(DEV), w, wa, k // 32), f"{t}x{n}x{k}")


def test_rows_of_any_size(qs):
    """Rows and weight rows from the smallest values to the largest the formats
    hold keep their own scale; zeros, NaN and infinities stay in their rows."""
    t, n, k = 600, 3600, 1024
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
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight("q8_0", torch.from_numpy(packed).to(DEV)))
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[4]).any()
    assert (y[2] == 0).all() and (y[5] == 0).all() and (y[6:, 2] == 0).all()
    keep = [0, 1] + list(range(6, t))
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64("q8_0", packed))
    want, bound = bounds(torch.from_numpy(ref.rows64(q[keep], s[keep])).to(DEV), w, wa, k // 32)
    assert ((y[keep].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,t,n,k", [("bf16", 700, 3100, 1024), ("f16", 700, 3100, 1024), ("bf16", 2049, 2560, 1280),
                                         ("f16", 140, 15100, 1056)])
def test_adapters(qs, dtype, t, n, k):
    """Packed sequences and mixed rows; ranks from 1 to 128."""
    qtype = "q4_0" if k % 256 else "q5_k"
    packed = ref.random_packed(qtype, n, k, t)
    q, s = ref.random_rows(t, k, 1)
    ranks = [128, 8, 40, 16, 64, 3, 1]
    made = make_adapters(ranks, n, k, TORCH[dtype], 3)
    bank = qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in made])
    rng = np.random.default_rng(t)
    ids = (np.searchsorted(np.sort(rng.integers(0, t, 9)), np.arange(t), side="right") % 8 - 1).astype(np.int32)
    ids[t // 2:t // 2 + 70] = rng.integers(-1, 9, 70)
    print(dtype, t, n, k, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)), adapters=bank,
                         ids=torch.from_numpy(ids).to(DEV))
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64(qtype, packed))
    want, bound = bounds(torch.from_numpy(ref.rows64(q, s)).to(DEV), w, wa, k // 32)
    delta, more = ref.adapters64(ref.rows64(q, s), [(a.double().numpy(), b.double().numpy(), c) for a, b, c in made], ids, n)
    delta, more = torch.from_numpy(delta).to(DEV), torch.from_numpy(more).to(DEV)
    check(y, want + delta, bound + more + ref.ROUND["bf16"] * delta.abs(), f"{dtype} {t}x{n}x{k}")
