"""What a low-rank adapter adds, alone: on a weight of zeros, with one value in
each row of A and one in each row of B, a result is a product of four numbers,
so that what each path keeps of scale * A x shows in full."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, TORCH, rows_on

pytestmark = pytest.mark.gpu

# dot products; tiles whole, in parts and of 64 columns; laid-out factors in 64 x
# 64, in 128 x 128 by eight waves and by four, two planes, minima
PATHS = [("q8_0", 1, 33), ("q4_k", 8, 130), ("q8_0", 20, 70), ("q4_k", 64, 2100), ("q6_k", 300, 300), ("q8_0", 513, 300),
         ("q4_k", 1030, 2100), ("q6_k", 4000, 2060), ("q2_k", 150, 9000)]
K = 512


def zero_weight(qs, qtype, n):
    size = ref.BYTES[qtype] * (K // (32 if qtype == "q8_0" else 256))
    return qs.PackedWeight(qtype, torch.zeros((n, size), dtype=torch.uint8, device=DEV))


def picks(rng, n, ranks, dtype):
    """Adapters of one value a row: (A, B, scale), and where and what they are."""
    made, places = [], []
    for i, r in enumerate(ranks):
        a, b = torch.zeros((r, K)), torch.zeros((n, r))
        col, av = rng.permutation(K)[:r], rng.uniform(0.5, 2, r)
        rank, bv = rng.integers(0, r, n), rng.uniform(-2, 2, n)
        a[np.arange(r), col] = torch.from_numpy(av).float()
        b[np.arange(n), rank] = torch.from_numpy(bv).float()
        made.append((a.to(dtype), b.to(dtype), 0.3 * (i + 1)))
        places.append((col, rank))
    return made, places


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("qtype,t,n", PATHS)
def test_a_x_keeps_its_bits(qs, qtype, t, n, dtype):
    """An f32 result. Roundings of a term, relative: the row's scale and the
    adapter's (1 U each), B's product and the sums of its at most three pieces,
    U each, twice that where a matrix instruction cuts: 8; two more are allowed,
    and with f16 adapters the roundings of the pieces' common scale and the result's: 4."""
    rng = np.random.default_rng(t)
    made, places = picks(rng, n, [16, 5, 40], TORCH[dtype])
    q, s = ref.random_rows(t, K, 2)
    ids = (np.arange(t) % 4 - 1).astype(np.int32) if t > 1 else np.array([2], np.int32)
    bank = qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in made])
    print(qtype, t, n, dtype, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), zero_weight(qs, qtype, n), dtype=torch.float32, adapters=bank,
                         ids=torch.from_numpy(ids).to(DEV)).double().cpu().numpy()
    x, want = ref.rows64(q, s), np.zeros((t, n))
    for i, ((a, b, c), (col, rank)) in enumerate(zip(made, places)):
        a, b = a.double().numpy(), b.double().numpy()
        v = np.float64(np.float32(c)) * x[:, col] * a[np.arange(len(col)), col]
        want[ids == i] = (v[:, rank] * b[np.arange(n), rank])[ids == i]
    off = np.abs(y - want) / np.maximum(np.abs(want), 1e-30)
    print("off by", off.max() / ref.U, "of 2^-24")
    assert (off <= (10 if dtype == "bf16" else 14) * ref.U).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("qtype,t,n", PATHS)
def test_the_largest_and_infinite_a_x(qs, qtype, t, n, dtype):
    """A x that rounds to infinity in bf16 but is finite (its product with B is
    too), and one that overflows: an infinity of B's sign, on every path."""
    r = 8
    a, b = torch.zeros((r, K)), torch.full((n, r), 2.0 ** -4)
    a[0, 5], a[1, 70], a[2, 40] = 1.0, 100.0, 1.0
    b[n // 2:] *= -1
    bank = qs.AdapterBank([(a.to(DEV, TORCH[dtype]), b.to(DEV, TORCH[dtype]), 1.0)])
    q, s = np.zeros((t, K), np.int8), np.ones((t, K // 32), np.float32)
    q[:, 5] = 1
    s[0, 0] = 3.4e38                    # finite; over bf16's largest number
    if t > 2:
        s[1, 2], q[1, 70], q[1, 40] = 3e38, 1, 3        # times 100 over f32's, with finite ones beside it
        q[2, 5], q[2, 40] = 7, 1
    print(qtype, t, n, dtype, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), zero_weight(qs, qtype, n), dtype=torch.float32, adapters=bank,
                         ids=torch.zeros((t,), dtype=torch.int32, device=DEV)).cpu().numpy()
    sign = np.where(np.arange(n) < n // 2, 1.0, -1.0)
    assert (np.abs(y[0] / (sign * (np.float32(3.4e38) / 16)) - 1) <= 14 * ref.U).all()
    if t > 2:
        assert (y[1] == sign * np.inf).all()
        assert (y[2] == sign * 0.5).all() and (y[3:] == sign / 16).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("qtype,t,n", PATHS)
def test_all_bits_of_a_x(qs, qtype, t, n, dtype):
    """Scales of 24 bits times powers of two: every step is exact, and so is the result."""
    r, rng = 40, np.random.default_rng(t)
    a, b = torch.zeros((r, K)), torch.zeros((n, r))
    col, rank = rng.permutation(K)[:r], rng.integers(0, r, n)
    a[np.arange(r), col] = torch.from_numpy(2.0 ** rng.integers(-2, 3, r)).float()
    b[np.arange(n), rank] = torch.from_numpy(2.0 ** rng.integers(-2, 3, n) * rng.choice([-1, 1], n)).float()
    bank = qs.AdapterBank([(a.to(DEV, TORCH[dtype]), b.to(DEV, TORCH[dtype]), 0.5)])
    q = (2 ** rng.integers(0, 7, (t, K))).astype(np.int8)
    s = rng.uniform(0.5, 2, (t, K // 32)).astype(np.float32)
    print(qtype, t, n, dtype, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), zero_weight(qs, qtype, n), dtype=torch.float32, adapters=bank,
                         ids=torch.zeros((t,), dtype=torch.int32, device=DEV)).double().cpu().numpy()
    a, b = a.double().numpy(), b.double().numpy()
    want = 0.5 * (ref.rows64(q, s)[:, col] * a[np.arange(r), col])[:, rank] * b[np.arange(n), rank]
    assert np.array_equal(y, want)
