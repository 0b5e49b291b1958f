"""An infinite scale, of a row or of a block of the weight, stands for no values:
what it reaches is NaN, whichever way a product runs; nothing else changes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, rows_on

pytestmark = pytest.mark.gpu

# dot products, tiles, laid-out factors of exact codes and, with a bf16 result, of f16
PATHS = [(1, 40, "f32"), (7, 700, "bf16"), (40, 300, "f32"), (600, 400, "f32"), (900, 7010, "bf16")]


def run(qs, qtype, packed, q, s, dtype):
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)),
                         dtype=torch.float32 if dtype == "f32" else torch.bfloat16)
    return y.float().cpu().numpy()


@pytest.mark.parametrize("qtype", ["q8_0", "q4_k", "q6_k", "iq3_s"])
@pytest.mark.parametrize("t,n,dtype", PATHS)
def test_of_a_row(qs, qtype, t, n, dtype):
    k = 1024
    packed = ref.random_packed(qtype, n, k, 1)
    q, s = ref.random_rows(t, k, 2)
    q = np.maximum(np.abs(q), 1)        # no 0 to make a NaN of
    print(qtype, t, n, dtype, flush=True)
    clean = run(qs, qtype, packed, q, s, dtype)
    s[t // 2, 7] = np.inf
    if t > 3:
        s[0, 0], s[t - 1, 31] = -np.inf, np.inf
    y = run(qs, qtype, packed, q, s, dtype)
    hit = np.isinf(s).any(1)
    assert np.isnan(y[hit]).all()
    assert np.array_equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("qtype", sorted(ref.BYTES))
@pytest.mark.parametrize("t,n,dtype", PATHS)
def test_of_a_block(qs, qtype, t, n, dtype):
    """Each f16 field of a block in turn (d, and the minimum where there is one)."""
    k = 1024
    packed = ref.random_packed(qtype, n, k, 1)
    size, blocks = ref.BYTES[qtype], k // ref.BLOCK[qtype]
    q, s = ref.random_rows(t, k, 2)
    q = np.maximum(np.abs(q), 1)
    print(qtype, t, n, dtype, flush=True)
    clean = run(qs, qtype, packed, q, s, dtype)
    b = packed.reshape(n, blocks, size)
    hit = np.zeros(n, bool)
    at = {"q6_k": (208,), "q3_k": (108,), "q2_k": (80, 82), "q4_1": (0, 2), "q5_1": (0, 2), "q4_k": (0, 2),
          "q5_k": (0, 2)}.get(qtype, (0,))
    for i, place in enumerate(at):
        for row, block, value in ((3 + 4 * i, 0, np.inf), (n - 2 - 5 * i, blocks - 1, -np.inf), (n // 2 + i, blocks // 2, np.inf)):
            b[row, block, place:place + 2] = np.array([value], np.float16).view(np.uint8)
            hit[row] = True
    y = run(qs, qtype, packed, q, s, dtype)
    assert np.isnan(y[:, hit]).all()
    assert np.array_equal(y[:, ~hit], clean[:, ~hit])
