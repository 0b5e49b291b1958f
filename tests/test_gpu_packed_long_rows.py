"""A few rows that are too long for the dot products' place in LDS, or long
enough that tiles take them: with and without adapters, against a 64-bit
computation with the bounds of the other products' tests."""

from __future__ import annotations

import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, check, rows_on, run_adapters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qtype", ["q8_0", "q4_k", "iq2_s"])
@pytest.mark.parametrize("t,n,k", [(1, 40, 65536), (1, 33, 131072), (3, 70, 14592), (4, 70, 40960), (5, 2100, 4352), (8, 130, 4096),
                                   (8, 130, 14592), (7, 40, 65536)])
def test_long_rows(qs, qtype, t, n, k):
    print(qtype, t, n, k, flush=True)
    packed = ref.random_packed(qtype, n, k, 1)
    q, s = ref.random_rows(t, k, 2)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)), dtype=torch.float32)
    check(y, *ref.linear64(qtype, packed, q, s, "f32"), f"{qtype} {t}x{n}x{k}")
    run_adapters(qs, qtype, t, n, k, "bf16", "f32", [16, 5], [i % 3 - 1 if t > 1 else 1 for i in range(t)])
