"""The caller's choice of exact codes for large products with a bf16 result
(exact=True), which otherwise take factors rounded to f16."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, TORCH, make_adapters, rows_on

pytestmark = pytest.mark.gpu


def bound_of_exact(x, w, wa, groups):
    """linear64's bound of a bf16 result, on the GPU."""
    y = x @ w.T
    return y, (groups + 14) * ref.U * (x.abs() @ wa.T) * 1.01 + ref.ROUND["bf16"] * y.abs() + 1e-30


@pytest.mark.parametrize("qtype,t,n,k,adapters", [
    ("q5_k", 509, 2560, 9728, None), ("q4_k", 2049, 2560, 1280, None), ("q2_k", 140, 46000, 1024, None),
    ("q8_0", 700, 9300, 1056, None), ("q6_k", 2047, 2560, 2560, "bf16"), ("q4_0", 900, 7010, 1056, "f16")])
def test_exact_codes(qs, qtype, t, n, k, adapters):
    """Rounded once: the f32 result's bits, rounded; within the bound of an
    exact product. Without `exact` the call takes f16 factors: other bits."""
    print(qtype, t, n, k, adapters, flush=True)
    packed = ref.random_packed(qtype, n, k, t)
    q, s = ref.random_rows(t, k, n)
    rows, weight = rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV))
    more = {}
    if adapters:
        made = make_adapters([128, 8, 40], n, k, TORCH[adapters], 3)
        more = dict(adapters=qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in made]),
                    ids=torch.from_numpy((np.arange(t) * 5 // t - 1).astype(np.int32)).to(DEV))
    y = qs.packed_linear(rows, weight, exact=True, **more)
    assert y.dtype == torch.bfloat16
    assert torch.equal(y, qs.packed_linear(rows, weight, dtype=torch.float32, **more).to(torch.bfloat16))
    assert not torch.equal(y, qs.packed_linear(rows, weight, **more))
    if not adapters:
        w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64(qtype, packed))
        want, bound = bound_of_exact(torch.from_numpy(ref.rows64(q, s)).to(DEV), w, wa, k // 32)
        assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", sorted(TORCH))
@pytest.mark.parametrize("t", [1, 40, 600])
def test_nothing_else_changes(qs, t, dtype):
    """Where codes are exact anyway `exact` is no other call."""
    n, k = 1030, 512
    rows = rows_on(qs, *ref.random_rows(t, k, 1))
    weight = qs.PackedWeight("q4_k", torch.from_numpy(ref.random_packed("q4_k", n, k, 1)).to(DEV))
    print(t, dtype, flush=True)
    assert torch.equal(qs.packed_linear(rows, weight, dtype=TORCH[dtype], exact=True),
                       qs.packed_linear(rows, weight, dtype=TORCH[dtype]))
