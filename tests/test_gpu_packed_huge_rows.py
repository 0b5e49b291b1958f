"""Rows whose values come close to f32's largest, with weights small enough for
finite results: 3.4e38 is passed by the sum of a group's codes times its scale, and
by 128 times a scale, though by no value."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref
from test_gpu_packed_f16 import bounds
from test_gpu_packed_f16 import check as check16
from test_gpu_packed_linear import DEV, check, rows_on

pytestmark = pytest.mark.gpu


def case(qtype, t, n, k):
    """Scales whose 127-fold is finite and whose 128-fold is not; codes of one sign in the first group."""
    packed = ref.random_packed(qtype, n, k, 1)
    blocks = packed.reshape(-1, ref.BYTES[qtype])
    rng = np.random.default_rng(2)
    for at in ref.HALVES.get(qtype, (0,)):
        blocks[:, at:at + 2] = rng.uniform(1e-6, 2e-6, len(blocks)).astype(np.float16)[:, None].view(np.uint8)
    q, s = ref.random_rows(t, k, 3)
    q = np.maximum(q, -127)
    q[:, :32] = 127
    s[t // 2:] = np.float32(2.67e36)
    with np.errstate(over="ignore"):
        assert np.isfinite(np.float32(127) * s).all() and not np.isfinite(np.float32(128) * s[-1]).any()
    return packed, q, s


@pytest.mark.parametrize("qtype", ["q4_1", "q2_k", "q5_k", "q6_k", "q8_0"])
@pytest.mark.parametrize("t,n", [(2, 40), (40, 300), (64, 2100), (600, 400), (1030, 2100)])
def test_exact_codes(qs, qtype, t, n):
    k = 512
    packed, q, s = case(qtype, t, n, k)
    print(qtype, t, n, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)), dtype=torch.float32)
    check(y, *ref.linear64(qtype, packed, q, s, "f32"), f"{qtype} {t}x{n}x{k}")


@pytest.mark.parametrize("qtype", ["q5_1", "q4_k", "q8_0"])
def test_f16_factors(qs, qtype):
    t, n, k = 900, 7010, 1024
    packed, q, s = case(qtype, t, n, k)
    rows, weight = rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV))
    print(qtype, t, n, flush=True)
    y = qs.packed_linear(rows, weight)
    assert not torch.equal(y, qs.packed_linear(rows, weight, exact=True))
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64(qtype, packed))
    want, bound = bounds(torch.from_numpy(ref.rows64(q, s)).to(DEV), w, wa, k // 32)
    half = t // 2           # by themselves: the others' norm is lost beside theirs
    for at in (slice(0, half), slice(half, t)):
        check16(y[at], want[at], bound[at], f"{qtype} rows {at.start} to {at.stop}")
