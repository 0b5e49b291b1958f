"""Products of f16 factors and of exact codes where neither can be taken for the
other: every format at a size past the rule for f16 factors, and weights of more
than one slice of the layout, each compared with the call's exact form too."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref
from test_gpu_packed_exact import bound_of_exact
from test_gpu_packed_f16 import bounds, check
from test_gpu_packed_linear import DEV, TORCH, make_adapters, rows_on

pytestmark = pytest.mark.gpu

SHAPES = [(140, 46200), (900, 7011), (2100, 3001)]


def both(qs, rows, weight, **more):
    """The result of f16 factors and of exact codes; fails where the call takes the same path twice."""
    y, exact = qs.packed_linear(rows, weight, **more), qs.packed_linear(rows, weight, exact=True, **more)
    assert not torch.equal(y, exact), "no f16 factors at this size"
    return y, exact


@pytest.mark.parametrize("i,qtype", list(enumerate(sorted(ref.BYTES))))
def test_every_format(qs, i, qtype):
    t, n = SHAPES[i % len(SHAPES)]
    k = 1056 if ref.BLOCK[qtype] == 32 else 1024
    print(qtype, t, n, k, flush=True)
    packed = ref.random_packed(qtype, n, k, i)
    q, s = ref.random_rows(t, k, i)
    y, exact = both(qs, rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)))
    x = torch.from_numpy(ref.rows64(q, s)).to(DEV)
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64(qtype, packed))
    check(y, *bounds(x, w, wa, k // 32), f"{qtype} {t}x{n}x{k}")
    want, bound = bound_of_exact(x, w, wa, k // 32)
    assert ((exact.double() - want).abs() <= bound).all()


SLICE = 1 << 26         # values of a weight that are laid out at a time


@pytest.mark.parametrize("qtype,t,n,k,f16", [("q2_k", 129, 66000, 1024, True), ("iq2_xs", 160, 66000, 1024, True),
                                             ("q4_k", 129, 263000, 256, False), ("q6_k", 130, 131500, 512, False)])
def test_weights_of_two_slices(qs, qtype, t, n, k, f16):
    """With adapters, whose rows of B are not sliced."""
    assert n * k > SLICE
    print(qtype, t, n, k, flush=True)
    packed = ref.random_packed(qtype, n, k, 5)
    q, s = ref.random_rows(t, k, 6)
    rows, weight = rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV))
    made = make_adapters([40, 8], n, k, torch.bfloat16, 7)
    ids = (np.arange(t) % 3 - 1).astype(np.int32)
    more = dict(adapters=qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in made]), ids=torch.from_numpy(ids).to(DEV))
    x = torch.from_numpy(ref.rows64(q, s)).to(DEV)
    w, wa = (torch.from_numpy(v).to(DEV) for v in ref.weight64(qtype, packed))
    delta, more_off = (torch.from_numpy(v).to(DEV) for v in ref.adapters64(
        ref.rows64(q, s), [(a.double().numpy(), b.double().numpy(), c) for a, b, c in made], ids, n))
    want, bound = bound_of_exact(x, w, wa, k // 32)
    off = more_off + ref.ROUND["bf16"] * delta.abs()
    if f16:
        y, exact = both(qs, rows, weight, **more)
        check(y, want + delta, bounds(x, w, wa, k // 32)[1] + off, f"{qtype} {t}x{n}x{k}")
    else:
        exact = qs.packed_linear(rows, weight, **more)
    assert ((exact.double() - want - delta).abs() <= bound + off).all()
