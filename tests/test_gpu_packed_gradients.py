"""Tensors that ask for gradients, on the GPU: a bank holds copies without a
graph, `out` is refused, and under no_grad everything runs."""

from __future__ import annotations

import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, make_adapters, rows_on

pytestmark = pytest.mark.gpu


def test_bank_of_trainable_adapters(qs):
    n, k, t = 70, 256, 5
    made = [(a.to(DEV).requires_grad_(), b.to(DEV).requires_grad_(), c)
            for a, b, c in make_adapters([8, 5], n, k, torch.bfloat16, 1)]
    bank = qs.AdapterBank(made)
    assert not bank.a.requires_grad and not bank.b.requires_grad and bank.a.grad_fn is None and bank.b.grad_fn is None
    rows = rows_on(qs, *ref.random_rows(t, k, 2))
    weight = qs.PackedWeight("q4_k", torch.from_numpy(ref.random_packed("q4_k", n, k, 1)).to(DEV))
    ids = torch.tensor([0, 1, -1, 0, 1], dtype=torch.int32, device=DEV)
    y = qs.packed_linear(rows, weight, adapters=bank, ids=ids)
    with torch.no_grad():
        for a, b, _ in made:
            a.mul_(3), b.mul_(0)
    assert torch.equal(qs.packed_linear(rows, weight, adapters=bank, ids=ids), y)       # copies, made once
    one = qs.AdapterBank(made[:1])          # a single adapter whose rank needs no padding is copied too
    assert one.a.data_ptr() != made[0][0].data_ptr() and not one.a.requires_grad


def test_out_and_no_grad(qs):
    n, k, t = 70, 256, 5
    x = torch.randn((t, k), device=DEV, dtype=torch.bfloat16).requires_grad_()
    norm = torch.ones(k, device=DEV).requires_grad_()
    weight = qs.PackedWeight("q4_k", torch.from_numpy(ref.random_packed("q4_k", n, k, 1)).to(DEV))
    rows = rows_on(qs, *ref.random_rows(t, k, 2))
    with pytest.raises(ValueError, match="no gradient"):
        qs.packed_linear(rows, weight, out=torch.empty((t, n), device=DEV, dtype=torch.bfloat16).requires_grad_())
    with torch.no_grad():
        got, h = qs.rms_norm_q8(x, norm, residual=x)
    want, total = qs.rms_norm_q8(x.detach(), norm.detach(), residual=x.detach())
    assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale) and torch.equal(h, total)
