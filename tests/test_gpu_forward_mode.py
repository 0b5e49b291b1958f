"""Forward mode on the GPU: the cache's operators and results that are written to refuse a tensor with a tangent."""

from __future__ import annotations

import contextlib

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("mode", [contextlib.nullcontext, torch.no_grad])
def test_a_tangent_is_refused(qs, mode):
    cache = qs.KVCache(2, 16, 2, 64)
    x, q = torch.full((3, 2, 64), 127.0, device=DEV), torch.zeros((1, 4, 64), device=DEV)      # held exactly, of step 1
    slots, tables, lengths = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0, 1, 2], [[0, 1]], [3]))
    with mode(), forward_ad.dual_level():
        d = lambda v: forward_ad.make_dual(v, torch.ones_like(v))  # noqa: E731
        for call in (lambda: qs.kv_write(cache, d(x), x, slots), lambda: qs.kv_write(cache, x, d(x), slots),
                     lambda: qs.kv_attention(d(q), cache, tables, lengths), lambda: qs.kv_attention(d(q) * 2, cache, tables, lengths),
                     lambda: qs.kv_attention(q, cache, tables, lengths, out=d(q.clone()))):
            with pytest.raises(ValueError, match="tangent"):
                call()
        qs.kv_write(cache, d(x).detach(), x, slots)
        assert (qs.kv_attention(d(q).detach(), cache, tables, lengths) == 127.0).all()
    assert (qs.kv_attention(q, cache, tables, lengths) == 127.0).all()
