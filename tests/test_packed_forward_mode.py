"""Tensors with a tangent of forward mode are refused, whether gradients are recorded or not: results would come
without theirs (no GPU needed: the check comes before the device's)."""

from __future__ import annotations

import contextlib

import pytest
import torch
from torch.autograd import forward_ad


@pytest.mark.parametrize("mode", [contextlib.nullcontext, torch.no_grad])
def test_a_tangent_is_refused(qs, mode):
    x, w = torch.ones((2, 64)), torch.ones(64)
    with mode(), forward_ad.dual_level():
        d = lambda v: forward_ad.make_dual(v, torch.ones_like(v))  # noqa: E731
        for call in (lambda: qs.rms_norm_q8(d(x), w), lambda: qs.rms_norm_q8(x, d(w)), lambda: qs.rms_norm_q8(x, w, residual=d(x)),
                     lambda: qs.rms_norm_q8(d(x) * 2, w), lambda: qs.q8_rows(d(x)),
                     lambda: qs.Q8Rows(x.to(torch.int8), d(torch.ones((2, 2)))), lambda: qs.packed_linear(d(x), None)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        for call in (lambda: qs.rms_norm_q8(x, w), lambda: qs.q8_rows(d(x).detach())):
            with pytest.raises(ValueError, match="ROCm device"):
                call()
    with pytest.raises(ValueError, match="ROCm device"):
        qs.rms_norm_q8(x, w)
