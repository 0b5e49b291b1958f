"""The operators on packed weights have no gradient: a tensor that asks for one
is refused while gradients are recorded, not taken out of its graph unsaid (no
GPU needed: the check comes before the device's)."""

from __future__ import annotations

import pytest
import torch

NO_GRADIENT = "no gradient"


def test_refused_while_gradients_are_recorded(qs):
    x, w = torch.ones((2, 64)), torch.ones(64)
    t = lambda v: v.clone().requires_grad_()  # noqa: E731
    with pytest.raises(ValueError, match=NO_GRADIENT):
        qs.rms_norm_q8(t(x), w)
    with pytest.raises(ValueError, match=NO_GRADIENT):
        qs.rms_norm_q8(x, t(w))
    with pytest.raises(ValueError, match=NO_GRADIENT):
        qs.rms_norm_q8(x, w, residual=t(x))
    with pytest.raises(ValueError, match=NO_GRADIENT):
        qs.rms_norm_q8(t(x) * 2, w)             # part of a graph, not a leaf
    with pytest.raises(ValueError, match=NO_GRADIENT):
        qs.q8_rows(t(x))
    with pytest.raises(ValueError, match=NO_GRADIENT):
        qs.Q8Rows(x.to(torch.int8), t(torch.ones((2, 2))))
    with pytest.raises(ValueError, match=NO_GRADIENT):
        qs.packed_linear(t(x), None)


@pytest.mark.parametrize("off", [torch.no_grad, torch.inference_mode])
def test_taken_where_none_is_recorded(qs, off):
    """A model's parameters ask for gradients by default; a server runs under
    no_grad. Here the next check, the device's, is what refuses."""
    x, w = torch.ones((2, 64)).requires_grad_(), torch.ones(64).requires_grad_()
    with off():
        with pytest.raises(ValueError, match="ROCm device"):
            qs.rms_norm_q8(x, w, residual=x)
        with pytest.raises(ValueError, match="ROCm device"):
            qs.Q8Rows(x.detach().to(torch.int8), torch.ones((2, 2)).requires_grad_())
