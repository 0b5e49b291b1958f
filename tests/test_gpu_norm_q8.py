"""RMS norm to 8-bit rows and the rows' values, against plain computations."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda:0"


def plain_codes(x, weight, residual):
    """Codes and steps with f32 operations on the CPU (each IEEE-rounded, as the kernel's)."""
    h = x.float().cpu()
    if residual is not None:
        h = h + residual.float().cpu()
    u = (h if weight is None else h * weight.cpu()).reshape(h.shape[0], -1, 32)
    a = u.abs().amax(2, keepdim=True) / 127
    return torch.where(a > 0, torch.round(u / a), 0.0).clamp(-127, 127), a, h


def check(rows, total, x, weight, residual, eps):
    t, k = x.shape
    codes, a, h = plain_codes(x, weight, residual)
    assert torch.equal(rows.q.cpu().float(), codes.reshape(t, k))
    if total is not None:
        assert torch.equal(total.cpu(), h.to(x.dtype))
    h = h.double()
    r = 1.0 if weight is None else 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    want = a.double()[:, :, 0] * r
    # k squares and their sum, the mean, the root (halving the error), two products
    bound = (k / 2 + 8) * ref.U * want.abs()
    assert ((rows.scale.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", sorted(TORCH))
@pytest.mark.parametrize("t,k,residual", [(1, 32, False), (1, 2560, True), (2, 96, True), (5, 4096, False), (333, 416, True),
                                          (3, 2048, True), (2, 2080, False), (2047, 64, True), (2048, 64, True),
                                          (2051, 2560, False), (2100, 9728, True), (1, 131072, True)])
def test_codes_scales_and_sum(qs, t, k, residual, dtype):
    print(t, k, residual, dtype, flush=True)
    g = torch.Generator().manual_seed(t + k)
    x = (torch.randn((t, k), generator=g) * torch.exp(torch.randn((t, 1), generator=g))).to(TORCH[dtype])
    res = torch.randn((t, k), generator=g).to(TORCH[dtype]) if residual else None
    w = 1 + 0.3 * torch.randn((k,), generator=g)
    got = qs.rms_norm_q8(x.to(DEV), w.to(DEV), eps=1e-5, residual=None if res is None else res.to(DEV))
    rows, total = got if residual else (got, None)
    check(rows, total, x, w, res, 1e-5)
    if t < 400:
        check(qs.q8_rows(x.to(DEV)), None, x, None, None, 0.0)


@pytest.mark.parametrize("t", [3, 2100])
def test_zero_rows_and_zero_groups(qs, t):
    x = torch.randn((t, 128), generator=torch.Generator().manual_seed(1))
    x[0] = 0
    x[1, 32:64] = 0
    w = torch.ones(128)
    rows = qs.rms_norm_q8(x.to(DEV), w.to(DEV))
    check(rows, None, x, w, None, 1e-6)
    assert (rows.values()[0] == 0).all() and (rows.values()[1, 32:64] == 0).all()
    zero = qs.rms_norm_q8(x[:1].to(DEV), w.to(DEV), eps=0.0)     # 0 / 0: no values, as plain
    assert (zero.q == 0).all() and torch.isnan(zero.scale).all()


@pytest.mark.parametrize("t", [4, 2100])
def test_nan_and_infinity_stay_where_the_plain_form_has_them(qs, t):
    x = torch.randn((t, 96), generator=torch.Generator().manual_seed(2))
    x[1, 40], x[2, 40], x[3, 7] = float("nan"), float("inf"), float("-inf")
    w = torch.ones(96)
    v = qs.rms_norm_q8(x.to(DEV), w.to(DEV)).values().cpu()
    assert torch.isfinite(v[0]).all() and torch.isfinite(v[4:]).all()
    assert torch.isnan(v[1]).all()                      # a NaN is in the row's mean
    assert torch.isnan(v[2, 32:64]).all() and (v[2, :32] == 0).all() and (v[2, 64:] == 0).all()
    assert torch.isnan(v[3, :32]).all() and (v[3, 32:] == 0).all()
    v = qs.q8_rows(x.to(DEV)).values().cpu()            # without a norm only the group is lost
    assert torch.isnan(v[1, 32:64]).all() and torch.isfinite(v[1, :32]).all() and torch.isfinite(v[1, 64:]).all()
    assert torch.isnan(v[2, 32:64]).all() and torch.isfinite(v[2, 64:]).all()


def test_tiny_and_huge_values(qs):
    """Steps in the subnormal range (codes capped at 127) and squares that overflow."""
    x = torch.zeros((3, 64))
    x[0, :5] = torch.tensor([190.0, 100.0, -190.0, 64.0, 0.0]) * 2.0 ** -149
    x[1] = 3e38
    x[2] = 1e-30
    rows = qs.q8_rows(x.to(DEV))
    check(rows, None, x, None, None, 0.0)
    assert rows.q[0, 0] == 127 and rows.q[0, 2] == -127
    v = qs.rms_norm_q8(x.to(DEV), torch.ones(64, device=DEV)).values().cpu()
    assert (v[1] == 0).all() and torch.isfinite(v).all()


def test_layouts(qs):
    g = torch.Generator().manual_seed(5)
    big = torch.randn((40, 256), generator=g).to(DEV, torch.bfloat16)
    w = (1 + 0.1 * torch.randn((160,), generator=g)).to(DEV)
    want = None
    base = big[:, 32:192].contiguous()
    off = torch.empty(40 * 160 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(40, 160).copy_(base)
    turned = base.t().contiguous().t()
    for x in (base, big[:, 32:192], off, turned):
        rows, total = qs.rms_norm_q8(x, w, residual=x)
        got = (rows.q, rows.scale, total)
        if want is None:
            want = got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = torch.full((1, 160), 0.5, device=DEV).expand(40, 160)
    assert torch.equal(qs.q8_rows(one).q, torch.full((40, 160), 127, dtype=torch.int8, device=DEV))
    empty = qs.rms_norm_q8(base[:0], w)
    assert empty.q.shape == (0, 160) and empty.values().shape == (0, 160)


@pytest.mark.parametrize("dtype", sorted(TORCH))
@pytest.mark.parametrize("t,k", [(1, 32), (7, 96), (130, 2560)])
def test_values(qs, t, k, dtype):
    q, s = ref.random_rows(t, k, t)
    rows = qs.Q8Rows(torch.from_numpy(q).to(DEV), torch.from_numpy(s).to(DEV))
    want = (torch.from_numpy(q).float() * torch.from_numpy(np.repeat(s, 32, 1))).to(TORCH[dtype])
    assert torch.equal(rows.values(TORCH[dtype]).cpu(), want)
