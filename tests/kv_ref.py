"""The quantised key-value cache in 64 bits, from the packed blocks of the
framework's own quantizers (test infrastructure)."""

from __future__ import annotations

import math

import torch

from dequant import dequantize

DEV = "cuda:0"


def values64(qs, kind: str, x):
    """What x (t, heads, d) stands for once it is quantised, f64 on the CPU."""
    t, heads, d = x.shape
    packed = qs.QUANT_TYPES[kind].make_kernel(torch.device(DEV), None)(x.reshape(t * heads, d).contiguous())
    return torch.from_numpy(dequantize(kind, packed.cpu().numpy(), t * heads)).double().reshape(t, heads, d)


def keys_values(t: int, heads: int, d: int, dtype, seed: int, spread: float = 1.0):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn((2, t, heads, d), generator=g)
    k[..., 5] *= 6
    return (k * spread).to(DEV, dtype), v.to(DEV, dtype)


def fill(qs, cache, lengths, dtype, seed, pages=None, poison=False):
    """Write sequences of `lengths` to pages in a shuffled order; the tables
    (int32, -1 past a sequence's pages) and each sequence's keys and values, f64.
    poison: every slot that no sequence has holds NaN."""
    p = cache.page_size
    if poison:
        t = cache.pages * p
        bad = torch.full((t, cache.heads, cache.head_dim), math.nan, dtype=dtype, device=DEV)
        qs.kv_write(cache, bad, bad, torch.arange(t, dtype=torch.int32, device=DEV))
    counts = [-(-n // p) for n in lengths]
    order = (torch.randperm(cache.pages, generator=torch.Generator().manual_seed(seed)) if pages is None else pages).tolist()
    tables = torch.full((len(lengths), max(counts) if counts else 0), -1, dtype=torch.int32)
    rows = []
    for i, n in enumerate(lengths):
        own, order = order[:counts[i]], order[counts[i]:]
        tables[i, :counts[i]] = torch.tensor(own, dtype=torch.int32)
        at = torch.arange(n)
        slots = (torch.tensor(own + [0])[at // p] * p + at % p).to(torch.int32)
        k, v = keys_values(n, cache.heads, cache.head_dim, dtype, seed * 1000 + i)
        qs.kv_write(cache, k, v, slots.to(DEV))
        rows.append((values64(qs, cache.k_type, k), values64(qs, cache.v_type, v)) if n else (k.cpu().double(), v.cpu().double()))
    return tables.to(DEV), rows


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def attention64(q, rows, scale=None, window=0, offset=0.0, wide=False):
    """(y, how far a kernel's y may be off) for q (b, n, query heads, d) and each
    sequence's (keys, values).

    What a kernel may add up to, with u = 2^-24:
    - a score s = scale sum q K: a sum of d products in f32 (at most d + 8 roundings
      of u of the sum of magnitudes A), q to 22 bits where it is f32 (2^-22 A), and
      4 roundings of s itself: e_s = ((d + 8) u + 2^-22) A + 4 u |s|;
    - p = exp(s - top): e_s for s and for the top, one rounding of each of s, top and
      their difference in powers of two, the exponential's own 2 u:
      e_p = 2 max e_s + 4 u max |s| + 4 u, relative, on numerator and denominator;
    - P = p step to 21 bits: 2^-21; then a sum of P c over L slots in f32, 32 at a
      time, over waves and workgroups: (L / 32 + 96) u, of magnitudes with the
      offset of four-bit codes (c + 8, so |V| + 8 step), the denominator's the same;
    - y is rounded once to its type."""
    b, n, hq, d = q.shape
    q64 = q.detach().cpu().double()
    y, far = torch.zeros_like(q64), torch.zeros_like(q64)
    scale = 1 / math.sqrt(d) if scale is None else scale
    u = 2.0 ** -24
    for i, (k, v) in enumerate(rows):
        length, heads = k.shape[0], k.shape[1]
        for j in range(n):
            last = length - n + j + 1
            first = max(0, last - window) if window else 0
            if last <= first:
                continue
            kk = k[first:last].repeat_interleave(hq // heads, 1)       # (L, hq, d)
            vv = v[first:last].repeat_interleave(hq // heads, 1)
            s = scale * torch.einsum("lhd,hd->hl", kk, q64[i, j])
            a = abs(scale) * torch.einsum("lhd,hd->hl", kk.abs(), q64[i, j].abs())
            e_s = ((d + 8) * u + (2.0 ** -22 if wide else 0.0)) * a + 4 * u * s.abs()
            e_p = 2 * e_s.amax(1) + 4 * u * s.abs().amax(1) + 4 * u
            p = torch.softmax(s, 1)
            y[i, j] = torch.einsum("hl,lhd->hd", p, vv)
            size = torch.einsum("hl,lhd->hd", p, vv.abs()) + offset * p.mul(_steps(vv)).sum(1)[:, None]
            far[i, j] = (2 * e_p[:, None] + 2.0 ** -21 + 2 * ((last - first) / 32 + 96) * u) * size
    return y, far + HALF_STEP[q.dtype] * (y.abs() + far) + 2.0 ** -24 * (q.dtype == torch.float16)


def _steps(v):
    """A bound of the values' steps, (hq, L): a block's largest value is at least seven of them."""
    return (v.abs().amax(2) / 7).transpose(0, 1)


def check(got, want, far):
    """Off by no more than `far`; NaN where the result is (an infinite query's)."""
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    got, want, far = (x.masked_fill(want.isnan(), 0.0) for x in (got, want, far))
    off = (got - want).abs()
    worst = (off / far.clamp_min(1e-300)).nan_to_num(math.inf).max().item() if off.numel() else 0.0
    print(f"off by {off.max().item() if off.numel() else 0:.3g}, {worst:.3g} of what is allowed", flush=True)
    assert worst <= 1.0, worst
