"""What the attention over the key-value cache keeps of its factors: results against 64
bits, 16-bit ones to their own rounding and no more than f32 sums beside it."""

from __future__ import annotations

import math

import pytest
import torch

import kv_ref as ref
from kv_ref import DEV

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DIGITS = {torch.bfloat16: 8, torch.float16: 11, torch.float32: 24}


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def half_spacing(x, dtype):
    """Half the distance between neighbours of dtype at |x|: what its rounding may take, at most half of what eps says."""
    low = -14 if dtype == torch.float16 else -126
    return torch.exp2((torch.frexp(x.abs().clamp_min(2.0 ** low))[1] - DIGITS[dtype] - 1).double())


def bound(q, rows, scale=None, window=0, offset=0.0):
    """(y, how far off a result may be) as in ref.attention64 for f32 sums, and the type's own rounding."""
    want, far = ref.attention64(q.float(), rows, scale, window, offset, q.dtype == torch.float32)
    return want, far + half_spacing(want.abs() + far, q.dtype)


def held(qs, cache, k, v, dtype=torch.float32):
    """Writes rows to the cache's first slots: what it holds of them, f64, and the table of its pages."""
    qs.kv_write(cache, k.to(DEV, dtype), v.to(DEV, dtype), torch.arange(len(k), dtype=torch.int32, device=DEV))
    rows = ref.values64(qs, cache.k_type, k.to(DEV, dtype)), ref.values64(qs, cache.v_type, v.to(DEV, dtype))
    return [rows], torch.arange(cache.pages, dtype=torch.int32, device=DEV)[None]


U = 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,below", [("q8_0", 9), ("q4_0", 11)])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_small_terms_of_values_beside_large_ones(qs, dtype, kind, below, d):
    """Eight slots of each 32 have codes of +-1 whose steps are powers of two and cancel; the others' steps are 2^below
    smaller, of eleven bits. All scores are 0 and every sum, in any order, is a whole number of the smallest
    step under 2^24 of them, so that f32 sums are exact: what is left are four roundings of f32, and the type's own."""
    g = torch.Generator().manual_seed(d)
    heads, n, top = 8, 64, 127.0 if kind == "q8_0" else -8.0
    step = (1024 + torch.randint(0, 1024, (n, heads, 1, 1), generator=g)).float() / 1024 * 2.0 ** -below
    codes = torch.randint(-7, 8, (n, heads, d // 32, 32), generator=g).float()
    for i in range(0, n, 32):
        large = i + torch.randperm(32, generator=g)[:8]
        step[large] = 1.0
        codes[large] = torch.tensor([1.0, -1.0] * 4).view(8, 1, 1, 1)
    codes[..., 0] = top
    v = (codes * step).view(n, heads, d)
    cache = qs.KVCache(4, 16, heads, d, "q8_0", kind)
    rows, table = held(qs, cache, torch.zeros_like(v), v)
    assert torch.equal(rows[0][1], v.double())
    y = qs.kv_attention(torch.ones((1, 1, heads, d), dtype=dtype, device=DEV), cache, table, ints(n))
    want = v.double().mean(0)[None, None]
    ref.check(y, want, 4 * U * want.abs() + half_spacing(want, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,below", [("q8_0", 11), ("q4_0", 13)])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_small_terms_of_scores_beside_large_ones(qs, dtype, kind, below, d):
    """Eight values of a query are 1 and meet codes of +-1 that cancel, the others are 2^-below and of eight bits, which
    every type has: each block's sum is a whole number of the smallest under 2^24 of them, exact in f32. Then a
    score is off by its blocks' sum and three roundings, (d / 32 + 4) u of the sum of their magnitudes, and the
    rest is as in ref.attention64."""
    g = torch.Generator().manual_seed(d)
    heads, group, n = 4, 4, 45
    codes = torch.randint(-7, 8, (n, heads, d // 32, 32), generator=g).float()
    codes[..., 1:9] = torch.tensor([1.0, -1.0] * 4)
    codes[..., 0] = 127.0 if kind == "q8_0" else -8.0
    k = (codes * (1024 + torch.randint(0, 1024, (n, heads, d // 32, 1), generator=g)).float() / 1024).view(n, heads, d)
    q = (128 + torch.randint(0, 128, (heads * group, d // 32, 32), generator=g)).float() / 128 * 2.0 ** -below
    q[..., 1:9] = 1.0
    q[..., 0] = 0.0
    q = q.view(1, 1, heads * group, d)
    cache = qs.KVCache(3, 16, heads, d, kind, "q8_0")
    rows, table = held(qs, cache, k, torch.randn((n, heads, d), generator=g))
    assert torch.equal(rows[0][0], k.double())
    scale = 2.0 ** below / (4 * math.sqrt(d))
    y = qs.kv_attention(q.to(DEV, dtype), cache, table, ints(n), scale=scale)
    blocks = (rows[0][0].repeat_interleave(group, 1) * q[0].double()).view(n, heads * group, d // 32, 32).sum(3) * scale
    s, a, v = blocks.sum(2), blocks.abs().sum(2), rows[0][1].repeat_interleave(group, 1)
    e_s = (d // 32 + 4) * U * a.amax(0) + 4 * U * s.abs().amax(0)
    p = torch.softmax(s, 0)[..., None]
    want, size = (p * v).sum(0), (p * v.abs()).sum(0)
    far = (2 * (2 * e_s + 4 * U)[:, None] + 2.0 ** -21 + 2 * (2 + 96) * U) * size
    ref.check(y[0, 0], want, far + half_spacing(want.abs() + far, dtype))


def weighted(qs, cache, scores, v, queries, dtype, length=None, batch=2):
    """Attention over rows whose keys are one value, so that a score is one product: sequences of the same rows, the
    `queries` of a head 1, 1/2, 1/4 ... in the key's place. Returns y and the result in 64 bits with what an
    f32 computation may be off by: a score by four roundings, the rest as in ref.attention64; a slot's P to 2^-21."""
    n, heads, d = v.shape
    k = torch.zeros((n, heads, d))
    k[:, :, 0] = scores if scores.dim() == 2 else scores[:, None]
    rows, table = held(qs, cache, k, v)
    q = torch.zeros((batch, 1, heads * queries, d))
    q[..., 0] = 2.0 ** -torch.arange(queries).repeat(heads)
    length = n if length is None else length
    y = qs.kv_attention(q.to(DEV, dtype), cache, table.expand(batch, -1), ints(*[length] * batch), scale=1.0)
    s = (rows[0][0][:length, :, None, :1] * q[0, 0].view(heads, queries, d)[None, :, :, :1].double())[..., 0]
    far = 2 * (2 * 4 * U * s.abs().amax(0) + 4 * U) + 2.0 ** -21 + 2 * (length / 32 + 96) * U
    p = torch.softmax(s, 0)
    vv = rows[0][1][:length, :, None]
    want, size = (p[..., None] * vv).sum(0), (p[..., None] * vv.abs()).sum(0)
    want, far = want.view(heads * queries, d), (far[..., None] * size).view(heads * queries, d)
    return y[:, 0], want.expand(batch, -1, -1), (far + half_spacing(want.abs() + far, dtype)).expand(batch, -1, -1)


@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
@pytest.mark.parametrize("seed", range(4))
def test_two_slots_of_many_heads(qs, kind, seed):
    """So many P that some of them round to half way between two f16: both parts of such a one belong together."""
    scores = torch.randn((2, 512), generator=torch.Generator().manual_seed(seed)) * 2
    ref.check(*weighted(qs, qs.KVCache(1, 16, 512, 64, "q8_0", kind), scores, positive(2, 512, 64, seed), 8, torch.float32, batch=1))


def positive(n, heads, d, seed):
    return torch.randn((n, heads, d), generator=torch.Generator().manual_seed(seed)).abs() + 0.1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("large,small", [(60.0, 1.0), (100.0, 0.02), (1e4, 1e-2)])
def test_blocks_of_other_sizes(qs, dtype, kind, d, large, small):
    """A block of small values is as exact as if there were no large ones beside it."""
    v = positive(760, 2, d, 1)
    v[..., 32:] *= small
    v[..., :32] *= large
    scores = torch.randn(760, generator=torch.Generator().manual_seed(2)) * 2
    ref.check(*weighted(qs, qs.KVCache(48, 16, 2, d, "q8_0", kind), scores, v, 4, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
@pytest.mark.parametrize("queries", [4, 12])
@pytest.mark.parametrize("at", [(7, 500), (0, 1), (758, 759)])
@pytest.mark.parametrize("times", [5e3, 1e6])
def test_large_values_of_no_weight(qs, dtype, kind, queries, at, times):
    """Two slots whose scores are 60 below the others' do not show, however large their values."""
    v = positive(760, 2, 128, 3) * 0.02
    scores = torch.randn(760, generator=torch.Generator().manual_seed(4))
    for i in at:
        v[i] *= times
        scores[i] = -60.0
    ref.check(*weighted(qs, qs.KVCache(48, 16, 2, 128, "q8_0", kind), scores, v, 1 if queries == 4 else queries, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("queries", [3, 13])
@pytest.mark.parametrize("slope", [-40.0, -8.0, 0.0, 8.0, 40.0])
def test_sizes_that_change_along_a_sequence(qs, dtype, kind, d, queries, slope):
    """Scores that rise or fall, and blocks whose values rise, fall, or are nothing for a while, over six steps of
    each wave, and over one."""
    n = 760
    v = positive(n, 2, d, 5)
    along = torch.linspace(-1, 1, n)[:, None, None]
    for b in range(d // 32):
        part = v[..., 32 * b:32 * b + 32]
        part *= (10.0 ** (2 * along), 10.0 ** (-2 * along), torch.ones_like(along), (along > 0.3).float(), (along < -0.3).float(),
                 torch.zeros_like(along), 10.0 ** (3 * along.abs() - 3), (along.abs() < 0.001).float())[(b + 3) % 8]
    scores = torch.linspace(0, 1, n) * slope + torch.randn(n, generator=torch.Generator().manual_seed(6))
    cache = qs.KVCache(48, 16, 2, d, "q8_0", kind)
    for length in (n, 130):
        ref.check(*weighted(qs, cache, scores, v, queries, dtype, length))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["q8_0", "q4_0"])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_a_block_of_nan_beside_numbers(qs, dtype, kind, d):
    """A NaN in a value that a query sees makes its block of the result NaN, and nothing of the others less exact."""
    v = positive(300, 2, d, 7) * 0.05
    v[100, :, 3] = math.nan
    scores = torch.randn(300, generator=torch.Generator().manual_seed(8)) * 3
    y, want, far = weighted(qs, qs.KVCache(20, 16, 2, d, "q8_0", kind), scores, v, 4, dtype)
    assert y[..., :32].isnan().all()
    ref.check(y[..., 32:], want[..., 32:], far[..., 32:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length,columns", [(2, 1), (40, 3), (40, 70), (700, 70)])
@pytest.mark.parametrize("value,scale", [(-math.inf, 0.1), (math.inf, -0.1), (-2.0, math.inf), (2.0, -math.inf), (-2e38, 1e3)])
def test_scores_that_are_all_minus_infinity(qs, dtype, length, columns, value, scale):
    """NaN, as the softmax of them is, and zeros only where a query sees nothing: the first of three new tokens of two."""
    if dtype == torch.float16 and abs(value) > 1e30 and value > -math.inf and value < math.inf:
        pytest.skip("no such f16")
    cache = qs.KVCache(70, 16, 2, 64, "q8_0", "q4_0")
    k, v = torch.zeros((length, 2, 64)), torch.randn((length, 2, 64), generator=torch.Generator().manual_seed(1))
    k[..., 0] = torch.rand((length, 2), generator=torch.Generator().manual_seed(2)) + 1
    if abs(value) == math.inf:      # a zero of a key would make the score NaN
        k += 1
    qs.kv_write(cache, k.to(DEV), v.to(DEV), torch.arange(length, dtype=torch.int32, device=DEV))
    q = torch.zeros((1, 3, 4, 64))
    q[..., 0] = value
    q[:, :, 3, 0] = 0.5 if abs(scale) < 1e3 else value
    y = qs.kv_attention(q.to(DEV, dtype), cache, torch.arange(columns, dtype=torch.int32, device=DEV)[None], ints(length), scale=scale)
    sees = torch.arange(3) >= 3 - length
    assert torch.equal(y.isnan().all(3).cpu()[0, :, :3], sees[:, None].expand(3, 3)) and not y[:, ~sees].any()
    if abs(scale) < 1e3:
        assert not y[:, :, 3].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("power", [127, 120, -120, -130])
def test_scales_near_the_ends_of_f32(qs, dtype, power):
    """Where scale log2(e) is out of range, and where scale is subnormal, scores of usual sizes are right."""
    cache = qs.KVCache(13, 16, 2, 64, "q8_0", "q4_0")
    k, v = ref.keys_values(200, 2, 64, torch.float32, 11)
    rows, table = held(qs, cache, k, v)
    q = (torch.randn((1, 2, 6, 64), generator=torch.Generator().manual_seed(12)) * 2.0 ** (-power - 3)).to(DEV, dtype)
    scale = 1.5 * 2.0 ** power
    want, far = bound(q, rows, scale)
    ref.check(qs.kv_attention(q, cache, table, ints(200), scale=scale), want, far)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, 3e4])
def test_what_another_query_sees_does_not_matter(qs, dtype, bad):
    """Bit for bit: keys and values of the last new tokens, of a window's slots before an earlier one's, of nothing."""
    cache = qs.KVCache(9, 16, 2, 128, "q8_0", "q8_0")
    k, v = ref.keys_values(100, 2, 128, torch.float32, 9)
    rows, table = held(qs, cache, k, v)
    q = torch.randn((1, 4, 6, 128), generator=torch.Generator().manual_seed(10)).to(DEV, dtype)
    for window in (0, 20):
        y = qs.kv_attention(q, cache, table, ints(100), window=window)
        kept = cache.data.clone()
        at = [98, 99, 100, 120] + ([0, 60, 76] if window else [])       # the first one sees those above 96 - window
        x = torch.full((len(at), 2, 128), bad, device=DEV)
        qs.kv_write(cache, x, x, ints(*at))
        z = qs.kv_attention(q, cache, table, ints(100), window=window)
        assert torch.equal(z[:, :2], y[:, :2])
        assert not torch.equal(z[:, 2:], y[:, 2:])
        cache.data.copy_(kept)
