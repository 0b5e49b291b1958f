"""The quantised key-value cache on the GPU: rows written and read back are what
the framework's quantizers make of them, and the attention over the cache is that
of these values in 64 bits."""

from __future__ import annotations

import math
import threading

import pytest
import torch

import kv_ref as ref
from kv_ref import DEV

pytestmark = pytest.mark.gpu
TYPES = ["q8_0", "q4_0"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---- rows ----

@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("k_type,v_type,dtype", [("q8_0", "q4_0", torch.bfloat16), ("q4_0", "q8_0", torch.float16),
                                                 ("q8_0", "q8_0", torch.float32), ("q4_0", "q4_0", torch.float32)])
@pytest.mark.parametrize("heads,t,page", [(1, 1, 16), (3, 37, 32), (8, 130, 64)])
def test_rows_are_the_quantizers(qs, d, k_type, v_type, dtype, heads, t, page):
    """Bit for bit, in any slots; what has no slot is left out, and the others' slots stay as they were."""
    cache = qs.KVCache(7, page, heads, d, k_type, v_type)
    k, v = ref.keys_values(t, heads, d, dtype, 1)
    slots = torch.randperm(7 * page, generator=torch.Generator().manual_seed(t))[:t].to(torch.int32).to(DEV)
    if t > 4:
        slots[2], slots[3], slots[4] = -1, 7 * page, -2 ** 31
    qs.kv_write(cache, k, v, slots)
    held = ((slots >= 0) & (slots < 7 * page)).cpu()
    got = qs.kv_read(cache, slots, dtype=torch.float32)
    for x, kind, y in ((k, k_type, got[0]), (v, v_type, got[1])):
        assert y.shape == (t, heads, d)
        assert torch.equal(y.cpu().double(), ref.values64(qs, kind, x) * held[:, None, None])
    others = torch.tensor([s for s in range(7 * page) if s not in set(slots.tolist())], dtype=torch.int32, device=DEV)
    for y in qs.kv_read(cache, others, dtype=torch.float32):
        assert not y.any()
    for out in (torch.float16, torch.bfloat16):
        for x, y in zip(got, qs.kv_read(cache, slots, dtype=out)):
            assert torch.equal(x.to(out), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("power", [-20, -6, 0, 7])
def test_ties_are_the_quantizers(qs, dtype, kind, power):
    """Bit for bit: largest magnitudes of either sign in a block, codes half way between two."""
    g = torch.Generator().manual_seed(power + 30)
    x = torch.randint(-255, 256, (1200, 2, 64), generator=g).float() / 2
    x[:400] = torch.randint(-2, 3, (400, 2, 64), generator=g).float()
    x[400:600] = (x[400:600] / 16).round() * 8.5
    x[600:800, :, ::7] = 127.0
    x[800:1000, :, 5::32] = -127.0
    x[1100:] = 0.0
    x[1150:, 0, 3] = -0.0
    x = (x * 2.0 ** power).to(DEV, dtype)
    cache = qs.KVCache(5, 256, 2, 64, kind)
    slots = torch.arange(1200, dtype=torch.int32, device=DEV)
    for rows in (slots[:700], slots[700:], slots):     # a row or several at a time
        qs.kv_write(cache, x[rows.long()], x[rows.long()].flip(2).contiguous(), rows)
        got = qs.kv_read(cache, rows, dtype=torch.float32)
        for y, z in zip(got, (x, x.flip(2))):
            assert torch.equal(y.cpu().double(), ref.values64(qs, kind, z[rows.long()].contiguous()))


@pytest.mark.parametrize("t", [2, 50, 300, 2000, 9000])
def test_a_slot_twice_holds_the_last_row(qs, t):
    """Also across the rows of different workgroups and launches."""
    heads, d = 2, 64
    cache = qs.KVCache(5, 64, heads, d, "q8_0", "q4_0")
    k, v = ref.keys_values(t, heads, d, torch.bfloat16, 2)
    slots = torch.randint(0, min(320, max(1, t // 3)), (t,), generator=torch.Generator().manual_seed(3)).to(torch.int32)
    last = {s: i for i, s in enumerate(slots.tolist())}
    qs.kv_write(cache, k, v, slots.to(DEV))
    rows = torch.tensor(list(last.values()))
    got = qs.kv_read(cache, slots[rows].to(DEV), dtype=torch.float32)
    assert torch.equal(got[0].cpu().double(), ref.values64(qs, "q8_0", k[rows.to(DEV)]))
    assert torch.equal(got[1].cpu().double(), ref.values64(qs, "q4_0", v[rows.to(DEV)]))


def test_rows_in_any_layout(qs):
    """Parts of a fused projection, heads apart, rows backwards, an odd start, flat rows."""
    heads, d, t = 3, 64, 21
    fused = torch.randn((t, 5 * heads * d + 8), generator=torch.Generator().manual_seed(4)).to(DEV, torch.bfloat16)
    slots = torch.arange(t, dtype=torch.int32, device=DEV)
    w = heads * d
    layouts = [(fused[:, w:2 * w], fused[:, 2 * w:3 * w]), (fused[:, 3:w + 3], fused[:, w + 5:2 * w + 5]),
               (fused[:, :w].view(t, heads, d), fused[:, w:2 * w].view(t, heads, d)),
               (fused[:, :w].reshape(t, d, heads).transpose(1, 2), fused[:, w:2 * w].flip(0).view(t, heads, d)),
               (fused[:1, :w].expand(t, w), fused[:, 0:2 * w:2])]
    for k, v in layouts:
        cache = qs.KVCache(1, 32, heads, d, "q4_0", "q8_0")
        qs.kv_write(cache, k, v, slots)
        got = qs.kv_read(cache, slots, dtype=torch.float32)
        assert torch.equal(got[0].cpu().double(), ref.values64(qs, "q4_0", k.reshape(t, heads, d)))
        assert torch.equal(got[1].cpu().double(), ref.values64(qs, "q8_0", v.reshape(t, heads, d)))
    again = qs.kv_read(cache, torch.stack([slots, slots], 1)[:, 0], dtype=torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("kind", TYPES)
def test_values_that_no_block_holds(qs, kind):
    """A NaN, an infinity and a step over f16's largest number make their block NaN, and no other; zeros and
    steps under f16's smallest give zeros."""
    x = torch.ones((6, 1, 64), device=DEV)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 7], x[3, 0, 1] = math.nan, math.inf, -math.inf, 3e38
    x[4] = 0.0
    x[5] = 1e-30
    cache = qs.KVCache(1, 16, 1, 64, kind)
    qs.kv_write(cache, x, x, ints(0, 1, 2, 3, 4, 5))
    for y in qs.kv_read(cache, ints(0, 1, 2, 3, 4, 5), dtype=torch.float32):
        bad = torch.zeros((6, 2), dtype=torch.bool)
        bad[0, 0] = bad[1, 1] = bad[2, 0] = bad[3, 0] = True
        assert torch.equal(y.view(6, 2, 32).isnan().all(2).cpu(), bad) and torch.equal(y.view(6, 2, 32).isnan().any(2).cpu(), bad)
        assert not y[4:].any()


def test_pages_may_be_copied(qs):
    """To another cache too; a cache may use bytes that it is given."""
    k, v = ref.keys_values(32, 2, 128, torch.float16, 5)
    a = qs.KVCache(3, 16, 2, 128, "q8_0", "q4_0")
    qs.kv_write(a, k, v, torch.arange(32, dtype=torch.int32, device=DEV))
    b = qs.KVCache(4, 16, 2, 128, "q8_0", "q4_0", data=torch.zeros((4, a.data.shape[1]), dtype=torch.uint8, device=DEV))
    b.data[3] = a.data[0]
    b.data[0] = a.data[1]
    slots = torch.arange(16, dtype=torch.int32, device=DEV)
    got = qs.kv_read(b, torch.cat([slots + 48, slots]), dtype=torch.float32)
    want = qs.kv_read(a, torch.cat([slots, slots + 16]), dtype=torch.float32)
    assert all(torch.equal(x, y) and x.any() for x, y in zip(got, want))


def test_slots_of_positions(qs):
    cache = qs.KVCache(5, 16, 1, 64)
    tables = ints(3, 1, -1, 0, 9, 2).view(2, 3)
    at = ints(0, 17, 33, -1, 48, 5, 16, 47, 15, 1 << 20).view(2, 5)
    want = [[48, 17, -1, -1, -1], [5, -1, 47, 15, -1]]
    assert cache.slots(tables, at).tolist() == want and cache.slots(tables, at.long()).tolist() == want
    assert cache.slots(tables[:, :0], at).tolist() == [[-1] * 5] * 2


def test_nothing_to_do(qs):
    cache = qs.KVCache(1, 16, 2, 64)
    none = torch.empty((0, 2, 64), device=DEV)
    qs.kv_write(cache, none, none, ints())
    assert qs.kv_read(cache, ints())[0].shape == (0, 2, 64)
    assert qs.kv_attention(torch.empty((0, 4, 64), device=DEV), cache, ints().view(0, 3), ints()).shape == (0, 4, 64)
    assert qs.kv_attention(torch.empty((2, 0, 4, 64), device=DEV), cache, ints(0, 0).view(2, 1), ints(1, 1)).shape == (2, 0, 4, 64)
    y = qs.kv_attention(torch.ones((2, 4, 64), device=DEV), cache, ints().view(2, 0), ints(5, 0))
    assert y.shape == (2, 4, 64) and not y.any()


# ---- attention ----

def attend(qs, cache, lengths, hq, n, dtype, seed, window=0, scale=None, poison=True, spread=1.0):
    """Checks a call against 64 bits, its tables as wide as they need be and wider, so that short lengths are split
    too; slots that no sequence has hold NaN. Returns what to call again."""
    tables, rows = ref.fill(qs, cache, lengths, dtype, seed, poison=poison)
    q = (spread * torch.randn((len(lengths), n, hq, cache.head_dim), generator=torch.Generator().manual_seed(seed))).to(DEV, dtype)
    print(cache.k_type, cache.v_type, cache.head_dim, lengths, hq, n, dtype, window, flush=True)
    want, far = ref.attention64(q, rows, scale, window, 8.0 if cache.v_type == "q4_0" else 0.0, dtype == torch.float32)
    more = torch.full((len(lengths), -(-1024 // cache.page_size)), -1, dtype=torch.int32, device=DEV)
    for table in (torch.cat([tables, more], 1), tables):
        y = qs.kv_attention(q[:, 0] if n == 1 else q, cache, table, ints(*lengths), scale=scale, window=window)
        ref.check(y.view(q.shape), want, far)
    return q, tables, y


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("k_type", TYPES)
@pytest.mark.parametrize("v_type", TYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention(qs, d, k_type, v_type, dtype):
    """Lengths from none over one to several pages, around the ends of steps and pages."""
    lengths = [33, 0, 1, 2, 15, 16, 17, 31, 32, 63, 64, 65, 100, 257]
    attend(qs, qs.KVCache(60, 16, 2, d, k_type, v_type), lengths, 8, 1, dtype, 1)


@pytest.mark.parametrize("heads,group", [(1, 1), (1, 7), (1, 8), (2, 9), (3, 5), (1, 16), (2, 17), (1, 40), (1, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_heads(qs, heads, group, dtype):
    attend(qs, qs.KVCache(20, 32, heads, 64, "q8_0", "q4_0"), [90, 5, 300], heads * group, 1, dtype, 2)


@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 16])
@pytest.mark.parametrize("group", [1, 3, 4])
@pytest.mark.parametrize("window", [0, 1, 7, 33, 1000])
def test_new_tokens_and_windows(qs, n, group, window):
    """Also sequences shorter than their new tokens, whose first ones are before the start."""
    attend(qs, qs.KVCache(30, 16, 2, 128, "q8_0", "q8_0"), [70, 0, 1, 3, 16, 40, 129], 2 * group, n, torch.float16, 3, window)


@pytest.mark.parametrize("page", [16, 64, 256, 1024])
@pytest.mark.parametrize("k_type,v_type", [("q8_0", "q8_0"), ("q4_0", "q4_0"), ("q8_0", "q4_0")])
def test_long(qs, page, k_type, v_type):
    lengths = [5003, 1, 1500, 0, 2049]
    attend(qs, qs.KVCache(sum(-(-n // page) for n in lengths) + 2, page, 2, 128, k_type, v_type), lengths, 8, 1, torch.float32, 4)


@pytest.mark.parametrize("batch", [1, 200, 700])
def test_batches(qs, batch):
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 40, (batch,), generator=g).tolist()
    lengths[batch // 2] = 900
    attend(qs, qs.KVCache(sum(-(-n // 16) for n in lengths) + 1, 16, 1, 64, "q8_0", "q4_0"), lengths, 3, 1, torch.bfloat16, 5)


@pytest.mark.parametrize("batch,heads,d,longest", [(300, 8, 64, 200), (300, 8, 128, 2500), (600, 8, 64, 900), (100, 24, 64, 700)])
def test_many_segments(qs, batch, heads, d, longest):
    """More heads of sequences than workgroups: whole ones to a wave each, and long ones among them split."""
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 25, (batch,), generator=g).tolist()
    lengths[0], lengths[batch // 3], lengths[-1] = longest, longest // 2 + 1, 0
    attend(qs, qs.KVCache(sum(-(-n // 32) for n in lengths) + 1, 32, heads, d, "q8_0", "q4_0"), lengths, heads * 2, 1, torch.bfloat16, 14)


@pytest.mark.parametrize("length", [1, 100, 257, 1000, 4097])
@pytest.mark.parametrize("window", [0, 40, 600])
@pytest.mark.parametrize("table", [0, 50])
def test_a_lone_sequence(qs, length, window, table):
    """Its tables as wide as it needs, and far wider."""
    cache = qs.KVCache(100, 64, 2, 128, "q4_0", "q8_0")
    tables, rows = ref.fill(qs, cache, [length], torch.float16, 15, poison=True)
    wide = torch.full((1, tables.shape[1] + table), -1, dtype=torch.int32, device=DEV)
    wide[:, :tables.shape[1]] = tables
    q = torch.randn((1, 2, 10, 128), generator=torch.Generator().manual_seed(15)).to(DEV, torch.float16)
    y = qs.kv_attention(q, cache, wide, ints(length), window=window)
    want, far = ref.attention64(q, rows, window=window)
    ref.check(y, want, far)


@pytest.mark.parametrize("heads,d,length", [(1, 64, 30000), (1, 256, 20001), (2, 128, 70001)])
def test_a_head_of_many_parts(qs, heads, d, length):
    attend(qs, qs.KVCache(-(-length // 256) + 1, 256, heads, d, "q8_0", "q4_0"), [length], 3 * heads, 2, torch.bfloat16, 17)


@pytest.mark.parametrize("heads,d,t", [(1, 64, 1500), (1, 256, 5000), (3, 192, 1030), (33, 64, 1100)])
@pytest.mark.parametrize("slots", [40, 100000])
def test_many_rows_of_few_and_of_many_slots(qs, heads, d, t, slots):
    """Most of them again and again, and in any order; the last row of a slot stays."""
    cache = qs.KVCache(-(-slots // 1024), 1024, heads, d, "q4_0", "q8_0")
    k, v = ref.keys_values(t, heads, d, torch.float16, 18)
    at = torch.randint(-3, slots, (t,), generator=torch.Generator().manual_seed(t)).to(torch.int32)
    last = {s: i for i, s in enumerate(at.tolist()) if s >= 0}
    qs.kv_write(cache, k, v, at.to(DEV))
    rows = torch.tensor(list(last.values()))
    got = qs.kv_read(cache, at[rows].to(DEV), dtype=torch.float32)
    for x, kind, y in ((k, "q4_0", got[0]), (v, "q8_0", got[1])):
        assert torch.equal(y.cpu().double(), ref.values64(qs, kind, x[rows.to(DEV)]))


def test_out_may_be_q(qs):
    cache = qs.KVCache(80, 16, 2, 64, "q8_0")
    lengths = [400, 3, 0, 700]
    tables, _ = ref.fill(qs, cache, lengths, torch.bfloat16, 16)
    q = torch.randn((4, 3, 12, 64), generator=torch.Generator().manual_seed(16)).to(DEV, torch.bfloat16)
    want = qs.kv_attention(q, cache, tables, ints(*lengths))
    assert qs.kv_attention(q, cache, tables, ints(*lengths), out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spread", [1e-30, 1e-4, 30.0, 2e4])
def test_large_and_small_queries(qs, dtype, spread):
    """Scores from all alike to one that takes all."""
    if dtype == torch.float16 and spread < 1e-4:
        spread = 1e-5
    attend(qs, qs.KVCache(20, 16, 2, 128, "q8_0", "q8_0"), [200, 50], 4, 1, dtype, 6, spread=spread)
    attend(qs, qs.KVCache(20, 16, 2, 128, "q4_0", "q4_0"), [200, 50], 4, 1, dtype, 6, spread=spread, scale=-0.02)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spread,scale", [(0.0, 0.1), (1.0, 0.0), (1.0, -3.0), (1e-20, 1e20)])
def test_scales_and_queries_of_zeros(qs, dtype, spread, scale):
    attend(qs, qs.KVCache(70, 16, 2, 64, "q8_0", "q4_0"), [300, 1, 0, 700], 6, 2, dtype, 19, spread=spread, scale=scale)


@pytest.mark.parametrize("window", [2 ** 31 - 2, 2 ** 31, 2 ** 63, 2 ** 64 + 1])
def test_windows_longer_than_all(qs, window):
    attend(qs, qs.KVCache(70, 16, 2, 64, "q8_0", "q4_0"), [300, 1, 0, 700], 6, 2, torch.bfloat16, 20, window=window)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e3])
@pytest.mark.parametrize("kind", TYPES)
def test_large_and_small_values(qs, size, kind):
    """Values whose steps change by orders along a sequence: the smallest first, then the largest in its middle."""
    cache = qs.KVCache(10, 16, 1, 64, kind)
    k, v = ref.keys_values(150, 1, 64, torch.float32, 7)
    v[:70] *= 1e-3
    v *= size
    qs.kv_write(cache, k, v, torch.arange(150, dtype=torch.int32, device=DEV))
    q = torch.randn((1, 1, 4, 64), generator=torch.Generator().manual_seed(8)).to(DEV)
    for length in (60, 150):
        y = qs.kv_attention(q, cache, torch.arange(10, dtype=torch.int32, device=DEV)[None], ints(length))
        rows = [(ref.values64(qs, kind, k[:length]), ref.values64(qs, kind, v[:length]))]
        want, far = ref.attention64(q, rows, offset=8.0 if kind == "q4_0" else 0.0, wide=True)
        ref.check(y, want, far)


def test_lengths_and_pages_that_are_not(qs):
    """Lengths below 0 and over the table, pages that are not in the cache: seen by no query."""
    cache = qs.KVCache(8, 16, 1, 64, "q8_0")
    k, v = ref.keys_values(128, 1, 64, torch.bfloat16, 9)
    qs.kv_write(cache, k, v, torch.arange(128, dtype=torch.int32, device=DEV))
    q = torch.randn((5, 1, 2, 64), generator=torch.Generator().manual_seed(9)).to(DEV, torch.bfloat16)
    tables = ints(0, 1, 2, 3, 1, 2, 3, 4, 3, -1, 5, 8, -2 ** 31, 2 ** 31 - 1, 6, 7, -1, -1, -1, -1).view(5, 4)
    y = qs.kv_attention(q, cache, tables, ints(-3, 2 ** 31 - 1, 60, 64, 64))
    k64, v64 = ref.values64(qs, "q8_0", k), ref.values64(qs, "q8_0", v)
    at = [torch.arange(0), torch.arange(16, 80), torch.cat([torch.arange(48, 64), torch.arange(80, 96)]), torch.arange(96, 128),
          torch.arange(0)]
    want, far = ref.attention64(q, [(k64[i], v64[i]) for i in at])
    ref.check(y, want, far)
    assert not y[0].any() and not y[4].any()


def test_unseen_positions_do_not_matter(qs):
    """NaN in the keys and values of positions that an earlier new token, a window or a length leaves out."""
    cache = qs.KVCache(9, 16, 1, 64, "q8_0", "q4_0")
    tables, rows = ref.fill(qs, cache, [100], torch.bfloat16, 10)
    q = torch.randn((1, 4, 2, 64), generator=torch.Generator().manual_seed(10)).to(DEV, torch.bfloat16)
    bad = torch.full((1, 1, 64), math.nan, device=DEV)
    for window in (0, 20):
        y = qs.kv_attention(q, cache, tables, ints(100), window=window)
        want, far = ref.attention64(q, rows, window=window, offset=8.0)
        ref.check(y, want, far)
        held = cache.data.clone()
        for position in ([98, 99] + ([0, 60, 75] if window else [])):
            qs.kv_write(cache, bad, bad, cache.slots(tables, ints(position)[None])[0])
        z = qs.kv_attention(q, cache, tables, ints(100), window=window)
        assert z[0, 2:].isnan().all()
        # a NaN step among a step's values changes the power of two that p is taken to: f32's last bits
        ref.check(z[:, :2], want[:, :2], far[:, :2])
        cache.data.copy_(held)


def test_queries_in_any_layout(qs):
    heads, d, b, n = 2, 64, 3, 2
    cache = qs.KVCache(9, 16, heads, d, "q8_0")
    tables, rows = ref.fill(qs, cache, [40, 3, 20], torch.bfloat16, 11)
    lengths = ints(40, 3, 20)
    fused = torch.randn((b * n, 1000), generator=torch.Generator().manual_seed(11)).to(DEV, torch.bfloat16)
    w = 4 * d
    for q in (fused[:, 8:8 + w].view(b, n, 4, d), fused[:, 3:3 + w].view(b, n, 4, d), fused[:, :w].view(n, b, 4, d).transpose(0, 1),
              fused[:, :w].view(b, n, d, 4).transpose(2, 3), fused[:1, :w].view(1, 1, 4, d).expand(b, n, 4, d)):
        y = qs.kv_attention(q, cache, tables, lengths)
        assert torch.equal(y, qs.kv_attention(q.contiguous(), cache, tables, lengths))
        want, far = ref.attention64(q, rows)
        ref.check(y, want, far)
    q = fused[:b, 16:16 + w].view(b, 4, d)
    y = qs.kv_attention(q, cache, tables, lengths)
    assert torch.equal(y, qs.kv_attention(q.contiguous()[:, None], cache, tables, lengths)[:, 0])
    wide = torch.full((b, 8), -1, dtype=torch.int32, device=DEV)
    wide[:, ::2][:, :tables.shape[1]] = tables
    twice = torch.stack([lengths, lengths], 1)[:, 0]
    assert torch.equal(y, qs.kv_attention(q, cache, wide[:, ::2][:, :tables.shape[1]], twice))
    out = torch.full_like(y, 7)
    assert qs.kv_attention(q, cache, tables, lengths, out=out) is out and torch.equal(out, y)


def test_over_four_gigabytes(qs):
    """Pages past 2^32 bytes."""
    cache = qs.KVCache(1030, 1024, 8, 256, "q8_0", "q8_0")
    assert cache.data.numel() > 2 ** 32
    pages = torch.tensor([1029, 0, 1028, 985, 986, 987])
    tables, rows = ref.fill(qs, cache, [2500, 70], torch.bfloat16, 12, pages=pages)
    q = torch.randn((2, 1, 8, 256), generator=torch.Generator().manual_seed(12)).to(DEV, torch.bfloat16)
    want, far = ref.attention64(q, rows)
    ref.check(qs.kv_attention(q, cache, tables, ints(2500, 70)), want, far)
    slots = cache.slots(tables[:1], torch.arange(2500, device=DEV)[None])[0]
    assert torch.equal(qs.kv_read(cache, slots, dtype=torch.float32)[0].cpu().double(), rows[0][0])


def test_python_refuses(qs):
    """Types, shapes, places and gradients."""
    cache = qs.KVCache(2, 16, 2, 64)
    x, slots, q = torch.ones((3, 2, 64), device=DEV), ints(0, 1, 2), torch.ones((1, 4, 64), device=DEV)
    tables, lengths = ints(0, 1).view(1, 2), ints(3)
    write = lambda k=x, v=x, s=slots: qs.kv_write(cache, k, v, s)  # noqa: E731
    for call, word in ((lambda: write(k=x.double()), "dtype"), (lambda: write(v=x.half()), "alike"), (lambda: write(k=x[:2]), "rows"),
                       (lambda: write(s=slots[:2]), "rows"), (lambda: write(s=slots.long()), "int32"), (lambda: write(k=x.cpu()), "is on cpu"),
                       (lambda: write(s=slots.cpu()), "is on cpu"), (lambda: write(v=x[:, :1]), "must be"), (lambda: write(k=x[0]), "must be"),
                       (lambda: write(k=x.clone().requires_grad_()), "requires a gradient"),
                       (lambda: write(v=x.clone().requires_grad_()), "requires a gradient"), (lambda: qs.kv_read(cache, slots.long()), "int32"),
                       (lambda: qs.kv_read(cache, slots.cpu()), "is on cpu"), (lambda: qs.kv_read(cache, slots, dtype=torch.int8), "dtype")):
        with pytest.raises(ValueError, match=word):
            call()
    attend = lambda q=q, t=tables, n=lengths, **k: qs.kv_attention(q, cache, t, n, **k)  # noqa: E731
    for call, word in ((lambda: attend(q=q.double()), "dtype"), (lambda: attend(q=q[0]), "q must be"), (lambda: attend(q=q[:, :3]), "heads"),
                       (lambda: attend(q=q[:, :0]), "heads"), (lambda: attend(q=torch.ones((1, 4, 128), device=DEV)), "heads"),
                       (lambda: attend(q=torch.ones((1, 17, 4, 64), device=DEV)), "at most 16"), (lambda: attend(q=q.cpu()), "is on cpu"),
                       (lambda: attend(t=tables.long()), "int32"), (lambda: attend(t=tables[0]), "int32"), (lambda: attend(t=tables.cpu()), "is on cpu"),
                       (lambda: attend(n=lengths.long()), "int32"), (lambda: attend(n=ints(1, 2)), "1 sequences"),
                       (lambda: attend(t=tables.view(2, 1)), "1 sequences"), (lambda: attend(window=-1), "window"),
                       (lambda: attend(out=torch.ones((1, 4, 64), device=DEV).half()), "out must be"),
                       (lambda: attend(out=torch.ones((1, 4, 128), device=DEV)[..., :64]), "out must be"),
                       (lambda: attend(q=q.clone().requires_grad_()), "requires a gradient"),
                       (lambda: attend(out=q.clone().requires_grad_()), "requires a gradient")):
        with pytest.raises(ValueError, match=word):
            call()
    with pytest.raises(qs.QuantSpecError, match="query heads"):
        attend(q=torch.ones((1, 258, 64), device=DEV))
    with torch.no_grad():
        write(k=x.clone().requires_grad_())
        attend(q=q.clone().requires_grad_())


def test_a_cache_stays_what_it_is(qs):
    cache = qs.KVCache(2, 16, 1, 64)
    for name in ("data", "pages", "page_size", "heads", "k_type"):
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, getattr(cache, name))


def test_threads_share_a_cache(qs):
    """Reads from several threads at once, each on a stream of its own: the bits of a call alone."""
    cache = qs.KVCache(60, 16, 2, 64, "q8_0", "q4_0")
    calls = []
    for i, lengths in enumerate(([300], [20, 40], [5] * 8, [400, 1, 7])):
        tables = torch.randint(0, 60, (len(lengths), 30), generator=torch.Generator().manual_seed(i)).to(DEV, torch.int32)
        q = torch.randn((len(lengths), 6, 64), generator=torch.Generator().manual_seed(i)).to(DEV, torch.bfloat16)
        calls.append((q, tables, ints(*lengths)))
    k, v = ref.keys_values(960, 2, 64, torch.bfloat16, 17)
    qs.kv_write(cache, k, v, torch.arange(960, dtype=torch.int32, device=DEV))
    wants = [qs.kv_attention(q, cache, t, n) for q, t, n in calls]
    torch.cuda.synchronize()
    faults = []

    def work(i):
        try:
            q, t, n = calls[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    y = qs.kv_attention(q, cache, t, n)
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(y, wants[i]):
                        faults.append(i)
        except BaseException as e:          # noqa: BLE001 - shown by the test's own thread
            faults.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    assert not any(th.is_alive() for th in threads) and not faults, faults


# ---- streams and graphs ----

def test_another_stream(qs):
    cache = qs.KVCache(20, 16, 2, 128, "q8_0", "q4_0")
    q, tables, y = attend(qs, cache, [100, 60], 8, 1, torch.bfloat16, 13)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        z = [qs.kv_attention(q, cache, tables, ints(100, 60)) for _ in range(10)]
    s.synchronize()
    assert all(torch.equal(x.view_as(y), y) for x in z)


def test_a_decode_step_in_a_graph(qs):
    """Write and attention captured once, replayed over new tokens and lengths, with eager calls between; a
    second graph of the same cache beside it."""
    heads, d, hq, b = 2, 64, 6, 3
    cache, eager = (qs.KVCache(30, 16, heads, d, "q8_0", "q8_0") for _ in range(2))
    lengths = [30, 0, 77]
    tables = torch.arange(30, dtype=torch.int32, device=DEV).view(3, 10)
    for c in (cache, eager):
        for i, n in enumerate(lengths):
            k, v = ref.keys_values(n, heads, d, torch.bfloat16, 20 + i)
            qs.kv_write(c, k, v, c.slots(tables[i:i + 1], torch.arange(n, device=DEV)[None])[0])
    q, k, v = (torch.zeros((b, h, d), dtype=torch.bfloat16, device=DEV) for h in (hq, heads, heads))
    at, n = ints(*lengths), ints(1, 1, 1)

    def step(c, q, k, v, at):
        qs.kv_write(c, k, v, c.slots(tables, at[:, None])[:, 0].contiguous())
        return qs.kv_attention(q, c, tables, at + 1)

    kept = cache.data.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, q, k, v, at)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step(cache, q, k, v, at))
    cache.data.copy_(kept)
    for i in range(6):
        g = torch.Generator().manual_seed(100 + i)
        new = [torch.randn(x.shape, generator=g).to(DEV, torch.bfloat16) for x in (q, k, v)]
        for x, y in zip((q, k, v), new):
            x.copy_(y)
        graphs[i % 2].replay()
        want = step(eager, *new, at)
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want) and torch.equal(cache.data, eager.data), i
        at += n
