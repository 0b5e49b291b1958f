"""Products of 8-bit rows with packed weights, and the low-rank adapters
beside them, against a plain 64-bit computation."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda:0"


def rows_on(qs, q, s):
    return qs.Q8Rows(torch.from_numpy(q).to(DEV), torch.from_numpy(s).to(DEV))


def check(got, want, bound, what):
    g = got.double().cpu().numpy()
    assert g.shape == want.shape, what
    worst = np.max(np.abs(g - want) / bound) if want.size else 0.0
    print(f"{what}: worst error {worst:.3f} of its bound", flush=True)
    assert np.isfinite(g).all() and worst <= 1.0, what


@pytest.mark.parametrize("qtype", sorted(ref.BYTES))
def test_decoded_values_one_by_one(qs, qtype):
    """Row i of the identity picks value i of every weight row."""
    k, n = 256, 37
    packed = ref.random_packed(qtype, n, k, 3)
    q, s = np.eye(k, dtype=np.int8), np.ones((k, k // 32), np.float32)
    print(qtype, flush=True)
    w = qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV))
    rows = rows_on(qs, q, s)
    want, bound = ref.linear64(qtype, packed, q, s, "f32")
    check(qs.packed_linear(rows, w, dtype=torch.float32), want, bound, f"{qtype} all rows")
    for i in (0, 100, 255):
        check(qs.packed_linear(rows[i:i + 1], w, dtype=torch.float32), want[i:i + 1], bound[i:i + 1], f"{qtype} row {i}")


@pytest.mark.parametrize("t,n,blocks,dtype", [
    (1, 1, 1, "f32"), (1, 67, 5, "bf16"), (2, 33, 3, "f16"), (3, 130, 2, "f32"), (4, 31, 9, "bf16"),
    (5, 95, 3, "f32"), (32, 32, 2, "bf16"), (33, 129, 3, "f16"), (61, 260, 2, "f32"), (200, 257, 2, "bf16")])
@pytest.mark.parametrize("qtype", sorted(ref.BYTES))
def test_small_shapes(qs, qtype, t, n, blocks, dtype):
    """Rows and columns that no tile divides; row lengths of one block up (for
    32-value blocks lengths that are odd multiples of 32)."""
    k = blocks * ref.BLOCK[qtype]
    packed = ref.random_packed(qtype, n, k, t * 7 + n)
    q, s = ref.random_rows(t, k, t + n)
    print(qtype, t, n, k, dtype, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)), dtype=TORCH[dtype])
    check(y, *ref.linear64(qtype, packed, q, s, dtype), f"{qtype} {t}x{n}x{k} {dtype}")


@pytest.mark.parametrize("qtype,t,n,k,dtype", [
    ("q4_k", 129, 12289, 256, "f32"), ("q6_k", 129, 12289, 256, "bf16"), ("q8_0", 300, 9000, 288, "f16"),
    ("q2_k", 257, 8193, 512, "bf16"), ("iq2_xs", 513, 4097, 512, "f16"), ("q5_1", 1025, 2049, 160, "bf16"),
    ("q4_k", 700, 6000, 768, "bf16"), ("q4_0", 511, 12000, 96, "bf16"), ("iq3_s", 640, 5001, 256, "f32"),
    ("q6_k", 16, 4096, 9728, "f32"), ("q4_k", 1, 9728, 2560, "f32"), ("q5_k", 2, 2560, 9728, "f32")])
def test_larger_shapes(qs, qtype, t, n, k, dtype):
    packed = ref.random_packed(qtype, n, k, n)
    q, s = ref.random_rows(t, k, t)
    print(qtype, t, n, k, dtype, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)), dtype=TORCH[dtype])
    check(y, *ref.linear64(qtype, packed, q, s, dtype), f"{qtype} {t}x{n}x{k} {dtype}")


@pytest.mark.parametrize("t", [1, 4, 6, 40, 300])
def test_a_row_does_not_depend_on_its_neighbours(qs, t):
    """NaN and infinite scales, zero rows and extreme codes stay in their rows."""
    qtype, n, k = "q4_k", 2100, 512
    packed = ref.random_packed(qtype, n, k, 1)
    q, s = ref.random_rows(t, k, 2)
    q[0] = -128
    s[-1, 3] = np.nan
    if t > 2:
        s[1, 0] = np.inf
        q[2] = 0
    print(t, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)),
                         dtype=torch.float32).cpu().numpy()
    assert np.isnan(y[-1]).all()
    keep = [i for i in range(t - 1) if not (t > 2 and i == 1)]
    if t > 2:
        assert not np.isfinite(y[1]).any() and (y[2] == 0).all()
    want, bound = ref.linear64(qtype, packed, q[keep], s[keep], "f32")
    if keep:
        assert (np.abs(y[keep] - want) <= bound).all()


def test_empty_and_output_buffers(qs):
    packed = torch.from_numpy(ref.random_packed("q8_0", 40, 64, 1)).to(DEV)
    w = qs.PackedWeight("q8_0", packed)
    none = qs.Q8Rows(torch.empty((0, 64), dtype=torch.int8, device=DEV), torch.empty((0, 2), device=DEV))
    assert qs.packed_linear(none, w).shape == (0, 40)
    assert qs.packed_linear(none, qs.PackedWeight("q8_0", packed[:0])).shape == (0, 0)
    q, s = ref.random_rows(9, 64, 5)
    rows = rows_on(qs, q, s)
    out = torch.full((9, 40), 7.0, dtype=torch.float16, device=DEV)
    assert qs.packed_linear(rows, w, dtype=torch.float16, out=out) is out
    assert torch.equal(out, qs.packed_linear(rows, w, dtype=torch.float16))
    # a slice of the weight's rows is a weight; a slice of the rows is rows
    part = qs.packed_linear(rows[2:5], qs.PackedWeight("q8_0", packed[3:21]), dtype=torch.float32)
    want, bound = ref.linear64("q8_0", packed[3:21].cpu().numpy(), q[2:5], s[2:5], "f32")
    check(part, want, bound, "slices")


def test_float_rows_go_to_8_bits_first(qs):
    x = torch.randn((7, 256), generator=torch.Generator().manual_seed(1)).to(DEV, torch.bfloat16)
    w = qs.PackedWeight("q6_k", torch.from_numpy(ref.random_packed("q6_k", 50, 256, 1)).to(DEV))
    assert torch.equal(qs.packed_linear(x, w), qs.packed_linear(qs.q8_rows(x), w))


def test_offsets_past_32_bits(qs):
    """A weight of over 2^31 bytes and a result of over 2^31 bytes: the last
    rows and columns are the ones a 32-bit offset would miss."""
    k, n = 9728, 210000                       # 2.17 GB of Q8_0
    part = ref.random_packed("q8_0", 100, k, 4)
    data = torch.from_numpy(part).to(DEV).repeat(n // 100, 1)
    w = qs.PackedWeight("q8_0", data)
    for t in (1, 6):
        q, s = ref.random_rows(t, k, t)
        print("past 32 bits", t, flush=True)
        y = qs.packed_linear(rows_on(qs, q, s), w, dtype=torch.float32)
        want, bound = ref.linear64("q8_0", part, q, s, "f32")
        check(y[:, -100:], want, bound, f"last columns, {t} rows")
        assert torch.equal(y[:, :100], y[:, -100:])
    del data, w
    t, n, k = 5400, 200000, 32                # 2.16 GB of bf16 results
    part = ref.random_packed("q4_0", 100, k, 5)
    w = qs.PackedWeight("q4_0", torch.from_numpy(part).to(DEV).repeat(n // 100, 1))
    q, s = ref.random_rows(t, k, 3)
    print("past 32 bits, result", flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), w)
    want, bound = ref.linear64("q4_0", part, q[-50:], s[-50:], "bf16")
    check(y[-50:, -100:], want, bound, "last rows and columns")


def make_adapters(ranks, n, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    made = []
    for i, r in enumerate(ranks):
        a = (torch.randn((r, k), generator=g) / k ** 0.5).to(dtype)
        b = torch.randn((n, r), generator=g).to(dtype)
        made.append((a, b, 0.25 * (i + 1)))
    return made


def run_adapters(qs, qtype, t, n, k, dtype, out, ranks, ids, seed=0):
    packed = ref.random_packed(qtype, n, k, seed)
    q, s = ref.random_rows(t, k, seed + 1)
    made = make_adapters(ranks, n, k, TORCH[dtype], seed)
    bank = qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in made])
    ids = np.asarray(ids, np.int32)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)), dtype=TORCH[out],
                         adapters=bank, ids=torch.from_numpy(ids).to(DEV))
    want, bound = ref.linear64(qtype, packed, q, s, out)
    delta, more = ref.adapters64(ref.rows64(q, s), [(a.double().numpy(), b.double().numpy(), c) for a, b, c in made],
                                 ids, n)
    check(y, want + delta, bound + more + ref.ROUND[out] * np.abs(delta), f"{qtype} {t}x{n}x{k} {dtype} {out} {ranks[:4]}")
    return y, bank


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("t,n,k", [(1, 70, 256), (3, 33, 512), (4, 515, 256), (17, 64, 512), (40, 300, 256), (150, 5000, 512),
                                   (300, 8193, 256), (513, 1025, 768)])
def test_adapters_of_each_row(qs, t, n, k, dtype, out):
    """Ranks from 1 up, odd ones among them; rows without an adapter, and ids
    outside the bank, which mean none too."""
    ranks = [1, 16, 5, 64, 8, 33]
    ids = np.random.default_rng(t).integers(-1, len(ranks) + 1, t)
    ids[0] = 3
    if t > 2:
        ids[1], ids[2] = -2 ** 31, 2 ** 31 - 1
    print(t, n, k, dtype, out, flush=True)
    run_adapters(qs, "q4_k", t, n, k, dtype, out, ranks, ids)


@pytest.mark.parametrize("qtype,t,n,k,dtype", [("q6_k", 700, 2560, 1024, "bf16"), ("q8_0", 300, 4100, 96, "f16"),
                                               ("q4_0", 2000, 3000, 128, "bf16")])
def test_adapters_of_packed_sequences(qs, qtype, t, n, k, dtype):
    """Sequences one after another: runs of rows with one adapter, of lengths
    from one row up, some without an adapter."""
    rng = np.random.default_rng(t)
    cuts = np.sort(rng.integers(0, t, 9))
    ids = (np.searchsorted(cuts, np.arange(t), side="right") % 7) - 1
    print(qtype, t, n, k, dtype, flush=True)
    run_adapters(qs, qtype, t, n, k, dtype, "bf16" if dtype == "bf16" else "f16", [128, 8, 40, 16, 64, 3], ids)


@pytest.mark.parametrize("t", [1, 20, 300])
def test_rows_without_an_adapter_keep_their_bits(qs, t):
    """A NaN in an adapter stays in its rows, and rows without one come out as without a bank."""
    n, k = 2100, 256
    packed = torch.from_numpy(ref.random_packed("q4_k", n, k, 1)).to(DEV)
    rows = rows_on(qs, *ref.random_rows(t, k, 2))
    a, b, c = make_adapters([16], n, k, torch.bfloat16, 1)[0]
    a[3, 5] = float("nan")
    bank = qs.AdapterBank([(a.to(DEV), b.to(DEV), c)])
    ids = torch.full((t,), -1, dtype=torch.int32, device=DEV)
    w = qs.PackedWeight("q4_k", packed)
    plain = qs.packed_linear(rows, w)
    assert torch.equal(qs.packed_linear(rows, w, adapters=bank, ids=ids), plain)
    ids[t // 2] = 0
    y = qs.packed_linear(rows, w, adapters=bank, ids=ids)
    assert torch.isnan(y[t // 2]).all()
    keep = [i for i in range(t) if i != t // 2]
    assert torch.equal(y[keep], plain[keep])


def test_streams_graphs_and_repeats(qs):
    """Work on a side stream, calls that share no buffers at once, and a graph
    replayed with the program's own work between: the same bits every time."""
    n, k = 1300, 512
    w = qs.PackedWeight("q5_k", torch.from_numpy(ref.random_packed("q5_k", n, k, 1)).to(DEV))
    bank = qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in make_adapters([16, 40], n, k, torch.bfloat16, 1)])
    x = torch.randn((90, k), generator=torch.Generator().manual_seed(3)).to(DEV, torch.bfloat16)
    weight = torch.ones((k,), device=DEV)
    ids = (torch.arange(90, device=DEV) % 3 - 1).to(torch.int32)

    def layer():
        rows, h = qs.rms_norm_q8(x, weight, residual=x)
        return qs.packed_linear(rows, w, adapters=bank, ids=ids), h

    want = [v.clone() for v in layer()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        many = [layer() for _ in range(5)]
    here = [layer() for _ in range(5)]
    torch.cuda.synchronize()
    for got in many + here:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = layer()
    for i in range(4):
        y.zero_(), h.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = layer()
        assert torch.equal(y, want[0]) and torch.equal(h, want[1]) and torch.equal(eager[0], want[0]), i
