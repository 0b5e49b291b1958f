"""Products with packed weights at the sizes where a different tile, or a
different split of the groups, costs least: each against a 64-bit computation
with the bounds of the other products' tests."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, TORCH, check, make_adapters, rows_on

pytestmark = pytest.mark.gpu

# tiles that decode the weight, of 32 and of 64 columns, in 1 to 8 parts with a
# shorter last one; above 128 rows and a round of such tiles, or 512 rows,
# laid-out factors in tiles of 64 x 64, of 128 x 128 by eight waves and by four
SHAPES = [(12, 70, 4352), (33, 2047, 768), (61, 1024, 2560), (64, 2048, 512), (65, 2050, 1312), (100, 4100, 2336),
          (128, 2304, 1056), (70, 8200, 544), (150, 8192, 512), (192, 1500, 1056), (193, 600, 800), (140, 8300, 256),
          (300, 1500, 544), (500, 2048, 256), (513, 640, 288), (700, 1030, 544),
          (129, 515, 1312), (1030, 2100, 256), (2000, 3100, 96), (400, 1000, 800)]


@pytest.mark.parametrize("t,n,k", SHAPES)
def test_tiles_and_parts(qs, t, n, k):
    for qtype in ("q8_0", "q4_1") if k % 256 else ("q4_k", "q6_k", "iq2_xs"):
        packed = ref.random_packed(qtype, n, k, t)
        q, s = ref.random_rows(t, k, n)
        print(qtype, t, n, k, flush=True)
        y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)), dtype=torch.float16)
        check(y, *ref.linear64(qtype, packed, q, s, "f16"), f"{qtype} {t}x{n}x{k}")


@pytest.mark.parametrize("t,n,k", [s for s in SHAPES if s[0] * s[1] < 2 << 20])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_adapters_with_them(qs, dtype, t, n, k):
    """Rows of one adapter next to rows of all; steps of 32 ranks go round the waves that share a tile."""
    qtype = "q5_1" if k % 256 else "q2_k"
    packed = ref.random_packed(qtype, n, k, t)
    q, s = ref.random_rows(t, k, n)
    made = make_adapters([72, 8, 130, 33], n, k, TORCH[dtype], 5)
    bank = qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in made])
    ids = np.where(np.arange(t) < t // 2, 2, np.arange(t) % 6 - 1).astype(np.int32)
    print(dtype, t, n, k, flush=True)
    y = qs.packed_linear(rows_on(qs, q, s), qs.PackedWeight(qtype, torch.from_numpy(packed).to(DEV)), dtype=torch.float32,
                         adapters=bank, ids=torch.from_numpy(ids).to(DEV))
    want, bound = ref.linear64(qtype, packed, q, s, "f32")
    delta, more = ref.adapters64(ref.rows64(q, s), [(a.double().numpy(), b.double().numpy(), c) for a, b, c in made], ids, n)
    check(y, want + delta, bound + more + ref.ROUND["f32"] * np.abs(delta), f"{dtype} {t}x{n}x{k}")
