"""Calls from several threads at once, each on a stream of its own, on one weight
and one bank: the bits of a call alone."""

from __future__ import annotations

import threading

import pytest
import torch

import packed_ref as ref
from test_gpu_packed_linear import DEV, make_adapters

pytestmark = pytest.mark.gpu


def test_threads_share_a_weight(qs):
    n, k, threads = 1030, 512, 6
    weight = qs.PackedWeight("q4_k", torch.from_numpy(ref.random_packed("q4_k", n, k, 1)).to(DEV))
    bank = qs.AdapterBank([(a.to(DEV), b.to(DEV), c) for a, b, c in make_adapters([16, 40], n, k, torch.bfloat16, 1)])
    norm = torch.linspace(0.5, 1.5, k, device=DEV)
    inputs, wants, faults = [], [], []

    def layer(x, ids):
        rows, h = qs.rms_norm_q8(x, norm, residual=x)
        return qs.packed_linear(rows, weight, adapters=bank, ids=ids), h

    for i in range(threads):
        t = (1, 5, 40, 300, 520, 700)[i]
        x = torch.randn((t, k), generator=torch.Generator().manual_seed(i)).to(DEV, torch.bfloat16)
        inputs.append((x, (torch.arange(t, device=DEV) % 3 - 1).to(torch.int32)))
        wants.append(layer(*inputs[-1]))
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for j in range(20):
                    got = layer(*inputs[i])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, wants[i])):
                        faults.append((i, j))
                    with pytest.raises(qs.QuantSpecError, match="multiple of 32"):      # a message of this thread's own
                        qs.q8_rows(inputs[i][0][:, :40 + 8 * (i % 2) + 1])
        except BaseException as e:          # noqa: BLE001 - shown by the test's own thread
            faults.append((i, repr(e)))

    all_of_them = [threading.Thread(target=work, args=(i,)) for i in range(threads)]
    for th in all_of_them:
        th.start()
    for th in all_of_them:
        th.join(60)
    assert not any(th.is_alive() for th in all_of_them) and not faults, faults
