"""A feed-forward block on packed weights, as a server runs it: requests with
and without low-rank adapters in one batch.

    python examples/packed_ffn.py                              # random weights, quantized here
    python examples/packed_ffn.py --gguf model-Q4_K_M.gguf --block 3

    rows, h = norm of (x + h), in 8 bits      rms_norm_q8
    g, u    = rows gate^T, rows up^T          packed_linear, up with each row's adapter
    y       = (silu(g) * u) down^T            packed_linear, which takes its rows to 8 bits first

Prints the error against the same block in 64 bits (with random weights) and
the GPU time of a call, captured in a graph, for each number of rows.
"""

from __future__ import annotations

import argparse
import importlib
import sys
from dataclasses import dataclass
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch

qs = importlib.import_module("quant-studio_amd")
DEV = "cuda:0"


@dataclass
class Ffn:
    norm: torch.Tensor          # (k,) float32
    gate: qs.PackedWeight
    up: qs.PackedWeight
    down: qs.PackedWeight
    adapters: qs.AdapterBank | None = None      # of up

    def __call__(self, x, h, ids=None):
        """(y, x + h) for rows x (t, k) and the residual h; ids: each row's adapter, -1 for none."""
        rows, h = qs.rms_norm_q8(x, self.norm, residual=h)
        bank = None if ids is None else self.adapters
        gate = qs.packed_linear(rows, self.gate)
        up = qs.packed_linear(rows, self.up, adapters=bank, ids=ids)
        return qs.packed_linear(torch.nn.functional.silu(gate) * up, self.down), h


def random_ffn(k: int, ff: int, types=("q4_k", "q4_k", "q6_k"), seed: int = 0):
    """A block of random weights, each packed by its type's quantizer, and the weights."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    dense = [(torch.randn(s, generator=g, device=DEV) / s[1] ** 0.5).to(torch.bfloat16) for s in ((ff, k), (ff, k), (k, ff))]
    packed = [qs.PackedWeight(t, qs.QUANT_TYPES[t].make_kernel(torch.device(DEV), None)(w).view(w.shape[0], -1))
              for t, w in zip(types, dense)]
    return Ffn(1 + 0.1 * torch.randn((k,), generator=g, device=DEV), *packed), dense


def ffn_of_gguf(path: str, block: int) -> Ffn:
    """The block as it lies in a GGUF file."""
    gguf = importlib.import_module("quant-studio_amd.gguf_io").GGUFReader(path)
    names = {int(q.ggml_type): name for name, q in qs.QUANT_TYPES.items()}
    tensors = {t.name: t for t in gguf.tensors}

    def packed(what):
        t = tensors[f"blk.{block}.ffn_{what}.weight"]
        if int(t.ggml_type) not in names:
            raise ValueError(f"{t.name} is {t.ggml_type.name}, not a packed type")
        return qs.PackedWeight(names[int(t.ggml_type)], torch.from_numpy(t.rows().copy()).to(DEV))
    norm = torch.from_numpy(tensors[f"blk.{block}.ffn_norm.weight"].array().copy()).to(DEV, torch.float32)
    return Ffn(norm, packed("gate"), packed("up"), packed("down"))


def random_adapters(k: int, n: int, ranks, seed: int = 1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [((torch.randn((r, k), generator=g, device=DEV) / k ** 0.5).to(torch.bfloat16),
             (0.1 * torch.randn((n, r), generator=g, device=DEV)).to(torch.bfloat16), 1.0) for r in ranks]


def microseconds(call, calls: int = 20) -> float:
    for _ in range(3):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            call()
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / calls)
    return min(times)


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--gguf", help="take the block from this file instead of random weights")
    p.add_argument("--block", type=int, default=0)
    p.add_argument("--embd", type=int, default=2560)
    p.add_argument("--ff", type=int, default=9728)
    p.add_argument("--rows", type=int, nargs="+", default=[1, 8, 64, 512])
    p.add_argument("--ranks", type=int, nargs="+", default=[16, 64, 8, 32])
    a = p.parse_args(argv)
    dense = None
    if a.gguf:
        ffn = ffn_of_gguf(a.gguf, a.block)
    else:
        ffn, dense = random_ffn(a.embd, a.ff)
    k = ffn.norm.shape[0]
    made = random_adapters(k, ffn.up.n, a.ranks)
    ffn.adapters = qs.AdapterBank(made)
    for t in a.rows:
        g = torch.Generator(device=DEV).manual_seed(t)
        x, h = (torch.randn((t, k), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        ids = torch.randint(-1, len(made), (t,), generator=g, device=DEV).to(torch.int32)
        y, total = ffn(x, h, ids)
        line = f"{t:5d} rows: {microseconds(lambda: ffn(x, h, ids)):8.1f} us, {microseconds(lambda: ffn(x, h)):8.1f} without adapters"
        if dense is not None:
            want = plain(ffn, [w.double() for w in dense], made, x, h, ids)
            line += f"; off the unpacked weights' result by {((y.double() - want).norm() / want.norm()).item():.4f}"
        print(line, flush=True)
    return 0


def plain(ffn: Ffn, weights, adapters, x, h, ids):
    """The block in 64 bits with these gate, up and down."""
    gate, up, down = weights
    s = x.double() + h.double()
    s = s * torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6) * ffn.norm.double()
    u = s @ up.T
    for i, (a, b, c) in enumerate(adapters):
        mine = ids == i
        u[mine] += c * (s[mine] @ a.double().T @ b.double().T)
    return (torch.nn.functional.silu(s @ gate.T) * u) @ down.T


if __name__ == "__main__":
    raise SystemExit(main())
