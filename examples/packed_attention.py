"""An attention block on packed weights with a quantised key-value cache, as a
server runs it: sequences of any lengths in the pages of one cache.

    python examples/packed_attention.py                        # random weights, quantized here
    python examples/packed_attention.py --gguf model-Q4_K_M.gguf --block 3 --heads 32

    rows, h  = norm of (x + h), in 8 bits              rms_norm_q8
    q, k, v  = rows Wq^T, rows Wk^T, rows Wv^T          packed_linear
    q, k     turned by their positions
    cache   <- k, v, quantised                          kv_write
    a        = attention of q over the cache            kv_attention
    y        = a Wo^T                                   packed_linear

A prompt goes through in runs of 16 tokens, which kv_attention takes at once. Prints
the error against the same block in 64 bits (with random weights) and the GPU time
of a decode step, captured in a graph, for each number of sequences.
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


def turned(x, positions, base: float = 10000.0):
    """x (t, heads, d) with each pair (i, i + d / 2) turned by its position's angle."""
    half = x.shape[-1] // 2
    angle = positions[:, None, None] * base ** (-torch.arange(half, device=x.device, dtype=positions.dtype) / half)
    c, s, (a, b) = angle.cos(), angle.sin(), x.to(positions.dtype).split(half, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@dataclass
class Attention:
    norm: torch.Tensor          # (k,) float32
    q: qs.PackedWeight
    k: qs.PackedWeight
    v: qs.PackedWeight
    o: qs.PackedWeight
    cache: qs.KVCache

    def __call__(self, x, h, tables, lengths):
        """(y, x + h) for n new tokens of each of b sequences: rows x, h (b * n, k), pages
        tables (b, m), lengths (b,) with the new tokens counted."""
        b, d = len(lengths), self.cache.head_dim
        n = len(x) // b
        at = lengths[:, None] - n + torch.arange(n, device=x.device, dtype=torch.int32)
        rows, h = qs.rms_norm_q8(x, self.norm, residual=h)
        q, k, v = (qs.packed_linear(rows, w).view(b * n, -1, d) for w in (self.q, self.k, self.v))
        positions = at.reshape(-1).float()
        q, k = turned(q, positions).to(x.dtype), turned(k, positions).to(x.dtype)
        qs.kv_write(self.cache, k, v, self.cache.slots(tables, at).view(-1))
        a = qs.kv_attention(q.view(b, n, -1, d), self.cache, tables, lengths)
        return qs.packed_linear(a.view(b * n, -1), self.o), h

    def prompt(self, x, h, tables):
        """The block over a whole prompt of each sequence, x and h (b, t, k): y and x + h."""
        b, t, width = x.shape
        ys, hs = [], []
        for i in range(0, t, 16):
            n = min(16, t - i)
            lengths = torch.full((b,), i + n, dtype=torch.int32, device=x.device)
            y, r = self(x[:, i:i + n].reshape(b * n, width), h[:, i:i + n].reshape(b * n, width), tables, lengths)
            ys.append(y.view(b, n, width))
            hs.append(r.view(b, n, width))
        return torch.cat(ys, 1), torch.cat(hs, 1)


def new_cache(sequences: int, positions: int, heads: int, d: int, types, page: int = 64):
    """A cache with room for `positions` of each sequence, and tables of pages in a shuffled order."""
    each = -(-positions // page)
    cache = qs.KVCache(sequences * each, page, heads, d, *types, device=DEV)
    order = torch.randperm(sequences * each, generator=torch.Generator().manual_seed(0))
    return cache, order.view(sequences, each).to(DEV, torch.int32)


def random_weights(width: int, heads: int, kv_heads: int, d: int, types=("q4_k", "q4_k", "q6_k", "q4_k"), seed: int = 0):
    """Norm, packed q, k, v and o, and the four before they were packed."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    shapes = ((heads * d, width), (kv_heads * d, width), (kv_heads * d, width), (width, heads * d))
    dense = [(torch.randn(s, generator=g, device=DEV) / s[1] ** 0.5).to(torch.bfloat16) for s in shapes]
    packed = [qs.PackedWeight(t, qs.QUANT_TYPES[t].make_kernel(torch.device(DEV), None)(w).view(w.shape[0], -1))
              for t, w in zip(types, dense)]
    return 1 + 0.1 * torch.randn((width,), generator=g, device=DEV), packed, dense


def weights_of_gguf(path: str, block: int):
    """Norm and packed q, k, v and o as they lie in a GGUF file."""
    gguf = importlib.import_module("quant-studio_amd.gguf_io").GGUFReader(path)
    names = {int(q.ggml_type): name for name, q in qs.QUANT_TYPES.items()}
    tensors = {t.name: t for t in gguf.tensors}

    def packed(what):
        t = tensors[f"blk.{block}.attn_{what}.weight"]
        if int(t.ggml_type) not in names:
            raise ValueError(f"{t.name} is {t.ggml_type.name}, not a packed type")
        return qs.PackedWeight(names[int(t.ggml_type)], torch.from_numpy(t.rows().copy()).to(DEV))
    norm = torch.from_numpy(tensors[f"blk.{block}.attn_norm.weight"].array().copy()).to(DEV, torch.float32)
    return norm, [packed(w) for w in ("q", "k", "v", "output")]


def plain(norm, weights, x, h, d: int):
    """The block over whole sequences x, h (b, t, k) in 64 bits with these q, k, v and o, nothing quantised."""
    b, t, width = x.shape
    r = x.double() + h.double()
    r = r * torch.rsqrt((r * r).mean(2, keepdim=True) + 1e-6) * norm.double()
    q, k, v = ((r @ w.double().T).view(b * t, -1, d) for w in weights[:3])
    positions = torch.arange(t, device=x.device, dtype=torch.float64).repeat(b)
    q, k, v = (y.view(b, t, -1, d).transpose(1, 2) for y in (turned(q, positions), turned(k, positions), v))
    group = q.shape[1] // k.shape[1]
    s = q @ k.repeat_interleave(group, 1).transpose(2, 3) / d ** 0.5
    s = s.masked_fill(torch.ones((t, t), dtype=torch.bool, device=x.device).triu(1), -torch.inf)
    a = torch.softmax(s, 3) @ v.repeat_interleave(group, 1)
    return a.transpose(1, 2).reshape(b, t, -1) @ weights[3].double().T


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
    p.add_argument("--heads", type=int, default=32)
    p.add_argument("--kv-heads", type=int, default=8)
    p.add_argument("--head-dim", type=int, default=128)
    p.add_argument("--types", nargs=2, default=["q8_0", "q8_0"], help="of the cache's keys and values")
    p.add_argument("--sequences", type=int, nargs="+", default=[1, 16, 64])
    p.add_argument("--context", type=int, default=2048)
    a = p.parse_args(argv)
    d, dense = a.head_dim, None
    if a.gguf:
        norm, packed = weights_of_gguf(a.gguf, a.block)
        d = packed[0].n // a.heads
    else:
        norm, packed, dense = random_weights(a.embd, a.heads, a.kv_heads, d)
    width, kv_heads = norm.shape[0], packed[1].n // d
    g = torch.Generator(device=DEV).manual_seed(1)
    if dense is not None:
        t = min(50, a.context)
        cache, tables = new_cache(2, t, kv_heads, d, a.types)
        x, h = torch.randn((2, 2, t, width), generator=g, device=DEV).to(torch.bfloat16)
        y, _ = Attention(norm, *packed, cache).prompt(x, h, tables)
        want = plain(norm, dense, x, h, d)
        print(f"a prompt of {t} tokens: off the result without quantisation by {((y.double() - want).norm() / want.norm()).item():.4f}",
              flush=True)
    for b in a.sequences:
        cache, tables = new_cache(b, a.context, kv_heads, d, a.types)
        block = Attention(norm, *packed, cache)
        kv = torch.randn((2, a.context * b, kv_heads, d), generator=g, device=DEV).to(torch.bfloat16)
        at = torch.arange(a.context, device=DEV).expand(b, -1)
        qs.kv_write(cache, kv[0], kv[1], cache.slots(tables, at).view(-1))
        x, h = torch.randn((2, b, width), generator=g, device=DEV).to(torch.bfloat16)
        lengths = torch.full((b,), a.context, dtype=torch.int32, device=DEV)
        print(f"{b:4d} sequences of {a.context} positions: {microseconds(lambda: block(x, h, tables, lengths)):8.1f} us a token of each, "
              f"{microseconds(lambda: qs.kv_attention(q_of(block, b, x.dtype), cache, tables, lengths)):8.1f} of it attention", flush=True)
    return 0


def q_of(block: Attention, b: int, dtype):
    return torch.zeros((b, block.q.n // block.cache.head_dim, block.cache.head_dim), dtype=dtype, device=DEV)


if __name__ == "__main__":
    raise SystemExit(main())
