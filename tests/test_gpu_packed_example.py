"""The example that runs the operators on packed weights together."""

from __future__ import annotations

import importlib
import importlib.util
import sys
from pathlib import Path

import pytest
import torch

from dequant import dequantize

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(qs):
    spec = importlib.util.spec_from_file_location("packed_ffn", Path(__file__).resolve().parent.parent / "examples" / "packed_ffn.py")
    module = importlib.util.module_from_spec(spec)
    sys.modules["packed_ffn"] = module      # its dataclass looks its module up
    spec.loader.exec_module(module)
    return module


def unpacked(w):
    return torch.from_numpy(dequantize(w.name, w.data.cpu().numpy(), w.n)).to("cuda:0")


@pytest.mark.parametrize("t", [1, 7, 50, 130])
def test_block(example, t):
    """Against the block in 64 bits on the values that the packed weights hold.
    What is left are the rows in 8 bits: steps of max|u| / 127 of 32 values,
    which are off by 1/sqrt(12) of a step: 0.7% where the largest is 3 times the
    rms (the norm's rows, once in the gate and once in up), 1.1% at 5 times (the
    down product's rows), with bf16's 0.2% under 1.6% together; twice that is allowed."""
    k, ff = 512, 1280
    ffn, _ = example.random_ffn(k, ff)
    made = example.random_adapters(k, ff, [16, 24, 8])
    ffn.adapters = example.qs.AdapterBank(made)
    g = torch.Generator(device="cuda:0").manual_seed(t)
    x, h = (torch.randn((t, k), generator=g, device="cuda:0").to(torch.bfloat16) for _ in range(2))
    ids = torch.randint(-1, 3, (t,), generator=g, device="cuda:0").to(torch.int32)
    weights = [unpacked(w) for w in (ffn.gate, ffn.up, ffn.down)]
    print(t, flush=True)
    y, total = ffn(x, h, ids)
    want = example.plain(ffn, weights, made, x, h, ids)
    off = ((y.double() - want).norm() / want.norm()).item()
    print("off by", off)
    assert off <= 0.032
    assert torch.equal(total, x + h)
    y0, _ = ffn(x, h)
    want0 = example.plain(ffn, weights, [], x, h, ids)
    assert ((y0.double() - want0).norm() / want0.norm()).item() <= 0.032


def test_block_of_a_file(example, tmp_path):
    """The same bits from a GGUF file's tensors as from the quantizers'."""
    gguf = importlib.import_module("quant-studio_amd.gguf_io")
    types = importlib.import_module("quant-studio_amd.gguf_types")
    ffn, _ = example.random_ffn(256, 512)
    tensors = []
    for what, w in (("gate", ffn.gate), ("up", ffn.up), ("down", ffn.down)):
        tensors.append((f"blk.2.ffn_{what}.weight", (w.k, w.n), types.GGMLQuantizationType(w.ggml_type), w.data.cpu().numpy()))
    tensors.append(("blk.2.ffn_norm.weight", (256,), types.GGMLQuantizationType.F32, ffn.norm.cpu().numpy()))
    path = tmp_path / "block.gguf"
    gguf.write_gguf(path, "llama", [], tensors)
    again = example.ffn_of_gguf(str(path), 2)
    x = torch.randn((3, 256), generator=torch.Generator().manual_seed(1)).to("cuda:0", torch.bfloat16)
    assert all(torch.equal(a, b) for a, b in zip(ffn(x, x), again(x, x)))


def test_command(example, capsys):
    assert example.main(["--embd", "256", "--ff", "512", "--rows", "1", "40", "--ranks", "8"]) == 0
    assert "40 rows" in capsys.readouterr().out
