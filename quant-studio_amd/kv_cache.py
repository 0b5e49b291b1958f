"""A quantised key-value cache and the attention over it: the other half of a
layer on packed weights.

    cache = KVCache(pages, 64, kv_heads, head_dim, "q8_0", "q4_0")
    slots = cache.slots(tables, positions)                 # where a step's tokens go
    kv_write(cache, k, v, slots)                           # quantised as they are written
    y = kv_attention(q, cache, tables, lengths)            # one new token of each sequence
    k, v = kv_read(cache, slots)                           # values, for a prompt's attention

The reference ends at the GGUF file and has none of this. Every function is one
call into the gfx950 library (C ABI in include/quant_studio.h) on torch's current
stream; nothing is synchronised, and every failure raises. These are serving
forms: codes carry no gradient, and a tensor that requires one is refused while
gradients are recorded, one with a tangent of forward mode always.
"""

from __future__ import annotations

import ctypes
import math

from . import packed
from .packed import _call, _device_of, _fail, _no_gradient, _same_device, _type_id

_TYPES = {"q8_0": 8, "q4_0": 2}         # QS_TYPE_* of include/quant_studio.h
torch = forward_ad = None


def _lib():
    global torch, forward_ad
    lib = packed._lib()
    torch, forward_ad = packed.torch, packed.forward_ad
    return lib


class _Cache(ctypes.Structure):
    """qs_kv_cache of include/quant_studio.h."""
    _fields_ = [("k_type", ctypes.c_int32), ("v_type", ctypes.c_int32), ("heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("page_size", ctypes.c_int32), ("pages", ctypes.c_int32),
                ("data", ctypes.c_void_p)]


class KVCache:
    """Pages of quantised keys and values on a ROCm device: page_size slots each,
    a slot holds a key and a value of `heads` heads of head_dim values (64, 128,
    192 or 256). k_type, v_type: "q8_0" or "q4_0" (v_type None: as k_type); codes
    and steps are those of the quantizers of these names.

    data: uint8 (pages, bytes of a page), zeros at first, or a tensor to use as it
    is. A page may be copied to another (data[j] = data[i]), of a cache of the same
    sizes too; the order of a page's bytes is the library's own. What a cache is does
    not change: its attributes cannot be set."""

    __slots__ = ("pages", "page_size", "heads", "head_dim", "k_type", "v_type", "data", "_c", "_ref", "_dev", "_work")

    def __init__(self, pages: int, page_size: int, heads: int, head_dim: int, k_type: str = "q8_0",
                 v_type: str | None = None, device=None, data=None):
        lib = _lib()
        v_type = k_type if v_type is None else v_type
        for name in (k_type, v_type):
            if name not in _TYPES:
                raise ValueError(f"KVCache: unsupported type {name!r}: one of {', '.join(sorted(_TYPES))}")
        for name, n in (("pages", pages), ("page_size", page_size), ("heads", heads), ("head_dim", head_dim)):
            if not 0 < n < 1 << 31:
                raise ValueError(f"KVCache: {name} {n} is not in 1..2^31 - 1")
        size = lib.qs_kv_page_bytes(_TYPES[k_type], _TYPES[v_type], heads, head_dim, page_size)
        if size < 0:
            _fail()
        if pages * page_size >= 1 << 31:
            raise ValueError(f"KVCache: {pages} pages of {page_size} slots are 2^31 slots or more")
        if data is None:
            data = torch.zeros((pages, size), dtype=torch.uint8, device="cuda" if device is None else device)
        elif data.dtype != torch.uint8 or tuple(data.shape) != (pages, size) or not data.is_contiguous() \
                or data.data_ptr() % 16:
            raise ValueError(f"KVCache: data must be contiguous uint8 {(pages, size)} on a 16-byte boundary, "
                             f"got {data.dtype} {tuple(data.shape)}")
        self._dev = _device_of(data, "KVCache")
        if device is not None and torch.device(device) not in (data.device, torch.device("cuda")):
            raise ValueError(f"KVCache: data is on {data.device}, not {device}")
        self.pages, self.page_size, self.heads, self.head_dim = pages, page_size, heads, head_dim
        self.k_type, self.v_type, self.data = k_type, v_type, data
        self._c = _Cache(_TYPES[k_type], _TYPES[v_type], heads, head_dim, page_size, pages, data.data_ptr())
        self._ref = ctypes.byref(self._c)
        self._work = {}         # (sequences, new tokens, query heads, table columns) -> workspace bytes

    def __setattr__(self, name, value):
        if hasattr(self, "_work"):      # the last one set
            raise AttributeError(f"KVCache: {name} cannot be set: the calls would go on with what it was")
        object.__setattr__(self, name, value)

    def slots(self, tables, positions):
        """int32 slots of positions (b, n) of sequences whose pages are tables
        (b, m): -1 where a position is negative or past its table, or its page not
        in the cache. Plain torch operations."""
        entry = torch.div(positions, self.page_size, rounding_mode="floor").long()
        held = (positions >= 0) & (entry < tables.shape[1])
        if tables.shape[1] == 0:
            return torch.full_like(positions, -1, dtype=torch.int32)
        page = tables.gather(1, torch.where(held, entry, 0))
        held &= (page >= 0) & (page < self.pages)
        return torch.where(held, page * self.page_size + positions % self.page_size, -1).to(torch.int32)


def _rows(what: str, name: str, x, cache: KVCache):
    """(x, its row stride in bytes): rows of heads * head_dim values in a layout the C call takes."""
    width, esz = cache.heads * cache.head_dim, x.element_size()
    if x.dim() == 3:
        if x.shape[1] != cache.heads or x.shape[2] != cache.head_dim:
            raise ValueError(f"{what}: {name} must be (t, {cache.heads}, {cache.head_dim}), got {tuple(x.shape)}")
    elif x.dim() != 2 or x.shape[1] != width:
        raise ValueError(f"{what}: {name} must be (t, {cache.heads}, {cache.head_dim}) or (t, {width}), got {tuple(x.shape)}")
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, width * esz
    t = x.shape[0]
    dense = x.stride(-1) == 1 and (x.dim() == 2 or x.shape[1] == 1 or x.stride(1) == cache.head_dim)
    if not dense or x.data_ptr() % 16 or (t > 1 and (x.stride(0) < width or x.stride(0) * esz % 16)):
        x = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
    return x, (x.stride(0) if t > 1 else width) * esz


def _ints(what: str, name: str, x, dims: int, dev: int):
    if x.dtype != torch.int32 or x.dim() != dims:
        raise ValueError(f"{what}: {name} must be int32 with {dims} dimension(s), got {x.dtype} {tuple(x.shape)}")
    if x.get_device() != dev:
        _same_device(dev, what, name, x)


def kv_write(cache: KVCache, k, v, slots) -> None:
    """Quantise rows of keys and values into the cache's slots.

    k, v: (t, heads, head_dim), or (t, heads * head_dim), float32 / float16 /
    bfloat16, any strides (layouts the C call does not take are copied first).
    slots: (t,) int32; a row whose slot is not in the cache, such as -1, is left out,
    and of rows with the same slot the last one is written. A NaN, an infinity or a
    step over float16's largest number makes the values of its block of 32 NaN."""
    lib = _lib()
    src = _type_id(k.dtype, "kv_write")
    if k.requires_grad or v.requires_grad or forward_ad._current_level >= 0:
        _no_gradient("kv_write", "k", k)
        _no_gradient("kv_write", "v", v)
    dev = cache._dev
    if k.get_device() != dev or v.get_device() != dev:
        _same_device(dev, "kv_write", "k", k)
        _same_device(dev, "kv_write", "v", v)
    if k.dtype != v.dtype:
        raise ValueError(f"kv_write: k and v must be alike, got {k.dtype} and {v.dtype}")
    _ints("kv_write", "slots", slots, 1, dev)
    t = slots.shape[0]
    if k.shape != (t, cache.heads, cache.head_dim) or v.shape != k.shape or not k.is_contiguous() or not v.is_contiguous() \
            or (k.data_ptr() | v.data_ptr()) % 16:
        k, k_stride = _rows("kv_write", "k", k, cache)
        v, v_stride = _rows("kv_write", "v", v, cache)
        if k.shape[0] != t or v.shape[0] != t:
            raise ValueError(f"kv_write: {k.shape[0]} and {v.shape[0]} rows for {t} slots")
    else:
        k_stride = v_stride = cache.heads * cache.head_dim * k.element_size()
    if not slots.is_contiguous():
        slots = slots.contiguous()
    _call(dev, lib.qs_kv_write, cache._ref, src, k.data_ptr(), k_stride, v.data_ptr(), v_stride, slots.data_ptr(), t)


def kv_read(cache: KVCache, slots, dtype=None):
    """The keys and values that slots (t,) int32 hold, two (t, heads, head_dim) of
    dtype (bfloat16 by default). A slot that is not in the cache gives zeros."""
    lib = _lib()
    dtype = torch.bfloat16 if dtype is None else dtype
    dst = _type_id(dtype, "kv_read")
    dev = cache._dev
    _ints("kv_read", "slots", slots, 1, dev)
    if not slots.is_contiguous():
        slots = slots.contiguous()
    t = len(slots)
    k = cache.data.new_empty((t, cache.heads, cache.head_dim), dtype=dtype)
    v = torch.empty_like(k)
    _call(dev, lib.qs_kv_read, cache._ref, slots.data_ptr(), t, dst, k.data_ptr(), v.data_ptr())
    return k, v


_SIZES = 256        # of workspaces that a cache remembers


def _workspace(cache: KVCache, key) -> int:
    need = _lib().qs_kv_attention_workspace(cache._ref, *key)
    if need < 0:
        _fail()
    if len(cache._work) >= _SIZES:
        cache._work.clear()
    cache._work[key] = need
    return need


def kv_attention(q, cache: KVCache, tables, lengths, scale: float | None = None, window: int = 0, out=None):
    """Attention of each sequence's last n tokens (n at most 16) over its slots,
    which hold those tokens' keys and values already. Returns q's shape and type.

    q: (b, query heads, head_dim), one new token each, or (b, n, query heads,
    head_dim); float32 / float16 / bfloat16; query head h reads key/value head
    h // (query heads / heads).
    tables: (b, m) int32, the page of each run of page_size positions; positions of
    a page that is not in the cache, such as -1, are seen by no query.
    lengths: (b,) int32, the new tokens counted, cut to 0 .. m * page_size. Token i of
    n is at position P = length - n + i and sees positions up to P, with a window those
    above P - window; one that sees none gives zeros, one whose scores are all
    -infinity NaN. What lies at other positions does not matter, whatever it is.
    scale: 1 / sqrt(head_dim) by default.
    out: a contiguous tensor of q's shape and type to write instead of a new one."""
    lib = _lib()
    kind = _type_id(q.dtype, "kv_attention")
    if q.requires_grad or forward_ad._current_level >= 0:
        _no_gradient("kv_attention", "q", q)
    dev, d = cache._dev, cache.head_dim
    if q.get_device() != dev:
        _same_device(dev, "kv_attention", "q", q)
    shape = q.shape
    if len(shape) == 3:
        b, heads, width = shape
        n = 1
    elif len(shape) == 4:
        b, n, heads, width = shape
    else:
        raise ValueError(f"kv_attention: q must be (b, heads, {d}) or (b, n, heads, {d}), got {tuple(shape)}")
    if width != d or heads == 0 or heads % cache.heads:
        raise ValueError(f"kv_attention: q has {heads} heads of {width} values, the cache {cache.heads} of {d}")
    if n > 16:
        raise ValueError(f"kv_attention: {n} new tokens of a sequence, at most 16")
    _ints("kv_attention", "tables", tables, 2, dev)
    _ints("kv_attention", "lengths", lengths, 1, dev)
    rows, m = tables.shape
    if rows != b or len(lengths) != b:
        raise ValueError(f"kv_attention: {rows} tables and {len(lengths)} lengths for {b} sequences")
    if window < 0:
        raise ValueError(f"kv_attention: window {window} < 0")
    esz = q.element_size()
    stride = heads * d
    if not q.is_contiguous() or q.data_ptr() % 16:
        # tokens at one stride from each other, heads side by side
        between = q.stride(-3) if n > 1 or len(shape) == 3 else q.stride(0)
        if q.stride(-1) != 1 or (heads > 1 and q.stride(-2) != d) or q.data_ptr() % 16 or between * esz % 16 \
                or between < stride or (n > 1 and b > 1 and q.stride(0) != n * between):
            q = torch.empty(shape, dtype=q.dtype, device=q.device).copy_(q)
        else:
            stride = between
    table_stride = m
    if not tables.is_contiguous():
        if (m > 1 and tables.stride(1) != 1) or (b > 1 and tables.stride(0) < m):
            tables = tables.contiguous()
        elif b > 1:
            table_stride = tables.stride(0)
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    key = (b, n, heads, m)
    need = cache._work.get(key)
    if need is None:
        need = _workspace(cache, key)
    work_ptr = None
    if need:
        work = cache.data.new_empty((need,))
        work_ptr = work.data_ptr()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.shape != shape or not out.is_contiguous() or not out.is_cuda or out.get_device() != dev:
        raise ValueError(f"kv_attention: out must be contiguous {q.dtype} {tuple(shape)} on cuda:{dev}")
    else:
        _no_gradient("kv_attention", "out", out)
    _call(dev, lib.qs_kv_attention, cache._ref, kind, q.data_ptr(), stride * esz, b, n, heads, tables.data_ptr(), m,
          table_stride, lengths.data_ptr(), 1 / math.sqrt(d) if scale is None else scale, min(window, 1 << 62),
          out.data_ptr(), out.numel() * esz, work_ptr, need)
    return out
