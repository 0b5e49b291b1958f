"""A layer on packed weights: what a program does with the blocks that the
quantizers write.

    rows, h = rms_norm_q8(x, norm_weight, residual=h)      # 8-bit rows, x + h
    w = PackedWeight("q4_k", QUANT_TYPES["q4_k"].make_kernel(dev, None)(w_bf16))
    y = packed_linear(rows, w)                             # (t, n) bf16
    y = packed_linear(rows, w, adapters=bank, ids=ids)     # with each row's adapter

The reference ends at the GGUF file and has none of this. Every function is
calls into the gfx950 library (C ABI in include/quant_studio.h) on torch's
current stream; nothing is synchronised, and every failure raises. These are
serving forms: 8-bit rows and packed weights carry no gradient.
"""

from __future__ import annotations

import contextlib
import ctypes

MAX_VALUES_PER_CALL = 1 << 34


def _fail():
    from . import QuantSpecError, last_error
    raise QuantSpecError(last_error())


def _type_id(dtype, what: str) -> int:
    from . import _src_id
    t = _src_id(dtype)
    if t is None:
        raise ValueError(f"{what}: unsupported dtype {dtype} (float32, float16 or bfloat16)")
    return t


def _on_device(x):
    """The launch needs x's device to be the current one."""
    import torch
    if x.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(x.device)


def _need_rocm(x, what: str) -> None:
    if x.device.type != "cuda":
        raise ValueError(f"{what}: needs tensors on a ROCm device, got one on {x.device}")


def _stream(x) -> int:
    import torch
    return torch.cuda.current_stream(x.device).cuda_stream


def _same_device(x, what: str, **others) -> None:
    for name, o in others.items():
        if o is not None and o.device != x.device:
            raise ValueError(f"{what}: {name} is on {o.device}, the rows on {x.device}")


def _dense(x):
    """x, or a fresh copy where it is not contiguous or starts off a 16-byte boundary."""
    import torch
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x
    return torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)


def _strided(x):
    """(x, its row stride in bytes) in a layout the C call takes: unit stride
    along k, rows on 16-byte boundaries."""
    n, k = x.shape
    esz = x.element_size()
    if x.numel() and ((k > 1 and x.stride(1) != 1) or x.data_ptr() % 16 or
                      (n > 1 and (x.stride(0) < k or (x.stride(0) * esz) % 16))):
        import torch
        x = torch.empty((n, k), dtype=x.dtype, device=x.device).copy_(x)
    return x, (x.stride(0) if n > 1 else k) * esz


class Q8Rows:
    """Rows in 8 bits: codes q (t, k) int8 and scales (t, k // 32) f32, on a
    ROCm device; row r stands for q[r, i] * scale[r, i // 32]."""

    __slots__ = ("q", "scale")

    def __init__(self, q, scale):
        import torch
        if q.dim() != 2 or q.dtype != torch.int8 or q.shape[1] % 32 or q.shape[1] == 0:
            raise ValueError(f"Q8Rows: q must be int8 (t, k) with k a multiple of 32, got {q.dtype} {tuple(q.shape)}")
        if scale.dtype != torch.float32 or tuple(scale.shape) != (q.shape[0], q.shape[1] // 32):
            raise ValueError(f"Q8Rows: scale must be float32 {(q.shape[0], q.shape[1] // 32)}, "
                             f"got {scale.dtype} {tuple(scale.shape)}")
        _need_rocm(q, "Q8Rows")
        _same_device(q, "Q8Rows", scale=scale)
        self.q, self.scale = _dense(q), scale.contiguous()

    @property
    def shape(self):
        return self.q.shape

    @property
    def device(self):
        return self.q.device

    def __len__(self):
        return self.q.shape[0]

    def __getitem__(self, rows: slice) -> "Q8Rows":
        return Q8Rows(self.q[rows], self.scale[rows])

    def values(self, dtype=None):
        """The values the rows stand for, (t, k) of dtype (float32 by default)."""
        import torch
        from . import library
        dtype = torch.float32 if dtype is None else dtype
        dst = _type_id(dtype, "Q8Rows.values")
        t, k = self.q.shape
        out = torch.empty((t, k), dtype=dtype, device=self.q.device)
        with _on_device(self.q):
            if library().qs_q8_values(self.q.data_ptr(), self.scale.data_ptr(), t, k, dst, out.data_ptr(),
                                      _stream(self.q)) != 0:
                _fail()
        return out


def _rows_q8(what: str, x, weight, eps: float, residual, want_sum: bool):
    import torch
    from . import library
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be 2-D (t, k), got shape {tuple(x.shape)}")
    src = _type_id(x.dtype, what)
    _need_rocm(x, what)
    _same_device(x, what, weight=weight, residual=residual)
    t, k = x.shape
    if weight is not None and (weight.dtype != torch.float32 or tuple(weight.shape) != (k,)):
        raise ValueError(f"{what}: weight must be float32 ({k},), got {weight.dtype} {tuple(weight.shape)}")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError(f"{what}: residual must be {x.dtype} {tuple(x.shape)}, "
                         f"got {residual.dtype} {tuple(residual.shape)}")
    x, stride = _strided(x)
    rstride = 0
    if residual is not None:
        residual, rstride = _strided(residual)
    if weight is not None:
        weight = _dense(weight)
    q = torch.empty((t, k), dtype=torch.int8, device=x.device)
    scale = torch.empty((t, k // 32), dtype=torch.float32, device=x.device)
    total = torch.empty((t, k), dtype=x.dtype, device=x.device) if want_sum else None
    with _on_device(x):
        rc = library().qs_rms_norm_q8(src, x.data_ptr(), t, k, stride,
                                      None if residual is None else residual.data_ptr(), rstride,
                                      None if weight is None else weight.data_ptr(), eps,
                                      None if total is None else total.data_ptr(), q.data_ptr(), scale.data_ptr(),
                                      _stream(x))
    if rc != 0:
        _fail()
    return Q8Rows(q, scale), total


def rms_norm_q8(x, weight, eps: float = 1e-6, residual=None):
    """RMS norm of the rows of x (t, k), or of x + residual, to 8-bit rows.

    h = x + residual; u = h * weight; each 32 values of u get the step
    a = max|u| / 127 and the codes rint(u / a); their scale is
    a / sqrt(mean(h^2) + eps). All in float32 whatever x's type.
    x, residual: float32 / float16 / bfloat16, any strides (layouts the C call
    does not take are copied first); weight: (k,) float32; k a multiple of 32.
    Returns Q8Rows, or (Q8Rows, h in x's type) with a residual."""
    rows, total = _rows_q8("rms_norm_q8", x, weight, eps, residual, residual is not None)
    return rows if residual is None else (rows, total)


def q8_rows(x) -> Q8Rows:
    """The rows of x (t, k) as they are, in 8 bits (rms_norm_q8 without the
    norm): the input of a projection that no norm precedes."""
    return _rows_q8("q8_rows", x, None, 0.0, None, False)[0]


class PackedWeight:
    """A packed weight: the bytes (n, row bytes) of a registered type, as a
    quant_fn returns them or a GGUF tensor holds them, on a ROCm device. The
    bytes are used where they are; nothing is laid out again."""

    __slots__ = ("name", "ggml_type", "data", "n", "k")

    def __init__(self, name: str, data):
        import torch
        from . import QUANT_TYPES
        from .gguf_types import QUANT_SIZES
        if name not in QUANT_TYPES:
            raise ValueError(f"PackedWeight: unknown type {name!r}: one of {', '.join(sorted(QUANT_TYPES))}")
        if data.dim() != 2 or data.dtype != torch.uint8:
            raise ValueError(f"PackedWeight: data must be uint8 (n, row bytes), got {data.dtype} {tuple(data.shape)}")
        _need_rocm(data, "PackedWeight")
        blk, size = QUANT_SIZES[QUANT_TYPES[name].ggml_type]
        if data.shape[1] == 0 or data.shape[1] % size:
            raise ValueError(f"PackedWeight: rows of {data.shape[1]} bytes are not blocks of {size} ({name})")
        self.name = name
        self.ggml_type = int(QUANT_TYPES[name].ggml_type)
        # what the C call takes: blocks of whole words on 4-byte boundaries, others on 2-byte ones
        align = 2 if size % 4 else 4
        self.data = data if data.is_contiguous() and data.data_ptr() % align == 0 else _dense(data)
        self.n, self.k = data.shape[0], data.shape[1] // size * blk


class AdapterBank:
    """Low-rank adapters of one weight: a list of (A (r, k), B (n, r), scale),
    float16 or bfloat16 (all alike), on a ROCm device; ranks may differ. They
    are laid side by side once, ranks padded with zeros to multiples of 8."""

    __slots__ = ("n", "k", "dtype", "ranks", "a", "b", "offsets", "scales", "_c")

    def __init__(self, adapters):
        import torch
        adapters = list(adapters)
        if not adapters:
            raise ValueError("AdapterBank: no adapters")
        a0, b0, _ = adapters[0]
        self.k, self.n, self.dtype = a0.shape[-1], b0.shape[0], a0.dtype
        if self.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"AdapterBank: unsupported dtype {self.dtype} (float16 or bfloat16)")
        _need_rocm(a0, "AdapterBank")
        self.ranks, parts_a, parts_b, scales, offsets = [], [], [], [], [0]
        for i, (a, b, scale) in enumerate(adapters):
            r = a.shape[0]
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != self.k or tuple(b.shape) != (self.n, r) or r == 0:
                raise ValueError(f"AdapterBank: adapter {i}: A {tuple(a.shape)} and B {tuple(b.shape)} are not "
                                 f"(r, {self.k}) and ({self.n}, r)")
            if a.dtype != self.dtype or b.dtype != self.dtype:
                raise ValueError(f"AdapterBank: adapter {i}: {a.dtype} / {b.dtype}, the first is {self.dtype}")
            _same_device(a0, "AdapterBank", A=a, B=b)
            pad = -r % 8
            parts_a.append(torch.nn.functional.pad(a, (0, 0, 0, pad)))
            parts_b.append(torch.nn.functional.pad(b, (0, pad)).reshape(-1))
            scales.append(float(scale))
            offsets.append(offsets[-1] + r + pad)
            self.ranks.append(r)
        widest = max(j - i for i, j in zip(offsets, offsets[1:]))
        if widest > 4096:
            raise ValueError(f"AdapterBank: rank {widest} is over 4096")
        self.a, self.b = torch.cat(parts_a), torch.cat(parts_b)
        self.offsets = torch.tensor(offsets, dtype=torch.int32, device=a0.device)
        self.scales = torch.tensor(scales, dtype=torch.float32, device=a0.device)
        self._c = _Adapters(len(adapters), _type_id(self.dtype, "AdapterBank"), widest, self.a.data_ptr(),
                            self.b.data_ptr(), self.offsets.data_ptr(), self.scales.data_ptr())

    def __len__(self):
        return len(self.ranks)


class _Adapters(ctypes.Structure):
    """qs_adapters of include/quant_studio.h."""
    _fields_ = [("count", ctypes.c_int32), ("type", ctypes.c_int32), ("max_rank", ctypes.c_int32),
                ("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("offsets", ctypes.c_void_p),
                ("scales", ctypes.c_void_p)]


def packed_linear(rows, weight: PackedWeight, dtype=None, adapters: AdapterBank | None = None, ids=None, out=None):
    """y = x W^T, (t, n) of dtype (bfloat16 by default), for 8-bit rows x (or a
    float tensor (t, k), which goes through q8_rows first) and a packed weight.

    adapters, ids: each row's low-rank adapter beside the product,
    y[r] += scale * B (A x[r]) for adapter ids[r] (int32 (t,), on the rows'
    device; a value outside 0 .. len(adapters) - 1, such as -1, means none).
    out: a contiguous (t, n) tensor to write instead of a new one."""
    import torch
    from . import library
    if not isinstance(rows, Q8Rows):
        rows = q8_rows(rows)
    q, scale = rows.q, rows.scale
    t, k = q.shape
    dtype = torch.bfloat16 if dtype is None else dtype
    dst = _type_id(dtype, "packed_linear")
    if weight.k != k:
        raise ValueError(f"packed_linear: rows of {k} values, the weight's have {weight.k}")
    _same_device(q, "packed_linear", weight=weight.data)
    if (adapters is None) != (ids is None):
        raise ValueError("packed_linear: adapters and ids go together")
    bank = None
    if adapters is not None:
        if adapters.n != weight.n or adapters.k != k:
            raise ValueError(f"packed_linear: adapters of a ({adapters.n}, {adapters.k}) weight, "
                             f"this one is ({weight.n}, {k})")
        if ids.dtype != torch.int32 or tuple(ids.shape) != (t,):
            raise ValueError(f"packed_linear: ids must be int32 ({t},), got {ids.dtype} {tuple(ids.shape)}")
        _same_device(q, "packed_linear", adapters=adapters.a, ids=ids)
        ids = ids.contiguous()
        bank = ctypes.byref(adapters._c)
    need = library().qs_packed_linear_workspace(weight.ggml_type, weight.n, k, t, dst,
                                                0 if bank is None else adapters._c.max_rank)
    if need < 0:
        _fail()
    work = torch.empty((need,), dtype=torch.uint8, device=q.device) if need else None
    if out is None:
        out = torch.empty((t, weight.n), dtype=dtype, device=q.device)
    elif out.dtype != dtype or tuple(out.shape) != (t, weight.n) or not out.is_contiguous() or out.device != q.device:
        raise ValueError(f"packed_linear: out must be contiguous {dtype} {(t, weight.n)} on {q.device}")
    with _on_device(q):
        rc = library().qs_packed_linear(weight.ggml_type, weight.data.data_ptr(), weight.n, k, q.data_ptr(),
                                        scale.data_ptr(), t, dst, out.data_ptr(), out.numel() * out.element_size(),
                                        bank, None if ids is None else ids.data_ptr(),
                                        None if work is None else work.data_ptr(),
                                        need, _stream(q))
    if rc != 0:
        _fail()
    return out
