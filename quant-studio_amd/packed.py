"""A layer on packed weights: what a program does with the blocks that the
quantizers write.

    rows, h = rms_norm_q8(x, norm_weight, residual=h)      # 8-bit rows, x + h
    w = PackedWeight("q4_k", QUANT_TYPES["q4_k"].make_kernel(dev, None)(w_bf16))
    y = packed_linear(rows, w)                             # (t, n) bf16
    y = packed_linear(rows, w, adapters=bank, ids=ids)     # with each row's adapter

The reference ends at the GGUF file and has none of this. Every function is
calls into the gfx950 library (C ABI in include/quant_studio.h) on torch's
current stream; nothing is synchronised, and every failure raises. These are
serving forms: 8-bit rows and packed weights carry no gradient, and a tensor that
requires one is refused while gradients are recorded.

A decode step makes hundreds of these calls, each a few microseconds of GPU
work, so what Python does per call counts as much: devices are compared as
numbers, sizes asked once, and nothing is checked twice.
"""

from __future__ import annotations

import ctypes

torch = None            # imported with the library when a function is first called
_L = None
_TYPE_ID: dict = {}     # dtype -> source type id of the C ABI
_EXACT = 0x100          # QS_EXACT of include/quant_studio.h


def _lib():
    global torch, _L
    if _L is None:
        import torch as t
        from . import library
        lib = library()
        _TYPE_ID.update({t.float32: 0, t.float16: 1, t.bfloat16: 30})
        torch, _L = t, lib
    return _L


def _fail():
    from . import QuantSpecError, last_error
    raise QuantSpecError(last_error())


def _type_id(dtype, what: str) -> int:
    t = _TYPE_ID.get(dtype)
    if t is None:
        raise ValueError(f"{what}: unsupported dtype {dtype} (float32, float16 or bfloat16)")
    return t


def _device_of(x, what: str) -> int:
    if not x.is_cuda:
        raise ValueError(f"{what}: needs tensors on a ROCm device, got one on {x.device}")
    return x.get_device()


def _same_device(dev: int, what: str, name: str, x) -> None:
    if not x.is_cuda or x.get_device() != dev:
        raise ValueError(f"{what}: {name} is on {x.device}, the rows on cuda:{dev}")


def _no_gradient(what: str, name: str, x) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: {name} requires a gradient and there is no gradient through 8-bit rows: "
                         "detach it, or call under torch.no_grad()")


def _call(dev: int, fn, *args) -> None:
    """fn(*args, the current stream of device dev) with dev the current device."""
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if torch._C._cuda_getDevice() == dev:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc != 0:
        _fail()


def _dense(x):
    """x, or a fresh copy where it is not contiguous or starts off a 16-byte boundary."""
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x
    return torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)


def _strided(x):
    """(x, its row stride in bytes) in a layout the C call takes: unit stride
    along k, rows on 16-byte boundaries."""
    n, k = x.shape
    esz = x.element_size()
    if x.is_contiguous() and x.data_ptr() % 16 == 0 and (n <= 1 or k * esz % 16 == 0):
        return x, k * esz
    if x.numel() and ((k > 1 and x.stride(1) != 1) or x.data_ptr() % 16 or
                      (n > 1 and (x.stride(0) < k or (x.stride(0) * esz) % 16))):
        x = torch.empty((n, k), dtype=x.dtype, device=x.device).copy_(x)
    return x, (x.stride(0) if n > 1 else k) * esz


class Q8Rows:
    """Rows in 8 bits: codes q (t, k) int8 and scales (t, k // 32) f32, on a
    ROCm device; row r stands for q[r, i] * scale[r, i // 32]."""

    __slots__ = ("t", "k", "_q", "_scale", "_both", "_dev", "_q_ptr", "_scale_ptr")

    def __init__(self, q, scale):
        _lib()
        if q.dim() != 2 or q.dtype != torch.int8 or q.shape[1] % 32 or q.shape[1] == 0:
            raise ValueError(f"Q8Rows: q must be int8 (t, k) with k a multiple of 32, got {q.dtype} {tuple(q.shape)}")
        if scale.dtype != torch.float32 or tuple(scale.shape) != (q.shape[0], q.shape[1] // 32):
            raise ValueError(f"Q8Rows: scale must be float32 {(q.shape[0], q.shape[1] // 32)}, "
                             f"got {scale.dtype} {tuple(scale.shape)}")
        _no_gradient("Q8Rows", "scale", scale)
        self._dev = _device_of(q, "Q8Rows")
        _same_device(self._dev, "Q8Rows", "scale", scale)
        self.t, self.k = q.shape
        self._q, self._scale, self._both = _dense(q), scale.contiguous(), None
        self._q_ptr, self._scale_ptr = self._q.data_ptr(), self._scale.data_ptr()

    @property
    def q(self):
        if self._q is None:         # the norm's rows: codes, then scales, in one allocation
            self._q = self._both[:self.t * self.k].view(torch.int8).view(self.t, self.k)
        return self._q

    @property
    def scale(self):
        if self._scale is None:
            self._scale = self._both[self.t * self.k:].view(torch.float32).view(self.t, self.k // 32)
        return self._scale

    @property
    def shape(self):
        return torch.Size((self.t, self.k))

    @property
    def device(self):
        return torch.device("cuda", self._dev)

    def __len__(self):
        return self.t

    def __getitem__(self, rows: slice) -> "Q8Rows":
        return Q8Rows(self.q[rows], self.scale[rows])

    def values(self, dtype=None):
        """The values the rows stand for, (t, k) of dtype (float32 by default)."""
        lib = _lib()
        dtype = torch.float32 if dtype is None else dtype
        dst = _type_id(dtype, "Q8Rows.values")
        t, k = self.t, self.k
        out = (self._q if self._both is None else self._both).new_empty((t, k), dtype=dtype)
        _call(self._dev, lib.qs_q8_values, self._q_ptr, self._scale_ptr, t, k, dst, out.data_ptr())
        return out


def _rows_q8(what: str, x, weight, eps: float, residual):
    lib = _lib()
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be 2-D (t, k), got shape {tuple(x.shape)}")
    src = _type_id(x.dtype, what)
    _no_gradient(what, "x", x)
    if weight is not None:
        _no_gradient(what, "weight", weight)
    if residual is not None:
        _no_gradient(what, "residual", residual)
    dev = _device_of(x, what)
    t, k = x.shape
    weight_ptr = residual_ptr = total_ptr = total = None
    if weight is not None:
        _same_device(dev, what, "weight", weight)
        if weight.dtype != torch.float32 or weight.dim() != 1 or weight.shape[0] != k:
            raise ValueError(f"{what}: weight must be float32 ({k},), got {weight.dtype} {tuple(weight.shape)}")
        weight = _dense(weight)
        weight_ptr = weight.data_ptr()
    x, stride = _strided(x)
    rstride = 0
    if residual is not None:
        _same_device(dev, what, "residual", residual)
        if residual.dtype != x.dtype or residual.shape != x.shape:
            raise ValueError(f"{what}: residual must be {x.dtype} {tuple(x.shape)}, "
                             f"got {residual.dtype} {tuple(residual.shape)}")
        residual, rstride = _strided(residual)
        total = x.new_empty((t, k))
        residual_ptr, total_ptr = residual.data_ptr(), total.data_ptr()
    both = x.new_empty((t * k + t * (k // 32) * 4,), dtype=torch.uint8)
    ptr = both.data_ptr()
    _call(dev, lib.qs_rms_norm_q8, src, x.data_ptr(), t, k, stride, residual_ptr, rstride, weight_ptr, eps, total_ptr, ptr,
          ptr + t * k)
    rows = object.__new__(Q8Rows)       # as the call left them: nothing to check
    rows.t, rows.k, rows._q, rows._scale, rows._both, rows._dev = t, k, None, None, both, dev
    rows._q_ptr, rows._scale_ptr = ptr, ptr + t * k
    return rows, total


def rms_norm_q8(x, weight, eps: float = 1e-6, residual=None):
    """RMS norm of the rows of x (t, k), or of x + residual, to 8-bit rows.

    h = x + residual; u = h * weight; each 32 values of u get the step
    a = max|u| / 127 and the codes rint(u / a); their scale is
    a / sqrt(mean(h^2) + eps). All in float32 whatever x's type.
    x, residual: float32 / float16 / bfloat16, any strides (layouts the C call
    does not take are copied first); weight: (k,) float32; k a multiple of 32.
    Returns Q8Rows, or (Q8Rows, h in x's type) with a residual."""
    rows, total = _rows_q8("rms_norm_q8", x, weight, eps, residual)
    return rows if residual is None else (rows, total)


def q8_rows(x) -> Q8Rows:
    """The rows of x (t, k) as they are, in 8 bits (rms_norm_q8 without the
    norm): the input of a projection that no norm precedes."""
    return _rows_q8("q8_rows", x, None, 0.0, None)[0]


class PackedWeight:
    """A packed weight: the bytes (n, row bytes) of a registered type, as a
    quant_fn returns them or a GGUF tensor holds them, on a ROCm device. The
    bytes are used where they are; nothing is laid out again."""

    __slots__ = ("name", "ggml_type", "data", "n", "k", "_dev", "_work")

    def __init__(self, name: str, data):
        _lib()
        from . import QUANT_TYPES
        from .gguf_types import QUANT_SIZES
        if name not in QUANT_TYPES:
            raise ValueError(f"PackedWeight: unknown type {name!r}: one of {', '.join(sorted(QUANT_TYPES))}")
        if data.dim() != 2 or data.dtype != torch.uint8:
            raise ValueError(f"PackedWeight: data must be uint8 (n, row bytes), got {data.dtype} {tuple(data.shape)}")
        self._dev = _device_of(data, "PackedWeight")
        blk, size = QUANT_SIZES[QUANT_TYPES[name].ggml_type]
        if data.shape[1] == 0 or data.shape[1] % size:
            raise ValueError(f"PackedWeight: rows of {data.shape[1]} bytes are not blocks of {size} ({name})")
        self.name = name
        self.ggml_type = int(QUANT_TYPES[name].ggml_type)
        # what the C call takes: blocks of whole words on 4-byte boundaries, others on 2-byte ones
        align = 2 if size % 4 else 4
        self.data = data if data.is_contiguous() and data.data_ptr() % align == 0 else _dense(data)
        self.n, self.k = data.shape[0], data.shape[1] // size * blk
        self._work = {}         # (rows, result type, rank) -> workspace bytes


class _Adapters(ctypes.Structure):
    """qs_adapters of include/quant_studio.h."""
    _fields_ = [("count", ctypes.c_int32), ("type", ctypes.c_int32), ("max_rank", ctypes.c_int32),
                ("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("offsets", ctypes.c_void_p),
                ("scales", ctypes.c_void_p)]


class AdapterBank:
    """Low-rank adapters of one weight: a list of (A (r, k), B (n, r), scale),
    float16 or bfloat16 (all alike), on a ROCm device; ranks may differ. They
    are laid side by side once, ranks padded with zeros to multiples of 8: copies,
    without gradients, which later changes of A and B do not reach."""

    __slots__ = ("n", "k", "dtype", "ranks", "a", "b", "offsets", "scales", "_c", "_dev")

    def __init__(self, adapters):
        _lib()
        adapters = list(adapters)
        if not adapters:
            raise ValueError("AdapterBank: no adapters")
        a0, b0, _ = adapters[0]
        self.k, self.n, self.dtype = a0.shape[-1], b0.shape[0], a0.dtype
        if self.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"AdapterBank: unsupported dtype {self.dtype} (float16 or bfloat16)")
        self._dev = _device_of(a0, "AdapterBank")
        self.ranks, parts_a, parts_b, scales, offsets = [], [], [], [], [0]
        for i, (a, b, scale) in enumerate(adapters):
            a, b = a.detach(), b.detach()
            r = a.shape[0]
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != self.k or tuple(b.shape) != (self.n, r) or r == 0:
                raise ValueError(f"AdapterBank: adapter {i}: A {tuple(a.shape)} and B {tuple(b.shape)} are not "
                                 f"(r, {self.k}) and ({self.n}, r)")
            if a.dtype != self.dtype or b.dtype != self.dtype:
                raise ValueError(f"AdapterBank: adapter {i}: {a.dtype} / {b.dtype}, the first is {self.dtype}")
            _same_device(self._dev, "AdapterBank", "A", a)
            _same_device(self._dev, "AdapterBank", "B", b)
            pad = -r % 8
            parts_a.append(torch.nn.functional.pad(a, (0, 0, 0, pad)) if pad else a)
            parts_b.append((torch.nn.functional.pad(b, (0, pad)) if pad else b).reshape(-1))
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


_SIZES = 256        # of workspaces that a weight remembers


def _workspace(weight: PackedWeight, t: int, dst: int, rank: int) -> int:
    """The workspace of a call in bytes, remembered until _SIZES others are:
    decoding asks for a few row counts again and again, prompts for any."""
    need = _lib().qs_packed_linear_workspace(weight.ggml_type, weight.n, weight.k, t, dst, rank)
    if need < 0:
        _fail()
    if len(weight._work) >= _SIZES:
        weight._work.clear()
    weight._work[(t, dst, rank)] = need
    return need


def packed_linear(rows, weight: PackedWeight, dtype=None, adapters: AdapterBank | None = None, ids=None, out=None,
                  exact: bool = False):
    """y = x W^T, (t, n) of dtype (bfloat16 by default), for 8-bit rows x (or a
    float tensor (t, k), which goes through q8_rows first) and a packed weight.

    adapters, ids: each row's low-rank adapter beside the product,
    y[r] += scale * B (A x[r]) for adapter ids[r] (int32 (t,), on the rows'
    device; a value outside 0 .. len(adapters) - 1, such as -1, means none).
    out: a contiguous (t, n) tensor to write instead of a new one.
    exact: large products with a bfloat16 result round both factors to float16
    (include/quant_studio.h has the sizes), which takes a half to two thirds of
    the time and, where the terms of a sum cancel, costs more than its rounding
    does; with exact=True they multiply exact codes, as all others do."""
    lib = _lib()
    if not isinstance(rows, Q8Rows):
        rows = q8_rows(rows)
    t, k, dev = rows.t, rows.k, rows._dev
    dtype = torch.bfloat16 if dtype is None else dtype
    dst = _type_id(dtype, "packed_linear") | (_EXACT if exact else 0)
    n = weight.n
    if weight.k != k:
        raise ValueError(f"packed_linear: rows of {k} values, the weight's have {weight.k}")
    if weight._dev != dev:
        _same_device(dev, "packed_linear", "weight", weight.data)
    if (adapters is None) != (ids is None):
        raise ValueError("packed_linear: adapters and ids go together")
    bank = ids_ptr = work_ptr = None
    rank = 0
    if adapters is not None:
        if adapters.n != n or adapters.k != k:
            raise ValueError(f"packed_linear: adapters of a ({adapters.n}, {adapters.k}) weight, this one is ({n}, {k})")
        if ids.dtype != torch.int32 or ids.dim() != 1 or ids.shape[0] != t:
            raise ValueError(f"packed_linear: ids must be int32 ({t},), got {ids.dtype} {tuple(ids.shape)}")
        _same_device(dev, "packed_linear", "ids", ids)
        if adapters._dev != dev:
            _same_device(dev, "packed_linear", "adapters", adapters.a)
        ids = ids.contiguous()
        ids_ptr, bank, rank = ids.data_ptr(), ctypes.byref(adapters._c), adapters._c.max_rank
    need = weight._work.get((t, dst, rank))
    if need is None:
        need = _workspace(weight, t, dst, rank)
    if need:
        work = weight.data.new_empty((need,))
        work_ptr = work.data_ptr()
    if out is None:
        out = weight.data.new_empty((t, n), dtype=dtype)
    elif out.dtype != dtype or tuple(out.shape) != (t, n) or not out.is_contiguous() or not out.is_cuda or out.get_device() != dev:
        raise ValueError(f"packed_linear: out must be contiguous {dtype} {(t, n)} on cuda:{dev}")
    else:
        _no_gradient("packed_linear", "out", out)
    _call(dev, lib.qs_packed_linear, weight.ggml_type, weight.data.data_ptr(), n, k, rows._q_ptr, rows._scale_ptr, t,
          dst, out.data_ptr(), out.numel() * out.element_size(), bank, ids_ptr, work_ptr, need)
    return out
