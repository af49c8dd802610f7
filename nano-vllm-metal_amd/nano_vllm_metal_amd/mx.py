"""Microscaled (MX) tensors and their products on the GPU (include/nvm_mx.h).

An ``MxTensor`` holds rows of block-scaled floating point: 32 consecutive
values share one power-of-two scale (E8M0), the values are E2M1 (``mxfp4``) or
E4M3 (``mxfp8``), as in the OCP Microscaling formats and in MLX's ``mxfp4``
weights.  ``mx_linear`` multiplies MX activations with MXFP4 weights on the
matrix cores; it stands beside ``quantized_linear``
(``layers/linear.py:92-126``), ``mx_swiglu`` beside ``quantized_swiglu`` and
``residual_rms_norm_mx`` beside ``residual_rms_norm``, with activations of
eight (or four) bits between them.  No CPU fallback.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

MX_BLOCK = 32
# nvm_mx_format and nvm_mx_dtype of include/nvm_mx.h
MX_FORMATS = {"mxfp4": 0, "mxfp8": 1}
MX_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_SHORT_SUMS = 16  # NVM_MX_SHORT_SUMS
_PER_BYTE = {"mxfp4": 2, "mxfp8": 1}
_MAX_PITCH = 1 << 20


def _pitch(n: int) -> int:
    """Bytes from one row of scales to the next: n / 32, rounded up to 16."""
    return -(-n // (16 * MX_BLOCK)) * 16


def _format(fmt: str) -> int:
    try:
        return MX_FORMATS[fmt]
    except KeyError:
        raise ValueError(f"MX format must be one of {sorted(MX_FORMATS)}, got {fmt!r}") from None


class MxTensor:
    """``codes`` uint8 ``[..., n]`` (mxfp8) or ``[..., n / 2]`` (mxfp4, the
    even value in the low half) and ``scales`` uint8 ``[..., n / 32]``, byte b
    standing for ``2 ** (b - 127)``, 255 for NaN.

    The kernels read scales in rows that start 16 bytes apart or a multiple;
    the tensors that this package returns lie so, others (a checkpoint's) are
    copied into that layout once, here.
    """

    # _base holds the codes; where a kernel wrote the tensor, the scales too, from
    # byte _split on, and codes and scales are views that are made when asked for
    # (each takes as long as an allocation, and operators pass pointers on).
    __slots__ = ("_base", "_split", "_codes", "_scales", "fmt", "shape", "rows", "pitch")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str):
        _format(fmt)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("MxTensor: codes and scales must be uint8")
        if codes.dim() < 1 or scales.dim() != codes.dim():
            raise ValueError("MxTensor: codes and scales must have the same number of dimensions")
        n = codes.shape[-1] * _PER_BYTE[fmt]
        if n == 0 or n % MX_BLOCK or scales.shape[:-1] != codes.shape[:-1] \
                or scales.shape[-1] * MX_BLOCK != n:
            raise ValueError(f"MxTensor: codes {tuple(codes.shape)} and scales "
                             f"{tuple(scales.shape)} are not rows of {fmt} blocks of {MX_BLOCK}")
        if codes.device != scales.device:
            raise ValueError("MxTensor: codes and scales must be on one device")
        pitch = _row_pitch(scales, n)
        if pitch is None:
            scales, pitch = _lay_out(scales, n), _pitch(n)
        self._base = self._codes = _packed(codes)
        self._split = None
        self._scales = scales
        self.fmt = fmt
        self.shape = torch.Size((*codes.shape[:-1], n))
        self.rows = codes.shape[:-1].numel()
        self.pitch = pitch

    @classmethod
    def _empty(cls, lead, rows: int, n: int, fmt: str, device) -> "MxTensor":
        """A tensor for a kernel to write: nothing to check or to copy."""
        t = cls.__new__(cls)
        t.pitch = pitch = _pitch(n)
        t._split = split = rows * (n // _PER_BYTE[fmt])
        t._base = torch.empty(split + rows * pitch, dtype=torch.uint8, device=device)
        t._codes = t._scales = None
        t.fmt = fmt
        t.shape = torch.Size((*lead, n))
        t.rows = rows
        return t

    def _view(self, width: int, pitch: int, offset: int) -> torch.Tensor:
        """Rows of ``width`` bytes, ``pitch`` apart, from a byte of the base on."""
        shape = self.shape
        if len(shape) == 2:
            return self._base.as_strided((shape[0], width), (pitch, 1), offset)
        lead, strides = shape[:-1], [1]
        for size in reversed(lead):
            strides.append(pitch)
            pitch *= max(size, 1)
        return self._base.as_strided((*lead, width), strides[::-1], offset)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            width = self.shape[-1] // _PER_BYTE[self.fmt]
            self._codes = self._view(width, width, 0)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._view(self.shape[-1] // MX_BLOCK, self.pitch, self._split)
        return self._scales

    def _pointers(self) -> Tuple[int, int]:
        """Addresses of codes and scales."""
        if self._split is None:
            return self._base.data_ptr(), self._scales.data_ptr()
        at = self._base.data_ptr()
        return at, at + self._split

    @property
    def device(self) -> torch.device:
        return self._base.device

    @property
    def in_features(self) -> int:
        return self.shape[-1]

    @property
    def out_features(self) -> int:
        return self.shape[-2]

    def to(self, device) -> "MxTensor":
        return MxTensor(self.codes.to(device), self.scales.to(device), self.fmt)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return mx_dequantize(self, dtype)

    def __reduce__(self):  # (copies: of what the views show, not of the views beside their base)
        return MxTensor, (self.codes, self.scales, self.fmt)

    def __repr__(self) -> str:
        return f"MxTensor({self.fmt}, shape={tuple(self.shape)}, device={self.device})"


def _row_pitch(scales: torch.Tensor, n: int) -> Optional[int]:
    """Bytes between rows of scales that lie as the kernels read them: rows a
    multiple of 16 bytes apart, up to ``_MAX_PITCH``, evenly over all leading
    dimensions, and the last row's padding inside the storage.  None for others."""
    if scales.stride(-1) != 1 and scales.shape[-1] > 1 or scales.data_ptr() % 16:
        return None
    need = _pitch(n)
    pitch = scales.stride(-2) if scales.dim() > 1 and scales.shape[-2] > 1 else need
    if pitch % 16 or not need <= pitch <= _MAX_PITCH:
        return None
    step = pitch
    for size, stride in zip(reversed(scales.shape[:-1]), reversed(scales.stride()[:-1])):
        if size > 1 and stride != step:
            return None
        step *= size
    rows = scales.shape[:-1].numel()
    last = scales.storage_offset() + max(rows - 1, 0) * pitch + need
    return pitch if rows == 0 or last <= scales.untyped_storage().nbytes() else None


def _lay_out(scales: torch.Tensor, n: int) -> torch.Tensor:
    pitch = _pitch(n)
    out = torch.zeros((*scales.shape[:-1], pitch), dtype=torch.uint8, device=scales.device)
    out = out[..., :n // MX_BLOCK]
    out.copy_(scales)
    return out


def _packed(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# (each operator: its tensors' device, whichever is current, and its stream)
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _index(a: torch.Tensor, b: torch.Tensor) -> int:
    """The one GPU of both."""
    index = a.get_device()
    if index < 0 or b.get_device() != index:
        _lib.require_device(a, b)
    return index


def mx_quantize(x: torch.Tensor, fmt: str = "mxfp8") -> MxTensor:
    """``x [..., n]`` (float16, bfloat16 or float32; n a multiple of 32) in MX:
    per block of 32 the scale ``2 ** (floor(log2(max |x|)) - emax)`` (emax 2
    for mxfp4, 8 for mxfp8) and the values divided by it, rounded to nearest
    even, saturating at 6 or 448.  A block that holds a NaN or an infinity
    stands for NaNs."""
    lib = _lib.load()
    code = _format(fmt)
    dev = _lib.require_device(x)
    dtype = MX_DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"mx_quantize: x must be float16, bfloat16 or float32, got {x.dtype}")
    shape = x.shape
    n = shape[-1] if shape else 0
    if n == 0 or n % MX_BLOCK:
        raise ValueError(f"mx_quantize: the last dimension must be a positive multiple of "
                         f"{MX_BLOCK}, got shape {tuple(shape)}")
    ld = n
    if not x.is_contiguous():
        if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= n \
                and x.stride(0) * x.element_size() % 16 == 0:
            ld = x.stride(0)
        else:
            x = x.contiguous()
    if x.data_ptr() % 16:
        x, ld = x.clone(memory_format=torch.contiguous_format), n
    rows = x.numel() // n
    index = dev.index
    if index != _current_device():
        with torch.cuda.device(index):
            return mx_quantize(x, fmt)
    out = MxTensor._empty(shape[:-1], rows, n, fmt, dev)
    codes, scales = out._pointers()
    _lib.check(lib.nvm_mx_quantize(x.data_ptr(), rows, n, ld, dtype, code, codes, scales, out.pitch,
                                   _raw_stream(index)))
    return out


def mx_dequantize(t: MxTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that ``t`` stands for, rounded once to ``dtype``."""
    lib = _lib.load()
    if type(t) is not MxTensor:
        raise ValueError("mx_dequantize: t must be an MxTensor")
    dev = _lib.require_device(t._base)
    code = MX_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"mx_dequantize: dtype must be float16, bfloat16 or float32, got {dtype}")
    index = dev.index
    if index != _current_device():
        with torch.cuda.device(index):
            return mx_dequantize(t, dtype)
    out = torch.empty(t.shape, dtype=dtype, device=dev)
    codes, scales = t._pointers()
    _lib.check(lib.nvm_mx_dequantize(codes, scales, t.pitch, t.rows, t.shape[-1], MX_FORMATS[t.fmt],
                                     code, out.data_ptr(), _raw_stream(index)))
    return out


def mx_embedding(tokens: torch.Tensor, table: MxTensor, dtype: torch.dtype) -> torch.Tensor:
    """The rows of ``table [V, D]`` for ``tokens``, rounded once to ``dtype``,
    ``[*tokens.shape, D]``: ``embedding`` of a table in MX.  Ids outside ``[0,
    V)`` give zero rows."""
    lib = _lib.load()
    if type(table) is not MxTensor or len(table.shape) != 2:
        raise ValueError("mx_embedding: table must be a two-dimensional MxTensor")
    index = _index(tokens, table._base)
    code = MX_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"mx_embedding: dtype must be float16, bfloat16 or float32, got {dtype}")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"mx_embedding: tokens must be int32 or int64, got {tokens.dtype}")
    if index != _current_device():
        with torch.cuda.device(index):
            return mx_embedding(tokens, table, dtype)
    V, D = table.shape
    if tokens.dtype == torch.int64:  # (an id that 32 bits would wrap stays outside)
        tokens = tokens.clamp(-1, V)
    ids = tokens.reshape(-1).to(torch.int32).contiguous()
    out = torch.empty((*tokens.shape, D), dtype=dtype, device=ids.device)
    codes, scales = table._pointers()
    _lib.check(lib.nvm_mx_embedding(ids.data_ptr(), ids.numel(), codes, scales, table.pitch, V, D,
                                    MX_FORMATS[table.fmt], code, out.data_ptr(),
                                    _raw_stream(index)))
    return out


def residual_rms_norm_mx(h: torch.Tensor, r: Optional[torch.Tensor], weight: torch.Tensor,
                         eps: float, fmt: str = "mxfp8") -> Tuple[torch.Tensor, MxTensor]:
    """``residual_rms_norm`` with an MX output: ``(h + r, rms_norm(h + r) *
    weight in MX)``; with ``r`` None, ``(h, rms_norm(h) * weight in MX)``.  The
    sum is rounded to the activation dtype, the norm is not before it is
    quantised."""
    lib = _lib.load()
    code = _format(fmt)
    dev = _lib.require_device(h, r, weight)
    dtype = _lib.dtype_code(h.dtype)
    shape = h.shape
    H = shape[-1] if shape else 0
    if H == 0 or H % MX_BLOCK:
        raise ValueError(f"residual_rms_norm_mx: the last dimension must be a positive multiple "
                         f"of {MX_BLOCK}, got shape {tuple(shape)}")
    if weight.numel() != H:
        raise ValueError(f"residual_rms_norm_mx: weight must have {H} elements")
    index = dev.index
    if index != _current_device():
        with torch.cuda.device(index):
            return residual_rms_norm_mx(h, r, weight, eps, fmt)
    hc = _packed(h)
    rc = h_out = None
    if r is not None:
        if r.shape != shape or r.dtype != h.dtype:
            raise ValueError("residual_rms_norm_mx: r must have the shape and dtype of h")
        rc = _packed(r)
        h_out = torch.empty_like(hc)
    w = _packed(weight if weight.dtype == h.dtype else weight.to(h.dtype))
    rows = hc.numel() // H
    out = MxTensor._empty(shape[:-1], rows, H, fmt, dev)
    codes, scales = out._pointers()
    _lib.check(lib.nvm_residual_rms_norm_mx(
        hc.data_ptr(), _lib.ptr(rc), w.data_ptr(), rows, H, float(eps), dtype, _lib.ptr(h_out),
        code, codes, scales, out.pitch, _raw_stream(index)))
    return (h if h_out is None else h_out), out


def mx_stack_outputs(*ws: MxTensor) -> MxTensor:
    """One weight for several projections of the same input: rows one behind
    the other."""
    if any(w.fmt != ws[0].fmt or w.shape[1:] != ws[0].shape[1:] for w in ws):
        raise ValueError("mx_stack_outputs: projections differ in format or input features")
    return MxTensor(torch.cat([w.codes for w in ws]), torch.cat([w.scales for w in ws]), ws[0].fmt)


def _activations(x: Union[MxTensor, torch.Tensor], op: str) -> MxTensor:
    if x.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"{op}: x must be an MxTensor, float16 or bfloat16, got {x.dtype}")
    return mx_quantize(x, "mxfp8")


def _check_weight(op: str, name: str, w: MxTensor, a: MxTensor) -> None:
    if type(w) is not MxTensor or w.fmt != "mxfp4" or len(w.shape) != 2:
        raise ValueError(f"{op}: {name} must be a two-dimensional mxfp4 MxTensor")
    if w.shape[1] != a.shape[-1]:
        raise ValueError(f"{op}: {name} has {w.shape[1]} input features, x has {a.shape[-1]}")


def mx_linear(x: Union[MxTensor, torch.Tensor], w: MxTensor,
              dtype: Optional[torch.dtype] = None,
              bias: Optional[torch.Tensor] = None, short_sums: bool = False) -> torch.Tensor:
    """``x . w^T (+ bias)``: ``x [..., N]`` in MX (16-bit activations are
    quantised to mxfp8 first), ``w [K, N]`` in mxfp4.  Float32 sums, one rounding to ``dtype``
    (float16, bfloat16 or float32; by default that of 16-bit activations, else
    bfloat16); ``bias [K]`` of any of these types is added to that, as by
    ``quantized_linear``, and the sum rounded again.  ``short_sums``: mxfp8 activations are summed by the scaled matrix
    instruction itself, at about twice the rate for many rows, and 2^-17 to
    2^-15 of a sum is lost, in a float32 output too (include/nvm_mx.h)."""
    lib = _lib.load()
    if type(x) is MxTensor:
        a = x
        dtype = torch.bfloat16 if dtype is None else dtype
    else:
        a = _activations(x, "mx_linear")
        dtype = x.dtype if dtype is None else dtype
    code = MX_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"mx_linear: dtype must be float16, bfloat16 or float32, got {dtype}")
    _check_weight("mx_linear", "w", w, a)
    if bias is not None and (bias.shape != w.shape[:1] or bias.dtype not in MX_DTYPES):
        raise ValueError(f"mx_linear: bias must be [{w.shape[0]}] of float16, bfloat16 or float32, "
                         f"got {tuple(bias.shape)} of {bias.dtype}")
    index = _index(a._base, w._base)
    if bias is not None and bias.get_device() != index:
        _lib.require_device(a._base, bias)
    if index != _current_device():
        with torch.cuda.device(index):
            return mx_linear(a, w, dtype, bias, short_sums)
    K, N = w.shape
    lead = a.shape
    out = torch.empty((lead[0], K) if len(lead) == 2 else (*lead[:-1], K), dtype=dtype,
                      device=a._base.device)
    ac, asc = a._pointers()
    wc, wsc = w._pointers()
    sums = _SHORT_SUMS if short_sums else 0
    _lib.check(lib.nvm_mx_matmul(ac, asc, a.pitch, MX_FORMATS[a.fmt] | sums, wc, wsc, w.pitch,
                                 a.rows, N, K, code, out.data_ptr(), _raw_stream(index)))
    return out if bias is None else (out + bias).to(dtype)


def mx_swiglu(x: Union[MxTensor, torch.Tensor], w_gate: MxTensor, w_up: MxTensor,
              fmt: str = "mxfp8", short_sums: bool = False) -> MxTensor:
    """``silu(x . gate^T) * (x . up^T)`` in MX, the input of a down projection
    (models/qwen3.py:176-184): ``x`` as for ``mx_linear``, both weights ``[K,
    N]`` in mxfp4, K a multiple of 32.  Everything up to the quantisation is
    float32, unless ``short_sums`` asks for sums as ``mx_linear`` says."""
    lib = _lib.load()
    code = _format(fmt)
    a = x if type(x) is MxTensor else _activations(x, "mx_swiglu")
    _check_weight("mx_swiglu", "w_gate", w_gate, a)
    _check_weight("mx_swiglu", "w_up", w_up, a)
    K, N = w_gate.shape
    if w_up.shape[0] != K or K == 0 or K % MX_BLOCK:
        raise ValueError(f"mx_swiglu: gate and up must have the same output features, a positive "
                         f"multiple of {MX_BLOCK}, got {K} and {w_up.shape[0]}")
    index = _index(a._base, w_gate._base)
    if w_up._base.get_device() != index:
        _lib.require_device(a._base, w_up._base)
    if index != _current_device():
        with torch.cuda.device(index):
            return mx_swiglu(a, w_gate, w_up, fmt, short_sums)
    out = MxTensor._empty(a.shape[:-1], a.rows, K, fmt, a._base.device)
    ac, asc = a._pointers()
    gc, gsc = w_gate._pointers()
    uc, usc = w_up._pointers()
    oc, osc = out._pointers()
    sums = _SHORT_SUMS if short_sums else 0
    _lib.check(lib.nvm_mx_swiglu(ac, asc, a.pitch, MX_FORMATS[a.fmt] | sums, gc, gsc, w_gate.pitch,
                                 uc, usc, w_up.pitch, a.rows, N, K, code, oc, osc, out.pitch,
                                 _raw_stream(index)))
    return out
