"""Microscaled (MX) tensors and their products on the GPU (include/nvm_mx.h).

An ``MxTensor`` holds rows of block-scaled floating point: 32 consecutive
values share one power-of-two scale (E8M0), the values are E2M1 (``mxfp4``) or
E4M3 (``mxfp8``), as in the OCP Microscaling formats and in MLX's ``mxfp4``
weights.  ``mx_linear`` multiplies MX activations with MXFP4 weights on the
scaled matrix instructions; it stands beside ``quantized_linear``
(``layers/linear.py:92-126``), ``mx_swiglu`` beside ``quantized_swiglu`` and
``residual_rms_norm_mx`` beside ``residual_rms_norm``, with activations of
eight (or four) bits between them.  No CPU fallback.
"""

from __future__ import annotations

import contextlib
from typing import Optional, Tuple, Union

import torch

from . import _lib

MX_BLOCK = 32
# nvm_mx_format and nvm_mx_dtype of include/nvm_mx.h
MX_FORMATS = {"mxfp4": 0, "mxfp8": 1}
MX_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_PER_BYTE = {"mxfp4": 2, "mxfp8": 1}


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

    __slots__ = ("codes", "scales", "fmt", "shape")

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
        codes = codes.contiguous()
        self.codes = codes if codes.data_ptr() % 16 == 0 else codes.clone()
        self.scales = scales if _scales_laid_out(scales, n) else _lay_out(scales, n)
        self.fmt = fmt
        self.shape = torch.Size((*codes.shape[:-1], n))

    @classmethod
    def _of(cls, codes, scales, fmt, shape) -> "MxTensor":
        """A tensor that a kernel wrote: nothing to check or to copy."""
        t = cls.__new__(cls)
        t.codes, t.scales, t.fmt, t.shape = codes, scales, fmt, shape
        return t

    @classmethod
    def _empty(cls, lead, n: int, fmt: str, device) -> "MxTensor":
        pitch = _pitch(n)
        codes = torch.empty((*lead, n // _PER_BYTE[fmt]), dtype=torch.uint8, device=device)
        scales = torch.empty((*lead, pitch), dtype=torch.uint8, device=device)
        if pitch * MX_BLOCK != n:
            scales = scales[..., :n // MX_BLOCK]
        return cls._of(codes, scales, fmt, torch.Size((*lead, n)))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def in_features(self) -> int:
        return self.shape[-1]

    @property
    def out_features(self) -> int:
        return self.shape[-2]

    @property
    def rows(self) -> int:
        return self.shape[:-1].numel()

    def to(self, device) -> "MxTensor":
        return MxTensor(self.codes.to(device), self.scales.to(device), self.fmt)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return mx_dequantize(self, dtype)

    def __repr__(self) -> str:
        return f"MxTensor({self.fmt}, shape={tuple(self.shape)}, device={self.device})"


def _row_pitch(scales: torch.Tensor, n: int) -> int:
    """Bytes between rows of a scale tensor in the kernels' layout."""
    return scales.stride(-2) if scales.dim() > 1 else _pitch(n)


def _scales_laid_out(scales: torch.Tensor, n: int) -> bool:
    """Whether rows start a multiple of 16 bytes apart, evenly over all leading
    dimensions, and the last row's padding is inside the storage."""
    if scales.stride(-1) != 1 and scales.shape[-1] > 1 or scales.data_ptr() % 16:
        return False
    pitch = _row_pitch(scales, n)
    if pitch % 16 or pitch < _pitch(n):
        return False
    step = pitch
    for size, stride in zip(reversed(scales.shape[:-1]), reversed(scales.stride()[:-1])):
        if stride != step:
            return False
        step *= size
    rows = scales.shape[:-1].numel()
    last = scales.storage_offset() + max(rows - 1, 0) * pitch + _pitch(n)
    return rows == 0 or last <= scales.untyped_storage().nbytes()


def _lay_out(scales: torch.Tensor, n: int) -> torch.Tensor:
    pitch = _pitch(n)
    out = torch.zeros((*scales.shape[:-1], pitch), dtype=torch.uint8, device=scales.device)
    out = out[..., :n // MX_BLOCK]
    out.copy_(scales)
    return out


def _rows(x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """x as 16-byte aligned rows (a copy where it is not), and the values from
    one row to the next."""
    n, per16 = x.shape[-1], 16 // x.element_size()
    if not x.is_contiguous() and not (x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= n
                                      and x.stride(0) % per16 == 0):
        x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x, (x.stride(0) if x.dim() == 2 and x.shape[0] > 1 else n)


def _on(device: torch.device):
    """The launch's device is the tensors', whichever is current."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def mx_quantize(x: torch.Tensor, fmt: str = "mxfp8") -> MxTensor:
    """``x [..., n]`` (float16, bfloat16 or float32; n a multiple of 32) in MX:
    per block of 32 the scale ``2 ** (floor(log2(max |x|)) - emax)`` (emax 2
    for mxfp4, 8 for mxfp8) and the values divided by it, rounded to nearest
    even, saturating at 6 or 448.  A block that holds a NaN or an infinity
    stands for NaNs."""
    lib = _lib.load()
    code = _format(fmt)
    dev = _lib.require_device(x)
    if x.dtype not in MX_DTYPES:
        raise ValueError(f"mx_quantize: x must be float16, bfloat16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] == 0 or x.shape[-1] % MX_BLOCK:
        raise ValueError(f"mx_quantize: the last dimension must be a positive multiple of "
                         f"{MX_BLOCK}, got shape {tuple(x.shape)}")
    n = x.shape[-1]
    xr, ld = _rows(x)
    with _on(dev):
        out = MxTensor._empty(x.shape[:-1], n, fmt, dev)
        _lib.check(lib.nvm_mx_quantize(xr.data_ptr(), out.rows, n, ld, MX_DTYPES[x.dtype], code,
                                       out.codes.data_ptr(), out.scales.data_ptr(), _pitch(n),
                                       _lib.stream_of(dev)))
    return out


def mx_dequantize(t: MxTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that ``t`` stands for, rounded once to ``dtype``."""
    lib = _lib.load()
    dev = _lib.require_device(t.codes, t.scales)
    if dtype not in MX_DTYPES:
        raise ValueError(f"mx_dequantize: dtype must be float16, bfloat16 or float32, got {dtype}")
    n = t.shape[-1]
    with _on(dev):
        out = torch.empty(t.shape, dtype=dtype, device=dev)
        _lib.check(lib.nvm_mx_dequantize(t.codes.data_ptr(), t.scales.data_ptr(),
                                         _row_pitch(t.scales, n), t.rows, n, MX_FORMATS[t.fmt],
                                         MX_DTYPES[dtype], out.data_ptr(), _lib.stream_of(dev)))
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
    H = h.shape[-1]
    if r is not None and (r.shape != h.shape or r.dtype != h.dtype):
        raise ValueError("residual_rms_norm_mx: r must have the shape and dtype of h")
    if weight.numel() != H:
        raise ValueError(f"residual_rms_norm_mx: weight must have {H} elements")
    hc = _packed(h)
    rc = None if r is None else _packed(r)
    w = _packed(weight if weight.dtype == h.dtype else weight.to(h.dtype))
    with _on(dev):
        out = MxTensor._empty(h.shape[:-1], H, fmt, dev) if H % MX_BLOCK == 0 and H else None
        if out is None:
            raise ValueError(f"residual_rms_norm_mx: the last dimension must be a positive "
                             f"multiple of {MX_BLOCK}, got {H}")
        h_out = torch.empty_like(hc) if r is not None else None
        _lib.check(lib.nvm_residual_rms_norm_mx(
            hc.data_ptr(), _lib.ptr(rc), w.data_ptr(), out.rows, H, float(eps),
            _lib.dtype_code(h.dtype), _lib.ptr(h_out), code, out.codes.data_ptr(),
            out.scales.data_ptr(), _pitch(H), _lib.stream_of(dev)))
    return (h if h_out is None else h_out), out


def _packed(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _activations(x: Union[MxTensor, torch.Tensor], op: str) -> MxTensor:
    if isinstance(x, MxTensor):
        return x
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{op}: x must be an MxTensor, float16 or bfloat16, got {x.dtype}")
    return mx_quantize(x, "mxfp8")


def _check_weight(op: str, name: str, w: MxTensor, n: int) -> None:
    if not isinstance(w, MxTensor) or w.fmt != "mxfp4" or len(w.shape) != 2:
        raise ValueError(f"{op}: {name} must be a two-dimensional mxfp4 MxTensor")
    if w.shape[1] != n:
        raise ValueError(f"{op}: {name} has {w.shape[1]} input features, x has {n}")


def mx_linear(x: Union[MxTensor, torch.Tensor], w: MxTensor,
              dtype: Optional[torch.dtype] = None,
              bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x . w^T (+ bias)``: ``x [..., N]`` in MX (16-bit activations are
    quantised to mxfp8 first), ``w [K, N]`` in mxfp4.  Exact products, float32
    sums, one rounding to ``dtype`` (float16, bfloat16 or float32; by default
    that of 16-bit activations, else bfloat16)."""
    lib = _lib.load()
    if dtype is None:
        dtype = torch.bfloat16 if isinstance(x, MxTensor) else x.dtype
    if dtype not in MX_DTYPES:
        raise ValueError(f"mx_linear: dtype must be float16, bfloat16 or float32, got {dtype}")
    a = _activations(x, "mx_linear")
    n = a.shape[-1]
    _check_weight("mx_linear", "w", w, n)
    dev = _lib.require_device(a.codes, w.codes)
    K = w.shape[0]
    with _on(dev):
        out = torch.empty((*a.shape[:-1], K), dtype=dtype, device=dev)
        _lib.check(lib.nvm_mx_matmul(
            a.codes.data_ptr(), a.scales.data_ptr(), _row_pitch(a.scales, n), MX_FORMATS[a.fmt],
            w.codes.data_ptr(), w.scales.data_ptr(), _row_pitch(w.scales, n), a.rows, n, K,
            MX_DTYPES[dtype], out.data_ptr(), _lib.stream_of(dev)))
    return out if bias is None else out + bias


def mx_swiglu(x: Union[MxTensor, torch.Tensor], w_gate: MxTensor, w_up: MxTensor,
              fmt: str = "mxfp8") -> MxTensor:
    """``silu(x . gate^T) * (x . up^T)`` in MX, the input of a down projection
    (models/qwen3.py:176-184): ``x`` as for ``mx_linear``, both weights ``[K,
    N]`` in mxfp4, K a multiple of 32.  Everything up to the quantisation is
    float32."""
    lib = _lib.load()
    code = _format(fmt)
    a = _activations(x, "mx_swiglu")
    n = a.shape[-1]
    _check_weight("mx_swiglu", "w_gate", w_gate, n)
    _check_weight("mx_swiglu", "w_up", w_up, n)
    K = w_gate.shape[0]
    if w_up.shape[0] != K or K == 0 or K % MX_BLOCK:
        raise ValueError(f"mx_swiglu: gate and up must have the same output features, a positive "
                         f"multiple of {MX_BLOCK}, got {K} and {w_up.shape[0]}")
    dev = _lib.require_device(a.codes, w_gate.codes, w_up.codes)
    with _on(dev):
        out = MxTensor._empty(a.shape[:-1], K, fmt, dev)
        _lib.check(lib.nvm_mx_swiglu(
            a.codes.data_ptr(), a.scales.data_ptr(), _row_pitch(a.scales, n), MX_FORMATS[a.fmt],
            w_gate.codes.data_ptr(), w_gate.scales.data_ptr(), _row_pitch(w_gate.scales, n),
            w_up.codes.data_ptr(), w_up.scales.data_ptr(), _row_pitch(w_up.scales, n), a.rows, n,
            K, code, out.codes.data_ptr(), out.scales.data_ptr(), _pitch(K),
            _lib.stream_of(dev)))
    return out
