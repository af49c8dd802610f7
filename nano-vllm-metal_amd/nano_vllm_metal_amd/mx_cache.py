"""The 4-bit KV cache on the GPU (include/nvm_mx_cache.h).

``MxPages`` holds a layer's keys or values in MXFP4, 4.25 bits a value: the
page pools of ``PagedKVCache(..., kv_bits=4)``.  ``qk_norm_rope_store_mx``
stands beside ``qk_norm_rope_store`` (``models/qwen3.py:103-133``) and
``paged_attention_mx`` beside ``paged_attention``
(``layers/attention.py:154-230``), over such pages; ``paged_kv_read_mx`` says
what stored rows stand for.  The reference's own quantised cache has eight
bits (``kv_bits``).  No CPU fallback.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .mx import MX_BLOCK, MxTensor, _current_device, _raw_stream, mx_dequantize

_INT_TYPES = {torch.uint8, torch.int8, torch.uint16, torch.int16, torch.uint32, torch.int32,
              torch.int64}
_CODES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # nvm_kv_dtype


class MxPages:
    """Pages ``[P, num_kv_heads, page_size, D]`` of keys or values in MXFP4:
    ``codes`` uint8 ``[..., D / 2]`` (E2M1, the even value in the low half) and
    ``scales`` uint8 ``[..., D / 32]``, byte b standing for ``2 ** (b - 127)``,
    255 for NaN.  Both contiguous: the store writes into them, wherever they lie at
    the call."""

    # _at: the addresses that were checked
    __slots__ = ("_codes", "_scales", "shape", "device", "_index", "_at")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("MxPages: codes and scales must be uint8")
        if codes.dim() != 4 or scales.dim() != 4 or codes.shape[:3] != scales.shape[:3]:
            raise ValueError("MxPages: codes [P, Hkv, page_size, D/2] and scales [P, Hkv, page_size, "
                             f"D/32], got {tuple(codes.shape)} and {tuple(scales.shape)}")
        D = 2 * codes.shape[3]
        if D == 0 or D % MX_BLOCK or scales.shape[3] * MX_BLOCK != D or 0 in codes.shape:
            raise ValueError(f"MxPages: codes {tuple(codes.shape)} and scales "
                             f"{tuple(scales.shape)} are not pages of blocks of {MX_BLOCK}")
        if codes.device != scales.device:
            raise ValueError("MxPages: codes and scales must be on one device")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("MxPages: codes and scales must be contiguous")
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("MxPages: codes and scales must be 16-byte aligned")
        self._codes, self._scales = codes, scales
        self.shape = torch.Size((*codes.shape[:3], D))
        self.device = codes.device
        self._index = codes.get_device()
        self._at = (codes.data_ptr(), scales.data_ptr())

    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    def _refresh(self) -> None:
        """Checks codes and scales that lie elsewhere than before (``set_``, ``data``)."""
        shape = self.shape
        self.__init__(self._codes, self._scales)
        if self.shape != shape:
            now, self.shape = self.shape, shape
            self._at = (0, 0)
            raise ValueError(f"MxPages: pages of {tuple(shape)} have become {tuple(now)}")

    @classmethod
    def zeros(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int,
              device="cuda") -> "MxPages":
        if head_dim % MX_BLOCK:
            raise ValueError(f"MxPages: head dim {head_dim} must be a multiple of {MX_BLOCK}")
        lead = (num_pages, num_kv_heads, page_size)
        return cls(torch.zeros((*lead, head_dim // 2), dtype=torch.uint8, device=device),
                   torch.zeros((*lead, head_dim // MX_BLOCK), dtype=torch.uint8, device=device))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What all the pages stand for, ``[P, num_kv_heads, page_size, D]``."""
        return mx_dequantize(MxTensor(self.codes, self.scales, "mxfp4"), dtype)

    def __reduce__(self):
        return MxPages, (self.codes, self.scales)

    def __repr__(self) -> str:
        return f"MxPages(shape={tuple(self.shape)}, device={self.device})"


def _check_pages(op: str, key_pages: MxPages, value_pages: MxPages) -> int:
    """The one GPU of both."""
    if type(key_pages) is not MxPages or type(value_pages) is not MxPages:
        raise ValueError(f"{op}: key_pages and value_pages must be MxPages")
    for p in (key_pages, value_pages):
        codes, scales = p._at
        if p._codes.data_ptr() != codes or p._scales.data_ptr() != scales:
            p._refresh()
    if key_pages.shape != value_pages.shape:
        raise ValueError(f"{op}: key and value pages differ in shape")
    index = key_pages._index
    if index < 0 or value_pages._index != index:
        _lib.require_device(key_pages.codes, value_pages.codes)
    return index


def _ints(op: str, name: str, t: torch.Tensor, n: int, index: int) -> torch.Tensor:
    """`n` int32 values in a row, on device `index`."""
    if t.dtype != torch.int32:
        if t.dtype not in _INT_TYPES:
            raise ValueError(f"{op}: {name} must be integers of at most 63 bits, got {t.dtype}")
        if t.dtype in (torch.int64, torch.uint32):  # (what 32 bits would wrap stays outside)
            t = t.to(torch.int64).clamp(-1, 0x7FFFFFFF)
        t = t.to(torch.int32)
    if t.numel() != n:
        raise ValueError(f"{op}: {name} must have {n} elements, got {t.numel()}")
    if t.get_device() != index:
        raise ValueError(f"{op}: {name} is not on the pages' device")
    return t if t.is_contiguous() else t.contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t if t.is_contiguous() else t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def qk_norm_rope_store_mx(qkv: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int,
                          q_norm: torch.Tensor, k_norm: torch.Tensor, eps: float,
                          positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                          page_ids: torch.Tensor, slots: torch.Tensor, key_pages: MxPages,
                          value_pages: MxPages, want_kv: bool = False,
                          out_dtype: Optional[torch.dtype] = None
                          ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``qk_norm_rope_store`` into 4-bit pages: ``qkv [..., (Hq + 2 Hkv) * D]``
    -> ``q [T, Hq, D]`` (and, with ``want_kv``, ``k, v [T, Hkv, D]``, not
    quantised) of ``out_dtype``, the dtype of ``qkv`` or float32, both holding
    values rounded once to the dtype of ``qkv``; k and v quantised into slots
    ``[page_ids[t], :, slots[t]]``.  k is not rounded before it is quantised.
    Slots outside the pages are not stored; what a slot holds that two tokens
    name is not specified."""
    op = "qk_norm_rope_store_mx"
    lib = _lib.load()
    index = _check_pages(op, key_pages, value_pages)
    P, Hkv, ps, D = key_pages.shape
    if Hkv != num_kv_heads or D != head_dim:
        raise ValueError(f"{op}: pages must be [P, {num_kv_heads}, page_size, {head_dim}], got "
                         f"{tuple(key_pages.shape)}")
    dtype = _lib.dtype_code(qkv.dtype)
    out_dtype = qkv.dtype if out_dtype is None else out_dtype
    if out_dtype != qkv.dtype and out_dtype != torch.float32:
        raise ValueError(f"{op}: out_dtype must be {qkv.dtype} or float32, got {out_dtype}")
    width = (num_heads + 2 * num_kv_heads) * D
    if num_heads <= 0 or qkv.dim() == 0 or qkv.shape[-1] != width:
        raise ValueError(f"{op}: qkv must be [..., {width}], got {tuple(qkv.shape)}")
    if q_norm.numel() != D or k_norm.numel() != D:
        raise ValueError(f"{op}: q_norm/k_norm must have {D} elements")
    if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != D // 2:
        raise ValueError(f"{op}: cos/sin must be [max_pos, {D // 2}]")
    for t in (qkv, q_norm, k_norm, cos, sin):
        if t.get_device() != index:
            _lib.require_device(key_pages.codes, t)
    if index != _current_device():
        with torch.cuda.device(index):
            return qk_norm_rope_store_mx(qkv, num_heads, num_kv_heads, head_dim, q_norm, k_norm,
                                         eps, positions, cos, sin, page_ids, slots, key_pages,
                                         value_pages, want_kv, out_dtype)
    # (converted operands are held until the call: a temporary's memory could
    # become the next one's)
    x = _aligned(qkv)
    T = x.numel() // width
    pos = _ints(op, "positions", positions, T, index)
    pages = _ints(op, "page_ids", page_ids, T, index)
    at = _ints(op, "slots", slots, T, index)
    qn = _aligned(q_norm if q_norm.dtype == qkv.dtype else q_norm.to(qkv.dtype))
    kn = _aligned(k_norm if k_norm.dtype == qkv.dtype else k_norm.to(qkv.dtype))
    c = _aligned(cos if cos.dtype == torch.float32 else cos.to(torch.float32))
    s = _aligned(sin if sin.dtype == torch.float32 else sin.to(torch.float32))
    dev = qkv.device
    q = torch.empty((T, num_heads, D), dtype=out_dtype, device=dev)
    k = torch.empty((T, Hkv, D), dtype=out_dtype, device=dev) if want_kv else None
    v = torch.empty((T, Hkv, D), dtype=out_dtype, device=dev) if want_kv else None
    kc, ks = key_pages._at
    vc, vs = value_pages._at
    _lib.check(lib.nvm_qk_norm_rope_store_mx(
        x.data_ptr(), T, num_heads, Hkv, D, qn.data_ptr(), kn.data_ptr(), eps, pos.data_ptr(),
        c.data_ptr(), s.data_ptr(), c.shape[0], pages.data_ptr(), at.data_ptr(), kc, ks, vc, vs, P,
        ps, dtype, _CODES[out_dtype], q.data_ptr(), _lib.ptr(k), _lib.ptr(v), _raw_stream(index)))
    return q, k, v


def paged_kv_read_mx(key_pages: MxPages, value_pages: MxPages, page_ids: torch.Tensor,
                     slots: torch.Tensor, dtype: torch.dtype = torch.float32
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """What the slots ``(page_ids[t], slots[t])`` stand for: ``k, v [T,
    num_kv_heads, D]``, rounded once to ``dtype`` (float16, bfloat16 or
    float32).  Slots outside the pages give zeros."""
    op = "paged_kv_read_mx"
    lib = _lib.load()
    index = _check_pages(op, key_pages, value_pages)
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"{op}: dtype must be float16, bfloat16 or float32, got {dtype}")
    if index != _current_device():
        with torch.cuda.device(index):
            return paged_kv_read_mx(key_pages, value_pages, page_ids, slots, dtype)
    P, Hkv, ps, D = key_pages.shape
    T = page_ids.numel()
    pages = _ints(op, "page_ids", page_ids, T, index)
    at = _ints(op, "slots", slots, T, index)
    k = torch.empty((T, Hkv, D), dtype=dtype, device=pages.device)
    v = torch.empty((T, Hkv, D), dtype=dtype, device=pages.device)
    kc, ks = key_pages._at
    vc, vs = value_pages._at
    _lib.check(lib.nvm_paged_kv_read_mx(kc, ks, vc, vs, P, Hkv, ps, D, pages.data_ptr(),
                                        at.data_ptr(), T, code, k.data_ptr(), v.data_ptr(),
                                        _raw_stream(index)))
    return k, v


def paged_attention_mx(query: torch.Tensor, key_pages: MxPages, value_pages: MxPages,
                       block_table: torch.Tensor, context_lens: torch.Tensor,
                       scale: Optional[float] = None, mask: Optional[str] = None,
                       out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``paged_attention`` over 4-bit pages: ``softmax(query . paged_key^T *
    scale) . paged_value``.

    ``query [B, num_heads, L, D]`` of float16, bfloat16 or float32 (read where
    it lies if its rows are contiguous and 16-byte aligned, so a transposed
    token-major query is not copied); ``block_table [B, max_pages]`` physical
    page ids (negative or beyond the pool: no page); ``context_lens [B]``;
    ``mask`` None or ``"causal"`` (query row i of L sees key positions j <= i +
    context_len - L).  Rows that see nothing are zero.  Sums are float32; the
    result is rounded once to ``out_dtype`` (by default the query's), ``[B,
    num_heads, L, D]`` as a view of ``[B, L, num_heads, D]``."""
    op = "paged_attention_mx"
    if mask is not None and mask != "causal":
        raise NotImplementedError(f"{op}: unsupported mask {mask!r}")
    lib = _lib.load()
    index = _check_pages(op, key_pages, value_pages)
    if query.dim() != 4:
        raise ValueError(f"{op}: query must be [B, num_heads, L, D], got {tuple(query.shape)}")
    B, Hq, L, D = query.shape
    P, Hkv, ps, Dk = key_pages.shape
    if Dk != D:
        raise ValueError(f"{op}: q and page tensors must have the same head dimension")
    if Hq == 0 or Hq % Hkv:
        raise ValueError(f"{op}: num_heads must be divisible by num_kv_heads")
    if block_table.dim() != 2 or context_lens.dim() != 1 or block_table.shape[0] != B \
            or context_lens.shape[0] != B:
        raise ValueError(f"{op}: block_table [B, max_pages] and context_lens [B] must match the "
                         "query batch")
    q_code = _CODES.get(query.dtype)
    out_dtype = query.dtype if out_dtype is None else out_dtype
    o_code = _CODES.get(out_dtype)
    if q_code is None or o_code is None:
        raise ValueError(f"{op}: query and out_dtype must be float16, bfloat16 or float32, got "
                         f"{query.dtype} and {out_dtype}")
    if query.get_device() != index:
        _lib.require_device(key_pages.codes, query)
    if index != _current_device():
        with torch.cuda.device(index):
            return paged_attention_mx(query, key_pages, value_pages, block_table, context_lens,
                                      scale, mask, out_dtype)
    max_pages = block_table.shape[1]
    bt = _ints(op, "block_table", block_table, B * max_pages, index)
    lens = _ints(op, "context_lens", context_lens, B, index)
    out = torch.empty((B, L, Hq, D), dtype=out_dtype, device=query.device)
    if out.numel() == 0:
        return out.transpose(1, 2)
    sb, sh, sl, sd = query.stride()
    unit = 4 if q_code == 2 else 8
    if sd != 1 or sb % unit or sh % unit or sl % unit or query.data_ptr() % 16:
        query = query.clone(memory_format=torch.contiguous_format)
        sb, sh, sl, _ = query.stride()
    size = _lib.workspace_size("nvm_paged_attention_mx_workspace_size", B, L, D, max_pages, ps, Hkv,
                               Hq)
    ws = torch.empty(size, dtype=torch.uint8, device=query.device) if size else None
    kc, ks = key_pages._at
    vc, vs = value_pages._at
    _lib.check(lib.nvm_paged_attention_mx(
        query.data_ptr(), q_code, sb, sh, sl, B, L, D, kc, ks, vc, vs, P, ps, bt.data_ptr(),
        max_pages, lens.data_ptr(), D ** -0.5 if scale is None else scale, mask is not None, Hkv,
        Hq, o_code, out.data_ptr(), _lib.ptr(ws), size, _raw_stream(index)))
    return out.transpose(1, 2)
