"""Log probabilities of tokens on the GPU (include/nvm_logprobs.h).

What a model answers beside a token: how probable it was, how undecided the
model, and what else it might have said.  ``LLM.generate`` calls it for
``SamplingParams.logprobs`` and ``LLM.score`` for a text's own tokens; it stands
beside ``sample`` (``layers/sampler.py``).  No CPU fallback.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

MAX_TOP_LOGPROBS = 64
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # nvm_logits_dtype
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # float32 [...]
    entropy: torch.Tensor       # float32 [...]
    top_ids: torch.Tensor       # int64 [..., top_k]
    top_logprobs: torch.Tensor  # float32 [..., top_k]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Of each row of ``logits [..., V]`` (float16, bfloat16 or float32), with
    ``p`` its softmax: ``log p`` of the row's token of ``tokens [...]`` (0 for one
    outside ``[0, V)``), the entropy ``-sum p log p`` in nats, and the ``top_k``
    (at most 64) most probable tokens with their ``log p``, in descending order of
    their logits, equal ones by ascending id.  A row with a NaN or +infinity, or
    of -infinities only, gives NaNs.  Rows of a two-dimensional ``logits`` may lie
    apart; others are made contiguous."""
    op = "token_logprobs"
    lib = _lib.load()
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise ValueError(f"{op}: logits must be float16, bfloat16 or float32, got {logits.dtype}")
    lead = tokens.shape
    if logits.dim() == 0 or logits.shape[:-1] != lead:
        raise ValueError(f"{op}: logits [..., V] and tokens [...] must match, got "
                         f"{tuple(logits.shape)} and {tuple(lead)}")
    V = logits.shape[-1]
    if V == 0:
        raise ValueError(f"{op}: rows of no logits")
    if not 0 <= top_k <= min(V, MAX_TOP_LOGPROBS):
        raise ValueError(f"{op}: top_k must be in [0, {min(V, MAX_TOP_LOGPROBS)}], got {top_k}")
    if tokens.dtype != torch.int64:
        if tokens.dtype.is_floating_point or tokens.dtype.is_complex or tokens.dtype == torch.bool:
            raise ValueError(f"{op}: tokens must be integers, got {tokens.dtype}")
        tokens = tokens.to(torch.int64)
    index = logits.get_device()
    if index < 0 or tokens.get_device() != index:
        _lib.require_device(logits, tokens)
    if index != _current_device():
        with torch.cuda.device(index):
            return token_logprobs(logits, tokens, top_k)
    ld = V
    if not logits.is_contiguous():
        if logits.dim() == 2 and logits.stride(1) == 1 and logits.stride(0) >= V:
            ld = logits.stride(0)
        else:
            logits = logits.contiguous()
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    N = tokens.numel()
    dev = logits.device
    lp = torch.empty(lead, dtype=torch.float32, device=dev)
    ent = torch.empty(lead, dtype=torch.float32, device=dev)
    ids = torch.empty((*lead, top_k), dtype=torch.int64, device=dev)
    top = torch.empty((*lead, top_k), dtype=torch.float32, device=dev)
    size = _lib.workspace_size("nvm_token_logprobs_workspace_size", N, V, code, top_k)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _lib.check(lib.nvm_token_logprobs(logits.data_ptr(), N, V, ld, code, tokens.data_ptr(), top_k,
                                      lp.data_ptr(), ent.data_ptr(), ids.data_ptr(), top.data_ptr(),
                                      _lib.ptr(ws), size, _raw_stream(index)))
    return TokenLogprobs(lp, ent, ids, top)
