"""token_logprobs without a GPU: what the entry points refuse."""

from __future__ import annotations

import ctypes

import pytest
import torch

A = 4096  # an aligned address that nothing reads: every call below is refused or empty
CALL = dict(x=A, N=3, V=1000, ld=1000, dtype=1, tokens=A, k=5, lp=A, ent=A, ids=A, top=A, ws=A,
            bytes=1 << 40, st=None)


def _lib():
    from nano_vllm_metal_amd import _lib

    return _lib, _lib.load()


@pytest.mark.parametrize("kw,code,msg", [
    ({"dtype": 3}, -1, "f16, bf16 or f32"),
    ({"dtype": -1}, -1, "f16, bf16 or f32"),
    ({"N": -1}, -1, "bad shape"),
    ({"V": 0}, -1, "bad shape"),
    ({"k": -1}, -1, "top_k"),
    ({"k": 11, "V": 10}, -1, "top_k"),
    ({"k": 65}, -2, "top_k at most 64"),
    ({"V": 1 << 31, "ld": 1 << 31}, -2, "too many"),
    ({"N": 1 << 24}, -2, "too many"),
    ({"ld": 999}, -1, "apart"),
    ({"x": None}, -1, "null pointer"),
    ({"tokens": None}, -1, "null pointer"),
    ({"ent": None}, -1, "null pointer"),
    ({"ids": None}, -1, "null pointer"),
    ({"x": A + 1}, -1, "aligned"),
    ({"x": A + 2, "dtype": 2}, -1, "aligned"),
])
def test_refusals(kw, code, msg):
    _, lib = _lib()
    assert lib.nvm_token_logprobs(*(CALL | kw).values()) == code
    assert msg in lib.nvm_last_error().decode()


def test_empty_batch_and_workspace():
    L, lib = _lib()
    assert lib.nvm_token_logprobs(*(CALL | {"N": 0, "x": None}).values()) == 0
    size = ctypes.c_size_t(7)
    assert lib.nvm_token_logprobs_workspace_size(0, 1000, 1, 5, ctypes.byref(size)) == 0
    assert size.value == 0
    assert lib.nvm_token_logprobs_workspace_size(1, 1000, 1, 5, None) == L.NVM_ERR_INVALID
    assert lib.nvm_token_logprobs_workspace_size(1, 1000, 9, 5, ctypes.byref(size)) == L.NVM_ERR_INVALID


def test_python_refusals():
    from nano_vllm_metal_amd import token_logprobs

    x, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU only"):
        token_logprobs(x, t)
    with pytest.raises(ValueError, match="float16, bfloat16 or float32"):
        token_logprobs(x.double(), t)
    with pytest.raises(ValueError, match="must match"):
        token_logprobs(x, t[:2])
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(x, t, 11)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(torch.zeros(3, 100), t, 65)
    with pytest.raises(ValueError, match="integers"):
        token_logprobs(x, t.float())
    with pytest.raises(ValueError, match="no logits"):
        token_logprobs(x[:, :0], t)
