"""The 4-bit cache and log probabilities without a GPU: calls that went wrong before
any kernel ran."""

from __future__ import annotations

import pytest
import torch


def _bytes(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


def test_pages_follow_their_tensors():
    """Codes and scales cannot be exchanged beside the addresses that were checked, and
    another storage of theirs is looked at again."""
    from nano_vllm_metal_amd import MxPages, paged_kv_read_mx

    p = MxPages.zeros(3, 2, 16, 64, "cpu")
    for name in ("codes", "scales"):
        with pytest.raises(AttributeError):
            setattr(p, name, _bytes(3, 2, 16, 32))
    i = torch.zeros(5, dtype=torch.int32)

    def refused(what):
        with pytest.raises(ValueError, match=what):
            paged_kv_read_mx(p, p, i, i)
        with pytest.raises(ValueError, match=what):  # (and not only once)
            paged_kv_read_mx(p, p, i, i)

    p.codes.data = _bytes(3, 2, 16, 32)
    refused("GPU only")
    assert p._at == (p.codes.data_ptr(), p.scales.data_ptr())
    p.codes.data, p.scales.data = _bytes(1, 2, 16, 32), _bytes(1, 2, 16, 2)
    refused("have become")
    p.codes.data = _bytes(3, 2, 16, 32)
    refused("MxPages: codes")
    p.scales.data = _bytes(3, 2, 16, 2)
    refused("GPU only")


def test_indices_of_every_type():
    """Values that 32 bits do not hold stay beyond every page, position and length;
    types that cannot be converted so are refused."""
    from nano_vllm_metal_amd.mx_cache import _ints

    for dt in (torch.uint8, torch.int8, torch.uint16, torch.int16, torch.uint32, torch.int32,
               torch.int64):
        got = _ints("op", "slots", torch.tensor([0, 1, 100], dtype=dt), 3, -1)
        assert got.dtype == torch.int32 and got.tolist() == [0, 1, 100]
    big = torch.tensor([2 ** 31, 2 ** 32 - 1, 2 ** 31 - 1], dtype=torch.uint32)
    assert _ints("op", "slots", big, 3, -1).tolist() == [2 ** 31 - 1] * 3
    big = torch.tensor([2 ** 31, 2 ** 32 + 5, -2 ** 32], dtype=torch.int64)
    assert _ints("op", "slots", big, 3, -1).tolist() == [2 ** 31 - 1, 2 ** 31 - 1, -1]
    for dt in (torch.uint64, torch.bool, torch.float32, torch.complex64):
        with pytest.raises(ValueError, match="slots must be integers"):
            _ints("op", "slots", torch.zeros(3, dtype=dt), 3, -1)


def test_most_query_rows():
    """A wavefront a query row: more than 2^32 - 256 threads are refused by name."""
    import ctypes

    from nano_vllm_metal_amd import _lib

    lib, size = _lib.load(), ctypes.c_size_t(7)

    def ask(rows):
        return lib.nvm_paged_attention_mx_workspace_size(rows, 1, 32, 1, 16, 1, 1, ctypes.byref(size))

    most = (2 ** 32 - 256) // 64
    assert ask(most) == _lib.NVM_OK and size.value == 0
    for rows in (most + 1, most + 3, 2 ** 26):
        assert ask(rows) == _lib.NVM_ERR_UNSUPPORTED
        assert "too many query rows" in lib.nvm_last_error().decode()


def test_cache_slots_outside_the_pages():
    """Sixteen bits, on the CPU: slots that are not there are not stored, nor taken for
    others counted from the end, and read as zeros."""
    from nano_vllm_metal_amd import PagedKVCache

    cache = PagedKVCache(1, 2, 8, 3, 4, torch.float32, "cpu")
    x = torch.arange(1.0, 1 + 6 * 16).reshape(1, 6, 2, 8)
    ids = torch.tensor([1, -1, 0, 4, 2, 2 ** 40])
    slots = torch.tensor([3, 0, -1, 0, 4, 1])
    cache.write(0, x, 2 * x, ids, slots)
    want = torch.zeros(3, 2, 4, 8)
    want[1, :, 3] = x[0, 0]
    assert torch.equal(cache.key_pages[0][:3], want)
    assert torch.equal(cache.value_pages[0][:3], 2 * want)
    k, v = cache.read(0, ids, slots)
    assert torch.equal(k[0], x[0, 0]) and torch.equal(v[0], 2 * x[0, 0])
    assert k.shape == (6, 2, 8) and not k[1:].any() and not v[1:].any()


def test_counts_of_alternatives_are_whole_numbers():
    """Refused before a request has pages, which it would keep."""
    import numpy as np

    from nano_vllm_metal_amd.llm import _check_top

    for n in (None, 0, 5, 64, np.int64(3)):
        _check_top("x", n, 1000)
    for n in (2.5, 3.0, "3", float("nan"), [1], torch.tensor(2.0)):
        with pytest.raises(ValueError, match="x must be in .*a whole number"):
            _check_top("x", n, 1000)
