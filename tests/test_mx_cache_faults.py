"""The 4-bit cache without a GPU: calls that went wrong before any kernel ran."""

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
