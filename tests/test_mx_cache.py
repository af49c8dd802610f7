"""The 4-bit KV cache without a GPU: what the entry points refuse, and the
oracle's own sanity."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import attention_oracle as AO
from oracle import mx_cache_oracle as C
from oracle import mx_oracle as MX


def _lib():
    from nano_vllm_metal_amd import _lib

    return _lib, _lib.load()


def _err(lib):
    return lib.nvm_last_error().decode()


A = 4096  # an aligned address that nothing reads: every call below is refused or empty

STORE = dict(qkv=A, T=4, Hq=8, Hkv=2, D=64, qw=A, kw=A, eps=1e-6, pos=A, cos=A, sin=A, max_pos=100,
             pages=A, slots=A, kc=A, ks=A, vc=A, vs=A, P=3, ps=16, dtype=1, out=1, q=A, k=None,
             v=None, st=None)


@pytest.mark.parametrize("kw,code,msg", [
    ({"dtype": 2}, -1, "dtype must be"),
    ({"out": 0}, -1, "out dtype"),
    ({"out": 3}, -1, "out dtype"),
    ({"T": -1}, -1, "bad shape"),
    ({"Hq": 0}, -1, "bad shape"),
    ({"max_pos": 0}, -1, "bad shape"),
    ({"Hkv": 0}, -1, "bad pages"),
    ({"P": 0}, -1, "bad pages"),
    ({"ps": 0}, -1, "bad pages"),
    ({"D": 0}, -1, "bad pages"),
    ({"D": 48}, -2, "head dim"),
    ({"D": 288}, -2, "head dim"),
    ({"P": 1 << 40}, -2, "pool too large"),
    ({"ps": 1 << 31}, -2, "pool too large"),
    ({"P": 1 << 30, "ps": 1 << 30}, -2, "pool too large"),
    ({"T": 1 << 40}, -2, "too many"),
    ({"Hq": 1 << 21}, -2, "too many"),
    ({"max_pos": 1 << 31}, -2, "too many"),
    ({"kc": None}, -1, "null page"),
    ({"vs": None}, -1, "null page"),
    ({"ks": A + 8}, -1, "aligned"),
    ({"qkv": None}, -1, "null pointer"),
    ({"pos": None}, -1, "null pointer"),
    ({"q": None}, -1, "null pointer"),
    ({"qkv": A + 2}, -1, "aligned"),
    ({"cos": A + 4}, -1, "aligned"),
    ({"v": A + 8}, -1, "aligned"),
])
def test_store_refusals(kw, code, msg):
    _, lib = _lib()
    assert lib.nvm_qk_norm_rope_store_mx(*(STORE | kw).values()) == code
    assert msg in _err(lib)


READ = dict(kc=A, ks=A, vc=A, vs=A, P=3, Hkv=2, ps=16, D=64, pages=A, slots=A, T=5, out=2, k=A, v=A,
            st=None)


@pytest.mark.parametrize("kw,code,msg", [
    ({"out": 3}, -1, "out dtype"),
    ({"P": -1}, -1, "bad pages"),
    ({"D": 33}, -2, "head dim"),
    ({"T": -2}, -1, "bad shape"),
    ({"T": 1 << 32}, -2, "too many"),
    ({"vc": None}, -1, "null page"),
    ({"slots": None}, -1, "null pointer"),
    ({"k": A + 4}, -1, "aligned"),
])
def test_read_refusals(kw, code, msg):
    _, lib = _lib()
    assert lib.nvm_paged_kv_read_mx(*(READ | kw).values()) == code
    assert msg in _err(lib)


ATTEND = dict(q=A, qt=1, sb=512, sh=64, sl=64, B=2, L=1, D=64, kc=A, ks=A, vc=A, vs=A, P=9, ps=16,
              bt=A, mp=4, lens=A, scale=0.125, causal=1, Hkv=2, Hq=8, ot=1, out=A, ws=A,
              bytes=1 << 40, st=None)


@pytest.mark.parametrize("kw,code,msg", [
    ({"qt": 3}, -1, "dtypes"),
    ({"ot": 3}, -1, "dtypes"),
    ({"Hq": 7}, -1, "divisible"),
    ({"Hkv": 0}, -1, "divisible"),
    ({"B": -1}, -1, "bad shape"),
    ({"L": 0}, -1, "bad shape"),
    ({"ps": 0}, -1, "bad shape"),
    ({"mp": -1}, -1, "bad shape"),
    ({"D": 40}, -2, "head dim"),
    ({"D": 512}, -2, "head dim"),
    ({"mp": 1 << 28}, -2, "capacity"),
    ({"B": 1 << 30}, -2, "too many"),
    ({"B": 1 << 20, "L": 1 << 20}, -2, "too many"),
    ({"P": 0}, -1, "bad pages"),
    ({"kc": None}, -1, "null page"),
    ({"vc": A + 1}, -1, "aligned"),
    ({"q": None}, -1, "null pointer"),
    ({"bt": None}, -1, "null pointer"),
    ({"lens": None}, -1, "null pointer"),
    ({"out": None}, -1, "null pointer"),
    ({"q": A + 2}, -1, "query rows"),
    ({"sh": 60}, -1, "query rows"),
    ({"qt": 2, "sl": 66}, -1, "query rows"),
])
def test_attention_refusals(kw, code, msg):
    _, lib = _lib()
    assert lib.nvm_paged_attention_mx(*(ATTEND | kw).values()) == code
    assert msg in _err(lib)


def test_empty_calls_do_nothing():
    L, lib = _lib()
    assert lib.nvm_qk_norm_rope_store_mx(*(STORE | {"T": 0, "qkv": None}).values()) == 0
    assert lib.nvm_paged_kv_read_mx(*(READ | {"T": 0, "k": None}).values()) == 0
    assert lib.nvm_paged_attention_mx(*(ATTEND | {"B": 0, "q": None}).values()) == 0
    size = ctypes.c_size_t(7)
    assert lib.nvm_paged_attention_mx_workspace_size(0, 1, 128, 9, 16, 4, 32, ctypes.byref(size)) == 0
    assert size.value == 0
    assert lib.nvm_paged_attention_mx_workspace_size(1, 1, 128, 9, 16, 4, 32, None) == L.NVM_ERR_INVALID


def test_pages_are_checked():
    from nano_vllm_metal_amd import MxPages

    def make(c, s, dt=torch.uint8):
        return MxPages(torch.zeros(c, dtype=dt), torch.zeros(s, dtype=torch.uint8))

    p = make((3, 2, 16, 32), (3, 2, 16, 2))
    assert p.shape == (3, 2, 16, 64)
    for bad in (lambda: make((3, 2, 16, 32), (3, 2, 16, 1)), lambda: make((3, 2, 16, 24), (3, 2, 16, 1)),
                lambda: make((3, 16, 32), (3, 16, 2)), lambda: make((0, 2, 16, 32), (0, 2, 16, 2)),
                lambda: make((3, 2, 16, 32), (3, 2, 8, 2)),
                lambda: make((3, 2, 16, 32), (3, 2, 16, 2), torch.int8),
                lambda: MxPages(p.codes.transpose(1, 2), p.scales.transpose(1, 2)),
                lambda: MxPages(p.codes.flatten()[1:1 + 16 * 32].reshape(1, 1, 16, 32),
                                torch.zeros(1, 1, 16, 2, dtype=torch.uint8)),
                lambda: MxPages.zeros(3, 2, 16, 48, "cpu")):
        with pytest.raises(ValueError, match="MxPages"):
            bad()


def test_python_refusals():
    """Everything is refused before any device work: CPU tensors at last."""
    from nano_vllm_metal_amd import (MxPages, paged_attention_mx, paged_kv_read_mx,
                                     qk_norm_rope_store_mx)

    p = MxPages.zeros(3, 2, 16, 64, "cpu")
    other = MxPages.zeros(4, 2, 16, 64, "cpu")
    i = torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU only"):
        paged_kv_read_mx(p, p, i, i)
    with pytest.raises(ValueError, match="differ in shape"):
        paged_kv_read_mx(p, other, i, i)
    with pytest.raises(ValueError, match="must be MxPages"):
        paged_kv_read_mx(p.codes, p.codes, i, i)
    q = torch.zeros(2, 8, 1, 64, dtype=torch.bfloat16)
    bt, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU only"):
        paged_attention_mx(q, p, p, bt, lens)
    with pytest.raises(NotImplementedError):
        paged_attention_mx(q, p, p, bt, lens, mask="window")
    with pytest.raises(ValueError, match="must be MxPages"):
        paged_attention_mx(q, q, q, bt, lens)
    with pytest.raises(ValueError, match="GPU only"):
        qk_norm_rope_store_mx(torch.zeros(5, 768, dtype=torch.bfloat16), 8, 2, 64, i, i, 1e-6, i, q, q,
                              i, i, p, p)


def test_oracle_attention_is_paged_attention_of_the_values():
    """Against the other oracle, over pages of float64 values."""
    g = torch.Generator().manual_seed(3)
    k, v = (C.random_pages(g, 12, 2, 16, 64) for _ in range(2))
    q = torch.randn(2, 4, 5, 64, generator=g)
    bt = torch.randperm(12, generator=g).reshape(2, 6).int()
    bt[1, 2] = -1
    lens = torch.tensor([70, 90], dtype=torch.int32)
    kd, vd = (MX.decode(c, s, "mxfp4").numpy() for c, s in (k, v))
    for causal in (False, True):
        got, bound = C.attention(q, k, v, bt, lens, 0.3, causal)
        want = AO.paged_attention(q.reshape(8, 5, 64).numpy(), kd, vd, bt.numpy(), lens.numpy(), 0.3,
                                  causal, 2, 4)
        assert torch.allclose(got.reshape(8, 5, 64), torch.from_numpy(want), rtol=1e-12, atol=1e-12)
        assert (bound > 0).all() and float(bound.max()) < 2e-2


def test_oracle_rotation():
    """Position zero leaves the normed row; a rotation keeps its length; half a
    turn changes its sign."""
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(3, 2, 64, generator=g), torch.ones(64)
    one, zero = torch.ones(3, 32), torch.zeros(3, 32)
    y, _ = C.norm_rope(x, w, one, zero, 0.0)
    assert torch.allclose(y, torch.nn.functional.rms_norm(x.double(), (64,), eps=0.0))
    z, size = C.norm_rope(x, w, -one, zero, 0.0)
    assert torch.equal(z, -y) and torch.equal(size, y.abs())
    a = torch.rand(3, 32, generator=g)
    r, _ = C.norm_rope(x, w, a.cos(), a.sin(), 0.0)
    assert torch.allclose(r.norm(dim=-1), y.norm(dim=-1), rtol=1e-6)
