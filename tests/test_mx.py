"""The microscaled path without a GPU: what the entry points refuse (before any
device work, so with pointers that are never read), how an ``MxTensor`` lies in
memory, the ``mxfp4`` checkpoint loader, and the 64-bit oracle itself."""

from __future__ import annotations

import json

import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

FMTS = ["mxfp4", "mxfp8"]
P = 1 << 20  # a 16-byte aligned address


def _lib():
    from nano_vllm_metal_amd import _lib

    return _lib, _lib.load()


# ---------------------------------------------------------------- the C entries

# entry -> (argument names in order, a valid call)
CALLS = {
    "quantize": dict(x=P, rows=4, n=64, x_ld=64, dtype=1, fmt=1, codes=P, scales=P, ld=16, st=None),
    "dequantize": dict(codes=P, scales=P, ld=16, rows=4, n=64, fmt=0, dtype=1, out=P, st=None),
    "embedding": dict(ids=P, T=3, codes=P, scales=P, ld=16, V=9, n=64, fmt=0, dtype=1, out=P,
                      st=None),
    "residual_rms_norm_mx": dict(h=P, r=P, w=P, T=4, H=64, eps=1e-6, dtype=1, h_out=P, fmt=1,
                                 codes=P, scales=P, ld=16, st=None),
    "matmul": dict(a=P, as_=P, a_ld=16, fmt=1, w=P, ws=P, w_ld=16, M=4, N=64, K=32, dtype=1, out=P,
                   st=None),
    "swiglu": dict(a=P, as_=P, a_ld=16, fmt=1, g=P, gs=P, g_ld=16, u=P, us=P, u_ld=16, M=4, N=64,
                   K=32, ofmt=1, out=P, out_s=P, o_ld=16, st=None),
}
BIG = 1 << 31

REFUSALS = [
    ("quantize", dict(dtype=3), -1, "dtype"), ("quantize", dict(fmt=2), -1, "format"),
    ("quantize", dict(n=48), -1, "multiple of 32"), ("quantize", dict(n=0), -1, "bad shape"),
    ("quantize", dict(rows=-1), -1, "bad shape"), ("quantize", dict(x=None), -1, "null pointer"),
    ("quantize", dict(x=P + 8), -1, "16-byte aligned"), ("quantize", dict(x_ld=32), -1, "overlap"),
    ("quantize", dict(x_ld=65), -1, "aligned"), ("quantize", dict(codes=None), -1, "null pointer"),
    ("quantize", dict(codes=P + 4), -1, "aligned"), ("quantize", dict(scales=P + 1), -1, "aligned"),
    ("quantize", dict(ld=2), -1, "multiple of 16 bytes apart"),
    ("quantize", dict(n=1024, x_ld=1024, ld=16), -1, "at least 32"),
    ("quantize", dict(ld=1 << 21), -1, "apart"),
    ("quantize", dict(n=1 << 21, x_ld=1 << 21, ld=1 << 16), -2, "too large"),
    ("quantize", dict(rows=BIG), -2, "too large"),
    ("quantize", dict(rows=BIG - 1), -2, "2^35"),
    ("quantize", dict(x_ld=1 << 41), -1, "aligned"),
    ("dequantize", dict(dtype=-1), -1, "dtype"), ("dequantize", dict(fmt=9), -1, "format"),
    ("dequantize", dict(out=None), -1, "out must be"), ("dequantize", dict(out=P + 2), -1, "out"),
    ("dequantize", dict(scales=None), -1, "null pointer"), ("dequantize", dict(n=33), -1, "shape"),
    ("dequantize", dict(rows=BIG - 1), -2, "2^35"), ("dequantize", dict(ld=0), -1, "apart"),
    ("embedding", dict(T=-1), -1, "bad shape"), ("embedding", dict(V=0), -1, "bad shape"),
    ("embedding", dict(ids=None), -1, "ids"), ("embedding", dict(codes=None), -1, "null pointer"),
    ("embedding", dict(V=BIG), -2, "too large"), ("embedding", dict(T=BIG), -1, "bad shape"),
    ("embedding", dict(T=BIG - 1), -2, "2^35"), ("embedding", dict(out=P + 8), -1, "out"),
    ("embedding", dict(n=16), -1, "bad shape"), ("embedding", dict(ld=8), -1, "apart"),
    ("residual_rms_norm_mx", dict(dtype=2), -1, "dtype"),
    ("residual_rms_norm_mx", dict(H=8224, ld=272), -2, "H at most 8192"),
    ("residual_rms_norm_mx", dict(T=1 << 24), -2, "T at most"),
    ("residual_rms_norm_mx", dict(H=40), -1, "multiple of 32"),
    ("residual_rms_norm_mx", dict(h=None), -1, "null pointer"),
    ("residual_rms_norm_mx", dict(w=None), -1, "null pointer"),
    ("residual_rms_norm_mx", dict(h_out=None), -1, "null pointer"),
    ("residual_rms_norm_mx", dict(h=P + 2), -1, "aligned"),
    ("residual_rms_norm_mx", dict(r=P + 2), -1, "aligned"),
    ("residual_rms_norm_mx", dict(fmt=-1), -1, "format"),
    ("residual_rms_norm_mx", dict(codes=None), -1, "null pointer"),
    ("matmul", dict(dtype=3), -1, "out_dtype"), ("matmul", dict(fmt=2), -1, "a format"),
    ("matmul", dict(N=40), -1, "multiple of 32"), ("matmul", dict(K=-1), -1, "bad shape of w"),
    ("matmul", dict(M=-2), -1, "bad shape of a"), ("matmul", dict(a=None), -1, "(a)"),
    ("matmul", dict(ws=None), -1, "(w)"), ("matmul", dict(w=P + 8), -1, "of w must be"),
    ("matmul", dict(a_ld=8), -1, "scale rows of a"), ("matmul", dict(w_ld=24), -1, "rows of w"),
    ("matmul", dict(out=None), -1, "out must be"), ("matmul", dict(out=P + 4), -1, "out must be"),
    ("matmul", dict(M=BIG - 1, K=BIG - 1), -2, "too many output tiles"),
    ("matmul", dict(M=1, K=BIG - 1), -2, "too many output tiles"),
    ("swiglu", dict(K=48), -1, "bad shape of output"), ("swiglu", dict(K=0), -1, "bad shape"),
    ("swiglu", dict(ofmt=5), -1, "output format"), ("swiglu", dict(fmt=5), -1, "a format"),
    ("swiglu", dict(g=None), -1, "(gate)"), ("swiglu", dict(us=None), -1, "(up)"),
    ("swiglu", dict(out=None), -1, "(output)"), ("swiglu", dict(o_ld=2), -1, "rows of output"),
    ("swiglu", dict(u_ld=17), -1, "rows of up"), ("swiglu", dict(N=2), -1, "bad shape"),
    ("swiglu", dict(M=BIG - 1, K=1 << 20, o_ld=1 << 15), -2, "too many output tiles"),
]


def _call(name, **over):
    _, lib = _lib()
    args = dict(CALLS[name], **over)
    fn = getattr(lib, "nvm_" + name if name.endswith("_mx") else "nvm_mx_" + name)
    return fn(*args.values()), lib.nvm_last_error().decode()


@pytest.mark.parametrize("name,over,code,msg", REFUSALS)
def test_entries_refuse(name, over, code, msg):
    rc, err = _call(name, **over)
    assert rc == code and msg in err, (rc, err)


@pytest.mark.parametrize("name,over", [
    ("quantize", dict(rows=0, x=None)), ("dequantize", dict(rows=0, out=None)),
    ("embedding", dict(T=0, ids=None)), ("residual_rms_norm_mx", dict(T=0, h=None)),
    ("matmul", dict(M=0, a=None)), ("matmul", dict(K=0, w=None)), ("swiglu", dict(M=0, a=None))])
def test_entries_of_nothing_are_no_ops(name, over):
    assert _call(name, **over)[0] == 0


# -------------------------------------------------------------------- MxTensor


def _mx(rows, n, fmt="mxfp4"):
    from nano_vllm_metal_amd import MxTensor

    codes = torch.randint(0, 256, (rows, n // (2 if fmt == "mxfp4" else 1)), dtype=torch.uint8)
    return MxTensor(codes, torch.randint(100, 150, (rows, n // 32), dtype=torch.uint8), fmt)


@pytest.mark.parametrize("n", [32, 64, 480, 512, 544, 1024, 2080])
@pytest.mark.parametrize("fmt", FMTS)
def test_tensor_lies_in_rows_of_16_bytes(n, fmt):
    from nano_vllm_metal_amd import MxTensor

    codes = torch.randint(0, 256, (5, n // (2 if fmt == "mxfp4" else 1)), dtype=torch.uint8)
    scales = torch.randint(0, 256, (5, n // 32), dtype=torch.uint8)
    t = MxTensor(codes, scales, fmt)
    pitch = -(-n // 512) * 16
    assert t.shape == (5, n) and t.rows == 5 and t.pitch == pitch
    assert t.in_features == n and t.out_features == 5
    assert torch.equal(t.scales, scales) and torch.equal(t.codes, codes)
    assert t.scales.stride(0) == pitch and t.scales.data_ptr() % 16 == 0
    assert t.scales.untyped_storage().nbytes() >= 5 * pitch
    again = MxTensor(t.codes, t.scales, fmt)  # lies well: nothing is copied
    assert again.scales.data_ptr() == t.scales.data_ptr()
    assert MxTensor(t.codes[2:], t.scales[2:], fmt).scales.data_ptr() == t.scales[2:].data_ptr()


def test_tensor_copies_what_the_kernels_could_not_read():
    from nano_vllm_metal_amd import MxTensor

    codes = torch.randint(0, 256, (6, 64), dtype=torch.uint8)  # mxfp8, two blocks
    wide = torch.randint(0, 256, (6, 32), dtype=torch.uint8)
    fine = MxTensor(codes, wide[:, :2], "mxfp8")
    assert fine.pitch == 32 and fine.scales.data_ptr() == wide.data_ptr()
    for scales in (wide[:, 1:3],                                  # not aligned
                   wide[:, ::16],                                 # not in a row
                   torch.empty(6 * 18, dtype=torch.uint8).view(6, 18)[:, :2],  # 18 bytes apart
                   wide.view(-1)[160 + 16:].as_strided((2, 2), (0, 1)).expand(2, 2)[:1],
                   wide.flip(0)[:, :2].t().contiguous().t(),      # columns
                   wide.new_zeros(6, 2)):
        t = MxTensor(codes[:scales.shape[0]], scales, "mxfp8")
        assert torch.equal(t.scales, scales) and t.pitch % 16 == 0
        assert t.scales.data_ptr() % 16 == 0 and t.scales.stride(-1) in (1, 16)
        assert t.scales.untyped_storage().nbytes() - t.scales.storage_offset() >= 16 * t.rows
    # rows further apart than the kernels take: copied
    far = torch.zeros(2, (1 << 20) + 16, dtype=torch.uint8)[:, :2]
    assert MxTensor(codes[:2], far, "mxfp8").pitch == 16
    near = torch.zeros(2, 1 << 20, dtype=torch.uint8)[:, :2]
    assert MxTensor(codes[:2], near, "mxfp8").pitch == 1 << 20
    # the last row's padding would lie behind the storage: copied
    tight = torch.zeros(5 * 16 + 2, dtype=torch.uint8).as_strided((6, 2), (16, 1))
    assert MxTensor(codes, tight, "mxfp8").scales.data_ptr() != tight.data_ptr()
    # codes: contiguous and aligned
    odd = torch.zeros(6 * 64 + 1, dtype=torch.uint8)[1:].view(6, 64)
    t = MxTensor(odd, wide[:, :2], "mxfp8")
    assert t.codes.data_ptr() % 16 == 0 and torch.equal(t.codes, odd)
    assert MxTensor(codes.t().contiguous().t(), wide[:, :2], "mxfp8").codes.is_contiguous()


def test_tensor_of_more_dimensions_and_of_none():
    from nano_vllm_metal_amd import MxTensor

    c = torch.zeros(2, 3, 64, dtype=torch.uint8)
    t = MxTensor(c, torch.zeros(2, 3, 2, dtype=torch.uint8), "mxfp8")
    assert t.shape == (2, 3, 64) and t.rows == 6 and t.scales.stride() == (48, 16, 1)
    assert MxTensor(c[:, :0], t.scales[:, :0], "mxfp8").rows == 0
    assert MxTensor(c[0, 0], t.scales[0, 0], "mxfp8").rows == 1
    part = t.scales[:, :2]  # rows 16, 16, 32 apart: copied
    assert MxTensor(c[:, :2], part, "mxfp8").scales.data_ptr() != part.data_ptr()
    moved = t.to("cpu")
    assert moved.shape == t.shape and "mxfp8" in repr(moved)


@pytest.mark.parametrize("lead", [(), (1,), (5,), (2, 3), (2, 0, 3), (0,)])
@pytest.mark.parametrize("n", [32, 544, 2048])
@pytest.mark.parametrize("fmt", FMTS)
def test_tensor_that_a_kernel_writes(lead, n, fmt):
    """Codes and scales are views of one buffer, codes first, of the layout that
    an MxTensor of tensors has."""
    import copy
    import pickle

    from nano_vllm_metal_amd import MxTensor

    rows = int(np.prod(lead, dtype=np.int64))
    t = MxTensor._empty(lead, rows, n, fmt, "cpu")
    width, pitch = n // (2 if fmt == "mxfp4" else 1), -(-n // 512) * 16
    t._base.copy_(torch.randint(0, 256, t._base.shape, dtype=torch.uint8))
    assert t._base.numel() == rows * (width + pitch) and t.pitch == pitch and t.rows == rows
    codes, scales = t.codes, t.scales
    assert codes.shape == (*lead, width) and scales.shape == (*lead, n // 32)
    assert codes.is_contiguous() and t.codes is codes and t.scales is scales
    assert torch.equal(codes.reshape(-1), t._base[:rows * width])
    assert torch.equal(scales.reshape(rows, n // 32),
                       t._base[rows * width:].view(rows, pitch)[:, :n // 32])
    assert t._pointers() == (t._base.data_ptr(), t._base.data_ptr() + rows * width)
    again = MxTensor(codes, scales, fmt)
    assert again.pitch == pitch and again.shape == t.shape and again.rows == rows
    if rows:
        assert again._pointers() == t._pointers()  # (nothing was copied)
    for other in (copy.deepcopy(t), pickle.loads(pickle.dumps(t)), copy.deepcopy(again)):
        assert torch.equal(other.codes, codes) and torch.equal(other.scales, scales)
        if rows:
            assert other._pointers()[0] != t._pointers()[0]
        codes2, scales2 = other._pointers()
        assert codes2 == other.codes.data_ptr() and (not rows or scales2 == other.scales.data_ptr())


def test_tensor_refuses():
    from nano_vllm_metal_amd import MxTensor

    u = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    for codes, scales, fmt, msg in [
            (u(2, 16), u(2, 1), "mxfp6", "format"), (u(2, 16).int(), u(2, 1), "mxfp4", "uint8"),
            (u(2, 16), u(2, 1).float(), "mxfp4", "uint8"), (u(2, 16), u(1), "mxfp4", "dimensions"),
            (u(2, 16), u(2, 2), "mxfp4", "blocks"), (u(2, 24), u(2, 1), "mxfp8", "blocks"),
            (u(2, 16), u(3, 1), "mxfp4", "blocks"), (u(2, 0), u(2, 0), "mxfp4", "blocks")]:
        with pytest.raises(ValueError, match=msg):
            MxTensor(codes, scales, fmt)


def test_operators_refuse_cpu_tensors_and_bad_arguments():
    from nano_vllm_metal_amd import (mx_dequantize, mx_embedding, mx_linear, mx_quantize,
                                     mx_swiglu, residual_rms_norm_mx)

    x, w, a = torch.zeros(3, 64, dtype=torch.bfloat16), _mx(32, 64), _mx(3, 64, "mxfp8")
    for f in (lambda: mx_quantize(x), lambda: mx_dequantize(a), lambda: mx_linear(a, w),
              lambda: mx_linear(x, w), lambda: mx_swiglu(a, w, w),
              lambda: residual_rms_norm_mx(x, None, x[0], 1e-6),
              lambda: mx_embedding(torch.zeros(2, dtype=torch.long), w, torch.bfloat16)):
        with pytest.raises(ValueError, match="GPU only"):
            f()
    for f, msg in [(lambda: mx_quantize(x, "int4"), "format"),
                   (lambda: mx_linear(x.float(), w), "x must be"),
                   (lambda: mx_linear(a, _mx(32, 64, "mxfp8")), "mxfp4 MxTensor"),
                   (lambda: mx_linear(a, x), "mxfp4 MxTensor"),
                   (lambda: mx_linear(a, _mx(32, 96)), "96 input features"),
                   (lambda: mx_linear(a, w, torch.float64), "dtype"),
                   (lambda: mx_swiglu(a, w, _mx(64, 64)), "same output features"),
                   (lambda: mx_swiglu(a, _mx(48, 64), _mx(48, 64)), "multiple of 32"),
                   (lambda: mx_swiglu(a, w, w, "mxfp6"), "format"),
                   (lambda: mx_embedding(torch.zeros(2), x, x.dtype), "two-dimensional")]:
        with pytest.raises(ValueError, match=msg):
            f()


def test_stacked_projections_and_mixed_weights():
    from nano_vllm_metal_amd import QuantizedWeights
    from nano_vllm_metal_amd.qwen3 import DenseMLP, stack_outputs

    a, b = _mx(3, 544), _mx(5, 544)
    t = stack_outputs(a, b)
    assert t.shape == (8, 544) and t.pitch == 32
    assert torch.equal(t.codes[3:], b.codes) and torch.equal(t.scales[:3], a.scales)
    with pytest.raises(ValueError, match="input features"):
        stack_outputs(a, _mx(3, 64))
    q = QuantizedWeights(torch.zeros(3, 1), torch.zeros(3, 1), 64, 4,
                         torch.zeros(3, 8, dtype=torch.int32))
    with pytest.raises(ValueError, match="all be MxTensors"):
        stack_outputs(a, q)
    with pytest.raises(ValueError, match="all be MxTensors"):
        DenseMLP(a, a, q)


# -------------------------------------------------------------------- the loader


def _checkpoint(tmp_path, H=64, I=96, V=40, tie=False, **quantization):
    """A one-layer dense model in mxfp4 mode, and the tensors it was made of."""
    from safetensors.torch import save_file

    g = np.random.default_rng(1)
    t = {}

    def mx(name, out, inn):
        t[f"{name}.weight"] = torch.from_numpy(
            g.integers(0, 1 << 32, (out, inn // 8), dtype=np.uint32))
        t[f"{name}.scales"] = torch.from_numpy(g.integers(110, 125, (out, inn // 32),
                                                          dtype=np.uint8))

    for p, o, i in (("q", 64, H), ("k", 32, H), ("v", 32, H), ("o", H, 64)):
        mx(f"model.layers.0.self_attn.{p}_proj", o, i)
    for p, o, i in (("gate", I, H), ("up", I, H), ("down", H, I)):
        mx(f"model.layers.0.mlp.{p}_proj", o, i)
    mx("model.embed_tokens", V, H)
    if not tie:
        mx("lm_head", V, H)
    for n, s in (("self_attn.q_norm", 32), ("self_attn.k_norm", 32), ("input_layernorm", H),
                 ("post_attention_layernorm", H)):
        t[f"model.layers.0.{n}.weight"] = torch.ones(s, dtype=torch.bfloat16)
    t["model.norm.weight"] = torch.ones(H, dtype=torch.bfloat16)
    cfg = dict(hidden_size=H, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1,
               head_dim=32, vocab_size=V, intermediate_size=I, tie_word_embeddings=tie,
               max_position_embeddings=64,
               quantization=dict(group_size=32, bits=4, mode="mxfp4", **quantization))

    def write():
        (tmp_path / "config.json").write_text(json.dumps(cfg))
        save_file(t, str(tmp_path / "model.safetensors"))

    return t, cfg, write


@pytest.mark.parametrize("tie", [False, True])
def test_mxfp4_checkpoint(tmp_path, tie):
    from nano_vllm_metal_amd import MxTensor, Qwen3Model

    t, cfg, write = _checkpoint(tmp_path, tie=tie)
    write()
    m = Qwen3Model.from_checkpoint(tmp_path, device="cpu")
    mlp, layer = m.layers[0].mlp, m.layers[0]
    assert mlp.mx and (m.lm_head is None) == tie and m.device.type == "cpu"
    for w, name in ((m.embed_w, "model.embed_tokens"), (mlp.w_down, "model.layers.0.mlp.down_proj"),
                    (layer.wo, "model.layers.0.self_attn.o_proj")):
        words, scales = t[f"{name}.weight"].numpy(), t[f"{name}.scales"]
        assert type(w) is MxTensor and w.fmt == "mxfp4" and torch.equal(w.scales, scales)
        # value i of a row is code i % 8 of word i / 8, from the low bits up
        codes = (words[:, :, None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
        assert np.array_equal(O.unpack(w.codes, "mxfp4").numpy(), codes.reshape(len(words), -1))
    assert layer.wqkv.shape == (128, 64)
    assert torch.equal(layer.wqkv.scales[96:], t["model.layers.0.self_attn.v_proj.scales"])


def test_modules_in_either_mode(tmp_path):
    """An entry of its own makes a module affine among mxfp4 ones."""
    from nano_vllm_metal_amd import MxTensor, QuantizedWeights, Qwen3Model

    t, cfg, write = _checkpoint(tmp_path)
    cfg["quantization"]["lm_head"] = {"group_size": 64, "bits": 4}
    for f in ("scales", "biases"):
        t[f"lm_head.{f}"] = torch.zeros(40, 1, dtype=torch.bfloat16)
    write()
    m = Qwen3Model.from_checkpoint(tmp_path, device="cpu")
    assert type(m.lm_head) is QuantizedWeights and type(m.embed_w) is MxTensor


@pytest.mark.parametrize("change,msg", [
    (lambda t, q: q.update(mode="nvfp4"), "neither"),
    (lambda t, q: q.update(group_size=64), "groups of 32"),
    (lambda t, q: q.update(bits=8), "4 bits"),
    (lambda t, q: t.update({"lm_head.biases": torch.zeros(40, 2)}), "no biases"),
    (lambda t, q: t.update({"lm_head.scales": torch.zeros(40, 2)}), "uint8"),
    (lambda t, q: t.update({"lm_head.scales": t["lm_head.scales"][:, :1].contiguous()}), "shapes"),
    (lambda t, q: t.update({"lm_head.weight": t["lm_head.weight"].float()}), "uint32"),
    (lambda t, q: t.pop("model.layers.0.mlp.up_proj.scales"), "not in the checkpoint"),
    (lambda t, q: q.update({"model.layers.0.mlp.up_proj": False}), "unquantised"),
])
def test_bad_mxfp4_checkpoints(tmp_path, change, msg):
    from nano_vllm_metal_amd import Qwen3Model

    t, cfg, write = _checkpoint(tmp_path)
    change(t, cfg["quantization"])
    write()
    with pytest.raises((ValueError, KeyError), match=msg):
        Qwen3Model.from_checkpoint(tmp_path, device="cpu")


def test_sparse_blocks_in_mxfp4_are_refused(tmp_path):
    from nano_vllm_metal_amd import Qwen3Model

    t, cfg, write = _checkpoint(tmp_path)
    cfg.update(num_experts=4, num_experts_per_tok=2, moe_intermediate_size=32)
    write()
    with pytest.raises(ValueError, match="sparse blocks take affine"):
        Qwen3Model.from_checkpoint(tmp_path, device="cpu")


def test_random_model_modes():
    from nano_vllm_metal_amd import MxTensor, Qwen3Config, Qwen3Model

    c = Qwen3Config(hidden_size=64, num_hidden_layers=2, num_attention_heads=2,
                    num_key_value_heads=1, head_dim=32, vocab_size=64, intermediate_size=4096,
                    max_position_embeddings=16)
    m = Qwen3Model.random(c, device="cpu", mode="mxfp4", std=0.02)
    w = m.layers[1].mlp.w_down
    assert type(w) is MxTensor and type(m.lm_head) is MxTensor
    # scales of 2^-8 and 2^-7, codes of 2.93 root mean square
    assert set(w.scales.unique().tolist()) == {119, 120}
    assert 0.015 < O.decode(w.codes, w.scales, "mxfp4").square().mean().sqrt().item() < 0.022
    with pytest.raises(ValueError, match="mode"):
        Qwen3Model.random(c, device="cpu", mode="int8")


# -------------------------------------------------------------------- the oracle


@pytest.mark.parametrize("fmt", FMTS)
def test_oracle_rounds_to_the_nearest_element(fmt):
    grid = O.elements(fmt)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 64, generator=g, dtype=torch.float64) * 3
    x[0, :32], x[1, 5] = 0.0, float("nan")
    x[2, :32] = torch.cat((grid[-1:] / 8, (grid[:-1] + grid[1:])[:31].mul(0.5).repeat(31)[:31] / 8))
    c, b = O.quantize(x, fmt)
    back = O.decode(O.pack(c, fmt), b.to(torch.uint8), fmt)
    assert (back[0, :32] == 0).all() and b[0, 0] == 0
    assert torch.isnan(back[1, :32]).all() and b[1, 0] == 255
    ok = torch.ones_like(x, dtype=torch.bool)
    ok[1, :32] = False
    scale = O.pow2(b - 127).repeat_interleave(32, -1)
    near = (x.abs()[..., None] / scale[..., None] - grid).abs()
    best = near.amin(-1)
    assert torch.equal(((back.abs() - x.abs()).abs() / scale)[ok], best[ok])
    # two as near: the even code
    tie = ok & ((near == best[..., None]).sum(-1) == 2)
    assert tie.any() and ((c[tie] & 1) == 0).all()
    O.check_quantized(O.pack(c, fmt)[3:], b[3:].to(torch.uint8), fmt, x[3:], torch.zeros_like(x[3:]))


@pytest.mark.parametrize("fmt", FMTS)
def test_oracle_check_sees_a_wrong_code_and_a_wrong_scale(fmt):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 64, generator=g, dtype=torch.float64)
    c, b = O.quantize(x, fmt)
    c[2, 7] ^= 1
    with pytest.raises(AssertionError, match="elements"):
        O.check_quantized(O.pack(c, fmt), b.to(torch.uint8), fmt, x, torch.zeros_like(x))
    c[2, 7] ^= 1
    b[1, 1] += 1
    with pytest.raises(AssertionError, match="scales"):
        O.check_quantized(O.pack(c, fmt), b.to(torch.uint8), fmt, x, torch.zeros_like(x))
