"""The microscaled (MX) operators, as performance cases.

A block of 32 consecutive values of a row shares one power-of-two scale (E8M0,
byte b stands for 2^(b - 127)); the values are E2M1 (``mxfp4``, two a byte,
the even one in the low half) or E4M3 (``mxfp8``).  Kinds:

* ``quant``      activations to MXFP8 (``mx_quantize``)
* ``roundtrip``  values to MXFP4 and back to what the codes stand for
  (``mx_quantize``, ``mx_dequantize``)
* ``norm``       residual add and RMSNorm with an MXFP8 output
  (``residual_rms_norm_mx``)
* ``linear``     MX activations times MXFP4 weights (``mx_linear``)
* ``swiglu``     gate and up products, SwiGLU, MXFP8 output (``mx_swiglu``)

Sizes are the repository's own: the attention projections and the dense MLP of
the Qwen3-30B-A3B configuration (hidden 2048, 32 query and 4 kv heads of 128,
intermediate 6144), prompts of up to 4096 tokens and decode batches, and
generic odd ones.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 32
EPS = 1e-6
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EMAX = {"mxfp4": 2, "mxfp8": 8}
# in, out: stacked q/k/v, attention output, dense gate or up, dense down
PROJECTIONS = [(2048, 5120), (4096, 2048), (2048, 6144), (6144, 2048)]
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_FLOPS = 2.1e11


def listed():
    return [
        # the attention output of one decoding request on its way to the output projection
        {"name": "quant8_1", "kind": "quant", "M": 1, "n": 4096, "dtype": "bf16"},
        # the same of a prompt of 4096 tokens
        {"name": "quant8_4096", "kind": "quant", "M": 4096, "n": 4096, "dtype": "bf16"},
        # a loader turning the dense down projection into MXFP4 and looking at what is left of it
        {"name": "weights4_down", "kind": "roundtrip", "M": 2048, "n": 6144, "dtype": "f32"},
        # an odd batch of fp16 values with a ragged row length
        {"name": "round4_777_f16", "kind": "roundtrip", "M": 777, "n": 1376, "dtype": "f16"},
        # the norm in front of a projection, a small decode batch
        {"name": "norm8_decode_8", "kind": "norm", "M": 8, "n": 2048, "dtype": "bf16"},
        # the same for a prompt, fp16
        {"name": "norm8_4096_f16", "kind": "norm", "M": 4096, "n": 2048, "dtype": "f16"},
        # the attention input projection of one decoding request: latency and the weight stream
        {"name": "linear_1", "kind": "linear", "M": 1, "n": 2048, "o": 5120, "fmt": "mxfp8", "dtype": "bf16"},
        # the attention output projection of an odd decode batch
        {"name": "linear_37_f16", "kind": "linear", "M": 37, "n": 4096, "o": 2048, "fmt": "mxfp8", "dtype": "f16"},
        # the attention input projection of a prompt
        {"name": "linear_4096", "kind": "linear", "M": 4096, "n": 2048, "o": 5120, "fmt": "mxfp8", "dtype": "bf16"},
        # the dense down projection of a ragged prompt with 4-bit activations
        {"name": "linear44_1500", "kind": "linear", "M": 1500, "n": 6144, "o": 2048, "fmt": "mxfp4", "dtype": "bf16"},
        # the dense MLP's first half, a decode batch
        {"name": "swiglu_8", "kind": "swiglu", "M": 8, "n": 2048, "o": 6144, "fmt": "mxfp8"},
        # the same for a prompt: the largest case
        {"name": "swiglu_4096", "kind": "swiglu", "M": 4096, "n": 2048, "o": 6144, "fmt": "mxfp8"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    return rng.choice([2048, 4096, 6144, BLOCK * rng.randint(1, 200), BLOCK * _log(rng, 1, 200)])


def draw(rng):
    kind = rng.choice(["quant", "roundtrip", "norm", "linear", "linear", "linear", "swiglu", "swiglu"])
    if kind in ("quant", "roundtrip"):
        return {"kind": kind, "M": _log(rng, 1, 4096), "n": _width(rng), "dtype": rng.choice(["bf16", "f16", "f32"])}
    if kind == "norm":
        return {"kind": kind, "M": _log(rng, 1, 4096), "n": _width(rng), "dtype": rng.choice(["bf16", "f16"])}
    n, o = rng.choice(PROJECTIONS)
    if rng.random() < 0.4:
        n = _width(rng)
        o = rng.randint(65, 6200) if kind == "linear" else BLOCK * rng.randint(3, 194)
    M, fmt = _log(rng, 1, 4096), rng.choice(["mxfp8", "mxfp8", "mxfp4"])
    if kind == "linear":
        M = min(M, int(MOST_FLOPS / (2 * n * o)))
        return {"kind": kind, "M": M, "n": n, "o": o, "fmt": fmt, "dtype": rng.choice(["bf16", "bf16", "f16"])}
    M = min(M, int(MOST_FLOPS / (4 * n * o)))
    return {"kind": kind, "M": M, "n": n, "o": o, "fmt": fmt}


# ------------------------------------------------------------------ plain form


def _floor_log2(x):
    """floor(log2(x)) of positive values, from their exponent (0 for zero)."""
    return torch.frexp(x)[1] - 1


def _pow2(e, dtype=torch.float32):
    return torch.ldexp(torch.ones((), dtype=dtype, device=e.device), e)


def _round_elements(v, fmt):
    """Values divided by their block's scale, to the nearest element value (ties to even, saturating)."""
    a = v.abs()
    if fmt == "mxfp4":
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        return (torch.round(a / step) * step).clamp(max=6.0) * torch.sign(v)
    step = _pow2(_floor_log2(a.clamp(min=2.0 ** -6)) - 3, v.dtype)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _quantize(x, fmt):
    """Element values [M, n] and exponents [M, n / 32] of x [M, n]."""
    g = x.reshape(x.shape[0], -1, BLOCK)
    amax = g.abs().amax(-1)
    e = torch.where(amax > 0, _floor_log2(amax) - EMAX[fmt], torch.full_like(amax, -127, dtype=torch.int32))
    e = e.clamp(-127, 127)
    # (two factors: 2^-e alone can leave the range of 32 bits)
    half = torch.div(-e, 2, rounding_mode="floor")
    v = g * _pow2(half, x.dtype)[..., None] * _pow2(-e - half, x.dtype)[..., None]
    return _round_elements(v, fmt).reshape(x.shape), e


def _values(q, e, dtype=torch.float32):
    return (q.to(dtype).reshape(q.shape[0], -1, BLOCK) * _pow2(e, dtype)[..., None]).reshape(q.shape)


def _decode(t, dtype=torch.float32):
    """What packed codes and scale bytes stand for."""
    codes, scales, fmt = t
    if fmt == "mxfp8":
        q = codes.view(torch.float8_e4m3fn).to(dtype)
    else:
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=codes.device)
        q = table[torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1).long()]
    return _values(q, scales.to(torch.int32) - 127, dtype)


def _pair(q, e):
    """MXFP8 element values and scales in the types that hold them."""
    return q.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain(s):
    kind = s["kind"]
    if kind == "quant":
        return _pair(*_quantize(s["x"].float(), "mxfp8"))
    if kind == "roundtrip":
        return _values(*_quantize(s["x"].float(), "mxfp4")).to(torch.bfloat16)
    if kind == "norm":
        h = (s["h"].float() + s["r"].float()).to(s["h"].dtype)
        # (64 bits: else a value next to a rounding border of 8 bits would go by the mean's last bit)
        v = h.double()
        x = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * s["w"].double()
        return (h, *_pair(*_quantize(x, "mxfp8")))
    a = _decode(s["a"])
    if kind == "linear":
        return (a @ _decode(s["w"]).T).to(s["dtype"])
    g, u = a @ _decode(s["g"]).T, a @ _decode(s["u"]).T
    return _pair(*_quantize(g / (1 + torch.exp(-g)) * u, "mxfp8"))


# ------------------------------------------------------------ the framework's


def _package():
    if "nano_vllm_metal_amd" in sys.modules:
        return sys.modules["nano_vllm_metal_amd"]
    at = str(Path(__file__).resolve().parent.parent / "nano-vllm-metal_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import nano_vllm_metal_amd

    return nano_vllm_metal_amd


def _mx(P, s, name):
    """The handle that a program keeps of an operand (weights from loading on, activations from the
    operator that made them); it refers to the state's own tensors."""
    t = s.get("mx " + name)
    if t is None:
        t = s["mx " + name] = P.MxTensor(*s[name])
    return t


def _held(t):
    return t.codes.view(torch.float8_e4m3fn), t.scales.view(torch.float8_e8m0fnu)


def _own(s):
    P, kind = _package(), s["kind"]
    if kind == "quant":
        return _held(P.mx_quantize(s["x"], "mxfp8"))
    if kind == "roundtrip":
        return P.mx_dequantize(P.mx_quantize(s["x"], "mxfp4"), torch.bfloat16)
    if kind == "norm":
        h, x = P.residual_rms_norm_mx(s["h"], s["r"], s["w"], EPS, "mxfp8")
        return (h, *_held(x))
    if kind == "linear":
        return P.mx_linear(_mx(P, s, "a"), _mx(P, s, "w"), s["dtype"])
    return _held(P.mx_swiglu(_mx(P, s, "a"), _mx(P, s, "g"), _mx(P, s, "u"), "mxfp8"))


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, device=DEVICE, generator=g)


def _activations(g, M, n):
    """Values as a layer hands them on: columns of different sizes, a few of them much larger."""
    gain = torch.exp(0.5 * _randn(g, n))
    gain = torch.where(torch.rand(n, device=DEVICE, generator=g) < 0.005, 20.0 * gain, gain)
    return _randn(g, M, n) * gain


def _pack(x, fmt):
    """(codes, scales, fmt) of values: rows of scales start 16 bytes apart or a multiple."""
    q, e = _quantize(x, fmt)
    if fmt == "mxfp8":
        codes = q.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        grid = torch.tensor(E2M1, device=x.device)
        c = torch.bucketize(q.abs(), grid).to(torch.uint8) + 8 * (q < 0).to(torch.uint8)
        codes = c[:, 0::2] | (c[:, 1::2] << 4)
    pitch = -(-e.shape[1] // 16) * 16
    scales = torch.zeros((e.shape[0], pitch), dtype=torch.uint8, device=x.device)
    scales[:, : e.shape[1]] = (e + 127).to(torch.uint8)
    return codes, scales[:, : e.shape[1]], fmt


def prepare(case, seed):
    g, kind, M, n = _gen(seed), case["kind"], case["M"], case["n"]
    state = {"kind": kind}
    if kind in ("quant", "roundtrip"):
        state["x"] = _activations(g, M, n).to(DTYPES[case["dtype"]])
    elif kind == "norm":
        dt = DTYPES[case["dtype"]]
        state |= {"h": (3 * _activations(g, M, n)).to(dt), "r": _randn(g, M, n).to(dt),
                  "w": (1 + 0.1 * _randn(g, n)).to(dt)}
    else:
        state["a"] = _pack(_activations(g, M, n), case["fmt"])
        # (weights of a size that keeps the products near one, as a trained layer's are)
        for name in ("w",) if kind == "linear" else ("g", "u"):
            state[name] = _pack(_randn(g, case["o"], n) * n ** -0.5, "mxfp4")
        if kind == "linear":
            state["dtype"] = DTYPES[case["dtype"]]
    return state


# -------------------------------------------------------- what a pass needs


def work(case):
    kind, M, n = case["kind"], case["M"], case["n"]
    held = {"mxfp8": 1 + 1 / BLOCK, "mxfp4": 0.5 + 1 / BLOCK}
    size = 4 if case.get("dtype") == "f32" else 2
    if kind == "quant":
        by, fl = M * n * (size + held["mxfp8"]), 2.0 * M * n
    elif kind == "roundtrip":
        by, fl = M * n * (size + 2), 3.0 * M * n
    elif kind == "norm":
        by, fl = M * n * (6 + held["mxfp8"]) + 2 * n, 7.0 * M * n
    elif kind == "linear":
        o = case["o"]
        by, fl = M * n * held[case["fmt"]] + o * n * held["mxfp4"] + 2 * M * o, 2.0 * M * n * o
    else:
        o = case["o"]
        by = M * n * held[case["fmt"]] + 2 * o * n * held["mxfp4"] + M * o * held["mxfp8"]
        fl = 4.0 * M * n * o
    return {"bytes": float(by), "flops": float(fl)}


# ------------------------------------------------------------ 64-bit results


def _grid(fmt):
    """Every non-negative element value in order; the place of a value is its code."""
    if fmt == "mxfp4":
        return torch.tensor(E2M1, dtype=torch.float64, device=DEVICE)
    i = torch.arange(127, device=DEVICE)
    m, x = (i & 7).double(), (i >> 3).double()
    return torch.where(i < 8, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(x - 7))


def _exact_quantize(x, fmt):
    """Element values and scales of x (64 bits), by the nearest place of the grid."""
    g = x.reshape(x.shape[0], -1, BLOCK)
    amax = g.abs().amax(-1).contiguous()
    e = ((amax.view(torch.int64) >> 52) - 1023 - EMAX[fmt]).clamp(-127, 127)
    scale = torch.exp2(e.double())
    a, grid = (g.abs() / scale[..., None]).contiguous(), _grid(fmt)
    middle = (grid[1:] + grid[:-1]) / 2
    low, high = torch.bucketize(a, middle), torch.bucketize(a, middle, right=True)
    place = torch.where(low % 2 == 0, low, high)
    return (torch.copysign(grid[place], g)).reshape(x.shape), scale


def _exact_values(t):
    codes, scales, fmt = t
    if fmt == "mxfp4":
        c = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.int64, device=codes.device)
        c[:, 0::2], c[:, 1::2] = codes & 15, codes >> 4
        sign, c = c >> 3, c & 7
    else:
        sign, c = (codes >> 7).long(), (codes & 127).long()
    v = torch.where(sign == 1, -_grid(fmt)[c], _grid(fmt)[c])
    return v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "quant":
        return _exact_quantize(s["x"].double(), "mxfp8")
    if kind == "roundtrip":
        q, scale = _exact_quantize(s["x"].double(), "mxfp4")
        return q * scale.repeat_interleave(BLOCK, dim=1)
    if kind == "norm":
        total = s["h"].double() + s["r"].double()
        h = total.to(s["h"].dtype).double()
        x = h * (h.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["w"].double()
        return (total, *_exact_quantize(x, "mxfp8"))
    a = _exact_values(s["a"])
    if kind == "linear":
        return a @ _exact_values(s["w"]).T
    g, u = a @ _exact_values(s["g"]).T, a @ _exact_values(s["u"]).T
    return _exact_quantize(g * torch.sigmoid(g) * u, "mxfp8")
