"""Workloads of the 8-bit floating point linear and of the norm in front of it.

* ``quant``: values to e4m3 with a scale for each block of 128, rows of
  activations (1 x 128) or weights (128 x 128);
* ``gemm``: the product of two such operands, with a bias;
* ``gn``: group norm with an activation, channels last, its result in 16 bits
  or as e4m3 blocks for the product behind it.

``own`` false computes them as elementary torch operations in 32 bits,
``own`` true as calls of the package's entry points.
"""

import importlib
import math
import os
import sys
import types

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
_ACTIVATIONS = {"none": 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = "comfyui-int-crush_b200"
_E4M3_MAX = 448.0
_AMAX_MIN = 1e-8


def _runtime():
    """The package's runtime (its directory name is not an identifier)."""
    if _PACKAGE not in sys.modules:
        pkg = types.ModuleType(_PACKAGE)
        pkg.__path__ = [os.path.join(_ROOT, _PACKAGE)]
        sys.modules[_PACKAGE] = pkg
    return importlib.import_module(_PACKAGE + "._b200_runtime")


def _up(n, m):
    return -(-n // m)


# ── cases ────────────────────────────────────────────────────────────────────

def _quant(name, M, K, rows, dtype):
    return {"name": name, "op": "quant", "M": M, "K": K, "rows": rows, "dtype": dtype}


def _gemm(name, M, K, N, bias, dtype):
    return {"name": name, "op": "gemm", "M": M, "K": K, "N": N, "bias": bias, "dtype": dtype}


def _gn(name, B, L, C, groups, act, dtype, fp8):
    return {"name": name, "op": "gn", "B": B, "L": L, "C": C, "groups": groups, "act": act, "dtype": dtype, "fp8": fp8}


def listed():
    return [
        # the vector of a timestep or of one token before a projection: the
        # smallest call, where the launch is what it costs
        _quant("quant_token", 1, 5120, 1, "bf16"),
        # a ragged batch whose rows end inside a block
        _quant("quant_ragged", 3003, 2600, 1, "fp16"),
        # a video block's tokens before its projections
        _quant("quant_video", 65520, 5120, 1, "bf16"),
        # a weight at load time
        _quant("quant_weight", 13824, 5120, 128, "bf16"),
        # one row through a square projection: the weight's bytes count
        _gemm("gemm_token", 1, 5120, 5120, True, "bf16"),
        # odd sizes in every direction, a last block of 40
        _gemm("gemm_odd", 1001, 2600, 1111, True, "fp16"),
        # the text tokens of an image block, the wide half of its MLP
        _gemm("gemm_text", 512, 4096, 12288, True, "bf16"),
        # its image and text tokens together, back from the wide half
        _gemm("gemm_image", 4608, 12288, 4096, False, "fp16"),
        # a video block's FFN projection
        _gemm("gemm_video", 65520, 5120, 13824, True, "bf16"),
        # the innermost level of a convolutional network, 16 x 16 positions
        _gn("gn_inner", 2, 256, 1280, 32, "silu", "fp16", False),
        # an odd image in front of a 1x1 projection, groups of 11 channels
        _gn("gn_odd_fp8", 3, 61 * 45, 352, 32, "none", "fp16", True),
        # a decoder's last level, 1024 x 1024 positions
        _gn("gn_decoder", 1, 1024 * 1024, 128, 32, "silu", "bf16", False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))


def draw(rng):
    op = rng.choice(["quant", "gemm", "gemm", "gn"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "quant":
        K = _log(rng, 8, 1792) * 8 - rng.choice([0, 0, 0, 3])
        if rng.random() < 0.3:
            c = _quant("", _log(rng, 64, 14336), K, 128, rng.choice(["fp16", "bf16", "fp32"]))
        else:
            c = _quant("", _log(rng, 1, min(65520, 65520 * 5120 // K)), K, 1, dtype)
    elif op == "gemm":
        K, N = (_log(rng, 8, 1792) * 8 - rng.choice([0, 0, 0, 3]) for _ in range(2))
        M = rng.choice([1, 2, 8, 16, 40]) if rng.random() < 0.25 else _log(rng, 1, min(65520, 65520 * 5120 * 13824 // (K * N)))
        c = _gemm("", M, K, N, rng.random() < 0.5, rng.choice([dtype, dtype, "fp32"]))
    else:
        groups = rng.choice([1, 8, 16, 32, 32, 32])
        C = groups * _log(rng, 2, 2560 // groups if groups > 1 else 640)
        B = _log(rng, 1, 8)
        c = _gn("", B, _log(rng, 1, min(1 << 20, 1024 * 1024 * 128 // (B * C))), C, groups,
                rng.choice(["none", "silu", "silu", "gelu", "gelu_tanh"]), dtype, rng.random() < 0.4)
    del c["name"]
    return c


# ── inputs ───────────────────────────────────────────────────────────────────

def _blocks(x, rows):
    """``x`` [M, K] as [M / rows, rows, K / 128, 128], filled up with zeros."""
    M, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % 128, 0, -M % rows))
    return x.view(_up(M, rows), rows, _up(K, 128), 128)


def _plain_quantize(x, rows):
    """e4m3 values and scales of a matrix in 32 bits."""
    M, K = x.shape
    b = _blocks(x, rows)
    top = b.abs().amax((1, 3)).clamp(min=_AMAX_MIN)
    s = top / torch.full_like(top, _E4M3_MAX)   # (a plain number would be multiplied by its reciprocal)
    q = (b / s[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(q.shape[0] * rows, -1)[:M, :K], s


def _held(x, rows):
    """Values in 32 bits as a program holds an operand: e4m3 rows that start at
    multiples of 16 bytes, the scales of activations block by block."""
    M, K = x.shape
    q, s = _plain_quantize(x, rows)
    buf = torch.zeros(M, _up(K, 16) * 16, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn)[:, :K]
    buf.copy_(q)
    return buf, s.t().contiguous().t() if rows == 1 else s.contiguous()


def prepare(case, seed):
    c = case
    dev = "cuda"
    dt = _DTYPES[c["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(mean, std, generator=g)

    if c["op"] == "quant":
        # activations with a few wide channels, or weights
        x = normal(c["M"], c["K"], dtype=dt, std=1.0 if c["rows"] == 1 else c["K"] ** -0.5)
        if c["rows"] == 1:
            x[:, torch.randint(0, c["K"], (1 + c["K"] // 200,), device=dev, generator=g)] *= 12
        s = {"x": x, "rows": c["rows"]}
    elif c["op"] == "gemm":
        M, K, N = c["M"], c["K"], c["N"]
        s = {"out": dt}
        x = normal(M, K)
        x[:, torch.randint(0, K, (1 + K // 200,), device=dev, generator=g)] *= 12
        s["x"], s["s_a"] = _held(x, 1)
        del x
        s["w"], s["s_w"] = _held(normal(N, K, std=K ** -0.5), 128)
        s["bias"] = normal(N, std=0.1, dtype=dt) if c["bias"] else None
    else:
        B, L, C = c["B"], c["L"], c["C"]
        x = normal(B, L, C, dtype=dt)
        x *= torch.empty(C, device=dev).uniform_(0.3, 3.0, generator=g).to(dt)
        x += normal(B, 1, C, std=0.7, dtype=dt)
        s = {"x": x, "weight": normal(C, mean=1.0, std=0.3, dtype=dt), "shift": normal(C, std=0.3, dtype=dt),
             "groups": c["groups"], "act": c["act"], "fp8": c["fp8"]}
    s["op"] = c["op"]
    return s


# ── one pass ─────────────────────────────────────────────────────────────────

def _plain_activation(y, act):
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _plain_product(x, w, s_w, s_a, bias, dtype):
    N, K = w.shape
    x = x.float() * s_a.repeat_interleave(128, 1)[:, :K]
    w = w.float() * s_w.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = x @ w.t()
    return (y if bias is None else y + bias.float()).to(dtype)


def _plain_group_norm(x, weight, shift, groups, act):
    B, L, C = x.shape
    x = x.float().view(B, L, groups, C // groups)
    d = x - x.mean((1, 3), keepdim=True)
    d = d * torch.rsqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    return _plain_activation(d.view(B, L, C) * weight.float() + shift.float(), act)


def run(state):
    s = state
    if own:
        rt = _runtime()
        if s["op"] == "quant":
            return rt.quantize_fp8_block(s["x"], rows=s["rows"])
        if s["op"] == "gemm":
            return rt.gemm_fp8_block(s["x"], s["w"], s["s_w"], s["s_a"], bias=s["bias"], out_dtype=s["out"])
        call = rt.fused_groupnorm_quantize if s["fp8"] else rt.group_norm
        return call(s["x"], s["groups"], s["weight"], s["shift"], eps=1e-5, activation=_ACTIVATIONS[s["act"]])
    if s["op"] == "quant":
        return _plain_quantize(s["x"].float(), s["rows"])
    if s["op"] == "gemm":
        return _plain_product(s["x"], s["w"], s["s_w"], s["s_a"], s["bias"], s["out"])
    y = _plain_group_norm(s["x"], s["weight"], s["shift"], s["groups"], s["act"])
    if not s["fp8"]:
        return y.to(s["x"].dtype)
    q, scale = _plain_quantize(y.flatten(0, 1), 1)
    return q.view(y.shape), scale.view(*y.shape[:2], -1)


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    c = case
    if c["op"] == "quant":
        M, K = c["M"], c["K"]
        # |x|, the maximum, the division
        return {"bytes": M * K * (_BYTES[c["dtype"]] + 1) + 4 * _up(M, c["rows"]) * _up(K, 128), "flops": 3 * M * K}
    if c["op"] == "gemm":
        M, K, N = c["M"], c["K"], c["N"]
        out = _BYTES[c["dtype"]]
        scales = 4 * _up(K, 128) * (M + _up(N, 128))
        return {"bytes": M * K + N * K + scales + M * N * out + (N * out if c["bias"] else 0), "flops": 2 * M * N * K}
    n, C = c["B"] * c["L"] * c["C"], c["C"]
    out = n + 4 * c["B"] * c["L"] * _up(C, 128) if c["fp8"] else 2 * n
    # two sums, the norm, the activation
    return {"bytes": 2 * n + out + 4 * C, "flops": n * (6 + (4 if c["act"] != "none" else 0) + (3 if c["fp8"] else 0))}


# ── the definitions in 64 bits ───────────────────────────────────────────────

def _exact_quantize(x, rows, stored):
    """Scales in 64 bits, and the e4m3 values nearest to x over the scale as it
    is stored (in 32 bits)."""
    M, K = x.shape
    out = torch.empty(M, K, dtype=torch.float64, device=x.device)
    scales = torch.empty(_up(M, rows), _up(K, 128), dtype=torch.float64, device=x.device)
    for at in range(0, scales.shape[1]):
        cols = x[:, at * 128:(at + 1) * 128].to(torch.float64)
        top = cols.abs().amax(1)
        if rows > 1:
            top = torch.nn.functional.pad(top, (0, -M % rows)).view(-1, rows).amax(1)
        scale = torch.maximum(top, torch.full_like(top, _AMAX_MIN)) / _E4M3_MAX
        scales[:, at] = scale
        held = scale.to(torch.float32).to(torch.float64) if stored else scale
        t = cols / held.repeat_interleave(rows)[:M, None]
        # 4 significant bits, the last one 2^-9 at least; ties to even
        step = torch.exp2(torch.frexp(t).exponent.clamp(min=-5).to(torch.float64) - 4)
        out[:, at * 128:(at + 1) * 128] = (torch.round(t / step) * step).clamp(-_E4M3_MAX, _E4M3_MAX)
    return out, scales


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "quant":
        return _exact_quantize(s["x"], case["rows"], True)
    if case["op"] == "gemm":
        M, K, N = case["M"], case["K"], case["N"]
        out = torch.zeros(M, N, dtype=f, device="cuda")
        if s["bias"] is not None:
            out += s["bias"].to(f)
        of_row = torch.arange(N, device="cuda") // 128
        for b in range(_up(K, 128)):
            part = s["x"][:, b * 128:(b + 1) * 128].to(f) * s["s_a"][:, b, None].to(f)
            out.addmm_(part, (s["w"][:, b * 128:(b + 1) * 128].to(f) * s["s_w"][of_row, b, None].to(f)).T)
        return out
    B, L, C = s["x"].shape
    y = torch.empty(B, L, C, dtype=f, device="cuda")
    n = C // case["groups"]
    for b in range(B):
        for i in range(0, C, n):
            x = s["x"][b, :, i:i + n].to(f)
            var, mean = torch.var_mean(x, correction=0)
            y[b, :, i:i + n] = (x - mean) / torch.sqrt(var + 1e-5) * s["weight"][i:i + n].to(f) + s["shift"][i:i + n].to(f)
    if case["act"] == "silu":
        y *= torch.sigmoid(y)
    elif case["act"] == "gelu":
        y *= torch.special.ndtr(y)
    elif case["act"] == "gelu_tanh":
        y *= torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    if not case["fp8"]:
        return y
    q, scale = _exact_quantize(y.flatten(0, 1), 1, False)
    return q.view(B, L, C), scale.view(B, L, -1)
