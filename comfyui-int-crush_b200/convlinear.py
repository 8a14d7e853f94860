"""Standalone quantised linear modules with the reference's ``convlinear.py``
interface (``ConvLinear4bit`` / ``ConvLinear8bit``: constructor arguments,
``weight`` / ``scale`` / ``bias`` buffers, ``from_float``, ``forward``;
``convlinear.py:22-42,73-109,154-199``).

Behaviour: ``from_float`` takes an ``nn.Linear``, rotates its weight rows
block-wise with the Hadamard transform (when ``rot_need``), optionally
permutes the input columns (PermuQuant, INT4 only), and quantises per output
row (INT4 packed two per byte, or INT8).  ``forward`` applies the same
rotation / permutation to the activations and multiplies with the
dequantised weight.

Here the INT4 module runs the B200 kernels end to end (one prep launch for
rotation + permutation, then the W4A16 GEMM with the bias fused; fp16 or
bf16 CUDA activations).  The INT8 module is a W8A16 layer: its activation
prep runs on the B200 prep kernel on CUDA, and the dequantised linear is
torch's, which is the reference's own arithmetic for this module.

``ConvLinearFP8`` is the third format: e4m3 weights with a scale for each
128 x 128 block; ``forward`` quantises the activations (1 x 128 blocks) and
multiplies on the B200 kernels, bias fused.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _quant_utils as _qu

__all__ = ["ConvLinear4bit", "ConvLinear8bit", "ConvLinearFP8"]

_INTEGERS = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}   # by size


def _rotated_weight(linear: nn.Linear, rot_need: bool, rot_size: int, perm: torch.Tensor | None) -> torch.Tensor:
    """The float32 weight in the rotated (and permuted) input basis the
    module's activations are prepared into."""
    if rot_need and not _qu.is_power_of_two(rot_size):
        raise ValueError(f"rot_size must be a power of 2, got {rot_size}")
    w = linear.weight.detach().float()
    if rot_need:
        w = _qu.rotate_activations(w, rot_size)
    return w if perm is None else w[:, perm]


class _QuantLinearBase(nn.Module):
    """Buffers and activation prep shared by the two module types."""

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor, rot_need: bool, bias: torch.Tensor | None,
                 rot_size: int, in_features: int, perm: torch.Tensor | None = None) -> None:
        super().__init__()
        self.in_features = in_features
        self.out_features = weight.shape[-2]
        self.rot_need = rot_need
        self.rot_size = rot_size
        self._perm = perm
        self.register_buffer("weight", weight)
        self.register_buffer("scale", scale)
        if bias is None:
            self.bias = None
        else:
            self.register_buffer("bias", bias)

    def _prepared(self, x2: torch.Tensor) -> torch.Tensor:
        """Rotation (and permutation): one prep launch on CUDA fp16 / bf16
        activations, the torch restatement elsewhere (CPU modules)."""
        rot = self.rot_size if self.rot_need else 0
        if not rot and self._perm is None:
            return x2
        if x2.is_cuda and x2.dtype in (torch.float16, torch.bfloat16):
            from . import _b200_runtime as rt
            perm = None if self._perm is None else self._perm.to(x2.device)
            _, _, xp, _ = rt.prep_quantize(x2, rot_size=rot, w_in=self.in_features, perm=perm, quantize=False,
                                           want_prep=True)
            return xp
        xp = _qu.rotate_activations(x2, rot) if rot else x2
        if xp.shape[-1] < self.in_features:
            xp = F.pad(xp, (0, self.in_features - xp.shape[-1]))
        return xp if self._perm is None else xp[..., self._perm.to(xp.device)]

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"rot_size={self.rot_size}, rot_need={self.rot_need}")


class ConvLinear8bit(_QuantLinearBase):
    """W8A16 linear: optional rotation, int8 weights with per-row scales."""

    def __init__(self, weight, scale, rot_need=True, bias=None, rot_size=256):
        super().__init__(weight, scale, rot_need, bias, rot_size, in_features=weight.shape[-1])

    def forward(self, x):
        xp = self._prepared(x.reshape(-1, x.shape[-1]))
        w = self.weight.to(xp.dtype) * self.scale.to(xp.dtype)
        y = F.linear(xp, w, None if self.bias is None else self.bias.to(xp.dtype))
        return y.reshape(*x.shape[:-1], -1)

    @staticmethod
    def from_float(module: nn.Linear, rot_need: bool = True, rot_size: int = 256) -> "ConvLinear8bit":
        w = _rotated_weight(module, rot_need, rot_size, None)
        s = _qu.calculate_scales_int8(w, w.shape[1])
        q = _qu.quantize_weights_int8(w, s, w.shape[1])
        b = None if module.bias is None else module.bias.detach().clone()
        return ConvLinear8bit(weight=q, scale=s, rot_need=rot_need, bias=b, rot_size=rot_size)


class ConvLinear4bit(_QuantLinearBase):
    """W4A16 linear: optional rotation and permutation, packed INT4 weights
    with per-row scales; B200 kernels only (CUDA fp16 / bf16 activations)."""

    def __init__(self, weight, scale, rot_need=True, bias=None, rot_size=256, perm=None, in_features=None):
        super().__init__(weight, scale, rot_need, bias, rot_size,
                         in_features=in_features if in_features is not None else weight.shape[-1] * 2, perm=perm)

    def forward(self, x):
        if not (x.is_cuda and x.dtype in (torch.float16, torch.bfloat16)):
            raise RuntimeError("ConvLinear4bit runs on the B200 kernels: float16 / bfloat16 CUDA activations "
                               f"required (got {x.dtype} on {x.device})")
        from . import _b200_runtime as rt
        xp = self._prepared(x.reshape(-1, x.shape[-1]))
        b = None if self.bias is None else self.bias.to(x.dtype)
        y = rt.gemm_w4a16(xp, self.weight, self.scale.reshape(-1, 1), bias=b, K=self.in_features)
        return y.reshape(*x.shape[:-1], -1)

    @staticmethod
    def from_float(module: nn.Linear, rot_need: bool = True, rot_size: int = 256,
                   perm: torch.Tensor | None = None) -> "ConvLinear4bit":
        w = _rotated_weight(module, rot_need, rot_size, perm)
        s = _qu.calculate_scales(w, w.shape[1])
        packed = _qu.pack_int4(_qu.quantize_weights(w, s, w.shape[1])).to(torch.uint8)
        b = None if module.bias is None else module.bias.detach().clone()
        return ConvLinear4bit(weight=packed, scale=s, rot_need=rot_need, bias=b, rot_size=rot_size, perm=perm,
                              in_features=w.shape[1])


class ConvLinearFP8(_QuantLinearBase):
    """W8A8 linear in e4m3: weights with a scale for each 128 x 128 block,
    activations quantised 1 x 128 in ``forward``; optional rotation.  B200
    kernels only (CUDA fp16 / bf16 activations).  ``weight`` [N, K] is kept with
    its rows filled up to a multiple of 16 bytes, as the kernel reads them; a
    state dict holds [N, K], and one with filled rows loads too."""

    def __init__(self, weight, scale, rot_need=False, bias=None, rot_size=256, in_features=None):
        K = weight.shape[-1] if in_features is None else in_features
        if weight.shape[-1] % 16:
            weight = self._filled(weight, K, -(-K // 16) * 16)
        super().__init__(weight, scale, rot_need, bias, rot_size, in_features=K)

    @staticmethod
    def _filled(weight, K, width):
        """The K columns of ``weight`` in rows of ``width``, zeros behind them."""
        rows = torch.zeros(weight.shape[0], width, dtype=torch.uint8, device=weight.device)
        rows[:, :K] = weight[:, :K].contiguous().view(torch.uint8)
        return rows.view(weight.dtype)

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        if self.weight.shape[1] != self.in_features:
            destination[prefix + "weight"] = destination[prefix + "weight"][:, :self.in_features].contiguous()

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        w = state_dict.get(prefix + "weight")
        if w is not None and w.shape == (self.out_features, self.in_features) != self.weight.shape:
            state_dict = {**state_dict, prefix + "weight": self._filled(w.to(self.weight.dtype), self.in_features, self.weight.shape[1])}
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)

    def _apply(self, fn, recurse=True):
        # a cast of the model's floating point tensors is not one of e4m3 values
        # or of their scales: they go through it as integers
        kept = {name: self._buffers[name] for name in ("weight", "scale")}
        for name, t in kept.items():
            self._buffers[name] = t.view(_INTEGERS[t.element_size()])
        try:
            super()._apply(fn, recurse)
        finally:
            for name, t in kept.items():
                now = self._buffers[name]
                # (`type` casts integers too: then only the device is taken over)
                self._buffers[name] = now.view(t.dtype) if now.dtype is _INTEGERS[t.element_size()] else t.to(now.device)
        return self

    def forward(self, x):
        if not (x.is_cuda and x.dtype in (torch.float16, torch.bfloat16)):
            raise RuntimeError("ConvLinearFP8 runs on the B200 kernels: float16 / bfloat16 CUDA activations "
                               f"required (got {x.dtype} on {x.device})")
        from . import _b200_runtime as rt
        q, s = rt.quantize_fp8_block(self._prepared(x.reshape(-1, x.shape[-1])))
        y = rt.gemm_fp8_block(q, self.weight[:, :self.in_features], self.scale, s, bias=self.bias, out_dtype=x.dtype)
        return y.reshape(*x.shape[:-1], self.out_features)

    @staticmethod
    def from_float(module: nn.Linear, rot_need: bool = False, rot_size: int = 256) -> "ConvLinearFP8":
        w = _rotated_weight(module, rot_need, rot_size, None)
        if w.is_cuda:
            from . import _b200_runtime as rt
            q, s = rt.quantize_fp8_block(w, rows=128)
        else:
            q, s = _qu.quantize_weights_fp8(w)
        b = None if module.bias is None else module.bias.detach().clone()
        return ConvLinearFP8(weight=q, scale=s, rot_need=rot_need, bias=b, rot_size=rot_size, in_features=w.shape[1])
