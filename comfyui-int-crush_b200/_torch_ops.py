"""``torch.library`` registrations of the B200 kernels (namespace ``intcrush_b200``).

The C ABI (``libintcrush_b200.so``, reached through ctypes in ``_lib``) is the
boundary; these custom ops wrap the same entry points so that the fused
prep / GEMM calls are single graph nodes for ``torch.compile`` and
``torch.export`` (with fake kernels for shape propagation), instead of
graph breaks at every ctypes call:

* ``intcrush_b200::prep_quantize(x, smoothrot?, perm?, smooth?, rot_size,
  w_in) -> (x_int8, s_a)`` -- ``_b200_runtime.prep_quantize``;
* ``intcrush_b200::gemm_a8(x_int8, w, s_w, s_a, bias?, out_dtype,
  group_size, repacked) -> out`` -- ``_b200_runtime.gemm_a8``;
* ``intcrush_b200::gemm_w4a16(x, packed, scale, group_size, w_layout) ->
  out`` -- ``_b200_runtime.gemm_w4a16``;
* ``intcrush_b200::qk_norm_rope(q, k, q_gamma?, k_gamma?, cos?, sin?, layout,
  positions?, eps) -> (q, k)``, ``intcrush_b200::cross_attention(q, k, v,
  kv_lens?, key_mask?, scale) -> out`` and ``intcrush_b200::lora_batched(x,
  down, up, ids, scales?, base?) -> out`` -- the functions of the same names;
* ``intcrush_b200::quantize_fp8_block(x, rows) -> (q, s)``,
  ``intcrush_b200::gemm_fp8_block(x, w, s_w, s_a, bias?, out_dtype) -> out``,
  ``intcrush_b200::group_norm(x, groups, weight?, bias?, eps, activation) -> y``
  and ``intcrush_b200::fused_groupnorm_quantize(...) -> (q, s)`` -- likewise (rows
  and scales in the layout that the product takes without a copy).

The ops mirror the reference runtime's callables (``_triton_runtime.py:
16-41,114-130``): CUDA tensors in, freshly allocated outputs, launch on the
current stream.  ``register()`` is idempotent; importing this module
registers the ops.
"""

from __future__ import annotations

import torch

from . import _b200_runtime as _rt

_NS = "intcrush_b200"
_DTYPES = {0: torch.float16, 1: torch.bfloat16, 2: torch.float32}
_CODES = {v: k for k, v in _DTYPES.items()}
_done = False


def register() -> None:
    global _done
    if _done:
        return

    @torch.library.custom_op(f"{_NS}::prep_quantize", mutates_args=())
    def prep_quantize(x: torch.Tensor, smoothrot: torch.Tensor | None, perm: torch.Tensor | None,
                      smooth: torch.Tensor | None, rot_size: int, w_in: int) -> tuple[torch.Tensor, torch.Tensor]:
        xq, s_a, _, _ = _rt.prep_quantize(x, smoothrot=smoothrot, rot_size=rot_size, w_in=w_in, perm=perm,
                                          smooth=smooth)
        return xq.contiguous(), s_a

    @prep_quantize.register_fake
    def _(x, smoothrot, perm, smooth, rot_size, w_in):
        M = x.numel() // x.shape[-1]
        return (x.new_empty((M, w_in), dtype=torch.int8), x.new_empty((M,), dtype=torch.float32))

    @torch.library.custom_op(f"{_NS}::gemm_a8", mutates_args=())
    def gemm_a8(x_int8: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor, s_a: torch.Tensor,
                bias: torch.Tensor | None, out_dtype: int, group_size: int, repacked: bool) -> torch.Tensor:
        return _rt.gemm_a8(x_int8, w, s_w, s_a, bias=bias, out_dtype=_DTYPES[out_dtype],
                           group_size=group_size or None, repacked=repacked)

    @gemm_a8.register_fake
    def _(x_int8, w, s_w, s_a, bias, out_dtype, group_size, repacked):
        return x_int8.new_empty((x_int8.shape[0], w.shape[0]), dtype=_DTYPES[out_dtype])

    @torch.library.custom_op(f"{_NS}::gemm_w4a16", mutates_args=())
    def gemm_w4a16(x: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, group_size: int,
                   w_layout: int) -> torch.Tensor:
        return _rt.gemm_w4a16(x, packed, scale, group_size=group_size or None, w_layout=w_layout)

    @gemm_w4a16.register_fake
    def _(x, packed, scale, group_size, w_layout):
        return x.new_empty((x.shape[0], packed.shape[0]), dtype=x.dtype)

    @torch.library.custom_op(f"{_NS}::qk_norm_rope", mutates_args=())
    def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_gamma: torch.Tensor | None, k_gamma: torch.Tensor | None,
                     cos: torch.Tensor | None, sin: torch.Tensor | None, layout: str,
                     positions: torch.Tensor | None, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
        return _rt.qk_norm_rope(q, k, q_gamma=q_gamma, k_gamma=k_gamma, cos=cos, sin=sin, layout=layout,
                                positions=positions, eps=eps)

    @qk_norm_rope.register_fake
    def _(q, k, q_gamma, k_gamma, cos, sin, layout, positions, eps):
        return q.new_empty(q.shape), k.new_empty(k.shape)

    @torch.library.custom_op(f"{_NS}::cross_attention", mutates_args=())
    def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_lens: torch.Tensor | None,
                        key_mask: torch.Tensor | None, scale: float) -> torch.Tensor:
        return _rt.cross_attention(q, k, v, kv_lens=kv_lens, key_mask=key_mask, scale=scale)

    @cross_attention.register_fake
    def _(q, k, v, kv_lens, key_mask, scale):
        return q.new_empty(q.shape)

    @torch.library.custom_op(f"{_NS}::lora_batched", mutates_args=())
    def lora_batched(x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, ids: torch.Tensor,
                     scales: torch.Tensor | None, base: torch.Tensor | None) -> torch.Tensor:
        return _rt.lora_batched(x, down, up, ids, scales, base=base)

    @lora_batched.register_fake
    def _(x, down, up, ids, scales, base):
        return x.new_empty((*x.shape[:-1], up.shape[1]))

    def e4m3(x, rows):
        # the layout of _b200_runtime._fp8_buffers
        K = x.shape[-1]
        kb = (K + 127) // 128
        lead = x.shape[:-1]
        n = x.numel() // K
        q = x.new_empty((n, (K + 15) // 16 * 16), dtype=torch.float8_e4m3fn)[:, :K].view(x.shape)
        if rows == 128:
            return q, x.new_empty(((n + 127) // 128, kb), dtype=torch.float32)
        return q, x.new_empty((kb, n), dtype=torch.float32).t().view(*lead, kb)

    @torch.library.custom_op(f"{_NS}::quantize_fp8_block", mutates_args=())
    def quantize_fp8_block(x: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
        return _rt.quantize_fp8_block(x, rows=rows)

    @quantize_fp8_block.register_fake
    def _(x, rows):
        return e4m3(x, rows)

    @torch.library.custom_op(f"{_NS}::gemm_fp8_block", mutates_args=())
    def gemm_fp8_block(x: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor, s_a: torch.Tensor,
                       bias: torch.Tensor | None, out_dtype: int) -> torch.Tensor:
        return _rt.gemm_fp8_block(x, w, s_w, s_a, bias=bias, out_dtype=_DTYPES[out_dtype])

    @gemm_fp8_block.register_fake
    def _(x, w, s_w, s_a, bias, out_dtype):
        return x.new_empty((*x.shape[:-1], w.shape[0]), dtype=_DTYPES[out_dtype])

    @torch.library.custom_op(f"{_NS}::group_norm", mutates_args=())
    def group_norm(x: torch.Tensor, groups: int, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float,
                   activation: int) -> torch.Tensor:
        return _rt.group_norm(x, groups, weight, bias, eps, activation)

    @group_norm.register_fake
    def _(x, groups, weight, bias, eps, activation):
        return x.new_empty(x.shape)

    @torch.library.custom_op(f"{_NS}::fused_groupnorm_quantize", mutates_args=())
    def fused_groupnorm_quantize(x: torch.Tensor, groups: int, weight: torch.Tensor | None, bias: torch.Tensor | None,
                                 eps: float, activation: int) -> tuple[torch.Tensor, torch.Tensor]:
        return _rt.fused_groupnorm_quantize(x, groups, weight, bias, eps, activation)

    @fused_groupnorm_quantize.register_fake
    def _(x, groups, weight, bias, eps, activation):
        return e4m3(x, 1)

    _done = True


def dtype_code(dtype: torch.dtype) -> int:
    """The ``out_dtype`` integer of ``gemm_a8`` for a torch dtype."""
    return _CODES[dtype]


register()

__all__ = ["register", "dtype_code"]
