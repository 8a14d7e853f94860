"""B200 kernel runtime: the drop-in replacement of ``_triton_runtime``.

Exports the same module attributes as the reference's
``_triton_runtime.py:16-41,114-130`` -- the availability flags
``TRITON_AVAILABLE, TRITON_INT4_UNPACK, TRITON_INT8_GEMM,
TRITON_INT4_INT8_UNPACK, TRITON_DYNQUANT, TRITON_W4A8_GEMM, TRITON_FUSED_QGD``,
the toggles ``USE_FUSED_W8A8`` and ``USE_CUDA_GRAPHS`` (env
``INTCRUSH_NO_CUDA_GRAPHS=1`` disables graphs, ``_triton_runtime.py:60-61``) and
the six kernel callables with their signatures -- but every callable runs the
hand-written sm_100a kernels of ``libintcrush_b200.so``.  A flag is True when
the library loaded and a CUDA device is present.  There is no CPU fallback:
an op given CPU tensors, or called while the library is missing, raises.

New fused ops beyond the reference's set: ``prep_quantize`` (SmoothRot +
Hadamard + pad + PermuQuant + smooth + per-token INT8 in one pass),
``gemm_a8`` (W8A8 / W4A8 with per-channel or group scales, bias and the
zero-point term fused), ``gemm_w4a16`` (weight-streaming W4A16 with the
low-rank residual fused), ``lowrank_down`` / ``lowrank_add``.  Beside the
projections: ``qk_norm_rope`` (head norms and rotation in one pass),
``cross_attention`` and ``lora_batched`` (an adapter per request).  The 8-bit
floating point linear: ``quantize_fp8_block``, ``gemm_fp8_block``, and
``group_norm`` / ``fused_groupnorm_quantize`` in front of it.
"""

from __future__ import annotations

import ctypes
import functools
import logging
import os

import torch

from . import _lib as L

log = logging.getLogger(__name__)

# ── availability flags (names of the reference runtime) ─────────────────────
try:
    L.lib()
    B200_LIBRARY_LOADED = True
    _load_error: str | None = None
except OSError as exc:  # pragma: no cover - depends on the build
    B200_LIBRARY_LOADED = False
    _load_error = str(exc)

B200_AVAILABLE = B200_LIBRARY_LOADED and torch.cuda.is_available()

TRITON_AVAILABLE = B200_AVAILABLE
TRITON_INT4_UNPACK = B200_AVAILABLE
TRITON_INT8_GEMM = B200_AVAILABLE
TRITON_INT4_INT8_UNPACK = B200_AVAILABLE
TRITON_DYNQUANT = B200_AVAILABLE
TRITON_W4A8_GEMM = B200_AVAILABLE
TRITON_FUSED_QGD = B200_AVAILABLE

USE_FUSED_W8A8: bool = False
USE_CUDA_GRAPHS: bool = True
if os.environ.get("INTCRUSH_NO_CUDA_GRAPHS", "0") == "1":
    USE_CUDA_GRAPHS = False

_DT = {torch.float16: L.IC_DTYPE_F16, torch.bfloat16: L.IC_DTYPE_BF16, torch.float32: L.IC_DTYPE_F32}


def _p(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _need_cuda(what: str, *ts: torch.Tensor | None) -> None:
    if not B200_LIBRARY_LOADED:
        raise RuntimeError(f"{what}: libintcrush_b200.so is not loaded ({_load_error})")
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{what}: intcrush_b200 ops run on CUDA tensors only (got {t.device})")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"{what}: tensors on different devices ({dev}, {t.device})")


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


class _LibraryOn:
    """The library's entry points, called with CUDA device ``index`` current."""

    def __init__(self, index: int):
        self._index = index

    def __getattr__(self, name: str):
        entry = getattr(L.lib(), name)

        def call(*args):
            with torch.cuda.device(self._index):
                return entry(*args)

        return call


def _lib(index: int):
    """The library for tensors of CUDA device ``index``: a launch on a default
    stream, the SM count and a kernel's attributes go by the current device,
    which need not be the tensors' (a thread starts on device 0)."""
    return L.lib() if index == _current_device() else _LibraryOn(index)


def _f32c(t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None:
        return None
    return t.to(torch.float32).contiguous()


def _round16(n: int) -> int:
    return (n + 15) // 16 * 16


# ── activation prep ──────────────────────────────────────────────────────────

def prep_quantize(
    x: torch.Tensor,
    *,
    smoothrot: torch.Tensor | None = None,
    rot_size: int = 0,
    w_in: int | None = None,
    perm: torch.Tensor | None = None,
    smooth: torch.Tensor | None = None,
    quantize: bool = True,
    want_prep: bool = False,
    want_rowsum: bool = False,
    s_a_out: torch.Tensor | None = None,
    x_int8_out: torch.Tensor | None = None,
    x_prep_out: torch.Tensor | None = None,
    norm: tuple | None = None,
):
    """One-pass activation prep (``_ops.py:337-365`` + ``_ops.py:529-533``) and
    per-token INT8 quantisation (``kernels/triton_quantize.py:151-198``).

    ``norm`` = ``("layer", gamma, beta_or_None, eps)`` or ``("rms", gamma,
    None, eps)`` normalises each row first (fp32 statistics, one rounding to
    x's dtype), in the same pass (``ic_prep_quant_norm``).

    Returns ``(x_int8, s_a, x_prep, rowsum)``; entries not requested are None.
    ``x_int8`` is ``[M, w_in]`` (a view of a buffer whose row stride is w_in
    rounded up to 16 bytes; the padding columns hold zeros).
    """
    _need_cuda("prep_quantize", x, smoothrot, perm, smooth)
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    if x2.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"prep_quantize: x must be float16/bfloat16, got {x2.dtype}")
    M, K = x2.shape
    Kr = K if not rot_size else -(-K // rot_size) * rot_size
    w_in = Kr if w_in is None else max(int(w_in), Kr)
    # the kernel indexes these vectors without bounds checks: check lengths here
    if smoothrot is not None and smoothrot.numel() != K:
        raise ValueError(f"prep_quantize: smoothrot has {smoothrot.numel()} entries, expected K={K}")
    if perm is not None and perm.numel() != w_in:
        raise ValueError(f"prep_quantize: perm has {perm.numel()} entries, expected w_in={w_in}")
    if smooth is not None and smooth.numel() != w_in:
        raise ValueError(f"prep_quantize: smooth has {smooth.numel()} entries, expected w_in={w_in}")
    if perm is not None and perm.dtype != torch.int32:
        perm = perm.to(torch.int32)
    perm = None if perm is None else perm.contiguous()
    x_int8 = s_a = x_prep = rowsum = None
    xq_full = None
    if quantize:
        ldq = _round16(w_in)
        if x_int8_out is not None:
            xq_full = x_int8_out
            if xq_full.shape[0] != M or xq_full.stride(0) < w_in or xq_full.dtype != torch.int8:
                raise ValueError("prep_quantize: x_int8_out must be int8 [M, >= w_in]")
        else:
            xq_full = torch.empty((M, ldq), dtype=torch.int8, device=x.device)
        s_a = s_a_out if s_a_out is not None else torch.empty(M, dtype=torch.float32, device=x.device)
        x_int8 = xq_full[:, :w_in]
    if want_prep:
        x_prep = x_prep_out if x_prep_out is not None else torch.empty((M, w_in), dtype=x2.dtype, device=x.device)
    if want_rowsum:
        rowsum = torch.empty(M, dtype=torch.float32, device=x.device)
    sr = _f32c(smoothrot)
    sm = _f32c(smooth)
    if norm is not None:
        kind, gamma, beta, eps = norm
        code = {"layer": 1, "rms": 2}[kind]
        if sm is not None:
            raise ValueError("prep_quantize: a norm with SmoothQuant factors is not supported")
        g = _f32c(gamma.reshape(-1))
        b = None if beta is None else _f32c(beta.reshape(-1))
        if g.numel() != K or (b is not None and b.numel() != K):
            raise ValueError("prep_quantize: gamma / beta must have K entries")
        _need_cuda("prep_quantize", g, b)
        st = _lib(x2.get_device()).ic_prep_quant_norm(
            _p(x2), _DT[x2.dtype], M, K, x2.stride(0), code, _p(g), _p(b), float(eps), _p(sr), int(rot_size), w_in,
            _p(perm), _p(xq_full), xq_full.stride(0) if xq_full is not None else 0, _p(s_a), _p(x_prep),
            _p(rowsum), _stream(x2))
        L.check(st, "ic_prep_quant_norm")
        return x_int8, s_a, x_prep, rowsum
    st = _lib(x2.get_device()).ic_prep_quant(
        _p(x2), _DT[x2.dtype], M, K, x2.stride(0), _p(sr), int(rot_size), w_in, _p(perm), _p(sm),
        _p(xq_full), xq_full.stride(0) if xq_full is not None else 0, _p(s_a), _p(x_prep), _p(rowsum),
        _stream(x2))
    L.check(st, "ic_prep_quant")
    return x_int8, s_a, x_prep, rowsum


def dynamic_quantize_activation(
    x: torch.Tensor,
    s_a_out: torch.Tensor | None = None,
    x_int8_out: torch.Tensor | None = None,
):
    """``kernels/triton_quantize.py:151-198``: per-token symmetric INT8.

    Rounding is half-to-even with IEEE division (the reference's CPU form,
    ``kernels/triton_quantize.py:43-54``).  Leading dimensions are restored
    like ``_reshape_if_needed``.
    """
    orig = x.shape
    x2 = x.reshape(-1, orig[-1])
    if s_a_out is not None and s_a_out.shape != (x2.shape[0],):
        s_a_out = None
    if x_int8_out is not None and x_int8_out.shape != x2.shape:
        x_int8_out = None
    x_int8, s_a, _, _ = prep_quantize(x2, s_a_out=s_a_out, x_int8_out=x_int8_out)
    if len(orig) > 2:
        x_int8 = x_int8.reshape(orig)
        s_a = s_a.reshape(orig[:-1])
    return x_int8, s_a


def _norm_quantize(x, norm, s_a_out, x_int8_out):
    orig = x.shape
    x2 = x.reshape(-1, orig[-1])
    if s_a_out is not None and s_a_out.shape != (x2.shape[0],):
        s_a_out = None
    if x_int8_out is not None and x_int8_out.shape != x2.shape:
        x_int8_out = None
    x_int8, s_a, _, _ = prep_quantize(x2, norm=norm, s_a_out=s_a_out, x_int8_out=x_int8_out)
    if len(orig) > 2:
        x_int8 = x_int8.reshape(orig)
        s_a = s_a.reshape(orig[:-1])
    return x_int8, s_a


def fused_layernorm_quantize(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor | None = None,
                             eps: float = 1e-5, s_a_out: torch.Tensor | None = None,
                             x_int8_out: torch.Tensor | None = None):
    """``kernels/triton_quantize.py:274-338``: LayerNorm + per-row INT8 in one
    pass.  Follows the reference's CPU form: normalised values are cast to
    x's dtype (fp16/bf16), then quantised half-to-even."""
    return _norm_quantize(x, ("layer", gamma, beta, eps), s_a_out, x_int8_out)


def fused_rmsnorm_quantize(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6,
                           s_a_out: torch.Tensor | None = None, x_int8_out: torch.Tensor | None = None):
    """``kernels/triton_quantize.py:395-451``: RMSNorm + per-row INT8 in one pass
    (CPU form: ``x / sqrt(mean(x^2) + eps) * gamma`` cast to x's dtype)."""
    return _norm_quantize(x, ("rms", gamma, None, eps), s_a_out, x_int8_out)


# ── GEMMs ────────────────────────────────────────────────────────────────────

def gemm_a8(
    x_int8: torch.Tensor,
    w: torch.Tensor,
    s_w: torch.Tensor,
    s_a: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
    group_size: int | None = None,
    rowsum: torch.Tensor | None = None,
    zp_corr: torch.Tensor | None = None,
    repacked: bool = False,
    splits: int | None = None,
    activation: int = 0,
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """``out = s_a[m] * sum_g s_w[n,g] * (xq @ w^T)_g + bias - rowsum (x) zp_corr``.

    ``activation`` (0 none, 1 SiLU, 2 GELU erf, 3 GELU tanh) and then
    ``residual`` ([M, N], any float dtype, unit column stride) are applied in
    fp32 in the epilogue before the output cast.

    ``w`` is int8 ``[N, K]`` or packed INT4 uint8 ``[N, K/2]``; ``s_w`` is
    ``[N]``/``[N,1]`` (per channel) or ``[N, G]`` (groups of ``group_size``,
    default ``ceil(K / G)`` rounded to a multiple of 128).

    ``splits`` cuts K into that many parts run as separate work units (split-K,
    fp32 partials in a workspace allocated here, then a reduce kernel); None
    picks it from the tile count so that small-M calls fill the GPU
    (``INTCRUSH_SPLITK=0`` turns that off).
    """
    _need_cuda("gemm_a8", x_int8, w, s_w, s_a, bias, out, rowsum, zp_corr)
    if x_int8.dtype != torch.int8:
        raise AssertionError(f"x_int8 must be int8, got {x_int8.dtype}")
    M, K = x_int8.shape
    if x_int8.stride(1) != 1:
        x_int8 = x_int8.contiguous()
    if w.dtype == torch.int8:
        kind = L.IC_W_INT8
        N = w.shape[0]
        if w.shape[1] != K:
            raise AssertionError(f"K mismatch: {K} vs {w.shape[1]}")
    elif w.dtype == torch.uint8:
        kind = L.IC_W_INT4R if repacked else L.IC_W_INT4
        N = w.shape[0]
        if w.shape[1] != (K + 1) // 2:
            raise AssertionError(f"packed K mismatch: {K} vs {w.shape[1]} bytes")
    else:
        raise AssertionError(f"w must be int8 or uint8 (packed int4), got {w.dtype}")
    if w.stride(1) != 1:
        w = w.contiguous()
    sw = s_w.to(torch.float32)
    if sw.dim() == 1:
        sw = sw.reshape(N, -1)
    sw = sw.reshape(N, -1).contiguous()
    G = sw.shape[1]
    if G > 1 and group_size is None:
        group_size = -(-K // G)
    gs = int(group_size) if G > 1 else K
    sa = s_a.to(torch.float32).contiguous()
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=x_int8.device)
    elif out.shape != (M, N) or out.stride(1) != 1:
        raise AssertionError(f"out shape mismatch: {tuple(out.shape)} vs ({M}, {N})")
    b = None if bias is None else bias.contiguous()
    rs = _f32c(rowsum)
    zc = _f32c(zp_corr)
    if splits is None:
        splits = _auto_splits(M, N, K, G, gs, x_int8.device, kind != L.IC_W_INT8)
    if activation or residual is not None:
        r = residual
        if r is not None:
            if r.shape != (M, N):
                raise AssertionError(f"residual shape mismatch: {tuple(r.shape)} vs ({M}, {N})")
            _need_cuda("gemm_a8", r)
            if r.stride(1) != 1:
                r = r.contiguous()
        ws = torch.empty(splits * M * N if splits > 1 else 0, dtype=torch.float32, device=x_int8.device)
        st = _lib(x_int8.get_device()).ic_gemm_a8_ex(
            _p(x_int8), M, K, x_int8.stride(0), _p(w), kind, N, w.stride(0), _p(sw), G, gs, _p(sa),
            _p(b), _DT[b.dtype] if b is not None else 0, _p(rs), _p(zc), int(activation),
            _p(r), _DT[r.dtype] if r is not None else 0, r.stride(0) if r is not None else 0,
            _p(out), _DT[out.dtype], out.stride(0), int(splits), _p(ws) if splits > 1 else None, ws.numel(),
            _stream(x_int8))
        L.check(st, "ic_gemm_a8_ex")
        return out
    if splits > 1:
        ws = torch.empty(splits * M * N, dtype=torch.float32, device=x_int8.device)
        st = _lib(x_int8.get_device()).ic_gemm_a8_splitk(
            _p(x_int8), M, K, x_int8.stride(0), _p(w), kind, N, w.stride(0), _p(sw), G, gs, _p(sa),
            _p(b), _DT[b.dtype] if b is not None else 0, _p(rs), _p(zc), _p(out), _DT[out.dtype], out.stride(0),
            int(splits), _p(ws), ws.numel(), _stream(x_int8))
        L.check(st, "ic_gemm_a8_splitk")
        return out
    st = _lib(x_int8.get_device()).ic_gemm_a8(
        _p(x_int8), M, K, x_int8.stride(0), _p(w), kind, N, w.stride(0), _p(sw), G, gs, _p(sa),
        _p(b), _DT[b.dtype] if b is not None else 0, _p(rs), _p(zc), _p(out), _DT[out.dtype], out.stride(0),
        _stream(x_int8))
    L.check(st, "ic_gemm_a8")
    return out


_SMS: dict = {}


def _num_sms(device: torch.device) -> int:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _SMS:
        _SMS[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return _SMS[idx]


def _auto_splits(M: int, N: int, K: int, G: int, gs: int, device: torch.device, int4: bool) -> int:
    """Split-K factor for ``gemm_a8``: 1 unless the output tiles cover less
    than half of the SMs; then the largest divisor of the K-block count (and
    of G for group scales) that keeps at least 4 K blocks per part and the
    work units within one wave."""
    if os.environ.get("INTCRUSH_SPLITK", "1") == "0":
        return 1
    grouped = G > 1
    # token-tile width as the library picks it (pick_bn in gemm_tc.cu)
    sms = _num_sms(device)
    bn = 32 if M <= 32 else 64 if M <= 64 else 128 if M <= 128 else (192 if grouped else 256)
    while bn > 64 and -(-M // bn) * -(-N // 128) * 2 < sms:
        bn = 128 if bn > 128 else 64
    tiles = -(-M // bn) * -(-N // 128)
    if tiles * 2 > sms:
        return 1
    nkb = -(-K // 128)
    best = 1
    for d in range(2, 17):
        if nkb % d or nkb // d < 4:
            continue
        if grouped and (K % gs or G % d):
            continue
        if tiles * d <= sms:
            best = d
    return best


def fused_int8_gemm_dequant(
    x_int8: torch.Tensor,
    w_int8: torch.Tensor,
    s_w: torch.Tensor,
    s_a: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    activation: int = 0,
    residual: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``kernels/triton_int8_gemm.py:135-205`` on tcgen05 (kind::i8), with
    the reference's epilogue: ``activation`` 0 none, 1 SiLU, 2 GELU (erf),
    plus 3 GELU with the tanh approximation; then ``+ residual``."""
    if activation not in (0, 1, 2, 3):
        raise ValueError(f"activation must be 0, 1, 2 or 3, got {activation}")
    return gemm_a8(x_int8, w_int8, s_w, s_a, bias=bias, out_dtype=out_dtype, out=out, activation=activation,
                   residual=residual)


def int8_gemm_int8out(
    x_int8: torch.Tensor,
    w_int8: torch.Tensor,
    s_w: torch.Tensor,
    s_a: torch.Tensor,
    c_out: torch.Tensor | None = None,
    s_c_out: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    activation: int = 0,
    group_size: int | None = None,
    repacked: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``kernels/triton_int8_gemm.py:472-536``: a GEMM whose output is
    re-quantised to int8 for the next GEMM of a chain (``s_c`` feeds it as
    ``s_a``).

    The scale is row-global: ``s_c[m] = max(max_n |y[m, n]|, 1e-8) / 127``
    over the whole output row, ``c = rint(y / s_c)`` (ties to even), so that
    ``(c, s_c)`` equals ``dynamic_quantize_activation`` of the fp32 output,
    which the reference's docstring promises.  (The reference kernel takes
    the max over one BLOCK_N tile and lets the tiles of a row race on
    ``s_c``.)  Weights may be int8 or packed INT4 (``group_size`` /
    ``repacked`` as in :func:`gemm_a8`).
    """
    _need_cuda("int8_gemm_int8out", x_int8, w_int8, s_w, s_a, c_out, s_c_out, bias)
    if x_int8.dtype != torch.int8:
        raise AssertionError(f"x_int8 must be int8, got {x_int8.dtype}")
    M, K = x_int8.shape
    if x_int8.stride(1) != 1:
        x_int8 = x_int8.contiguous()
    if w_int8.dtype == torch.int8:
        kind, N = L.IC_W_INT8, w_int8.shape[0]
        if w_int8.shape[1] != K:
            raise AssertionError(f"K mismatch: {K} vs {w_int8.shape[1]}")
    elif w_int8.dtype == torch.uint8:
        kind, N = (L.IC_W_INT4R if repacked else L.IC_W_INT4), w_int8.shape[0]
        if w_int8.shape[1] != (K + 1) // 2:
            raise AssertionError(f"packed K mismatch: {K} vs {w_int8.shape[1]} bytes")
    else:
        raise AssertionError(f"w must be int8 or uint8 (packed int4), got {w_int8.dtype}")
    w = w_int8 if w_int8.stride(1) == 1 else w_int8.contiguous()
    sw = s_w.to(torch.float32).reshape(N, -1).contiguous()
    G = sw.shape[1]
    if G > 1 and group_size is None:
        group_size = -(-K // G)
    gs = int(group_size) if G > 1 else K
    sa = s_a.to(torch.float32).contiguous()
    if c_out is not None:
        if c_out.shape != (M, N) or c_out.dtype != torch.int8 or c_out.stride(1) != 1:
            raise AssertionError(f"c_out must be int8 [{M}, {N}] with unit column stride")
        c = c_out
    else:
        c = torch.empty((M, N), dtype=torch.int8, device=x_int8.device)
    if s_c_out is not None:
        if s_c_out.shape != (M,) or s_c_out.dtype != torch.float32 or not s_c_out.is_contiguous():
            raise AssertionError(f"s_c_out must be contiguous float32 [{M}]")
        s_c = s_c_out
    else:
        s_c = torch.empty(M, dtype=torch.float32, device=x_int8.device)
    b = None if bias is None else bias.contiguous()
    ws = torch.empty(M * N + M, dtype=torch.float32, device=x_int8.device)
    st = _lib(x_int8.get_device()).ic_gemm_a8_int8out(
        _p(x_int8), M, K, x_int8.stride(0), _p(w), kind, N, w.stride(0), _p(sw), G, gs, _p(sa),
        _p(b), _DT[b.dtype] if b is not None else 0, int(activation), _p(c), c.stride(0), _p(s_c),
        _p(ws), ws.numel(), _stream(x_int8))
    L.check(st, "ic_gemm_a8_int8out")
    return c, s_c


def fused_w4a8_gemm_dequant(
    x_int8: torch.Tensor,
    w_int8: torch.Tensor,
    s_w: torch.Tensor,
    s_a: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``kernels/triton_w4a8_gemm.py:111-169``.  Accepts the unpacked int8
    weights of the reference or, without materialising them, packed INT4."""
    return gemm_a8(x_int8, w_int8, s_w, s_a, bias=bias, out_dtype=out_dtype, out=out)


def fused_quant_int8_gemm_dequant(
    x_fp16: torch.Tensor,
    w_int8: torch.Tensor,
    s_w: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``kernels/triton_int8_gemm.py:331-389``: quantise + GEMM + dequant."""
    if x_fp16.dtype not in (torch.float16, torch.bfloat16):
        raise AssertionError(f"x must be fp16/bf16, got {x_fp16.dtype}")
    x_int8, s_a, _, _ = prep_quantize(x_fp16)
    if out is not None and out.shape != (x_int8.shape[0], w_int8.shape[0]):
        out = None
    return gemm_a8(x_int8, w_int8, s_w, s_a, bias=bias, out_dtype=out_dtype, out=out)


def gemm_w4a16(
    x: torch.Tensor,
    packed: torch.Tensor,
    scale: torch.Tensor,
    group_size: int | None = None,
    bias: torch.Tensor | None = None,
    lr_mid: torch.Tensor | None = None,
    lr_up: torch.Tensor | None = None,
    lr_scale: float = 1.0,
    out: torch.Tensor | None = None,
    K: int | None = None,
    w_layout: int = 0,
    splits: int | None = None,
) -> torch.Tensor:
    """W4A16: ``T(x @ W^T (+ bias))`` then ``+= lr_scale * lr_mid @ lr_up^T``,
    T = x's dtype.  fp16: ``W = fp16(q * fp16(s))`` (the Triton unpack's
    product); bf16: ``W = bf16(q * s)`` from the fp32 product (the PyTorch
    path's dequantisation cast to the activation dtype).

    ``splits`` (M > 128 only): K parts run as separate work units with fp32
    partials in a workspace allocated here; None picks the count that fills
    the SMs (token tiles of 128), 1 runs unsplit.

    Replaces ``unpack_int4_to_float16`` + ``F.linear`` (``_ops.py:473-474``)
    and the PyTorch INT4 path (``_ops.py:483-491``).
    """
    _need_cuda("gemm_w4a16", x, packed, scale, bias, lr_mid, lr_up, out)
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"gemm_w4a16: activations must be float16 or bfloat16, got {x.dtype}")
    x2 = x if x.stride(-1) == 1 else x.contiguous()
    M, Kx = x2.shape
    K = Kx if K is None else K
    N = packed.shape[0]
    if packed.dtype != torch.uint8 or packed.shape[1] != (K + 1) // 2:
        raise AssertionError("packed must be uint8 [N, ceil(K/2)]")
    sc = scale.reshape(N, -1)
    if sc.dtype not in (torch.float16, torch.float32):
        sc = sc.to(torch.float32)
    sc = sc.contiguous()
    G = sc.shape[1]
    gs = int(group_size) if (G > 1 and group_size is not None) else (-(-K // G) if G > 1 else K)
    if out is None:
        out = torch.empty((M, N), dtype=x.dtype, device=x.device)
    elif out.dtype != x.dtype:
        raise TypeError("gemm_w4a16: out must have x's dtype")
    b = None if bias is None else bias.contiguous()
    mid = None if lr_mid is None else lr_mid.to(x.dtype).contiguous()
    up = None if lr_up is None else lr_up.to(x.dtype).contiguous()
    R = 0 if mid is None else mid.shape[1]
    if splits is None:
        splits = _w4a16_splits(M, N, K, x.device)
    ws = torch.empty(splits * M * N if (splits > 1 and M > 128) else 0, dtype=torch.float32, device=x.device)
    st = _lib(x2.get_device()).ic_gemm_w4a16_splitk(
        _p(x2), _DT[x.dtype], M, K, x2.stride(0), _p(packed), N, packed.stride(0), int(w_layout),
        _p(sc), _DT[sc.dtype],
        G, gs, _p(b), _DT[b.dtype] if b is not None else 0, _p(mid), _p(up), R, float(lr_scale),
        _p(out), out.stride(0), int(splits), _p(ws) if ws.numel() else None, ws.numel(), _stream(x2))
    L.check(st, "ic_gemm_w4a16_splitk")
    return out


def _w4a16_splits(M: int, N: int, K: int, device) -> int:
    """The split count ``ic_gemm_w4a16_splitk`` plans for splits = 0 (token
    tiles of 128, one work unit per SM, at most 8 parts dividing the 64-wide
    K blocks); 1 for the M <= 128 weight-stream kernel."""
    if M <= 128:
        return 1
    tiles = -(-M // 128) * -(-N // 128)
    s = max(1, min(8, _num_sms(device) // max(tiles, 1)))
    nkb = -(-K // 64)
    while s > 1 and nkb % s:
        s -= 1
    return s


def lowrank_down(x: torch.Tensor, down: torch.Tensor) -> torch.Tensor:
    """``mid = T(x @ down^T)`` (``F.linear(x_raw, down)``, ``_ops.py:242``),
    T = x's dtype (fp16 or bf16; other dtypes compute in fp16)."""
    _need_cuda("lowrank_down", x, down)
    dt = x.dtype if x.dtype in (torch.float16, torch.bfloat16) else torch.float16
    x2 = x.reshape(-1, x.shape[-1]).to(dt)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    d = down.to(dt).contiguous()
    M, K = x2.shape
    R = d.shape[0]
    mid = torch.empty((M, R), dtype=dt, device=x.device)
    st = _lib(x2.get_device()).ic_lowrank_down_ex(
        _p(x2), _DT[dt], M, K, x2.stride(0), _p(d), R, _p(mid), _stream(x2))
    L.check(st, "ic_lowrank_down_ex")
    return mid


def lowrank_add(out: torch.Tensor, mid: torch.Tensor, up: torch.Tensor, scale: float) -> torch.Tensor:
    """In place ``out = T(out + scale * mid @ up^T)`` (``out.addmm_``,
    ``_ops.py:243``); out fp16 or bf16, rank up to 256."""
    _need_cuda("lowrank_add", out, mid, up)
    if out.dtype not in (torch.float16, torch.bfloat16) or out.stride(1) != 1:
        raise TypeError("lowrank_add: out must be a row-major float16 / bfloat16 matrix")
    m = mid.to(out.dtype).contiguous()
    u = up.to(out.dtype).contiguous()
    M, N = out.shape
    st = _lib(out.get_device()).ic_lowrank_add_ex(
        _p(out), _DT[out.dtype], M, N, out.stride(0), _p(m), _p(u), m.shape[1], float(scale), _stream(out))
    L.check(st, "ic_lowrank_add_ex")
    return out


def quantize_weight(w: torch.Tensor, bits: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-row requantisation of a float weight on the device (the layout
    classes' ``quantize``, ``quant_layout.py:100-129,179-200``): returns
    (packed uint8 ``[N, ceil(K/2)]``, fp16 scales ``[N]``) for ``bits`` 4 and
    (int8 ``[N, K]``, fp32 scales ``[N]``) for 8."""
    _need_cuda("quantize_weight", w)
    if w.dim() != 2:
        raise AssertionError(f"weight must be 2-D, got {tuple(w.shape)}")
    wf = w.to(torch.float32)
    if wf.stride(1) != 1:
        wf = wf.contiguous()
    N, K = wf.shape
    if bits == 4:
        q = torch.empty((N, (K + 1) // 2), dtype=torch.uint8, device=w.device)
        s = torch.empty(N, dtype=torch.float16, device=w.device)
    elif bits == 8:
        q = torch.empty((N, K), dtype=torch.int8, device=w.device)
        s = torch.empty(N, dtype=torch.float32, device=w.device)
    else:
        raise ValueError(f"bits must be 4 or 8, got {bits}")
    st = _lib(wf.get_device()).ic_quantize_weight(
        _p(wf), N, K, wf.stride(0), int(bits), _p(q), q.stride(0), _p(s), _stream(wf))
    L.check(st, "ic_quantize_weight")
    return q, s


def lokr_add(out: torch.Tensor, x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, scale: float) -> torch.Tensor:
    """``out[t] (viewed [out_l, out_k]) += scale * (w1 @ x[t].view(in_m, in_n)) @ w2^T``
    in place (``_apply_lokr``, ``_ops.py:88-138``): ``w1`` [out_l, in_m],
    ``w2`` [out_k, in_n] (the reference's ``w2_t`` transposed), ``out``
    contiguous [M, out_l * out_k], ``x`` [M, in_m * in_n], all fp16 or bf16.
    The first product is rounded to the activation dtype, as the
    reference's matmul does."""
    _need_cuda("lokr_add", out, x, w1, w2)
    if out.dtype not in (torch.float16, torch.bfloat16) or {x.dtype, w1.dtype, w2.dtype} != {out.dtype}:
        raise TypeError("lokr_add: out, x, w1 and w2 must share one dtype, float16 or bfloat16")
    if not out.is_contiguous():
        raise AssertionError("lokr_add: out must be contiguous")
    if x.stride(1) != 1:
        x = x.contiguous()
    w1c, w2c = w1.contiguous(), w2.contiguous()
    M, N = out.shape
    out_l, in_m = w1c.shape
    out_k, in_n = w2c.shape
    temp = torch.empty(M * out_l * in_n, dtype=out.dtype, device=out.device)
    st = _lib(out.get_device()).ic_lokr_add(
        _p(out), _DT[out.dtype], M, N, _p(x), x.stride(0), x.shape[1], _p(w1c), out_l, in_m, _p(w2c), out_k, in_n,
        float(scale), _p(temp), temp.numel(), _stream(out))
    L.check(st, "ic_lokr_add")
    return out


def repack_int4(packed: torch.Tensor, K: int, layout: int) -> torch.Tensor:
    """Load-time nibble permutation of packed INT4 weights (``ic_repack_int4``):
    layout 0 feeds ``gemm_a8(..., repacked=True)``, layout 1 feeds
    ``gemm_w4a16(..., w_layout=1)``.  Same shape and size as the input."""
    _need_cuda("repack_int4", packed)
    p = packed.contiguous()
    out = torch.empty_like(p)
    st = _lib(p.get_device()).ic_repack_int4(
        _p(p), p.shape[0], K, p.stride(0), _p(out), out.stride(0), int(layout), _stream(p))
    L.check(st, "ic_repack_int4")
    return out


def unpack_int4_to_int8(packed: torch.Tensor, K: int) -> torch.Tensor:
    """``kernels/triton_int4_to_int8_unpack.py:55-81``."""
    _need_cuda("unpack_int4_to_int8", packed)
    p = packed.contiguous()
    N = p.shape[0]
    out = torch.empty((N, K), dtype=torch.int8, device=p.device)
    st = _lib(p.get_device()).ic_unpack_int4_to_int8(
        _p(p), N, K, p.stride(0), _p(out), _stream(p))
    L.check(st, "ic_unpack_int4_to_int8")
    return out


def unpack_int4_to_float16(packed: torch.Tensor, scale: torch.Tensor, K: int,
                           group_size: int | None = None) -> torch.Tensor:
    """``kernels/triton_int4_unpack.py:62-88`` (scale ``[N]``), extended to
    group scales ``[N, G]``."""
    _need_cuda("unpack_int4_to_float16", packed, scale)
    p = packed.contiguous()
    N = p.shape[0]
    sc = scale.reshape(N, -1)
    if sc.dtype not in (torch.float16, torch.float32):
        sc = sc.to(torch.float32)
    sc = sc.contiguous()
    G = sc.shape[1]
    gs = int(group_size) if group_size else -(-K // G)
    out = torch.empty((N, K), dtype=torch.float16, device=p.device)
    st = _lib(p.get_device()).ic_unpack_int4_to_f16(
        _p(p), N, K, p.stride(0), _p(sc), _DT[sc.dtype], G, gs, _p(out), _stream(p))
    L.check(st, "ic_unpack_int4_to_f16")
    return out


# ── attention-side operators ─────────────────────────────────────────────────

_MASKS = {torch.bool: L.IC_MASK_BOOL, torch.float16: L.IC_MASK_F16, torch.bfloat16: L.IC_MASK_BF16,
          torch.float32: L.IC_MASK_F32}
_ROPE = {"interleaved": L.IC_ROPE_INTERLEAVED, "half": L.IC_ROPE_HALF}
_DENSE = torch.contiguous_format
_HALF = {torch.float16: L.IC_DTYPE_F16, torch.bfloat16: L.IC_DTYPE_BF16}

# These calls are short on the device, so their host side is kept short too:
# plain integers for pointers, the raw stream handle, one ctypes array per set
# of strides.
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


@functools.lru_cache(maxsize=1024)
def _strides12(*strides):
    return (ctypes.c_int64 * 12)(*strides)


# Workspace floats by sizes (and device: the plans go by its SM count).
@functools.lru_cache(maxsize=4096)
def _workspace(name: str, index: int, *sizes: int) -> int:
    return getattr(_lib(index), name)(*sizes)


def _same_device(what: str, index: int, *ts: torch.Tensor | None) -> None:
    """All of ``ts`` on CUDA device ``index`` (as ``_need_cuda``)."""
    if index < 0 or not B200_LIBRARY_LOADED:
        _need_cuda(what, *ts)
        raise RuntimeError(f"{what}: intcrush_b200 ops run on CUDA tensors only")
    for t in ts:
        if t is not None and t.get_device() != index:
            _need_cuda(what, *ts)
            raise RuntimeError(f"{what}: tensors on different devices")


def _heads_ok(t: torch.Tensor) -> bool:
    """``t`` ([batch, tokens, heads, D]) can be read as it is: elements
    contiguous, 16-byte aligned rows, tokens apart."""
    b, l, h, d = t.stride()
    return d == 1 and not ((b | l | h) & 7 or t.data_ptr() & 15) and (l != 0 or t.shape[1] <= 1)


def _plain_ones(t: torch.Tensor) -> torch.Tensor:
    """``t`` with the strides of its dimensions of one entry, which say nothing
    and may be anything, as 0."""
    return t.as_strided(t.shape, tuple(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride())) + t.stride()[3:])


def _heads(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels read it; a copy where it is not."""
    b, l, h, d = t.stride()
    if d == 1 and l and not ((b | l | h) & 7 or t.data_ptr() & 15):   # (_heads_ok, in place)
        return t
    t = _plain_ones(t)
    return t if _heads_ok(t) else t.clone(memory_format=_DENSE)


def _out_heads(what: str, out: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    if out.shape != like.shape or out.dtype != like.dtype:
        raise ValueError(f"{what}: out must be {like.dtype} {tuple(like.shape)}, got {out.dtype} {tuple(out.shape)}")
    y = out if _heads_ok(out) else _plain_ones(out)
    if not _heads_ok(y) or any(s == 0 and n > 1 for s, n in zip(y.stride(), y.shape)):
        raise ValueError(f"{what}: out must have contiguous elements, strides that are multiples of 8 and a 16-byte "
                         f"aligned start, got strides {out.stride()}")
    return y


_INT32_MAX = 2**31 - 1


def _index(t: torch.Tensor) -> torch.Tensor:
    """``t`` as int32 on the way to the kernels, which check its range.  Wider
    integers saturate: a length past the keys stays past them, and an id or a
    position outside its range stays outside."""
    dt = t.dtype
    if dt is not torch.int32:
        if dt.is_floating_point or dt.is_complex or dt is torch.bool:
            raise TypeError(f"an index tensor must hold integers, got {dt}")
        if dt is torch.uint64:
            t = t.view(torch.int64)
            t = t.masked_fill(t < 0, _INT32_MAX)   # 2^63 and more
        elif dt is torch.uint32:
            t = t.to(torch.int64)
        if t.dtype is torch.int64:
            t = t.clamp(-_INT32_MAX - 1, _INT32_MAX)
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _fp32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _gamma16(what: str, t: torch.Tensor | None, D: int) -> torch.Tensor | None:
    if t is None:
        return None
    if t.numel() != D:
        raise ValueError(f"{what}: gamma has {t.numel()} entries, expected {D}")
    g = _fp32(t)
    return g.clone() if g.data_ptr() & 15 else g


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor | None = None,
    *,
    q_gamma: torch.Tensor | None = None,
    k_gamma: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    layout: str = "interleaved",
    positions: torch.Tensor | None = None,
    eps: float = 1e-6,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
):
    """RMS norm of every query and key head and the position rotation, one pass.

    ``q`` [B, L, H, D] and ``k`` [B, L, Hk, D] (fp16 / bf16, D a multiple of 8
    up to 256) may be strided views, e.g. of a fused QKV projection's output.
    Each head becomes ``x * rsqrt(mean(x^2) + eps) * gamma`` (gammas [D], None
    = ones) in fp32; then its first ``2 * cos.shape[-1]`` elements turn by the
    angles whose cosines and sines are in row ``positions[b, l]`` (default:
    ``l``) of the tables ``cos`` / ``sin`` [rows, rot / 2]: pairs
    ``(2i, 2i + 1)`` (``layout="interleaved"``) or ``(i, i + rot / 2)``
    (``"half"``).  Without tables only the norm is applied.

    A position outside the tables, whatever the width of its integers, gives
    NaN for its token and sets the library's device error word.  (int32
    positions are taken as they are, others cost a conversion.)  Returns
    ``(q, k)`` normalised, or only ``q`` without a ``k``; ``q_out`` / ``k_out``
    may be the inputs themselves.
    """
    index = q.get_device()
    _same_device("qk_norm_rope", index, q, k, q_gamma, k_gamma, cos, sin, positions, q_out, k_out)
    dtype = _HALF.get(q.dtype)
    if dtype is None:
        raise TypeError(f"qk_norm_rope: q must be float16/bfloat16, got {q.dtype}")
    if q.dim() != 4:
        raise ValueError(f"qk_norm_rope: q must be [batch, tokens, heads, D], got {tuple(q.shape)}")
    form = _ROPE.get(layout)
    if form is None:
        raise ValueError(f"qk_norm_rope: layout must be 'interleaved' or 'half', got {layout!r}")
    B, T, H, D = q.shape
    rot = rows = 0
    if (cos is None) != (sin is None):
        raise ValueError("qk_norm_rope: cos and sin come together")
    if cos is not None:
        if cos.shape != sin.shape or cos.dim() != 2:
            raise ValueError(f"qk_norm_rope: tables must be [rows, rot / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}")
        cos, sin = _fp32(cos), _fp32(sin)
        rows, rot = cos.shape
        rot *= 2
        if rows > _INT32_MAX:
            rows = _INT32_MAX   # as a position it is past every table (_index)
    if positions is not None:
        if positions.shape != (B, T):
            raise ValueError(f"qk_norm_rope: positions must be [{B}, {T}], got {tuple(positions.shape)}")
        positions = _index(positions)
    gq = _gamma16("qk_norm_rope", q_gamma, D)
    x = _heads(q)
    y = torch.empty_like(q, memory_format=_DENSE) if q_out is None else _out_heads("qk_norm_rope", q_out, q)
    if k is None:
        if k_gamma is not None or k_out is not None:
            raise ValueError("qk_norm_rope: k_gamma / k_out without a k")
        Hk, xk, yk, gk = 0, None, None, None
        strides = _strides12(*x.stride()[:3], *y.stride()[:3], 0, 0, 0, 0, 0, 0)
    else:
        if k.dim() != 4 or k.dtype != q.dtype or k.shape[:2] != (B, T) or k.shape[3] != D:
            raise ValueError(f"qk_norm_rope: k must be {q.dtype} [{B}, {T}, heads, {D}], got {k.dtype} {tuple(k.shape)}")
        Hk = k.shape[2]
        gk = _gamma16("qk_norm_rope", k_gamma, D)
        xk = _heads(k)
        yk = torch.empty_like(k, memory_format=_DENSE) if k_out is None else _out_heads("qk_norm_rope", k_out, k)
        strides = _strides12(*x.stride()[:3], *y.stride()[:3], *xk.stride()[:3], *yk.stride()[:3])
    st = _lib(index).ic_qk_norm_rope(
        x.data_ptr(), y.data_ptr(), H, None if xk is None else xk.data_ptr(), None if yk is None else yk.data_ptr(), Hk,
        dtype, B, T, D, strides, None if gq is None else gq.data_ptr(), None if gk is None else gk.data_ptr(), eps, form,
        rot, cos.data_ptr() if rot else None, sin.data_ptr() if rot else None, rows,
        None if positions is None else positions.data_ptr(), _raw_stream(index))
    if st:
        L.check(st, "ic_qk_norm_rope")
    y = y if q_out is None else q_out
    return y if k is None else (y, yk if k_out is None else k_out)


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    kv_lens: torch.Tensor | None = None,
    key_mask: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of ``q`` [B, Lq, H, D] to an encoder's states ``k`` / ``v``
    [B, Lk, Hk, D] (fp16 / bf16, D a multiple of 8 up to 128, H a multiple of
    Hk: query heads ``h`` share key head ``h // (H // Hk)``):
    ``softmax(scale * q k^T + mask) v`` with ``scale`` 1/sqrt(D) by default.

    ``kv_lens`` [B] (integers on the device): sample b sees keys below
    ``kv_lens[b]``.  ``key_mask`` [B, Lk] or [Lk]: bool (False = not seen) or
    float (added to the scores, -inf = not seen).  What ``k`` and ``v`` hold at
    keys that are not seen does not matter; a sample that sees none gets
    zeros.  All may be strided views.  Returns [B, Lq, H, D].
    """
    index = q.get_device()
    _same_device("cross_attention", index, q, k, v, kv_lens, key_mask, out)
    dtype = _HALF.get(q.dtype)
    if dtype is None or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"cross_attention: q, k and v must share one dtype, float16 or bfloat16, got {q.dtype}, "
                        f"{k.dtype}, {v.dtype}")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"cross_attention: q must be [B, Lq, H, D], k and v [B, Lk, Hk, D], got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    B, Lq, H, D = q.shape
    _, Lk, Hk, _ = k.shape
    if kv_lens is not None:
        if kv_lens.shape != (B,):
            raise ValueError(f"cross_attention: kv_lens must be [{B}], got {tuple(kv_lens.shape)}")
        kv_lens = _index(kv_lens)
    kind = ld = 0
    if key_mask is not None:
        kind = _MASKS.get(key_mask.dtype, 0)
        if not kind:
            raise TypeError(f"cross_attention: key_mask must be bool, float16, bfloat16 or float32, got {key_mask.dtype}")
        if key_mask.shape not in ((B, Lk), (Lk,)):
            raise ValueError(f"cross_attention: key_mask must be [{B}, {Lk}] or [{Lk}], got {tuple(key_mask.shape)}")
        if key_mask.stride(-1) != 1:
            key_mask = key_mask.contiguous()
        ld = key_mask.stride(0) if key_mask.dim() == 2 and B > 1 else 0
        if 0 < ld < Lk:
            key_mask = key_mask.contiguous()
            ld = Lk
    y = torch.empty_like(q, memory_format=_DENSE) if out is None else _out_heads("cross_attention", out, q)
    q, k, v = _heads(q), _heads(k), _heads(v)
    n = _workspace("ic_cross_attention_workspace", index, B, Lq, Lk, H, Hk, D, kind)
    # (sizes that are refused: the call below says why)
    ws = q.new_empty(2 * n) if n > 0 else None   # n floats, in 16-bit elements
    st = _lib(index).ic_cross_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(), dtype, B, Lq, Lk, H, Hk, D,
        _strides12(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *y.stride()[:3]),
        D ** -0.5 if scale is None else scale, None if kv_lens is None else kv_lens.data_ptr(),
        None if key_mask is None else key_mask.data_ptr(), kind, ld, None if ws is None else ws.data_ptr(), n,
        _raw_stream(index))
    if st:
        L.check(st, "ic_cross_attention")
    return y if out is None else out


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` as a [rows, width] matrix with contiguous rows."""
    if t.dim() != 2:
        t = t.flatten(0, -2) if t.dim() > 2 else t.view(1, width)
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= width) else t.contiguous()


def lora_batched(
    x: torch.Tensor,
    down: torch.Tensor,
    up: torch.Tensor,
    ids: torch.Tensor,
    scales: torch.Tensor | None = None,
    *,
    base: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``base + scales[a] * (x @ down[a]^T) @ up[a]^T`` with an adapter ``a`` of
    its own for every request (``a < 0``: none), fp32 sums, one rounding.

    ``x`` [..., K] (fp16 / bf16), ``down`` [n, R, K] and ``up`` [n, N, R] the
    adapters (smaller ranks padded with zeros, R up to 256), ``ids`` integers
    on the device: one per row of x, or fewer, each for an equal run of rows
    (one per sample of a batch).  ``base`` [..., N] is the shared projection's
    output (None: zeros); ``out`` [..., N] may be ``base``.  An id that names
    no adapter gives NaN for its rows and sets the library's device error
    word.  Same inputs give the same bits; a request's last bits may change
    with which adapters (not with what) its neighbours use, as the order of the
    fp32 sums goes by them.  (One adapter for all rows: :func:`lowrank_down` /
    :func:`lowrank_add`, ``_ops.py:236-244``.)
    """
    index = x.get_device()
    _same_device("lora_batched", index, x, down, up, ids, scales, base, out)
    dt = x.dtype
    dtype = _HALF.get(dt)
    if dtype is None or down.dtype != dt or up.dtype != dt:
        raise TypeError(f"lora_batched: x, down and up must share one dtype, float16 or bfloat16, got {dt}, {down.dtype}, "
                        f"{up.dtype}")
    if down.dim() != 3 or up.dim() != 3 or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2]:
        raise ValueError(f"lora_batched: down must be [n, R, K] and up [n, N, R], got {tuple(down.shape)}, {tuple(up.shape)}")
    n, R, K = down.shape
    N = up.shape[1]
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"lora_batched: x has {tuple(x.shape)[-1:]} columns, expected {K}")
    full = (*x.shape[:-1], N)
    x2 = _rows(x, K)
    M = x2.shape[0]
    S = ids.numel()
    if (S == 0) != (M == 0) or (S and M % S):
        raise ValueError(f"lora_batched: {S} adapter ids do not divide {M} rows")
    ids = _index(ids)
    if scales is not None:
        if scales.numel() != n:
            raise ValueError(f"lora_batched: {scales.numel()} scales for {n} adapters")
        scales = _fp32(scales)
    b2 = None
    if base is not None:
        if base.dtype != dt or base.shape != full:
            raise ValueError(f"lora_batched: base must be {dt} {full}, got {base.dtype} {tuple(base.shape)}")
        b2 = _rows(base, N)
    if out is None:
        out = torch.empty_like(base) if base is not None and base.is_contiguous() else x.new_empty(full)
        ldo = N
    else:
        if out.dtype != dt or out.shape != full:
            raise ValueError(f"lora_batched: out must be {dt} {full}, got {out.dtype} {tuple(out.shape)}")
        if M == 0 or N == 0:
            return out
        o2 = out.view(-1, N)   # raises where the leading dimensions do not fold
        ldo = o2.stride(0) if M > 1 else N
        if o2.stride(1) != 1 or ldo < N:
            raise ValueError(f"lora_batched: out must be row-major, got strides {out.stride()}")
    if M == 0 or N == 0:
        return out
    need = _workspace("ic_lora_batched_workspace", index, M, K, N, R, n)
    # (sizes that are refused: the call below says why)
    ws = x.new_empty(2 * max(need, 0))   # floats, in 16-bit elements
    if not down.is_contiguous():
        down = down.contiguous()
    if not up.is_contiguous():
        up = up.contiguous()
    st = _lib(index).ic_lora_batched(
        x2.data_ptr(), dtype, M, K, x2.stride(0) if M > 1 else K, down.data_ptr(), up.data_ptr(), R, n, ids.data_ptr(),
        M // S, None if scales is None else scales.data_ptr(), None if b2 is None else b2.data_ptr(),
        N if b2 is None or M == 1 else b2.stride(0), out.data_ptr(), N, ldo, ws.data_ptr(), need, _raw_stream(index))
    if st:
        L.check(st, "ic_lora_batched")
    return out


# ── 8-bit floating point linear ──────────────────────────────────────────────

_E4M3 = torch.float8_e4m3fn


# What a call's checks and sizes come to goes by shapes, strides and types alone:
# kept for calls of the same form, so that those of a few microseconds on the
# device are not waited for.
def _sizes(*values: int):
    return (ctypes.c_int64 * len(values))(*values)


def _row_major(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` [..., width] as a matrix with contiguous rows, a copy only where its
    strides need one."""
    t = t.reshape(-1, width)
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= width) else t.contiguous()


def _fp8_buffers(x: torch.Tensor, M: int, K: int, scale_rows: int, by_block: bool):
    """Uninitialised e4m3 rows [M, K] whose stride is K rounded up to 16 (the last
    one whole too), and scales [scale_rows, K / 128], stored block by block where
    ``by_block``, on the device of ``x``."""
    q = x.new_empty((M, _round16(K)), dtype=_E4M3)
    kb = -(-K // 128)
    s = x.new_empty_strided((scale_rows, kb), (1, scale_rows) if by_block else (kb, 1), dtype=torch.float32)
    return q[:, :K] if K & 15 else q, s


@functools.lru_cache(maxsize=4096)
def _quantize_form(dtype, shape, stride, rows):
    """Sizes for the library (None: a matrix has to be made of x first), and of the
    results."""
    what = "quantize_fp8_block"
    code = _DT.get(dtype)
    if code is None:
        raise TypeError(f"{what}: x must be float16, bfloat16 or float32, got {dtype}")
    if rows not in (1, 128):
        raise ValueError(f"{what}: rows must be 1 or 128, got {rows}")
    if not shape or shape[-1] == 0 or (rows == 128 and len(shape) != 2):
        raise ValueError(f"{what}: x must be {'[..., K]' if rows == 1 else '[N, K]'}, got {tuple(shape)}")
    if len(shape) != 2:
        return None, 0, 0, 0
    M, K = shape
    scale_rows = M if rows == 1 else -(-M // 128)
    if stride[1] != 1 and K > 1 or (M > 1 and stride[0] < K):
        return None, 0, 0, 0
    return _sizes(code, M, K, stride[0] if M > 1 else K, rows, _round16(K), *((1, M) if rows == 1 else (-(-K // 128), 1))), M, K, scale_rows


def quantize_fp8_block(x: torch.Tensor, *, rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values with an fp32 scale for each block of 128 along the last
    dimension: ``s = max(max |x|, 1e-8) / 448``, ``q = e4m3(x / s)`` with IEEE
    division, ties to even.

    ``rows=1`` (activations): ``x`` [..., K] (fp16 / bf16 / fp32) gives ``q``
    [..., K] and ``s`` [..., ceil(K / 128)].  ``rows=128`` (weights): ``x``
    [N, K] gives ``q`` [N, K] and ``s`` [ceil(N / 128), ceil(K / 128)], a scale
    for each 128 x 128 block.  Both are what :func:`gemm_fp8_block` takes: ``q``'s
    rows start at multiples of 16 bytes (it is a view where K is no multiple of
    16), activations' scales are stored block by block.

    A NaN makes its block's scale NaN, an infinity infinite; neither is lost
    in a product.  (INT8 per token: :func:`dynamic_quantize_activation`,
    ``kernels/triton_quantize.py:151-198``.)
    """
    index = x.get_device()
    _same_device("quantize_fp8_block", index, x)
    sizes, M, K, scale_rows = _quantize_form(x.dtype, x.shape, x.stride(), rows)
    if sizes is None:
        q, s = quantize_fp8_block(_row_major(x, x.shape[-1]), rows=rows)
        return (q, s) if x.dim() == 2 else (q.view(x.shape), s.view(*x.shape[:-1], s.shape[1]))
    q, s = _fp8_buffers(x, M, K, scale_rows, rows == 1)
    if M:
        st = _lib(index).ic_quantize_fp8_block(x.data_ptr(), q.data_ptr(), s.data_ptr(), sizes, _raw_stream(index))
        if st:
            L.check(st, "ic_quantize_fp8_block")
    return q, s


def _fp8_rows(t: torch.Tensor, K: int) -> torch.Tensor:
    """A copy of an e4m3 matrix whose rows start at multiples of 16 bytes."""
    rows = t.new_empty((t.shape[0], _round16(K)))[:, :K]
    rows.view(torch.uint8).copy_((t if t.stride(1) == 1 else t.contiguous()).view(torch.uint8))
    return rows


@functools.lru_cache(maxsize=4096)
def _product_form(x, w, s_w, s_a, bias, out_dtype, out):
    """Each a tensor's (dtype, shape, stride), or None: what to copy first (1: x, 2:
    w, 4: bias), sizes for the library, M and N."""
    what = "gemm_fp8_block"
    if x[0] is not _E4M3 or w[0] is not _E4M3:
        raise TypeError(f"{what}: x and w must be float8_e4m3fn, got {x[0]}, {w[0]}")
    if not x[1] or len(w[1]) != 2 or x[1][-1] != w[1][1] or w[1][1] == 0:
        raise ValueError(f"{what}: x must be [..., K] and w [N, K], got {tuple(x[1])}, {tuple(w[1])}")
    N, K = w[1]
    kb = -(-K // 128)
    lead = tuple(x[1][:-1])
    if s_a[1] != (*lead, kb) or s_w[1] != (-(-N // 128), kb):
        raise ValueError(f"{what}: scales must be {(*lead, kb)} and {(-(-N // 128), kb)}, got {tuple(s_a[1])}, {tuple(s_w[1])}")
    if s_a[0] is not torch.float32 or s_w[0] is not torch.float32:
        raise TypeError(f"{what}: scales must be float32, got {s_a[0]}, {s_w[0]}")
    code = _DT.get(out_dtype if out is None else out[0])
    if code is None:
        raise TypeError(f"{what}: the output must be float16, bfloat16 or float32, got {out_dtype if out is None else out[0]}")
    copies = bias_code = 0
    if bias is not None:
        bias_code = _DT.get(bias[0])
        if bias_code is None:
            raise TypeError(f"{what}: bias must be float16, bfloat16 or float32, got {bias[0]}")
        if bias[1] != (N,):
            raise ValueError(f"{what}: bias must be [{N}], got {tuple(bias[1])}")
        copies = 0 if bias[2][0] == 1 or N <= 1 else 4
    if out is not None and out[1] != (*lead, N):
        raise ValueError(f"{what}: out must be {(*lead, N)}, got {tuple(out[1])}")
    if len(lead) != 1:
        return copies, None, 0, N
    M = lead[0]
    ldo = N
    if out is not None and M and N:
        ldo = out[2][0] if M > 1 else N
        if (N > 1 and out[2][1] != 1) or ldo < N:
            raise ValueError(f"{what}: out must be row-major, got strides {out[2]}")
    ld = []
    for i, (t, rows) in enumerate(((x, M), (w, N))):
        if (t[2][1] != 1 and K > 1) or (rows > 1 and (t[2][0] & 15 or t[2][0] < K)):
            copies |= 1 << i
        ld.append(t[2][0] if rows > 1 else _round16(K))
    return copies, _sizes(M, K, N, *ld, ldo, *s_a[2], *s_w[2], bias_code, code), M, N


def gemm_fp8_block(
    x: torch.Tensor,
    w: torch.Tensor,
    s_w: torch.Tensor,
    s_a: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``out[m, n] = sum_b s_a[m, b] s_w[n // 128, b] (x @ w^T)_b + bias`` of e4m3
    operands with a scale for each block of 128, fp32 sums, one rounding.

    ``x`` [..., K] and ``w`` [N, K] are ``float8_e4m3fn``, ``s_a`` [..., KB] and
    ``s_w`` [ceil(N / 128), KB] fp32 with KB = ceil(K / 128), as
    :func:`quantize_fp8_block` returns them or as a checkpoint holds them (any
    strides; rows of ``x`` or ``w`` that do not start at multiples of 16 bytes
    are copied first).  ``bias`` [N] and ``out_dtype`` are fp16, bf16 or fp32;
    ``out`` [..., N] sets the latter.  Same inputs give the same bits.
    (INT8 and INT4 operands: :func:`gemm_a8`, ``kernels/triton_int8_gemm.py:135-205``.)
    """
    index = x.get_device()
    _same_device("gemm_fp8_block", index, x, w, s_w, s_a, bias, out)
    copies, sizes, M, N = _product_form(
        (x.dtype, x.shape, x.stride()), (w.dtype, w.shape, w.stride()), (s_w.dtype, s_w.shape, s_w.stride()),
        (s_a.dtype, s_a.shape, s_a.stride()), None if bias is None else (bias.dtype, bias.shape, bias.stride()),
        out_dtype, None if out is None else (out.dtype, out.shape, out.stride()))
    if sizes is None:   # rows first
        K, lead = w.shape[1], x.shape[:-1]
        if out is not None and out.numel() == 0:
            return out
        flat = None if out is None else out.view(-1, N)   # raises where the leading dimensions do not fold
        rows = x.reshape(-1, K) if lead.numel() else x.new_empty((0, K))
        y = gemm_fp8_block(rows, w, s_w, s_a.reshape(rows.shape[0], -(-K // 128)), bias, out_dtype, flat)
        return y.view(*lead, N) if out is None else out
    y = x.new_empty((M, N), dtype=out_dtype) if out is None else out
    if M == 0 or N == 0:
        return y
    xp, wp = x.data_ptr(), w.data_ptr()
    if copies or (xp | wp) & 15:
        if copies & 1 or xp & 15:
            x = _fp8_rows(x, w.shape[1])
        if copies & 2 or wp & 15:
            w = _fp8_rows(w, w.shape[1])
        if copies & 4:
            bias = bias.contiguous()
        return gemm_fp8_block(x, w, s_w, s_a, bias, out_dtype, y)
    st = _lib(index).ic_gemm_fp8_block(xp, wp, s_a.data_ptr(), s_w.data_ptr(), None if bias is None else bias.data_ptr(),
                                       y.data_ptr(), sizes, _raw_stream(index))
    if st:
        L.check(st, "ic_gemm_fp8_block")
    return y


def _rows_of(shape, stride):
    """(L, batch stride, row stride) of a [B, ..., C] tensor whose positions are
    evenly spaced rows with contiguous channels that do not overlap, else None."""
    C = shape[-1]
    if stride[-1] != 1 and C > 1:
        return None
    L, row = 1, C
    for n, s in zip(reversed(shape[1:-1]), reversed(stride[1:-1])):
        if n == 1:
            continue
        if L == 1:
            row = s
        elif s != L * row:
            return None
        L *= n
    return None if L > 1 and row < C else (L, stride[0], row)


def _overlap(n: int, far: int, m: int, near: int, width: int) -> bool:
    """Whether two of n x m runs of ``width`` elements, ``far`` and ``near`` apart,
    share one."""
    if n == 1 or m == 1:
        return (n > 1 and far < width) or (m > 1 and near < width)
    if near > far:
        n, far, m, near = m, near, n, far
    if near < width:
        return True
    last = (m - 1) * near
    for j in range(1, min(n, (last + width - 1) // far + 1)):
        i, r = divmod(j * far, near)     # the runs before and behind the j-th of the others
        if (i < m and r < width) or (i + 1 < m and near - r < width):
            return True
    return False


@functools.lru_cache(maxsize=4096)
def _norm_form(what, index, x, groups, weight, bias, activation, out, quantize):
    """x, weight, bias and out as (dtype, shape, stride) or None: what to copy first
    (1: x, 2: weight, 4: bias), sizes for the library, workspace floats."""
    dtype, shape, stride = x
    code = _HALF.get(dtype)
    if code is None:
        raise TypeError(f"{what}: x must be float16/bfloat16, got {dtype}")
    if len(shape) < 2:
        raise ValueError(f"{what}: x must be [batch, ..., channels], got {tuple(shape)}")
    if activation not in (0, 1, 2, 3):
        raise ValueError(f"{what}: activation must be 0 (none), 1 (SiLU), 2 (GELU erf) or 3 (GELU tanh), got {activation}")
    B, C = shape[0], shape[-1]
    if groups < 1 or C == 0 or C % groups:
        raise ValueError(f"{what}: {C} channels do not divide into {groups} groups")
    codes, copies = [], 0
    for i, t in enumerate((weight, bias)):
        codes.append(0 if t is None else _DT.get(t[0]))
        if codes[-1] is None:
            raise TypeError(f"{what}: weight and bias must be float16, bfloat16 or float32, got {t[0]}")
        if t is not None and t[1] != (C,):
            raise ValueError(f"{what}: weight and bias must be [{C}], got {tuple(t[1])}")
        if t is not None and t[2][0] != 1 and C > 1:
            copies |= 2 << i
    if out is not None and (out[1] != shape or out[0] != dtype):
        raise ValueError(f"{what}: out must be {dtype} {tuple(shape)}, got {out[0]} {tuple(out[1])}")
    if 0 in shape:
        return copies, None, 0
    rows = _rows_of(shape, stride)
    if rows is None:
        return copies | 1, None, 0
    T, x_batch, x_row = rows
    y_batch, y_row = T * C, C
    if out is not None:
        rows = _rows_of(shape, out[2])
        if rows is None or _overlap(B, rows[1], T, rows[2], C):
            raise ValueError(f"{what}: out must be channels last with rows that do not overlap, got strides {out[2]}")
        _, y_batch, y_row = rows
    n = _workspace("ic_group_norm_workspace", index, B, T, C, groups, int(quantize))
    # (sizes that are refused: the call says why)
    return copies, _sizes(code, B, T, C, x_batch, x_row, groups, *codes, activation, y_batch, y_row, _round16(C), 1, B * T, n), n


def _group_norm(what, x, groups, weight, bias, eps, activation, out, quantize):
    index = x.get_device()
    _same_device(what, index, x, weight, bias, out)
    copies, sizes, n = _norm_form(
        what, index, (x.dtype, x.shape, x.stride()), groups, None if weight is None else (weight.dtype, weight.shape, weight.stride()),
        None if bias is None else (bias.dtype, bias.shape, bias.stride()), activation,
        None if out is None else (out.dtype, out.shape, out.stride()), quantize)
    if copies:
        return _group_norm(what, x.contiguous() if copies & 1 else x, groups, weight.contiguous() if copies & 2 else weight,
                           bias.contiguous() if copies & 4 else bias, eps, activation, out, quantize)
    y = q = s = qp = sp = yp = None
    if quantize:
        rows, C = x.numel() // x.shape[-1], x.shape[-1]
        q, s = _fp8_buffers(x, rows, C, rows, True)
        qp, sp = q.data_ptr(), s.data_ptr()
    else:
        y = x.new_empty(x.shape) if out is None else out
        yp = y.data_ptr()
    if sizes is not None:
        ws = x.new_empty(n, dtype=torch.float32) if n > 0 else None
        st = _lib(index).ic_group_norm(
            x.data_ptr(), None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(), eps, yp, qp, sp,
            None if ws is None else ws.data_ptr(), sizes, _raw_stream(index))
        if st:
            L.check(st, "ic_group_norm")
    return y if not quantize else (q.view(x.shape), s.view(*x.shape[:-1], s.shape[1]))


def group_norm(
    x: torch.Tensor,
    groups: int,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    eps: float = 1e-5,
    activation: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` over all positions and
    the ``C // groups`` channels of each group of each sample, in fp32, one
    rounding.

    ``x`` [B, ..., C] (fp16 / bf16) has its channels last, e.g. [B, H, W, C] or
    [B, L, C]; a [B, C, H, W] tensor in ``torch.channels_last`` format comes as
    ``x.permute(0, 2, 3, 1)``, without a copy; one with channels first is copied.  ``weight`` and ``bias`` [C] are
    fp16, bf16 or fp32 (None: ones, zeros), ``activation`` 0 none, 1 SiLU, 2 GELU
    (erf), 3 GELU (tanh) as in :func:`gemm_a8`.  Returns a contiguous tensor;
    ``out`` may be ``x`` itself, but overlap it in no other way.  Up to 8192
    channels.
    """
    return _group_norm("group_norm", x, groups, weight, bias, eps, activation, out, False)


def fused_groupnorm_quantize(
    x: torch.Tensor,
    groups: int,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    eps: float = 1e-5,
    activation: int = 0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`group_norm` whose result goes to e4m3 blocks of 128 channels in the
    same pass: ``(q, s)`` as :func:`quantize_fp8_block` returns them, for
    :func:`gemm_fp8_block`.  Quantised from the fp32 values, without a rounding to
    ``x``'s type in between."""
    return _group_norm("fused_groupnorm_quantize", x, groups, weight, bias, eps, activation, None, True)


def device_error(clear: bool = True, device: torch.device | int | None = None) -> int:
    """Error code of ``device`` (default: the current one): 1 = a bounded wait
    timed out, 2 = a position or adapter id out of its range.  Where both
    happened 1 is reported first; ``clear`` takes out what is reported."""
    with torch.cuda.device(device):
        return L.read_device_error(clear)


__all__ = [
    "TRITON_AVAILABLE", "TRITON_INT4_UNPACK", "TRITON_INT8_GEMM", "TRITON_INT4_INT8_UNPACK",
    "TRITON_DYNQUANT", "TRITON_W4A8_GEMM", "TRITON_FUSED_QGD", "USE_FUSED_W8A8", "USE_CUDA_GRAPHS",
    "B200_AVAILABLE", "B200_LIBRARY_LOADED",
    "dynamic_quantize_activation", "fused_int8_gemm_dequant", "int8_gemm_int8out", "quantize_weight", "lokr_add",
    "fused_quant_int8_gemm_dequant",
    "fused_w4a8_gemm_dequant", "unpack_int4_to_int8", "unpack_int4_to_float16",
    "prep_quantize", "gemm_a8", "gemm_w4a16", "repack_int4", "lowrank_down", "lowrank_add", "device_error",
    "fused_layernorm_quantize", "fused_rmsnorm_quantize",
    "qk_norm_rope", "cross_attention", "lora_batched",
    "quantize_fp8_block", "gemm_fp8_block", "group_norm", "fused_groupnorm_quantize",
]
