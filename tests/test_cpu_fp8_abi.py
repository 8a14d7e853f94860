"""Host side of the 8-bit floating point linear without a GPU: workspace sizes
and the refusals of the C entry points, all before any CUDA call."""

import ctypes

import pytest

from _pkg import load

L = load("_lib")
P = ctypes.c_void_p(256)      # aligned stand-in pointers: never used
ODD = ctypes.c_void_p(264)
ODDER = ctypes.c_void_p(257)


def sizes(**kw):
    return (ctypes.c_int64 * len(kw))(*kw.values())


def call(entry, pointers, numbers, eps, kw):
    """The entry with what ``kw`` changes among pointers and sizes."""
    p, n = dict(pointers), dict(numbers)
    for k, v in kw.items():
        (p if k in p else n)[k] = v
    packed = None if n.pop("none", False) else sizes(**n)
    args = list(p.values())
    if eps is not None:
        args.insert(3, kw.get("eps", eps))
    n.pop("eps", None)
    return getattr(L.lib(), entry)(*args, packed, None)


def quant(**kw):
    return call("ic_quantize_fp8_block", dict(x=P, q=P, s=P),
                dict(dtype=0, M=8, K=300, ldx=300, rows=1, ldq=304, s_row=1, s_block=8), None, kw)


def gemm(**kw):
    return call("ic_gemm_fp8_block", dict(x=P, w=P, s_a=P, s_w=P, bias=P, out=P),
                dict(M=8, K=300, N=40, ldx=304, ldw=304, ldo=40, sa_row=1, sa_block=8, sw_row=3, sw_block=1, bias_dtype=0,
                     out_dtype=1), None, kw)


def norm(**kw):
    eps = kw.pop("eps", 1e-5)
    return call("ic_group_norm", dict(x=P, gamma=P, beta=P, y=P, q=None, s=None, ws=P),
                dict(dtype=0, B=2, L=16, C=64, x_batch=1024, x_row=64, groups=4, gamma_dtype=0, beta_dtype=2, activation=1,
                     y_batch=1024, y_row=64, ldq=0, s_row=0, s_block=0, elems=1 << 40), eps, kw)


def refused(status, code, text):
    assert status == code
    assert text in L.lib().ic_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    (dict(none=True), 1, "sizes"), (dict(dtype=1 << 32), 1, "dtype"),
    (dict(dtype=3), 1, "dtype"), (dict(dtype=-1), 1, "dtype"), (dict(M=-1), 1, "bad M"), (dict(K=0), 1, "bad M"),
    (dict(ldx=299), 1, "bad M"), (dict(rows=2), 1, "rows of a block"), (dict(x=None), 1, "NULL"), (dict(q=None), 1, "NULL"),
    (dict(s=None), 1, "NULL"), (dict(ldq=300), 1, "row stride"), (dict(ldq=312), 1, "row stride"), (dict(q=ODD), 1, "aligned"),
    (dict(x=ODDER), 1, "aligned"), (dict(dtype=2, x=ctypes.c_void_p(258)), 1, "aligned"), (dict(M=1 << 40), 2, "too many"),
    (dict(M=1 << 30, K=1 << 20, ldx=1 << 20, ldq=1 << 20), 2, "too many"), (dict(M=1 << 24, rows=128), 2, "too many"),
])
def test_quantize_refusals(change, code, text):
    refused(quant(**change), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(none=True), 1, "sizes"), (dict(out_dtype=1 << 32), 1, "f16"),
    (dict(M=-1), 1, "bad M"), (dict(N=-1), 1, "bad M"), (dict(K=0), 1, "bad M"), (dict(out_dtype=3), 1, "f16, bf16 or f32"),
    (dict(bias_dtype=-1), 1, "f16, bf16 or f32"), (dict(ldx=299), 1, "row stride"), (dict(ldw=288), 1, "row stride"),
    (dict(ldo=39), 1, "row stride"), (dict(x=None), 1, "NULL"), (dict(w=None), 1, "NULL"), (dict(s_a=None), 1, "NULL"),
    (dict(s_w=None), 1, "NULL"), (dict(out=None), 1, "NULL"), (dict(x=ODD), 1, "aligned"), (dict(w=ODD), 1, "aligned"),
    (dict(ldx=312), 1, "multiples of 16"), (dict(ldw=301), 1, "multiples of 16"), (dict(out=ODDER), 1, "aligned"),
    (dict(out_dtype=2, out=ctypes.c_void_p(258)), 1, "aligned"), (dict(bias=ODDER), 1, "aligned"), (dict(M=1 << 31), 2, "too large"),
    (dict(N=1 << 31, ldo=1 << 31), 2, "too large"), (dict(ldx=1 << 38), 2, "too large"), (dict(M=1 << 30, N=1 << 30, ldo=1 << 30), 2, "too large"),
])
def test_product_refusals(change, code, text):
    refused(gemm(**change), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(none=True), 1, "sizes"), (dict(activation=1 << 32), 1, "activation"),
    (dict(dtype=2), 1, "dtype"), (dict(B=-1), 1, "bad sizes"), (dict(L=-1), 1, "bad sizes"), (dict(C=0), 1, "bad sizes"),
    (dict(groups=0), 1, "bad sizes"), (dict(groups=5), 1, "bad sizes"), (dict(C=8256, x_row=8256, y_row=8256), 2, "8192"),
    (dict(B=1 << 30), 2, "too many"), (dict(L=1 << 40), 2, "too many"), (dict(B=1 << 20, L=1 << 20), 2, "too many"),
    (dict(gamma_dtype=3), 1, "gamma"), (dict(beta_dtype=-2), 1, "gamma"), (dict(activation=4), 1, "activation"),
    (dict(activation=-1), 1, "activation"), (dict(eps=-1.0), 1, "eps"), (dict(eps=float("nan")), 1, "eps"), (dict(x=None), 1, "NULL"),
    (dict(y=None), 1, "NULL"), (dict(q=P, s=P, ldq=64), 1, "one of"), (dict(y=None, q=P, ldq=64), 1, "NULL"),
    (dict(x_row=63), 1, "row stride"), (dict(y_row=63), 1, "row stride"), (dict(y_batch=0), 1, "overlaps"),
    (dict(x=ODDER), 1, "aligned"), (dict(beta=ctypes.c_void_p(258)), 1, "aligned"), (dict(y=None, q=ODD, s=P, ldq=64), 1, "aligned"),
    (dict(y=None, q=P, s=P, ldq=63), 1, "row stride"), (dict(L=200000, ws=None), 1, "workspace"),
    (dict(L=200000, elems=3), 1, "workspace"), (dict(L=200000, ws=ctypes.c_void_p(260)), 1, "workspace"),
])
def test_norm_refusals(change, code, text):
    refused(norm(**change), code, text)


def test_nothing_to_do_needs_no_pointers():
    assert quant(M=0, x=None, q=None, s=None) == 0
    assert gemm(M=0, x=None, w=None, s_a=None, s_w=None, out=None) == 0
    assert gemm(N=0, ldo=0, x=None, w=None, s_a=None, s_w=None, out=None) == 0
    assert norm(B=0, x=None, y=None, ws=None) == 0
    assert norm(L=0, x=None, y=None, ws=None) == 0


def test_workspaces():
    lib = L.lib()
    assert lib.ic_group_norm_workspace(0, 5, 64, 4, 0) == 0
    assert lib.ic_group_norm_workspace(2, 5, 64, 5, 0) == -1
    assert lib.ic_group_norm_workspace(2, 256, 1280, 32, 0) == 0      # kept in shared memory
    assert lib.ic_group_norm_workspace(2, 256, 1280, 32, 1) == 0
    n = lib.ic_group_norm_workspace(3, 1 << 20, 128, 32, 0)
    assert n > 3 and (n - 3) % (2 * 3 * 32) == 0     # statistics of runs of rows, tiles taken
