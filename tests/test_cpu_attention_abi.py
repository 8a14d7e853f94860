"""Host side of the attention-side operators without a GPU: workspace sizes and
the refusals of the C entry points, all before any CUDA call."""

import ctypes

import pytest

from _pkg import load

L = load("_lib")
P = ctypes.c_void_p(256)      # aligned stand-in pointers: never used
ODD = ctypes.c_void_p(264)
S12 = ctypes.c_int64 * 12


def strides(*changes):
    s = [64 * 4 * 16, 64 * 4, 64] * 4
    for i, v in changes:
        s[i] = v
    return S12(*s)


def qk(**kw):
    a = dict(q=P, q_out=P, H=4, k=P, k_out=P, Hk=4, dtype=0, B=2, L=16, D=64, strides=strides(), qg=None, kg=None,
             eps=1e-6, layout=0, rot=64, cos=P, sin=P, rows=16, pos=None, stream=None)
    a.update(kw)
    return L.lib().ic_qk_norm_rope(*a.values())


def attn(**kw):
    a = dict(q=P, k=P, v=P, out=P, dtype=1, B=2, Lq=16, Lk=16, H=4, Hk=4, D=64, strides=strides(), scale=1.0, lens=None,
             mask=None, kind=0, ld=0, ws=P, elems=1 << 40, stream=None)
    a.update(kw)
    return L.lib().ic_cross_attention(*a.values())


def lora(**kw):
    a = dict(x=P, dtype=0, M=8, K=64, ldx=64, down=P, up=P, R=8, n=2, ids=P, rows=1, scales=None, base=P, ldb=32, out=P,
             N=32, ldo=32, ws=P, elems=1 << 40, stream=None)
    a.update(kw)
    return L.lib().ic_lora_batched(*a.values())


def refused(status, code, text):
    assert status == code
    assert text in L.lib().ic_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=2), 1, "dtype"), (dict(dtype=-1), 1, "dtype"), (dict(B=-1), 1, "negative"), (dict(D=36), 2, "multiple of 8"),
    (dict(D=264), 2, "up to 256"), (dict(D=0), 2, "multiple of 8"), (dict(rot=66), 1, "rot"), (dict(rot=3), 1, "rot"),
    (dict(rot=-2), 1, "rot"), (dict(layout=2), 1, "layout"), (dict(strides=None), 1, "strides"), (dict(q=None), 1, "NULL"),
    (dict(k_out=None), 1, "NULL"), (dict(cos=None), 1, "tables"), (dict(rows=15), 1, "table rows"),
    (dict(rows=0, pos=P), 1, "empty"), (dict(q=ODD), 1, "aligned"), (dict(strides=strides((1, 260))), 1, "aligned"),
    (dict(strides=strides((11, 65))), 1, "aligned"), (dict(qg=ODD), 1, "aligned"), (dict(B=1 << 30, L=1 << 30), 2, "rows"),
    (dict(H=1 << 20), 2, "heads"),
])
def test_qk_refusals(change, code, text):
    if "rows" in change and change.get("pos") is None and text == "empty":
        change["pos"] = P
    if "L" in change:
        change.update(rows=1 << 40)
    refused(qk(**change), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=2), 1, "dtype"), (dict(B=-1), 1, "bad sizes"), (dict(H=6), 1, "bad sizes"), (dict(Hk=0), 1, "bad sizes"),
    (dict(D=136), 2, "up to 128"), (dict(D=20), 2, "multiple of 8"), (dict(kind=5, mask=P, ld=16), 1, "mask kind"),
    (dict(kind=-1), 1, "mask kind"), (dict(kind=1), 1, "NULL"), (dict(kind=1, mask=P, ld=15), 1, "ld_mask"),
    (dict(q=None), 1, "NULL"), (dict(v=None), 1, "NULL"), (dict(strides=None), 1, "strides"), (dict(k=ODD), 1, "aligned"),
    (dict(strides=strides((8, 20))), 1, "aligned"), (dict(Lq=1, Lk=9000, ws=None), 1, "workspace"),
    (dict(Lq=1, Lk=9000, elems=8), 1, "workspace"), (dict(kind=1, mask=P, ld=16, elems=0), 1, "workspace"),
    (dict(kind=1, mask=P, ld=16, ws=ctypes.c_void_p(260)), 1, "workspace"), (dict(Lq=1 << 40), 2, "too many"),
    (dict(B=1 << 29, Lq=1 << 20), 2, "too many"),
])
def test_attention_refusals(change, code, text):
    refused(attn(**change), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=2), 1, "dtype"), (dict(M=-1), 1, "bad M"), (dict(K=0), 1, "bad M"), (dict(n=0), 1, "bad M"),
    (dict(R=0), 2, "rank"), (dict(R=257), 2, "rank"), (dict(M=1 << 40), 2, "too large"), (dict(rows=0), 1, "rows_per_id"),
    (dict(ldx=63), 1, "stride"), (dict(ldb=31), 1, "stride"), (dict(ldo=31), 1, "stride"), (dict(x=None), 1, "NULL"),
    (dict(ids=None), 1, "NULL"), (dict(ws=None), 1, "workspace"), (dict(elems=3), 1, "workspace"),
])
def test_lora_refusals(change, code, text):
    refused(lora(**change), code, text)


def test_nothing_to_do_needs_no_pointers():
    assert qk(B=0, q=None, q_out=None, k=None, k_out=None) == 0
    assert qk(H=0, Hk=0, q=None, q_out=None, k=None, k_out=None) == 0
    assert attn(Lq=0, q=None, k=None, v=None, out=None, ws=None) == 0
    assert lora(M=0, x=None, out=None, ws=None) == 0
    assert lora(N=0, ldo=0, ldb=0, x=None, out=None, ws=None) == 0


def test_workspaces():
    lib = L.lib()
    assert lib.ic_cross_attention_workspace(0, 5, 5, 2, 2, 64, 0) == 0
    assert lib.ic_cross_attention_workspace(1, 1, 10, 2, 3, 64, 0) == -1
    assert lib.ic_cross_attention_workspace(4, 4096, 512, 24, 24, 128, 0) == 0
    # a mask's bias rows, padded to 128 keys, and the ends
    assert lib.ic_cross_attention_workspace(3, 4096, 300, 24, 24, 64, 1) == 3 * 384 + 4
    assert lib.ic_cross_attention_workspace(1, 1, 8192, 8, 8, 128, 0) % (8 * 130) == 0
    assert lib.ic_lora_batched_workspace(0, 64, 64, 8, 1) == 0
    assert lib.ic_lora_batched_workspace(8, 64, 64, 0, 1) == -1
    assert lib.ic_lora_batched_workspace(8, 64, 64, 12, 1) >= 8 * 16
