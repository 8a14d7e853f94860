"""Head norm + rotation, cross attention and many-request adapters against
plain 64-bit forms, at the sizes, masks, strides and orders where they can go
wrong.

Bounds.  With u the unit roundoff of the tensors' type (2^-11 fp16, 2^-8
bf16), an output y that is computed in fp32 and rounded once is within u |y| of
the exact value, plus the fp32 part; fp16 values below 2^-14 round by up to
2^-25.  Attention also rounds each weight p_j to that type for the product
with v, which adds at most u sum_j p_j |v_j|; its fp32 part (scores, exp2) is
below 3e-5 of the same sum.  The adapters' fp32 sums are within 2^-18 of the
sum of the absolute products (K up to 5120), and the split of mid into two
16-bit values within 2^-16 of |mid| |up|.
"""

import math

import pytest
import torch

from _pkg import load

pytestmark = pytest.mark.gpu
rt = load("_b200_runtime") if torch.cuda.is_available() else None

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DTYPES = [torch.float16, torch.bfloat16]
f64 = torch.float64


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def check(got, want, tol):
    assert torch.isfinite(want).all()
    assert torch.isfinite(got.double()).all()
    over = (got.double() - want).abs() - tol
    assert over.max().item() <= 0, f"{over.max().item():.3e} past the bound ({(over > 0).sum().item()} values)"


# ── head norm + rotation ─────────────────────────────────────────────────────

def qk_reference(x, gamma, cos, sin, layout, positions, eps):
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if gamma is not None:
        x = x * gamma.double()
    if cos is None:
        return x
    B, L = x.shape[:2]
    pos = torch.arange(L, device=x.device).expand(B, L) if positions is None else positions.long()
    c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]
    half = cos.shape[1]
    y = x.clone()
    for i in range(half):
        a, b = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
        y[..., a] = x[..., a] * c[..., i] - x[..., b] * s[..., i]
        y[..., b] = x[..., b] * c[..., i] + x[..., a] * s[..., i]
    return y


def qk_tolerance(want, dtype):
    return U[dtype] * want.abs() + TINY[dtype] + 2e-6 * want.abs().amax(-1, keepdim=True)


def tables(rows, rot, g):
    a = torch.rand(rows, rot // 2, device="cuda", generator=g) * 2 * math.pi
    return a.cos(), a.sin()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,L,H,Hk,D,rot,pos", [
    (1, 1, 1, 1, 8, 8, False), (1, 1, 32, 8, 128, 128, True), (2, 7, 3, 1, 40, 20, True), (3, 33, 9, 5, 64, 64, False),
    (1, 130, 24, 24, 128, 64, False), (2, 5, 17, 2, 72, 36, True), (1, 19, 4, 4, 96, 48, True), (1, 9, 2, 2, 256, 256, False),
    (2, 3, 8, 1, 80, 2, True), (1, 12, 5, 3, 256, 96, True),
])
def test_qk_norm_rope(B, L, H, Hk, D, rot, pos, layout, dtype):
    g = gen(B * 1000 + L + D)
    qkv = normal(g, B, L, (H + 2 * Hk) * D, dtype=dtype, std=1.7)
    q = qkv[..., :H * D].view(B, L, H, D)
    k = qkv[..., H * D:(H + Hk) * D].view(B, L, Hk, D)
    gq, gk = normal(g, D), normal(g, D)
    cos, sin = tables(L + 50, rot, g)
    positions = torch.randint(0, L + 50, (B, L), device="cuda", generator=g) if pos else None
    yq, yk = rt.qk_norm_rope(q, k, q_gamma=gq, k_gamma=gk, cos=cos, sin=sin, layout=layout, positions=positions, eps=1e-5)
    for y, x, gamma in ((yq, q, gq), (yk, k, gk)):
        want = qk_reference(x, gamma, cos, sin, layout, positions, 1e-5)
        assert y.is_contiguous() and y.dtype == dtype
        check(y, want, qk_tolerance(want, dtype))


@pytest.mark.parametrize("layout,rot", [("interleaved", 64), ("half", 64), ("half", 36)])
def test_qk_norm_rope_in_place_and_alone(layout, rot):
    """The output over the input (a view of the projection) gives the same
    bits; queries alone give what they give beside keys."""
    g = gen(5)
    qkv = normal(g, 2, 37, 11 * 64, dtype=torch.bfloat16)
    q, k = qkv[..., :8 * 64].view(2, 37, 8, 64), qkv[..., 8 * 64:10 * 64].view(2, 37, 2, 64)
    v = qkv[..., 10 * 64:].clone()
    cos, sin = tables(37, rot, g)
    yq, yk = rt.qk_norm_rope(q, k, cos=cos, sin=sin, layout=layout)
    assert torch.equal(rt.qk_norm_rope(q, cos=cos, sin=sin, layout=layout), yq)
    assert torch.equal(rt.qk_norm_rope(k, cos=cos, sin=sin, layout=layout), yk)
    zq, zk = rt.qk_norm_rope(q, k, cos=cos, sin=sin, layout=layout, q_out=q, k_out=k)
    assert zq.data_ptr() == q.data_ptr() and torch.equal(zq, yq) and torch.equal(zk, yk)
    assert torch.equal(qkv[..., 10 * 64:], v)


@pytest.mark.parametrize("view", ["transposed", "odd_stride", "odd_start"])
def test_qk_norm_rope_layouts_in_memory(view):
    g = gen(6)
    if view == "transposed":      # heads before tokens in memory
        q = normal(g, 2, 4, 21, 64, dtype=torch.float16).transpose(1, 2)
    elif view == "odd_stride":    # rows of 65 elements: copied before the kernel
        q = normal(g, 2, 21, 4, 65, dtype=torch.float16)[..., :64]
    else:
        q = normal(g, 2 * 21 * 4 * 64 + 3, dtype=torch.float16)[3:].view(2, 21, 4, 64)
    cos, sin = tables(21, 64, g)
    want = qk_reference(q, None, cos, sin, "half", None, 1e-6)
    check(rt.qk_norm_rope(q, cos=cos, sin=sin, layout="half"), want, qk_tolerance(want, torch.float16))


def test_qk_norm_only_zero_rows_and_empty():
    g = gen(7)
    q = normal(g, 1, 6, 3, 64, dtype=torch.float16)
    q[0, 2] = 0
    want = qk_reference(q, None, None, None, "half", None, 1e-6)
    y = rt.qk_norm_rope(q)
    check(y, want, qk_tolerance(want, torch.float16))
    assert (y[0, 2] == 0).all()
    assert rt.qk_norm_rope(q[:, :0]).shape == (1, 0, 3, 64)
    yq, yk = rt.qk_norm_rope(q, q[:, :, :0])
    assert torch.equal(yq, y) and yk.shape == (1, 6, 0, 64)


def test_qk_nan_and_inf_stay_in_their_head():
    g = gen(8)
    q = normal(g, 1, 4, 6, 64, dtype=torch.bfloat16)
    cos, sin = tables(4, 48, g)
    y = rt.qk_norm_rope(q, cos=cos, sin=sin, layout="half")
    q2 = q.clone()
    q2[0, 1, 2, 5] = math.nan
    q2[0, 3, 4, 60] = math.inf
    z = rt.qk_norm_rope(q2, cos=cos, sin=sin, layout="half")
    assert z[0, 1, 2].isnan().all()
    other = torch.ones(4, 6, dtype=torch.bool, device="cuda")
    other[1, 2] = other[3, 4] = False
    assert torch.equal(z[0][other], y[0][other])
    # x / inf: zeros beside the infinite element, NaN at it
    assert z[0, 3, 4, 60].isnan() and (z[0, 3, 4, :60] == 0).all()


def test_qk_position_outside_the_tables():
    """NaN for that token only, and the device error word; nothing is read."""
    g = gen(9)
    q = normal(g, 2, 3, 5, 128, dtype=torch.float16)
    cos, sin = tables(10, 128, g)
    pos = torch.tensor([[0, 10, 2], [-1, 9, 3]], device="cuda")
    assert rt.device_error() == 0
    y = rt.qk_norm_rope(q, cos=cos, sin=sin, positions=pos)
    assert rt.device_error() == 2 and rt.device_error() == 0
    bad = (pos < 0) | (pos > 9)
    assert y[bad].isnan().all()
    want = qk_reference(q, None, cos, sin, "interleaved", pos.clamp(0, 9), 1e-6)
    check(y[~bad], want[~bad], qk_tolerance(want[~bad], torch.float16))


def test_qk_refusals():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16, device="cuda")
    c = torch.zeros(4, 32, device="cuda")
    with pytest.raises(TypeError, match="float16/bfloat16"):
        rt.qk_norm_rope(q.float())
    with pytest.raises(ValueError, match="layout"):
        rt.qk_norm_rope(q, layout="pairs")
    with pytest.raises(ValueError, match="batch, tokens, heads"):
        rt.qk_norm_rope(q[0])
    with pytest.raises(ValueError, match="come together"):
        rt.qk_norm_rope(q, cos=c)
    with pytest.raises(ValueError, match="table rows"):
        rt.qk_norm_rope(q, cos=c[:3], sin=c[:3])
    with pytest.raises(ValueError, match="rot"):
        rt.qk_norm_rope(q, cos=c.repeat(1, 2), sin=c.repeat(1, 2))
    with pytest.raises(ValueError, match="gamma"):
        rt.qk_norm_rope(q, q_gamma=c[0])
    with pytest.raises(ValueError, match="positions"):
        rt.qk_norm_rope(q, cos=c, sin=c, positions=torch.zeros(1, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="k must be"):
        rt.qk_norm_rope(q, q[:, :3])
    with pytest.raises(RuntimeError, match="multiple of 8"):
        rt.qk_norm_rope(q[..., :36])
    with pytest.raises(RuntimeError, match="CUDA"):
        rt.qk_norm_rope(q.cpu())
    with pytest.raises(ValueError, match="out must"):
        rt.qk_norm_rope(q, q_out=q[:, :, :1].expand(1, 4, 2, 64))


# ── cross attention ──────────────────────────────────────────────────────────

def attention_reference(q, k, v, kv_lens=None, key_mask=None, scale=None):
    """(output, bound) in 64 bits, sample by sample and head by head."""
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Lq, H, D, dtype=f64, device="cuda")
    tol = torch.zeros_like(out)
    u, tiny = U[q.dtype], TINY[q.dtype]
    if key_mask is not None and key_mask.dim() == 1:
        key_mask = key_mask.expand(B, Lk)
    for b in range(B):
        seen = torch.arange(Lk, device="cuda") < (Lk if kv_lens is None else int(kv_lens[b]))
        add = torch.zeros(Lk, dtype=f64, device="cuda")
        if key_mask is not None:
            if key_mask.dtype == torch.bool:
                seen = seen & key_mask[b]
            else:
                seen = seen & (key_mask[b] != -math.inf)
                add = key_mask[b].double()
        if not seen.any():
            continue
        # a constant cancels in the softmax; taking it out first keeps 64 bits
        # exact where every mask value is a type's lowest (-3.4e38 + s is s lost)
        add = add - add[seen].max()
        for h in range(H):
            kk, vv = k[b, seen, h // (H // Hk)].double(), v[b, seen, h // (H // Hk)].double()
            s = q[b, :, h].double() @ kk.T * scale + add[seen]
            p = torch.softmax(s, -1)
            o = p @ vv
            out[b, :, h] = o
            tol[b, :, h] = (u + 3e-5) * (p @ vv.abs()) + u * o.abs() + tiny * (1 + vv.abs().sum(0))
    return out, tol


def attention_inputs(seed, B, Lq, Lk, H, Hk, D, dtype, qstd=1.0):
    g = gen(seed)
    q = normal(g, B, Lq, H, D, dtype=dtype, std=qstd)
    kv = normal(g, B, Lk, 2, Hk, D, dtype=dtype)
    return q, kv[:, :, 0], kv[:, :, 1], g


SHAPES = [
    (1, 1, 1, 1, 1, 8), (1, 1, 77, 8, 8, 64), (2, 1, 4100, 8, 2, 128), (3, 5, 1, 4, 2, 64), (1, 17, 130, 6, 3, 40),
    (2, 129, 77, 4, 4, 80), (1, 257, 333, 5, 1, 128), (2, 300, 512, 4, 2, 64), (1, 1000, 129, 3, 3, 96),
    (1, 64, 3001, 2, 1, 128), (1, 385, 1030, 2, 2, 128), (9, 2, 40, 33, 11, 32), (1, 700, 128, 7, 7, 64),
    (1, 129, 256, 4, 1, 72), (2, 513, 16, 2, 2, 128),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", SHAPES)
def test_cross_attention(B, Lq, Lk, H, Hk, D, dtype):
    q, k, v, _ = attention_inputs(1, B, Lq, Lk, H, Hk, D, dtype)
    want, tol = attention_reference(q, k, v)
    out = rt.cross_attention(q, k, v)
    assert out.is_contiguous() and out.dtype == dtype and rt.device_error() == 0
    check(out, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["lens", "bool", "add", "add_f32", "add_low", "add_inf", "lens_bool", "row_add"])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", [(4, 1, 300, 8, 2, 64), (3, 200, 77, 3, 3, 64), (4, 300, 520, 2, 1, 128),
                                            (3, 40, 2100, 2, 2, 80), (2, 600, 1500, 2, 2, 128)])
def test_cross_attention_masks(B, Lq, Lk, H, Hk, D, kind, dtype):
    """What is not seen holds NaN and infinities."""
    q, k, v, g = attention_inputs(2, B, Lq, Lk, H, Hk, D, dtype)
    lens = mask = None
    if "lens" in kind:
        lens = torch.tensor([Lk, 0, 1, Lk // 2 + 3][:B], device="cuda")
    if "bool" in kind:
        mask = torch.rand(B, Lk, device="cuda", generator=g) < 0.6
        mask[B - 1] = False
        mask[B - 1, Lk // 2] = True
        mask[0, -5:] = False
        if kind == "bool":
            mask[1] = False
    elif kind == "row_add":
        mask = normal(g, Lk, dtype=dtype)
        mask[::7] = -math.inf
    elif "add" in kind:
        mask = normal(g, B, Lk, dtype=torch.float32 if kind == "add_f32" else dtype, std=3.0)
        if kind == "add_low":
            mask[0] = torch.finfo(dtype).min        # every key at the lowest value
            mask[1, Lk // 3:] = torch.finfo(dtype).min
        if kind == "add_inf":
            mask[0] = -math.inf
            mask[1, ::2] = -math.inf
    seen = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
    if lens is not None:
        seen &= torch.arange(Lk, device="cuda") < lens[:, None]
    if mask is not None:
        seen &= (mask if mask.dtype == torch.bool else mask != -math.inf).expand(B, Lk)
    want, tol = attention_reference(q, k, v, lens, mask)
    k, v = k.clone(), v.clone()
    hidden = (~seen).nonzero()
    k[hidden[:, 0], hidden[:, 1]] = math.nan
    v[hidden[::2, 0], hidden[::2, 1]] = math.nan
    v[hidden[1::2, 0], hidden[1::2, 1]] = -math.inf
    out = rt.cross_attention(q, k, v, kv_lens=lens, key_mask=mask)
    check(out, want, tol)
    empty = ~seen.any(1)
    assert (out[empty] == 0).all()


@pytest.mark.parametrize("Lq", [1, 300])
def test_cross_attention_growing_scores(Lq):
    """Scores that rise by hundreds along the keys: every tile moves the
    running maximum."""
    B, Lk, H, D = 1, 900, 2, 64
    q, k, v, g = attention_inputs(3, B, Lq, Lk, H, H, D, torch.float16)
    ramp = torch.linspace(-300, 300, Lk, device="cuda")
    for mask in (ramp, ramp.flip(0), ramp[torch.randperm(Lk, device="cuda", generator=g)]):
        want, tol = attention_reference(q, k, v, None, mask)
        check(rt.cross_attention(q, k, v, key_mask=mask), want, tol)


@pytest.mark.parametrize("Lq,Lk", [(1, 200), (300, 200), (5, 4000)])
def test_cross_attention_large_scores_and_scale(Lq, Lk):
    q, k, v, _ = attention_inputs(4, 1, Lq, Lk, 2, 2, 128, torch.bfloat16, qstd=12.0)
    for scale in (None, 0.5, 0.0, -0.3):
        want, tol = attention_reference(q, k, v, scale=scale)
        # scores of a few hundred in fp32: 2^-24 of them, times ln 2, moves p
        check(rt.cross_attention(q, k, v, scale=scale), want, tol * 1.05)


def test_cross_attention_no_keys_no_queries():
    q, k, v, _ = attention_inputs(5, 2, 9, 4, 4, 2, 64, torch.float16)
    assert (rt.cross_attention(q, k[:, :0], v[:, :0]) == 0).all()
    assert (rt.cross_attention(q, k, v, kv_lens=torch.zeros(2, dtype=torch.int32, device="cuda")) == 0).all()
    assert rt.cross_attention(q[:, :0], k, v).shape == (2, 0, 4, 64)
    assert rt.cross_attention(q[:0], k[:0], v[:0]).shape == (0, 9, 4, 64)
    # lengths past the keys are the keys'
    full = rt.cross_attention(q, k, v)
    assert torch.equal(rt.cross_attention(q, k, v, kv_lens=torch.tensor([99, 4], device="cuda")), full)


@pytest.mark.parametrize("Lq", [1, 40, 300])
def test_cross_attention_nan_in_one_query_or_seen_key(Lq):
    q, k, v, _ = attention_inputs(6, 2, Lq, 150, 2, 2, 64, torch.bfloat16)
    plain = rt.cross_attention(q, k, v)
    q2 = q.clone()
    q2[1, Lq - 1, 1, 3] = math.nan
    got = rt.cross_attention(q2, k, v)
    assert got[1, Lq - 1, 1].isnan().all()
    got[1, Lq - 1, 1] = plain[1, Lq - 1, 1]
    assert torch.equal(got, plain)
    k2 = k.clone()
    k2[0, 149, 1, 0] = math.nan
    got = rt.cross_attention(q, k2, v)
    assert got[0, :, 1].isnan().all()
    got[0, :, 1] = plain[0, :, 1]
    assert torch.equal(got, plain)


@pytest.mark.parametrize("Lq", [3, 300])
def test_cross_attention_strides(Lq):
    g = gen(7)
    B, Lk, H, D = 2, 200, 4, 64
    q = normal(g, B, H, Lq, D, dtype=torch.float16).transpose(1, 2)        # heads first in memory
    k = normal(g, Lk, B, H, D, dtype=torch.float16).transpose(0, 1)        # tokens first
    v = normal(g, B, Lk, H, D + 1, dtype=torch.float16)[..., 1:]           # copied: odd strides
    out = torch.full((B, Lq, 2 * H, D), 7.0, dtype=torch.float16, device="cuda")
    want, tol = attention_reference(q, k, v)
    y = rt.cross_attention(q, k, v, out=out[:, :, ::2])
    assert y.data_ptr() == out.data_ptr()
    check(y, want, tol)
    assert (out[:, :, 1::2] == 7).all()
    # one sample's keys for the whole batch
    ke, ve = k[:1].expand(B, Lk, H, D), v[:1].expand(B, Lk, H, D)
    want, tol = attention_reference(q, ke, ve)
    check(rt.cross_attention(q, ke, ve), want, tol)


@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", [(1, 1, 8192, 4, 1, 128), (2, 500, 700, 3, 3, 64), (1, 100, 5000, 2, 2, 128)])
def test_cross_attention_same_bits_other_stream_and_graph(B, Lq, Lk, H, Hk, D):
    q, k, v, g = attention_inputs(8, B, Lq, Lk, H, Hk, D, torch.bfloat16)
    mask = torch.rand(B, Lk, device="cuda", generator=g) < 0.9
    first = rt.cross_attention(q, k, v, key_mask=mask)
    for _ in range(3):
        assert torch.equal(rt.cross_attention(q, k, v, key_mask=mask), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rt.cross_attention(q, k, v, key_mask=mask)
    side.synchronize()
    assert torch.equal(other, first)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(first)
    with torch.cuda.graph(graph):
        rt.cross_attention(q, k, v, key_mask=mask, out=out)
    out.zero_()
    graph.replay()
    assert torch.equal(out, first)
    # new inputs in the captured tensors
    q.mul_(-1)
    graph.replay()
    assert torch.equal(out, rt.cross_attention(q, k, v, key_mask=mask))
    torch.cuda.synchronize()


def test_cross_attention_refusals():
    q = torch.zeros(2, 4, 4, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(2, 6, 2, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(TypeError, match="one dtype"):
        rt.cross_attention(q, k.bfloat16(), k)
    with pytest.raises(TypeError, match="one dtype"):
        rt.cross_attention(q.float(), k.float(), k.float())
    with pytest.raises(ValueError, match="q must be"):
        rt.cross_attention(q, k, k[:, :5])
    with pytest.raises(ValueError, match="q must be"):
        rt.cross_attention(q, k[:1], k[:1])
    with pytest.raises(ValueError, match="heads"):
        rt.cross_attention(q, k[:, :, :1].expand(2, 6, 3, 64), k[:, :, :1].expand(2, 6, 3, 64))
    with pytest.raises(ValueError, match="kv_lens"):
        rt.cross_attention(q, k, k, kv_lens=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError, match="integers"):
        rt.cross_attention(q, k, k, kv_lens=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError, match="key_mask"):
        rt.cross_attention(q, k, k, key_mask=torch.zeros(2, 5, dtype=torch.bool, device="cuda"))
    with pytest.raises(TypeError, match="key_mask"):
        rt.cross_attention(q, k, k, key_mask=torch.zeros(2, 6, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="multiple of 8 up to 128"):
        rt.cross_attention(*(torch.zeros(1, 2, 2, 136, dtype=torch.float16, device="cuda"),) * 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        rt.cross_attention(q.cpu(), k, k)
    with pytest.raises(ValueError, match="out must"):
        rt.cross_attention(q, k, k, out=q[..., :32])


# ── adapters of many requests ────────────────────────────────────────────────

def lora_reference(x, down, up, ids, scales, base, rows):
    """(output, bound) in 64 bits; rows without an adapter keep base."""
    M, N = x.shape[0], up.shape[1]
    y = torch.zeros(M, N, dtype=f64, device="cuda") if base is None else base.double()
    tol = torch.zeros(M, N, dtype=f64, device="cuda")
    of_row = ids.long().repeat_interleave(rows)
    for a in range(down.shape[0]):
        r = (of_row == a).nonzero()[:, 0]
        s = 1.0 if scales is None else scales[a].double()
        xd, d, u = x[r].double(), down[a].double(), up[a].double()
        mid = xd @ d.T
        y[r] += s * (mid @ u.T)
        tol[r] += abs(s) * (2.0 ** -16 * (mid.abs() @ u.abs().T) + 2.0 ** -18 * ((xd.abs() @ d.abs().T) @ u.abs().T))
    return y, tol + U[x.dtype] * y.abs() + TINY[x.dtype]


def lora_inputs(seed, M, K, N, R, n, dtype):
    g = gen(seed)
    x, base = normal(g, M, K, dtype=dtype), normal(g, M, N, dtype=dtype)
    down = normal(g, n, R, K, dtype=dtype, std=K ** -0.5)
    up = normal(g, n, N, R, dtype=dtype, std=R ** -0.5)
    scales = torch.rand(n, device="cuda", generator=g) + 0.5
    return x, base, down, up, scales, g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,rows,K,N,R,n", [
    (1, 1, 8, 8, 1, 1), (1, 1, 512, 64, 16, 3), (16, 1, 1024, 520, 16, 8), (37, 1, 77, 33, 5, 4), (64, 1, 256, 264, 12, 40),
    (33, 11, 640, 96, 32, 2), (300, 100, 136, 1000, 24, 5), (2600, 650, 96, 72, 64, 3), (2500, 1, 264, 40, 20, 4),
    (700, 7, 1000, 300, 128, 6), (90, 3, 320, 136, 192, 3), (3000, 1500, 64, 344, 256, 2), (2777, 1, 61, 35, 9, 3),
    # from 4096 rows: tiles of 128 rows through shared memory, where the rows are aligned
    (4200, 1, 136, 200, 24, 5), (4230, 470, 1000, 136, 8, 3), (5120, 640, 72, 328, 64, 4), (4099, 4099, 520, 64, 16, 2),
    (4864, 2432, 2056, 104, 32, 2), (4100, 100, 64, 72, 40, 30), (4096, 64, 77, 200, 16, 3),
])
def test_lora_batched(M, rows, K, N, R, n, dtype):
    x, base, down, up, scales, g = lora_inputs(1, M, K, N, R, n, dtype)
    ids = torch.randint(-1, n, (M // rows,), device="cuda", generator=g)
    want, tol = lora_reference(x, down, up, ids, scales, base, rows)
    y = rt.lora_batched(x, down, up, ids, scales, base=base)
    check(y, want, tol)
    assert torch.equal(y[ids.repeat_interleave(rows) < 0], base[ids.repeat_interleave(rows) < 0])
    # the deltas alone, scale 1
    want, tol = lora_reference(x, down, up, ids, None, None, rows)
    check(rt.lora_batched(x, down, up, ids), want, tol)
    # over the base
    z = rt.lora_batched(x, down, up, ids, scales, base=base, out=base)
    assert z.data_ptr() == base.data_ptr() and torch.equal(z, y)


@pytest.mark.parametrize("M,rows", [(48, 1), (2600, 1300), (2600, 1), (4200, 1), (4500, 150), (5200, 1300)])
def test_lora_requests_do_not_touch_each_other(M, rows):
    """NaN and infinities in one request's rows or adapter reach no other
    request, and an id that names no adapter only its own rows."""
    dtype = torch.float16
    x, base, down, up, scales, g = lora_inputs(2, M, 200, 88, 16, 4, dtype)
    ids = torch.randint(-1, 3, (M // rows,), device="cuda", generator=g)
    ids[0], ids[1] = 1, 2
    clean = rt.lora_batched(x, down, up, ids, scales, base=base)
    of_row = ids.repeat_interleave(rows)
    down2, up2 = down.clone(), up.clone()
    down2[2, 3, 5] = math.nan
    up2[2, 7] = math.inf
    up2[3] = math.nan
    got = rt.lora_batched(x, down2, up2, ids, scales, base=base)
    assert not torch.isfinite(got[of_row == 2]).all()
    assert torch.equal(got[of_row != 2], clean[of_row != 2])
    x2 = x.clone()
    x2[M - 1] = math.nan
    got = rt.lora_batched(x2, down, up, ids, scales, base=base)
    assert torch.equal(got[:M - 1], clean[:M - 1])
    assert rt.device_error() == 0
    ids2 = ids.clone()
    ids2[1] = 4
    got = rt.lora_batched(x, down, up, ids2, scales, base=base)
    assert rt.device_error() == 2
    wrong = ids2.repeat_interleave(rows) == 4
    assert got[wrong].isnan().all() and torch.equal(got[~wrong], clean[~wrong])


def test_lora_fp16_range():
    """mid past fp16's range and far below it: the row's power of two keeps it."""
    M, K, N, R = 20, 64, 40, 16
    x, _, down, up, _, g = lora_inputs(3, M, K, N, R, 1, torch.float16)
    ids = torch.zeros(M, dtype=torch.int32, device="cuda")
    for s in (3e4, 1e-6):
        scales = torch.tensor([s], device="cuda")
        small_up = up if s < 1 else (up * 2.0 ** -14).half()
        want, tol = lora_reference(x * 8, down, small_up, ids, scales, None, 1)
        check(rt.lora_batched(x * 8, down, small_up, ids, scales), want, tol)


def test_lora_strides_batches_stream_and_graph():
    dtype = torch.bfloat16
    x, base, down, up, scales, g = lora_inputs(4, 60, 320, 160, 8, 3, dtype)
    ids = torch.tensor([2, -1, 0], device="cuda")
    plain = rt.lora_batched(x, down, up, ids, scales, base=base)
    # [batch, tokens, K] views of wider buffers
    wide = torch.zeros(3, 20, 328, dtype=dtype, device="cuda")
    wide[..., :320] = x.view(3, 20, 320)
    out = torch.full((60, 168), 5.0, dtype=dtype, device="cuda")
    y = rt.lora_batched(wide[..., :320], down, up, ids, scales, base=base.view(3, 20, 160),
                        out=out.view(3, 20, 168)[..., :160])
    assert y.shape == (3, 20, 160) and torch.equal(y.reshape(60, 160), plain) and (out[:, 160:] == 5).all()
    # rows at odd addresses take the element-wise loads: same sums
    odd = torch.zeros(60 * 321 + 1, dtype=dtype, device="cuda")[1:].view(60, 321)[:, :320]
    odd.copy_(x)
    assert torch.equal(rt.lora_batched(odd, down, up, ids, scales, base=base), plain)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rt.lora_batched(x, down, up, ids, scales, base=base)
    side.synchronize()
    assert torch.equal(other, plain)
    ids32 = ids.int()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = rt.lora_batched(x, down, up, ids32, scales, base=base)
    graph.replay()
    assert torch.equal(z, plain)
    ids32.copy_(torch.tensor([1, 1, -1]))   # other requests, same graph
    graph.replay()
    assert torch.equal(z, rt.lora_batched(x, down, up, ids32, scales, base=base))
    torch.cuda.synchronize()


def test_lora_refusals():
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    x, down, up = h(4, 64), h(2, 8, 64), h(2, 32, 8)
    with pytest.raises(TypeError, match="one dtype"):
        rt.lora_batched(x, down.bfloat16(), up, ids)
    with pytest.raises(ValueError, match="down must be"):
        rt.lora_batched(x, down, h(2, 32, 9), ids)
    with pytest.raises(ValueError, match="columns"):
        rt.lora_batched(h(4, 63), down, up, ids)
    with pytest.raises(ValueError, match="do not divide"):
        rt.lora_batched(x, down, up, ids[:3])
    with pytest.raises(TypeError, match="integers"):
        rt.lora_batched(x, down, up, ids.float())
    with pytest.raises(ValueError, match="scales"):
        rt.lora_batched(x, down, up, ids, torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="base must"):
        rt.lora_batched(x, down, up, ids, base=h(4, 31))
    with pytest.raises(ValueError, match="out must"):
        rt.lora_batched(x, down, up, ids, out=h(5, 32))
    with pytest.raises(RuntimeError, match="rank"):
        rt.lora_batched(x, h(2, 257, 64), h(2, 32, 257), ids)
    with pytest.raises(RuntimeError, match="CUDA"):
        rt.lora_batched(x, down, up, ids.cpu())
    assert rt.lora_batched(h(0, 64), down, up, ids[:0]).shape == (0, 32)


# ── together ─────────────────────────────────────────────────────────────────

def test_conditioned_attention_example():
    """INT8 projections with adapters, head norms and rotation, attention to
    ragged texts: within a few fp16 roundings (2^-11 each, four in a row) and
    the few INT8 steps that they flip (a step is 1/127 of a row's largest value,
    and one value in a thousand moves)."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(__file__), "..", "examples", "conditioned_attention.py")
    spec = importlib.util.spec_from_file_location("conditioned_attention", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main() < 4 * 2.0 ** -11


def test_torch_library_ops():
    load("_torch_ops")
    ops = torch.ops.intcrush_b200
    g = gen(20)
    q, k = normal(g, 2, 9, 4, 64, dtype=torch.float16), normal(g, 2, 9, 2, 64, dtype=torch.float16)
    cos, sin = tables(9, 64, g)
    got = ops.qk_norm_rope(q, k, None, None, cos, sin, "half", None, 1e-6)
    want = rt.qk_norm_rope(q, k, cos=cos, sin=sin, layout="half")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(ops.cross_attention(q, k, k, None, None, 0.125), rt.cross_attention(q, k, k))
    x, base, down, up, scales, _ = lora_inputs(21, 12, 64, 40, 8, 2, torch.float16)
    ids = torch.tensor([0, 1, -1], device="cuda")
    assert torch.equal(ops.lora_batched(x, down, up, ids, scales, base), rt.lora_batched(x, down, up, ids, scales, base=base))
    for op, args in ((ops.cross_attention, (q, k, k, None, None, 0.125)), (ops.lora_batched, (x, down, up, ids, None, None))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))
