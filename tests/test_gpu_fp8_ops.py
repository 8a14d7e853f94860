"""Block quantisation, the e4m3 product and the group norm against plain 64-bit
forms, at the sizes, strides and values where they can go wrong.

Bounds.  Quantisation is exact: scale and quotient are single IEEE operations.
With u the unit roundoff of the output type (2^-11 fp16, 2^-8 bf16, 2^-24
fp32), a product computed in fp32 and rounded once is within u |y| of the exact
value, plus its fp32 part: the tensor core's sums of 128 and the KB scaled
additions, below (2^-18 + (KB + 4) 2^-24) of the sum of absolute products; fp16
values below 2^-14 round by up to 2^-25.  Group norm: a thread's sums run over at
most 128 rows here, so that the mean is off by at most 2^-17 of the largest
distance R from it, and the sum of squares by 2^-16 of itself; both are joined
over few hundred entries in trees.  The mean itself is held in fp32, by a
thread, a CTA, a cluster and a sample: four times 2^-24 |mean| (what is summed are
differences from one of them).  With h = (x - mean) / std gamma that is
|gamma| / std (2^-16 R + 2^-22 |mean|) + 2^-16 |h| before the activation, whose slope is at most
1.13 and whose own error is below 2^-18 (1 + |h|).  e4m3 rounds by half a
step: 2^-4 of the value, or 2^-10 scales below 2^-6.
"""

import math

import pytest
import torch

from _pkg import load

pytestmark = pytest.mark.gpu
rt = load("_b200_runtime") if torch.cuda.is_available() else None

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}
HALF = [torch.float16, torch.bfloat16]
ALL = [torch.float16, torch.bfloat16, torch.float32]
f64 = torch.float64
E4M3 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def check(got, want, tol):
    assert torch.isfinite(want).all()
    assert torch.isfinite(got.double()).all()
    over = (got.double() - want).abs() - tol
    assert over.max().item() <= 0, f"{over.max().item():.3e} past the bound ({(over > 0).sum().item()} values)"


def same(a, b):
    """Equal as values, NaN with NaN."""
    return torch.equal(torch.nan_to_num(a.float(), nan=1e30), torch.nan_to_num(b.float(), nan=1e30)) and torch.equal(
        a.float().isnan(), b.float().isnan())


# ── quantisation ─────────────────────────────────────────────────────────────

def quantize_reference(x, rows):
    """On the CPU, in fp32 with IEEE division."""
    x = x.detach().cpu().float()
    M, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % 128, 0, -M % rows)).view(-(-M // rows), rows, -(-K // 128), 128)
    top = b.abs().amax((1, 3))
    s = torch.where(top < 1e-8, torch.tensor(1e-8), top) / torch.full_like(top, 448.0)
    q = b / s[:, None, :, None]
    return q.to(E4M3).reshape(-1, b.shape[2] * 128)[:M, :K], s


def check_quantized(q, s, x, rows):
    wq, ws = quantize_reference(x, rows)
    assert q.dtype is E4M3 and s.dtype is torch.float32
    assert same(s.cpu(), ws)
    assert same(q.cpu(), wq)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 5120), (3, 128), (5, 129), (16, 127), (17, 256), (33, 1000), (127, 301), (128, 136),
                                 (257, 2600), (1000, 384), (2000, 1288), (300, 14336)])
def test_quantize(M, K, rows, dtype):
    g = gen(M + 31 * K)
    x = normal(g, M, K, dtype=dtype)
    x[:, ::37] *= 20
    check_quantized(*rt.quantize_fp8_block(x, rows=rows), x, rows)


@pytest.mark.parametrize("dtype", HALF)
def test_quantize_every_quotient(dtype):
    """Every value of a 16-bit type over the scales of every significand that a
    block's largest value can have: the corrected quotients round as IEEE
    division does."""
    bits = torch.arange(2 ** 15, dtype=torch.int32)
    values = bits.to(torch.int16).view(dtype)
    values = values[torch.isfinite(values)].cuda()
    one = torch.arange(2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    tops = one[(one >= 1) & (one < 2)].cuda()
    small = values[values < 2]
    small = small[small > 2.0 ** -18]
    pad = -len(small) % 127
    small = torch.cat([small, small.new_zeros(pad)]).view(-1, 127)
    for top in tops.split(64):
        x = torch.cat([torch.minimum(small[None].expand(len(top), -1, -1), top[:, None, None]),
                       top[:, None, None].expand(-1, small.shape[0], 1)], -1).reshape(-1, 128)
        q, s = rt.quantize_fp8_block(x)
        want_s = x.float().amax(1, keepdim=True) / torch.full((len(x), 1), 448.0, device="cuda")
        assert torch.equal(s, want_s)
        assert torch.equal(q.float(), (x.float() / want_s).to(E4M3).float())


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_zeros_tiny_and_not_finite(rows, dtype):
    x = normal(gen(3), 256, 640, dtype=dtype)
    x[0:128, 0:128] = 0
    x[0:128, 128:256] *= 1e-6 if dtype == torch.float16 else 1e-12
    x[5, 300] = math.inf
    x[6, 400] = math.nan
    x[7, 401] = -math.inf
    x[130, 130] = -math.inf
    x[200, 639] = math.nan
    check_quantized(*rt.quantize_fp8_block(x, rows=rows), x, rows)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("view", ["columns", "odd_start", "transposed", "every_other", "expanded"])
def test_quantize_layouts(view, rows):
    g = gen(4)
    if view == "columns":
        x = normal(g, 130, 700, dtype=torch.bfloat16)[:, 64:64 + 304]
    elif view == "odd_start":
        x = normal(g, 130 * 304 + 3, dtype=torch.bfloat16)[3:].view(130, 304)
    elif view == "transposed":
        x = normal(g, 304, 130, dtype=torch.bfloat16).t()
    elif view == "every_other":
        x = normal(g, 260, 304, dtype=torch.bfloat16)[::2]
    else:
        x = normal(g, 1, 304, dtype=torch.bfloat16).expand(130, -1)
    check_quantized(*rt.quantize_fp8_block(x, rows=rows), x, rows)


def test_quantize_leading_dimensions_and_padding():
    x = normal(gen(5), 2, 3, 5, 300, dtype=torch.float16)
    q, s = rt.quantize_fp8_block(x)
    assert q.shape == x.shape and s.shape == (2, 3, 5, 3)
    check_quantized(q.reshape(-1, 300), s.reshape(-1, 3), x.view(-1, 300), 1)
    assert q.stride(-2) == 304     # rows filled up to 16 bytes, with zeros
    rows = torch.as_strided(q.view(torch.uint8), (30, 304), (304, 1))
    assert (rows[:, 300:] == 0).all()
    q1, s1 = rt.quantize_fp8_block(x[0, 0, 0])
    assert q1.shape == (300,) and s1.shape == (3,) and torch.equal(q1.float(), q[0, 0, 0].float())
    q0, s0 = rt.quantize_fp8_block(x[:, :0])
    assert q0.shape == (2, 0, 5, 300) and s0.shape == (2, 0, 5, 3)


def test_quantize_far_rows():
    """Offsets past 2^31 elements, and past 2^32."""
    x = torch.zeros(34000, 1 << 17, dtype=torch.float16, device="cuda")
    x[-1, -128:] = torch.arange(128, device="cuda")
    x[20000, 5] = -3
    q, s = rt.quantize_fp8_block(x)
    check_quantized(q[-1:], s[-1:], x[-1:], 1)
    check_quantized(q[20000:20001], s[20000:20001], x[20000:20001], 1)
    assert q[-2].float().abs().max() == 0


# ── product ──────────────────────────────────────────────────────────────────

def operands(g, M, K, N):
    x, w = normal(g, M, K), normal(g, N, K, std=K ** -0.5)
    x[:, ::53] *= 15
    return rt.quantize_fp8_block(x), rt.quantize_fp8_block(w, rows=128)


def product_reference(x, w, s_w, s_a, bias):
    """Exact value and the sum of the absolute products."""
    N, K = w.shape
    xd = x.to(f64) * s_a.to(f64).repeat_interleave(128, 1)[:, :K]
    wd = w.to(f64) * s_w.to(f64).repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y, size = xd @ wd.T, xd.abs() @ wd.abs().T
    if bias is not None:
        y, size = y + bias.to(f64), size + bias.to(f64).abs()
    return y, size


def product_tolerance(want, size, K, dtype):
    fp32 = (2.0 ** -18 + (-(-K // 128) + 4) * 2.0 ** -24) * size
    return U[dtype] * (want.abs() + fp32) + fp32 + TINY[dtype]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("M,K,N,bias", [
    (1, 1, 1, None), (1, 16, 8, torch.float32), (1, 5120, 640, torch.float16), (2, 128, 128, None), (7, 300, 129, torch.bfloat16),
    (31, 257, 1000, None), (64, 4096, 200, torch.float32), (127, 640, 256, torch.float16), (128, 2048, 384, None),
    (129, 130, 513, torch.bfloat16), (200, 1111, 77, torch.float32), (1000, 384, 1111, torch.float16), (513, 8200, 264, None),
    (4096, 128, 136, None), (3, 264, 14336, torch.bfloat16),
])
def test_product(M, K, N, bias, dtype):
    g = gen(M + 7 * K + 13 * N)
    (x, s_a), (w, s_w) = operands(g, M, K, N)
    b = None if bias is None else normal(g, N, dtype=bias)
    y = rt.gemm_fp8_block(x, w, s_w, s_a, bias=b, out_dtype=dtype)
    assert y.shape == (M, N) and y.dtype == dtype and y.is_contiguous()
    want, size = product_reference(x, w, s_w, s_a, b)
    check(y, want, product_tolerance(want, size, K, dtype))
    assert rt.device_error() == 0


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("M,K,N", [(4608, 520, 4096), (4609, 1000, 4111), (2048, 128, 10240), (20000, 200, 300), (2300, 1, 9000)])
def test_product_of_many_tiles(M, K, N, dtype):
    g = gen(M + K)
    (x, s_a), (w, s_w) = operands(g, M, K, N)
    b = normal(g, N, dtype=torch.bfloat16)
    y = rt.gemm_fp8_block(x, w, s_w, s_a, bias=b, out_dtype=dtype)
    want, size = product_reference(x, w, s_w, s_a, b)
    check(y, want, product_tolerance(want, size, K, dtype))
    assert torch.equal(y, rt.gemm_fp8_block(x, w, s_w, s_a, bias=b, out_dtype=dtype))
    assert rt.device_error() == 0


@pytest.mark.parametrize("M,N", [(5, 300), (300, 520), (4500, 4100)])
def test_product_layouts(M, N):
    """Scales and operands in other layouts, outputs between other columns."""
    K = 390
    g = gen(M)
    (x, s_a), (w, s_w) = operands(g, M, K, N)
    y = rt.gemm_fp8_block(x, w, s_w, s_a, out_dtype=torch.float16)
    assert s_a.stride() != s_a.contiguous().stride() or M == 1
    assert torch.equal(rt.gemm_fp8_block(x.contiguous(), w.contiguous(), s_w.t().contiguous().t(), s_a.contiguous(),
                                         out_dtype=torch.float16), y)
    wide = torch.zeros(M, 2 * K + 58, dtype=torch.uint8, device="cuda").view(E4M3)
    far = wide[:, 17:17 + K]            # rows that do not start at 16 bytes
    far.copy_(x)
    assert torch.equal(rt.gemm_fp8_block(far, w, s_w, s_a, out_dtype=torch.float16), y)
    near = torch.full((M, 512), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
    near[:, 64:64 + K] = x              # NaN behind and before the values
    assert torch.equal(rt.gemm_fp8_block(near[:, 64:64 + K], w, s_w, s_a, out_dtype=torch.float16), y)
    for lo, pad in ((0, 8), (8, 24), (3, 7), (1, 0)):
        buf = torch.full((M, N + lo + pad), -7.0, dtype=torch.float16, device="cuda")
        out = buf[:, lo:lo + N]
        assert rt.gemm_fp8_block(x, w, s_w, s_a, out=out) is out
        assert torch.equal(out, y)
        assert (buf[:, :lo] == -7).all() and (buf[:, lo + N:] == -7).all()


def test_product_rows_behind_the_last_are_left():
    g = gen(9)
    (x, s_a), (w, s_w) = operands(g, 70, 256, 200)
    for M in (1, 33, 70):
        buf = torch.full((80, 200), -7.0, dtype=torch.float32, device="cuda")
        rt.gemm_fp8_block(x[:M], w, s_w, s_a[:M], out=buf[:M])
        assert (buf[M:] == -7).all() and not (buf[:M] == -7).any()


def test_product_leading_dimensions_and_empty():
    g = gen(10)
    (x, s_a), (w, s_w) = operands(g, 30, 256, 72)
    y = rt.gemm_fp8_block(x, w, s_w, s_a)
    got = rt.gemm_fp8_block(x.view(2, 3, 5, 256), w, s_w, s_a.view(2, 3, 5, 2))
    assert got.shape == (2, 3, 5, 72) and torch.equal(got.view(30, 72), y)
    assert torch.equal(rt.gemm_fp8_block(x[3], w, s_w, s_a[3]), y[3])
    assert rt.gemm_fp8_block(x[:0], w, s_w, s_a[:0]).shape == (0, 72)
    assert rt.gemm_fp8_block(x, w[:0], s_w[:0], s_a).shape == (30, 0)


@pytest.mark.parametrize("M", [6, 500])
def test_product_of_what_is_not_finite(M):
    """NaN and infinite blocks reach their own rows and features, and no others."""
    g = gen(11)
    xf, wf = normal(g, M, 384), normal(g, 260, 384, std=0.05)
    clean = rt.gemm_fp8_block(*[rt.quantize_fp8_block(xf)[0], rt.quantize_fp8_block(wf, rows=128)[0],
                                rt.quantize_fp8_block(wf, rows=128)[1], rt.quantize_fp8_block(xf)[1]])
    xf[2, 200] = math.nan
    xf[4, 3] = math.inf
    x, s_a = rt.quantize_fp8_block(xf)
    w, s_w = rt.quantize_fp8_block(wf, rows=128)
    y = rt.gemm_fp8_block(x, w, s_w, s_a)
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[[2, 4]] = True
    assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])
    wf[130, 0] = math.nan
    w, s_w = rt.quantize_fp8_block(wf, rows=128)
    y = rt.gemm_fp8_block(x, w, s_w, s_a)
    assert y[:, 128:256].isnan().all() and torch.equal(y[~bad][:, :128], clean[~bad][:, :128])


def test_product_overflows_to_infinity_in_half():
    x = torch.full((3, 256), 448.0, device="cuda").to(E4M3)
    w = torch.full((5, 256), 448.0, device="cuda").to(E4M3)
    one = torch.ones(3, 2, device="cuda"), torch.ones(1, 2, device="cuda")
    assert torch.isinf(rt.gemm_fp8_block(x, w, one[1], one[0], out_dtype=torch.float16)).all()
    assert (rt.gemm_fp8_block(x, w, one[1], one[0], out_dtype=torch.float32) == 448.0 * 448 * 256).all()


def test_product_far_rows():
    """Output offsets past 2^31 elements."""
    M, N, K = 300000, 8000, 16
    x = torch.ones(M, K, device="cuda").to(E4M3)
    w = torch.ones(N, K, device="cuda").to(E4M3)
    s_a = torch.arange(M, device="cuda", dtype=torch.float32).remainder(128)[:, None].contiguous()
    s_w = torch.ones(-(-N // 128), 1, device="cuda")
    y = rt.gemm_fp8_block(x, w, s_w, s_a, out_dtype=torch.float16)
    for lo in range(0, M, 50000):
        assert (y[lo:lo + 50000] == (16 * s_a[lo:lo + 50000]).half()).all()


# ── group norm ───────────────────────────────────────────────────────────────

ACTS = [lambda y: y, lambda y: y * torch.sigmoid(y), lambda y: 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5))),
        lambda y: 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))]


def norm_reference(x, groups, weight, bias, eps, act):
    """Exact value and the bound of the fp32 computation."""
    B, C = x.shape[0], x.shape[-1]
    v = x.to(f64).reshape(B, -1, groups, C // groups)
    mean = v.mean((1, 3), keepdim=True)
    d = v - mean
    rstd = 1 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + eps)
    far = d.abs().amax((1, 3), keepdim=True)
    gamma = (torch.ones(C, device="cuda", dtype=f64) if weight is None else weight.to(f64)).view(groups, -1)
    h = d * rstd * gamma
    tol = 2.0 ** -16 * (far * rstd * gamma.abs() + h.abs()) + 2.0 ** -22 * mean.abs() * rstd * gamma.abs()
    y = h.reshape(x.shape)
    tol = tol.reshape(x.shape)
    if bias is not None:
        y = y + bias.to(f64)
    tol = 1.13 * (tol + 2.0 ** -22 * y.abs()) + 2.0 ** -18 * (1 + y.abs())
    return ACTS[act](y), tol


def check_norm(y, x, groups, weight, bias, eps, act):
    want, tol = norm_reference(x, groups, weight, bias, eps, act)
    check(y, want, U[x.dtype] * (want.abs() + tol) + tol + TINY[x.dtype])


def check_norm_quantized(q, s, x, groups, weight, bias, eps, act):
    want, tol = norm_reference(x, groups, weight, bias, eps, act)
    want, tol = want.reshape(-1, x.shape[-1]), tol.reshape(-1, x.shape[-1])
    q, s = q.reshape(want.shape), s.reshape(len(want), -1)
    for b in range(s.shape[1]):
        w, t = want[:, 128 * b:128 * b + 128], tol[:, 128 * b:128 * b + 128]
        top, off = w.abs().amax(1).clamp(min=1e-8), t.amax(1)
        scale = s[:, b].double()
        assert ((scale - top / 448).abs() <= off / 448 + 2.0 ** -23 * top).all()
        check(q[:, 128 * b:128 * b + 128].double() * scale[:, None], w,
              2.0 ** -4 * (w.abs() + t) + t + 2.0 ** -10 * scale[:, None] + 2.0 ** -22 * w.abs())


SIZES = [
    (1, (1,), 8, 8), (1, (5,), 16, 4), (2, (16, 16), 1280, 32), (3, (61, 45), 352, 32), (2, (77,), 44, 4), (1, (50,), 13, 1),
    (4, (3,), 5120, 32), (1, (1000,), 8192, 16), (2, (4096,), 320, 32), (1, (300, 301), 128, 32), (1, (9001,), 13, 13),
    (2, (2500,), 640, 1), (16, (64,), 96, 96), (1, (7000,), 2568, 8), (5, (513,), 264, 3),
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("B,space,C,groups", SIZES)
def test_group_norm(B, space, C, groups, act, dtype):
    g = gen(C + act)
    x = normal(g, B, *space, C, dtype=dtype, std=1.5) + normal(g, B, *[1] * len(space), C, dtype=dtype)
    weight, bias = normal(g, C, dtype=dtype), normal(g, C, dtype=torch.float32)
    y = rt.group_norm(x, groups, weight, bias, eps=1e-5, activation=act)
    assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
    check_norm(y, x, groups, weight, bias, 1e-5, act)
    assert torch.equal(y, rt.group_norm(x, groups, weight, bias, eps=1e-5, activation=act))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("B,space,C,groups", SIZES)
def test_group_norm_quantized(B, space, C, groups, act, dtype):
    g = gen(C + act + 1)
    x = normal(g, B, *space, C, dtype=dtype, std=1.5)
    weight, bias = normal(g, C, dtype=torch.float32), normal(g, C, dtype=dtype)
    q, s = rt.fused_groupnorm_quantize(x, groups, weight, bias, eps=1e-6, activation=act)
    assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-C // 128))
    check_norm_quantized(q, s, x, groups, weight, bias, 1e-6, act)


@pytest.mark.parametrize("space", [(64,), (200, 200)])
def test_group_norm_far_from_zero(space):
    """A mean a thousand times the deviation: the sums are of differences."""
    g = gen(21)
    x = (normal(g, 2, *space, 64, std=1.0) + 1000.0).half()
    check_norm(rt.group_norm(x, 8), x, 8, None, None, 1e-5, 0)
    x[0, 0] = -1000.0     # and a first value far from the others
    check_norm(rt.group_norm(x, 8), x, 8, None, None, 1e-5, 0)


@pytest.mark.parametrize("space", [(9,), (150, 150)])
def test_group_norm_constant_groups_and_none(space):
    x = torch.full((2, *space, 32), 3.25, dtype=torch.bfloat16, device="cuda")
    assert (rt.group_norm(x, 4) == 0).all()
    bias = torch.arange(32, device="cuda", dtype=torch.float32)
    assert (rt.group_norm(x, 4, None, bias) == bias.bfloat16()).all()
    q, s = rt.fused_groupnorm_quantize(x, 4)
    assert (q.float() == 0).all()
    assert rt.group_norm(x[:0], 4).shape == (0, *space, 32)
    q, s = rt.fused_groupnorm_quantize(x[:, :0], 4)
    assert q.numel() == 0 and s.numel() == 0


@pytest.mark.parametrize("space", [(40,), (150, 150)])
def test_group_norm_quantized_near_the_largest_value(space):
    x = torch.ones(1, *space, 256, device="cuda", dtype=torch.bfloat16)
    x[..., ::2] = -1                                             # mean 0, variance 1: y = +-weight / sqrt(1 + eps)
    weight = torch.full((256,), 3.3e38, device="cuda", dtype=torch.bfloat16)
    weight[128:] = 2.9e38
    q, s = rt.fused_groupnorm_quantize(x, 8, weight, eps=1e-5)
    want = weight.double()[::128] / (1 + 1e-5) ** 0.5 / 448
    assert ((s.double() - want).abs() <= 2.0 ** -20 * want).all()   # fewer than eight roundings of 2^-24 and an rsqrt of 2^-22
    assert torch.equal(q.float(), 448 * x.reshape(q.shape).float())


@pytest.mark.parametrize("space", [(40,), (150, 150)])
def test_group_norm_not_finite(space):
    """A NaN or an infinity makes its group of its sample NaN, and no other."""
    g = gen(22)
    x = normal(g, 3, *space, 64, dtype=torch.float16)
    clean = rt.group_norm(x, 8, activation=1)
    x.view(3, -1, 64)[0, 3, 9] = math.nan
    x.view(3, -1, 64)[2, -1, 63] = math.inf
    y = rt.group_norm(x, 8, activation=1)
    bad = torch.zeros(3, 64, dtype=torch.bool, device="cuda")
    bad[0, 8:16] = True
    bad[2, 56:64] = True
    y, clean = y.view(3, -1, 64), clean.view(3, -1, 64)
    at = bad[:, None].expand_as(y)
    assert y[at].isnan().all() and torch.equal(y[~at], clean[~at])


@pytest.mark.parametrize("space", [(6, 7), (130, 131)])
@pytest.mark.parametrize("view", ["channels_last", "padded_rows", "odd_rows", "columns", "transposed", "batch_apart", "rows_only"])
def test_group_norm_layouts(view, space):
    g = gen(23)
    C = 48
    if view == "channels_last":
        x = normal(g, 2, C, *space, dtype=torch.float16).to(memory_format=torch.channels_last).permute(0, 2, 3, 1)
        assert x.is_contiguous()
    elif view == "padded_rows":
        x = normal(g, 2, *space, 64, dtype=torch.float16)[..., 8:8 + C]
    elif view == "odd_rows":
        x = normal(g, 2, *space, 53, dtype=torch.float16)[..., 3:3 + C]
    elif view == "columns":
        x = normal(g, 2, space[0], 2 * space[1], C, dtype=torch.float16)[:, :, ::2]
    elif view == "transposed":
        x = normal(g, 2, C, *space, dtype=torch.float16).permute(0, 2, 3, 1)
    elif view == "batch_apart":
        x = normal(g, 6, *space, C, dtype=torch.float16)[::3]
    else:
        x = normal(g, 9, C, dtype=torch.float16)
    weight = normal(g, 2 * C)[::2]
    check_norm(rt.group_norm(x, 6, weight, activation=1), x, 6, weight, None, 1e-5, 1)
    check_norm_quantized(*rt.fused_groupnorm_quantize(x, 6, weight, activation=1), x, 6, weight, None, 1e-5, 1)


@pytest.mark.parametrize("space", [(64,), (190, 190)])
def test_group_norm_in_place_and_between_others(space):
    g = gen(24)
    x = normal(g, 2, *space, 64, dtype=torch.bfloat16)
    y = rt.group_norm(x, 4, activation=2)
    for lo, width in ((8, 80), (3, 71)):
        buf = torch.full((2, *space, width), -7.0, dtype=torch.bfloat16, device="cuda")
        out = buf[..., lo:lo + 64]
        assert rt.group_norm(x, 4, activation=2, out=out) is out
        assert torch.equal(out, y) and (buf[..., :lo] == -7).all() and (buf[..., lo + 64:] == -7).all()
    assert rt.group_norm(x, 4, activation=2, out=x) is x and torch.equal(x, y)


# ── together ─────────────────────────────────────────────────────────────────

def test_projection_behind_a_norm():
    """Group norm + SiLU to e4m3 blocks, then the product with a bias: a 1 x 1
    projection of an image, from a channels-last tensor."""
    g = gen(31)
    x = normal(g, 2, 320, 33, 41, dtype=torch.float16).to(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    gamma, beta = normal(g, 320, dtype=torch.float16), normal(g, 320, dtype=torch.float16)
    weight, bias = normal(g, 640, 320, std=320 ** -0.5), normal(g, 640, dtype=torch.float16)
    w, s_w = rt.quantize_fp8_block(weight, rows=128)
    q, s = rt.fused_groupnorm_quantize(x, 32, gamma, beta, activation=1)
    y = rt.gemm_fp8_block(q, w, s_w, s, bias=bias, out_dtype=torch.float16)
    assert y.shape == (2, 33, 41, 640)
    want, size = product_reference(q.reshape(-1, 320), w, s_w, s.reshape(-1, 3), bias)
    check(y.view(-1, 640), want, product_tolerance(want, size, 320, torch.float16))
    exact, tol = norm_reference(x, 32, gamma, beta, 1e-5, 1)
    wd = w.to(f64) * s_w.to(f64).repeat_interleave(128, 0).repeat_interleave(128, 1)[:, :320]
    off = 2.0 ** -4 * (exact.abs() + tol) + tol + 2.0 ** -9 * s.double().repeat_interleave(128, -1)[..., :320]
    full = exact @ wd.T + bias.to(f64)
    check(y, full, off @ wd.abs().T * (1 + 2.0 ** -10) + U[torch.float16] * full.abs() * 2 + 2.0 ** -14)


@pytest.mark.parametrize("rot,K", [(False, 300), (False, 256), (True, 256), (True, 200)])
@pytest.mark.parametrize("dtype", HALF)
def test_module(rot, K, dtype):
    conv = load("convlinear")
    g = gen(32)
    lin = torch.nn.Linear(K, 200).cuda()
    with torch.no_grad():
        lin.weight.copy_(normal(g, 200, K, std=K ** -0.5))
        lin.bias.copy_(normal(g, 200))
    m = conv.ConvLinearFP8.from_float(lin, rot_need=rot, rot_size=64).to(dtype)
    c = conv.ConvLinearFP8.from_float(lin.cpu(), rot_need=False) if not rot else None
    if c is not None:
        assert torch.equal(c.weight.float(), m.weight.float().cpu()) and torch.equal(c.scale, m.scale.cpu())
    assert m.weight.dtype is E4M3 and m.scale.dtype is torch.float32
    x = normal(g, 4, 7, K, dtype=dtype)
    y = m(x)
    assert y.shape == (4, 7, 200) and y.dtype == dtype
    xp = m._prepared(x.view(-1, K))
    q, s = rt.quantize_fp8_block(xp)
    w = m.weight[:, :m.in_features]
    want, size = product_reference(q, w, m.scale, s, m.bias)
    check(y.view(-1, 200), want, product_tolerance(want, size, m.in_features, dtype))


@pytest.mark.parametrize("M,L", [(3, 50), (700, 30000)])
def test_graph_stream_and_repeats(M, L):
    """The chain captured on a stream of its own, replayed over other inputs; two
    graphs in flight on two streams do not disturb each other."""
    g = gen(33)
    xs = [normal(g, 1, L, 64, dtype=torch.float16) for _ in range(2)]
    ys = [normal(g, M, 384, dtype=torch.bfloat16) for _ in range(2)]
    w, s_w = rt.quantize_fp8_block(normal(g, 500, 384), rows=128)

    def chain(x, y):
        a = rt.group_norm(x, 8, activation=1)
        b = rt.fused_groupnorm_quantize(x, 8)
        q, s = rt.quantize_fp8_block(y)
        return a, b[0].float(), b[1], rt.gemm_fp8_block(q, w, s_w, s)

    want = [chain(x, y) for x, y in zip(xs, ys)]
    torch.cuda.synchronize()
    runs = []
    for x, y in zip(xs, ys):
        sx, sy = torch.zeros_like(x), torch.zeros_like(y)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            chain(sx, sy)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = chain(sx, sy)
        sx.copy_(x)
        sy.copy_(y)
        runs.append((graph, stream, out))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, _, out), w_ in zip(runs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w_))
    assert rt.device_error() == 0


def test_torch_library_ops():
    load("_torch_ops")
    ops = torch.ops.intcrush_b200
    g = gen(34)
    x = normal(g, 2, 9, 300, dtype=torch.float16)
    q, s = ops.quantize_fp8_block(x, 1)
    rq, rs = rt.quantize_fp8_block(x)
    assert torch.equal(q.float(), rq.float()) and torch.equal(s, rs)
    w, s_w = ops.quantize_fp8_block(normal(g, 40, 300), 128)
    b = normal(g, 40, dtype=torch.float16)
    assert torch.equal(ops.gemm_fp8_block(q, w, s_w, s, b, 0), rt.gemm_fp8_block(rq, w, s_w, rs, bias=b, out_dtype=torch.float16))
    assert torch.equal(ops.group_norm(x, 4, None, None, 1e-5, 1), rt.group_norm(x, 4, activation=1))
    q, s = ops.fused_groupnorm_quantize(x, 4, None, None, 1e-5, 1)
    rq, rs = rt.fused_groupnorm_quantize(x, 4, activation=1)
    assert torch.equal(q.float(), rq.float()) and torch.equal(s, rs)
    # (opcheck's schema test compares by arithmetic, which torch lacks for e4m3)
    fake = dict(test_utils=("test_faketensor",))
    torch.library.opcheck(ops.gemm_fp8_block.default, (*rt.quantize_fp8_block(x[0])[:1], w, s_w, rt.quantize_fp8_block(x[0])[1], b, 1), **fake)
    torch.library.opcheck(ops.quantize_fp8_block.default, (x, 1), **fake)
    torch.library.opcheck(ops.quantize_fp8_block.default, (x[0], 128), **fake)
    torch.library.opcheck(ops.fused_groupnorm_quantize.default, (x, 4, None, None, 1e-5, 0), **fake)
    torch.library.opcheck(ops.group_norm.default, (x, 4, None, None, 1e-5, 0), test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("C,groups,L", [(8192, 8192, 700), (8192, 1, 300), (4096, 4096, 37), (8190, 2730, 64)])
def test_group_norm_widest(C, groups, L):
    g = gen(35)
    x = normal(g, 1, L, C, dtype=torch.bfloat16)
    check_norm(rt.group_norm(x, groups), x, groups, None, None, 1e-5, 0)
    check_norm_quantized(*rt.fused_groupnorm_quantize(x, groups), x, groups, None, None, 1e-5, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [9, 33, 100, 121, 128])
@pytest.mark.parametrize("K,N", [(2048, 1800), (5120, 2560), (4000, 3200), (2040, 4100), (1030, 6000), (8192, 100)])
def test_product_shared_by_clusters(K, N, M, dtype):
    """Few tiles: clusters of two to eight CTAs share the blocks; rows that a tile
    lacks are not staged."""
    g = gen(K + M)
    (x, s_a), (w, s_w) = operands(g, M, K, N)
    b = normal(g, N, dtype=torch.float16)
    y = rt.gemm_fp8_block(x, w, s_w, s_a, bias=b, out_dtype=dtype)
    want, size = product_reference(x, w, s_w, s_a, b)
    check(y, want, product_tolerance(want, size, K, dtype))
    assert torch.equal(y, rt.gemm_fp8_block(x, w, s_w, s_a, bias=b, out_dtype=dtype))
    assert rt.device_error() == 0


@pytest.mark.parametrize("B,L,C,groups", [(300, 7, 64, 8), (150, 6000, 32, 2), (2, 40000, 136, 17), (700, 1, 16, 16)])
def test_group_norm_of_many_samples(B, L, C, groups):
    g = gen(36)
    x = normal(g, B, L, C, dtype=torch.float16) + normal(g, B, 1, C, dtype=torch.float16)
    weight, bias = normal(g, C), normal(g, C)
    check_norm(rt.group_norm(x, groups, weight, bias, activation=1), x, groups, weight, bias, 1e-5, 1)
    check_norm_quantized(*rt.fused_groupnorm_quantize(x, groups, weight, bias), x, groups, weight, bias, 1e-5, 0)


def test_group_norm_one_sample_does_not_see_another():
    """A sample gives the same bits alone, in a batch and between others."""
    g = gen(37)
    x = normal(g, 3, 30000, 64, dtype=torch.bfloat16)
    y = rt.group_norm(x, 4, activation=3)
    z = x.clone()
    z[0], z[2] = 100, math.inf
    assert torch.equal(rt.group_norm(z, 4, activation=3)[1], y[1])


def test_wait_that_runs_out_is_not_set_by_these_calls():
    assert rt.device_error() == 0
