"""The 8-bit floating point linear and its norm at values far out: activations of
very negative values, zeros with a sign, blocks that are not finite.

Inputs of the norm alternate between 1 and -1 from row to row, so that y = +-weight
/ sqrt(1 + eps); statistics, factors and their products are fewer than eight
roundings of 2^-24 and an rsqrt of 2^-22, y is within D = 2^-20 of itself.  An
activation whose logarithm changes by S for a change of 1 in that of y is then
within (1 + S) D of its exact value, and its own exponent, of a few roundings of 2^-24,
half of that again; 2^-19 covers the approximate functions behind it.  What lies
below 2^-118 (SiLU of -86.6) may be any such value."""

import math

import pytest
import torch

import test_gpu_fp8_ops as ops
from _pkg import load

pytestmark = pytest.mark.gpu
rt = load("_b200_runtime") if torch.cuda.is_available() else None

f64 = torch.float64
E4M3 = torch.float8_e4m3fn
HALF = [torch.float16, torch.bfloat16]
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SPACES = [(40,), (1000, 1002)]     # one launch, two


def alternating(space, C, dtype):
    x = torch.ones(1, math.prod(space), C, device="cuda", dtype=dtype)
    x[:, 1::2] = -1
    return x.view(1, *space, C)


def exact(y, act):
    """Value, and how much its logarithm changes with that of y (for y < 0)."""
    u = math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
    if act == 1:
        return y * torch.sigmoid(y), y.abs()
    if act == 2:
        return y * 0.5 * torch.special.erfc(-y * math.sqrt(0.5)), y * y
    return y * torch.sigmoid(2 * u), 2 * math.sqrt(2 / math.pi) * (y.abs() + 3 * 0.044715 * y.abs() ** 3)


def check_tails(act, space, dtype):
    far = [1e15, 1e20, 1e30, 3e38] if dtype == torch.bfloat16 else [100.0, 3e4, 6e4]
    weight = torch.cat([torch.linspace(0.01, 14, 205), torch.linspace(14, 110, 97), torch.tensor(far + [1e4] * (18 - len(far)))]).cuda()
    x = alternating(space, 320, dtype)
    got = rt.group_norm(x, 1, weight, activation=act)
    assert torch.equal(got.view(-1, 320)[2:], got.view(-1, 320)[:-2])
    got = got.view(-1, 320)[:2].double()
    y = torch.stack([weight, -weight]).to(f64) / math.sqrt(1 + 1e-5)
    want, slope = exact(y, act)
    slope = torch.where(y < 0, slope, torch.full_like(y, 0.2)).clamp(max=1e6)
    off = want.abs() * (1.5 * (1 + slope) * 2.0 ** -20 + 2.0 ** -19) + 2.0 ** -118
    tol = U[dtype] * (want.abs() + off) + off + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert torch.isfinite(got).all()
    over = (got - want).abs() - tol
    assert over.max().item() <= 0, f"y = {y.flatten()[over.argmax()]}: {got.flatten()[over.argmax()]}, not {want.flatten()[over.argmax()]}"


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("space", SPACES)
@pytest.mark.parametrize("act", [1, 3])
def test_activation_of_very_negative_values(act, space, dtype):
    check_tails(act, space, dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("space", SPACES)
def test_gelu_of_negative_values(space, dtype):
    """Relative to the value, also where 1 + erf has no digits left."""
    check_tails(2, space, dtype)


@pytest.mark.parametrize("space", SPACES)
@pytest.mark.parametrize("act", [1, 2, 3])
def test_quantized_activation_of_very_negative_values(act, space):
    """Nothing is left of a block far below 0: its scale is the least one."""
    x = alternating(space, 384, torch.bfloat16)
    weight = torch.full((384,), 1e20, device="cuda")
    weight[128:256] = 50
    q, s = rt.fused_groupnorm_quantize(x, 1, weight, activation=act)
    q, s = q.view(-1, 384), s.view(-1, 3)
    least = torch.tensor(1e-8, dtype=torch.float32) / torch.tensor(448.0)
    assert (s[1::2] == least.item()).all() and (q[1::2].float() == 0).all()
    want = weight[::128].double() / math.sqrt(1 + 1e-5) / 448
    assert ((s[::2].double() - want).abs() <= 2.0 ** -18 * want).all() and (q[::2].float() == 448).all()


@pytest.mark.parametrize("dtype", HALF)
def test_quantize_every_quotient_to_its_byte(dtype):
    """Values of both signs down to a quarter of the border between 0 and the least
    e4m3 value (2^-10 scales), zeros of both signs, over the scales of every
    significand that a block's largest value can have: the bytes of e4m3(x / s)."""
    every = torch.arange(2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype).cuda()
    every = every[torch.isfinite(every)]
    tops = every[(every >= 1) & (every < 2)]
    small = every[(every < 2) & (every > 2.0 ** -21)]
    small = torch.cat([small, -small, small.new_tensor([0.0, -0.0])])
    small = torch.cat([small, small.new_full((-len(small) % 127,), -0.0)]).view(-1, 127)
    for top in tops.split(32):
        t = top[:, None, None]
        x = torch.cat([torch.maximum(torch.minimum(small[None].expand(len(top), -1, -1), t), -t), t.expand(-1, small.shape[0], 1)], -1)
        x = x.reshape(-1, 128)
        q, s = rt.quantize_fp8_block(x)
        want_s = x.float().amax(1, keepdim=True) / torch.full((len(x), 1), 448.0, device="cuda")
        assert torch.equal(s, want_s)
        assert torch.equal(q.view(torch.uint8), (x.float() / want_s).to(E4M3).view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_keeps_a_zeros_sign(rows, dtype):
    x = torch.randn(128, 300, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    x[:, ::3] = -0.0
    x[:, 1::3] = 0.0
    q, _ = rt.quantize_fp8_block(x, rows=rows)
    assert (q[:, ::3].view(torch.uint8) == 0x80).all() and (q[:, 1::3].view(torch.uint8) == 0).all()


@pytest.mark.parametrize("space", [7, 80000])
@pytest.mark.parametrize("layout", ["samples_between_rows", "rows_of_others_between"])
def test_group_norm_into_rows_that_interleave(layout, space):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, space, 64, device="cuda", generator=g).half()
    buf = torch.full((space * 128 + 512,), -7.0, dtype=torch.float16, device="cuda")
    strides = (64, 128, 1) if layout == "samples_between_rows" else (192, 128, 1)
    out = buf.as_strided((2, space, 64), strides)
    y = rt.group_norm(x, 4, activation=1)
    assert rt.group_norm(x, 4, activation=1, out=out) is out and torch.equal(out, y)
    assert (buf == -7).sum() == len(buf) - y.numel()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", [2, 3])
@pytest.mark.parametrize("B,space,C,groups", ops.SIZES)
def test_group_norm_quantized_behind_gelu(B, space, C, groups, act, dtype):
    g = ops.gen(C + act + 2)
    x = ops.normal(g, B, *space, C, dtype=dtype, std=1.5)
    weight, bias = ops.normal(g, C), ops.normal(g, C, dtype=dtype)
    q, s = rt.fused_groupnorm_quantize(x, groups, weight, bias, eps=1e-6, activation=act)
    ops.check_norm_quantized(q, s, x, groups, weight, bias, 1e-6, act)
    again = rt.fused_groupnorm_quantize(x, groups, weight, bias, eps=1e-6, activation=act)
    assert torch.equal(q.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(s, again[1])


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("space", [50, 100000])
def test_quantized_norm_of_what_is_not_finite(space, act):
    """A NaN makes the scales and values of its blocks NaN; an infinity its block's
    scale infinite, its own value NaN and the others 0.  Other blocks and samples
    keep their bits."""
    x = ops.normal(ops.gen(3), 3, space, 256, dtype=torch.float16)
    beta = torch.zeros(256, device="cuda")
    q0, s0 = rt.fused_groupnorm_quantize(x, 8, None, beta, activation=act)
    assert torch.isfinite(s0).all() and torch.isfinite(q0.float()).all()

    x[0, space // 3, 40] = math.nan            # group 1 of sample 0: its channels lie in block 0
    q, s = rt.fused_groupnorm_quantize(x, 8, None, beta, activation=act)
    assert s[0, :, 0].isnan().all() and q[0, :, :128].float().isnan().all()
    assert torch.equal(s[0, :, 1], s0[0, :, 1]) and torch.equal(q[0, :, 128:].float(), q0[0, :, 128:].float())
    assert torch.equal(s[1:], s0[1:]) and torch.equal(q[1:].float(), q0[1:].float())

    beta[200] = math.inf                       # a channel of block 1, in every sample
    q, s = rt.fused_groupnorm_quantize(x, 8, None, beta, activation=act)
    assert (s[..., 1] == math.inf).all() and q[..., 200].float().isnan().all()
    others = torch.cat([q[..., 128:200], q[..., 201:]], -1).float()
    assert (others == 0).all()
    assert torch.equal(s[1:, :, 0], s0[1:, :, 0]) and torch.equal(q[1:, :, :128].float(), q0[1:, :, :128].float())


@pytest.mark.parametrize("C,groups", [(56, 7), (64, 4)])
@pytest.mark.parametrize("rows", [2, 146, 2 * 73 * 16, 73 * 5 * 32, 73 * 16 * 296])
def test_group_norm_of_squares_beyond_the_range(rows, C, groups):
    """The variance is infinite, so that all that is left is the bias; not 0, which
    would make large numbers of the values."""
    x = alternating((rows,), C, torch.bfloat16) * 2e19
    bias = torch.arange(C, device="cuda", dtype=torch.float32)
    y = rt.group_norm(x, groups, None, bias)
    assert (y == bias.bfloat16()).all()
    # and about its end: the sum over a group is rows * C / groups * 2^110, which 32 bits
    # hold below 2^128; eps is nothing beside it
    x = alternating((rows,), C, torch.bfloat16) * 2.0 ** 55
    y = rt.group_norm(x, groups)
    inside = rows * C // groups < 2 ** 18
    assert (y.double() - inside * alternating((rows,), C, f64)).abs().max() <= 2.0 ** -8
