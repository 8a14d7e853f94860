"""Calls of the attention-side operators at the ends of their ranges: wide
index types, lengths without a limit, odd strides, long keys, mixed errors.

References and bounds are those of the operators' other tests (64-bit forms; u
the unit roundoff of the tensors' type)."""

import math

import pytest
import torch

from _pkg import load
from test_gpu_attention_ops import (U, attention_inputs, attention_reference, check, gen, lora_inputs, lora_reference, normal,
                                    qk_reference, qk_tolerance, tables)

pytestmark = pytest.mark.gpu
rt = load("_b200_runtime") if torch.cuda.is_available() else None


# ── wide integers ────────────────────────────────────────────────────────────

@pytest.mark.parametrize("Lq", [1, 200])
def test_lengths_without_a_limit(Lq):
    """Lengths past the keys are the keys', also where 32 bits do not hold
    them; negative ones see nothing."""
    q, k, v, _ = attention_inputs(30, 4, Lq, 90, 2, 2, 64, torch.float16)
    lens = torch.tensor([2**63 - 1, 2**32 + 5, -2**32 + 5, 7], device="cuda")
    want, tol = attention_reference(q, k, v, torch.tensor([90, 90, 0, 7]))
    got = rt.cross_attention(q, k, v, kv_lens=lens)
    check(got, want, tol)
    assert (got[2] == 0).all()


def test_wide_ids_and_positions_outside_their_range():
    g = gen(31)
    q = normal(g, 1, 4, 3, 64, dtype=torch.float16)
    cos, sin = tables(10, 64, g)
    pos = torch.tensor([[2**32 + 1, 3, -2**32 + 2, 2**63 - 1]], device="cuda")
    assert rt.device_error() == 0
    y = rt.qk_norm_rope(q, cos=cos, sin=sin, positions=pos)
    assert rt.device_error() == 2
    want = qk_reference(q, None, cos, sin, "interleaved", torch.full_like(pos, 3), 1e-6)
    check(y[:, 1], want[:, 1], qk_tolerance(want[:, 1], torch.float16))
    assert y[:, [0, 2, 3]].isnan().all()

    x, base, down, up, scales, _ = lora_inputs(32, 4, 64, 40, 8, 2, torch.float16)
    ids = torch.tensor([2**32 + 1, 1, -2**32 + 1, -1], device="cuda")   # none, 1, negative, negative
    got = rt.lora_batched(x, down, up, ids, scales, base=base)
    assert rt.device_error() == 2 and rt.device_error() == 0
    assert got[0].isnan().all()
    want, tol = lora_reference(x[1:], down, up, torch.tensor([1, -1, -1], device="cuda"), scales, base[1:], 1)
    check(got[1:], want, tol)
    assert torch.equal(got[2:], base[2:])


# ── the error word ───────────────────────────────────────────────────────────

@pytest.mark.parametrize("index_first", [True, False])
def test_error_word_keeps_both_codes(index_first):
    """A bad index and a wait that runs out: both are reported, the wait
    first, one a read."""
    import ctypes

    L = load("_lib")
    q = torch.zeros(1, 1, 1, 64, dtype=torch.float16, device="cuda")
    cos, sin = tables(4, 64, gen(33))

    def index():
        rt.qk_norm_rope(q, cos=cos, sin=sin, positions=torch.tensor([[4]], device="cuda"))

    def timeout():
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert L.lib().ic_selftest_wait_timeout(1_000_000, stream) == L.IC_OK

    assert rt.device_error() == 0
    for call in (index, timeout) if index_first else (timeout, index):
        call()
    torch.cuda.synchronize()
    assert rt.device_error(clear=False) == L.IC_DEV_ERR_TIMEOUT
    assert [rt.device_error() for _ in range(3)] == [L.IC_DEV_ERR_TIMEOUT, L.IC_DEV_ERR_INDEX, 0]


# ── a batch of one with an odd batch stride ──────────────────────────────────

@pytest.mark.parametrize("Lq", [1, 5, 200])
def test_one_sample_of_an_odd_buffer(Lq):
    """One sample cut from a buffer whose samples are an odd number of elements
    apart."""
    g = gen(34)
    H, D = 3, 64

    def cut(L):
        stride = L * H * D + 5
        return normal(g, 2 * stride, dtype=torch.float16).as_strided((1, L, H, D), (stride, H * D, D, 1))

    q, k, v, out = cut(Lq), cut(70), cut(70), cut(Lq)
    want, tol = attention_reference(q, k, v)
    assert rt.cross_attention(q, k, v, out=out) is out
    check(out, want, tol)
    cos, sin = tables(Lq, D, g)
    want = qk_reference(q, None, cos, sin, "half", None, 1e-6)
    check(rt.qk_norm_rope(q, cos=cos, sin=sin, layout="half"), want, qk_tolerance(want, torch.float16))


# ── fp16 weights ─────────────────────────────────────────────────────────────

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Lq,scale", [(1, 1.0), (1, -1.0), (20, -1.0), (38400, 1.0)])
def test_many_keys_of_little_weight(Lq, scale, dtype):
    """One key that outweighs each of 2^19 others by 2^25.5 but not all of them
    together (their sum is 1.1 percent of it).  A weight is held to 2^-8 (bf16)
    or 2^-11 and 2^-32 of the largest one (fp16)."""
    Lk, D = 2**19, 64
    g = gen(35)
    q = torch.zeros(1, 1, 1, D, dtype=dtype, device="cuda")
    k = torch.zeros(1, Lk, 1, D, dtype=dtype, device="cuda")
    q[..., 0] = 1
    k[0, 0, 0, 0] = 17.675 / scale
    v = torch.rand(1, Lk, 1, D, device="cuda", generator=g).to(dtype)
    v[0, 0] = 0
    s = k[0, :, 0, 0].double() * scale
    p = torch.softmax(s, 0)[:, None]
    vd = v[0, :, 0].double()
    want = (p * vd).sum(0)
    tol = (U[dtype] + 3e-5) * want + U[dtype] * want
    if dtype == torch.float16:
        tol = tol + 2.0**-25 + 2.0**-32 * p.max() * vd.sum(0)
    got = rt.cross_attention(q.expand(1, Lq, 1, D), k, v, scale=scale)
    assert rt.device_error() == 0
    check(got[0, :, 0], want.expand(Lq, D), tol)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Lq,later", [(1, 64), (200, 130)])
def test_scores_whose_steps_pass_the_room(Lq, later, dtype):
    """Scores of 2^27, where fp32 counts in steps of 16: the later key has 2^16
    times the weight of the first one and takes (nearly) all of the output."""
    Lk, D = 300, 64
    q = torch.zeros(1, Lq, 1, D, dtype=dtype, device="cuda")
    k = torch.zeros(1, Lk, 1, D, dtype=dtype, device="cuda")
    q[..., 0], q[..., 1] = 2.0**14, 4.0
    k[0, 0, 0, 0], k[0, 0, 0, 1] = 2.0**13, 4.0
    k[0, later, 0, 0], k[0, later, 0, 1] = 2.0**13, 8.0
    v = normal(gen(36), 1, Lk, 1, D, dtype=dtype)
    # the scale whose product with log2(e), in fp32, is 1: scores in log2 are q k
    e = torch.tensor(math.log2(math.e))
    scale = next(s.item() for s in (1 / e + torch.arange(-4, 5) * 2.0**-24) if (s * e).item() == 1.0)
    got = rt.cross_attention(q, k, v, scale=scale)
    a, b = v[0, 0, 0].double(), v[0, later, 0].double()
    want = (b + a * 2.0**-16) / (1 + 2.0**-16)
    tol = (U[dtype] + 3e-5) * (b.abs() + a.abs() * 2.0**-16) + U[dtype] * want.abs() + 2.0**-25 + 2.0**-32
    check(got[0, :, 0], want.expand(Lq, D), tol)


# ── adapters of the neighbours ───────────────────────────────────────────────

@pytest.mark.parametrize("M", [1024, 1500, 4200])
def test_neighbours_other_adapters(M):
    """Neighbours that change to other valid adapters: a request stays within
    the operator's bound (the order of its sums may change with their ids), and
    rows of other tiles of 128 keep their bits."""
    x, base, down, up, scales, g = lora_inputs(37, M, 1000, 72, 16, 6, torch.float16)
    few = torch.arange(M, device="cuda") // 300 % 2
    many = few.clone()
    many[128:256:2] = torch.randint(-1, 6, (64,), device="cuda", generator=g)
    one = rt.lora_batched(x, down, up, few, scales, base=base)
    two = rt.lora_batched(x, down, up, many, scales, base=base)
    for got, ids in ((one, few), (two, many)):
        want, tol = lora_reference(x, down, up, ids, scales, base, 1)
        check(got, want, tol)
    other = torch.ones(M, dtype=torch.bool, device="cuda")
    other[128:256] = False
    assert torch.equal(one[other], two[other])
    assert torch.equal(rt.lora_batched(x, down, up, many, scales, base=base), two)
