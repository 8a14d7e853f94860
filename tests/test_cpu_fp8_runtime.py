"""Host side of the 8-bit floating point linear without a GPU: what the runtime's
calls refuse, what they hand to the library and on which device; the weight
quantiser and the module."""

import pytest
import torch

from _pkg import load
from test_cpu_attention_runtime import lib  # noqa: F401  (the stub library on two devices)

rt = load("_b200_runtime")
conv = load("convlinear")
qu = load("_quant_utils")
E4M3 = torch.float8_e4m3fn


def half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


def e4m3(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4M3)


def scales(*shape):
    return torch.zeros(*shape)


def product(x=None, w=None, s_w=None, s_a=None, **kw):
    return rt.gemm_fp8_block(e4m3(4, 300) if x is None else x, e4m3(200, 300) if w is None else w,
                             scales(2, 3) if s_w is None else s_w, scales(4, 3) if s_a is None else s_a, **kw)


CALLS = {
    "quantize": lambda: rt.quantize_fp8_block(half(4, 300)),
    "quantize weight": lambda: rt.quantize_fp8_block(torch.zeros(200, 300), rows=128),
    "product": lambda: product(bias=half(200)),
    "group norm": lambda: rt.group_norm(half(2, 5, 64), 4, half(64), half(64)),
    "group norm to e4m3": lambda: rt.fused_groupnorm_quantize(half(2, 5, 64), 4),
}


@pytest.mark.parametrize("call", CALLS)
def test_calls_run_on_the_tensors_device(lib, call):  # noqa: F811
    CALLS[call]()
    assert lib.calls and {device for _, device, _ in lib.calls} == {1}
    assert lib.current == 0


@pytest.mark.parametrize("call,error,text", [
    (lambda: rt.quantize_fp8_block(torch.zeros(4, 8, dtype=torch.float64)), TypeError, "float16, bfloat16 or float32"),
    (lambda: rt.quantize_fp8_block(half(4, 8), rows=64), ValueError, "1 or 128"),
    (lambda: rt.quantize_fp8_block(half(4, 0)), ValueError, "must be"),
    (lambda: rt.quantize_fp8_block(torch.tensor(1.0)), ValueError, "must be"),
    (lambda: rt.quantize_fp8_block(half(2, 4, 8), rows=128), ValueError, r"\[N, K\]"),
    (lambda: product(x=half(4, 300)), TypeError, "float8_e4m3fn"),
    (lambda: product(w=torch.zeros(200, 300, dtype=torch.uint8)), TypeError, "float8_e4m3fn"),
    (lambda: product(x=torch.zeros(4, 300, dtype=torch.uint8).view(torch.float8_e5m2)), TypeError, "float8_e4m3fn"),
    (lambda: product(x=e4m3(4, 304)), ValueError, "must be"),
    (lambda: product(w=e4m3(2, 100, 300)), ValueError, "must be"),
    (lambda: product(s_a=scales(4, 2)), ValueError, "scales must be"),
    (lambda: product(s_a=scales(3, 3)), ValueError, "scales must be"),
    (lambda: product(s_w=scales(200, 3)), ValueError, "scales must be"),
    (lambda: product(s_w=scales(2, 3).half()), TypeError, "float32"),
    (lambda: product(s_a=scales(4, 3).double()), TypeError, "float32"),
    (lambda: product(out_dtype=torch.int8), TypeError, "output"),
    (lambda: product(out=half(4, 199)), ValueError, "out must be"),
    (lambda: product(out=half(200, 4).t()), ValueError, "row-major"),
    (lambda: product(out=half(1, 200).expand(4, 200)), ValueError, "row-major"),
    (lambda: product(bias=half(199)), ValueError, "bias"),
    (lambda: product(bias=torch.zeros(200, dtype=torch.int32)), TypeError, "bias"),
    (lambda: rt.group_norm(torch.zeros(2, 5, 64), 4), TypeError, "float16/bfloat16"),
    (lambda: rt.group_norm(half(64), 4), ValueError, "must be"),
    (lambda: rt.group_norm(half(2, 5, 64), 5), ValueError, "divide"),
    (lambda: rt.group_norm(half(2, 5, 64), 0), ValueError, "divide"),
    (lambda: rt.group_norm(half(2, 5, 64), 4, activation=4), ValueError, "activation"),
    (lambda: rt.group_norm(half(2, 5, 64), 4, half(32)), ValueError, "weight and bias"),
    (lambda: rt.group_norm(half(2, 5, 64), 4, None, torch.zeros(64, dtype=torch.int64)), TypeError, "weight and bias"),
    (lambda: rt.group_norm(half(2, 5, 64), 4, out=half(2, 5, 32)), ValueError, "out must be"),
    (lambda: rt.group_norm(half(2, 5, 64), 4, out=half(2, 64, 5).transpose(1, 2)), ValueError, "channels last"),
    (lambda: rt.group_norm(half(2, 5, 64), 4, out=half(2, 1, 64).expand(2, 5, 64)), ValueError, "overlap"),
    (lambda: rt.group_norm(half(2, 5, 64), 4, out=half(1, 5, 64).expand(2, 5, 64)), ValueError, "overlap"),
])
def test_refusals(lib, call, error, text):  # noqa: F811
    with pytest.raises(error, match=text):
        call()
    assert not [c for c in lib.calls if not c[0].endswith("workspace")]


def test_calls_without_a_gpu():
    for call in CALLS.values():
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("K,ld", [(256, 256), (300, 304), (1, 16)])
def test_layouts_handed_over(lib, K, ld):  # noqa: F811
    """Rows start at multiples of 16 bytes, whole in their storage; the quantiser's
    results go to the product without a copy."""
    q, s = rt.quantize_fp8_block(half(5, K))
    kb = -(-K // 128)
    assert q.shape == (5, K) and q.stride() == (ld, 1) and s.shape == (5, kb) and s.stride() == (1, 5)
    assert q.untyped_storage().nbytes() == 5 * ld
    w, s_w = rt.quantize_fp8_block(half(200, K), rows=128)
    assert w.stride() == (ld, 1) and s_w.shape == (2, kb) and s_w.is_contiguous()
    lib.calls.clear()
    rt.gemm_fp8_block(q, w, s_w, s)
    (_, _, a), = lib.calls
    assert a[:4] == (q.data_ptr(), w.data_ptr(), s.data_ptr(), s_w.data_ptr()) and a[4] is None
    assert list(a[6]) == [5, K, 200, ld, ld, 200, 1, 5, kb, 1, 0, 1]


def test_operands_that_need_a_copy(lib):  # noqa: F811
    x = torch.arange(5 * 301, dtype=torch.uint8).view(5, 301)[:, 1:].view(E4M3)
    rt.gemm_fp8_block(x, e4m3(200, 300), scales(2, 3), scales(5, 3))
    (_, _, a), = lib.calls
    assert a[0] != x.data_ptr() and a[0] % 16 == 0 and list(a[6])[3:5] == [304, 304]
    assert torch.equal(rt._fp8_rows(x, 300).view(torch.uint8), x.view(torch.uint8))


@pytest.mark.parametrize("shape,strides,want", [
    ((2, 6, 7, 48), None, (2016, 48)), ((2, 48), (48, 1), (48, 48)), ((2, 5, 48), (4800, 96, 1), (4800, 96)),
])
def test_norm_rows(lib, shape, strides, want):  # noqa: F811
    x = half(*shape) if strides is None else torch.zeros(20000, dtype=torch.float16).as_strided(shape, strides)
    y = rt.group_norm(x, 4)
    (_, _, a), = [c for c in lib.calls if c[0] == "ic_group_norm"]
    assert a[0] == x.data_ptr() and tuple(a[8])[4:6] == want and y.is_contiguous() and y.shape == shape


def test_empty(lib):  # noqa: F811
    q, s = rt.quantize_fp8_block(half(3, 0, 300))
    assert q.shape == (3, 0, 300) and s.shape == (3, 0, 3)
    assert product(x=e4m3(0, 300), s_a=scales(0, 3)).shape == (0, 200)
    assert product(w=e4m3(0, 300), s_w=scales(0, 3)).shape == (4, 0)
    assert rt.group_norm(half(0, 5, 64), 4).shape == (0, 5, 64)
    q, s = rt.fused_groupnorm_quantize(half(2, 0, 64), 4)
    assert q.shape == (2, 0, 64) and s.shape == (2, 0, 1)
    assert not [c for c in lib.calls if not c[0].endswith("workspace")]


@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (200, 300), (257, 129)])
def test_weight_quantiser(N, K):
    """Every value is within half a step of e4m3 at its block's scale."""
    g = torch.Generator().manual_seed(N)
    w = torch.randn(N, K, generator=g)
    q, s = qu.quantize_weights_fp8(w)
    assert q.shape == (N, K) and q.dtype is E4M3 and s.shape == (-(-N // 128), -(-K // 128))
    each = s.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    back = q.float() * each
    assert ((back - w).abs() <= 2.0 ** -4 * w.abs() + 2.0 ** -10 * each).all()
    assert (q.float().abs() <= 448).all()
    with pytest.raises(ValueError, match="2D"):
        qu.quantize_weights_fp8(w[0])


@pytest.mark.parametrize("K", [256, 300])
def test_module_on_the_host(K):
    lin = torch.nn.Linear(K, 200)
    m = conv.ConvLinearFP8.from_float(lin)
    q, s = qu.quantize_weights_fp8(lin.weight.detach())
    assert m.weight.shape == (200, -(-K // 16) * 16) and torch.equal(m.weight[:, :K].float(), q.float())
    assert (m.weight[:, K:].float() == 0).all() and torch.equal(m.scale, s)
    m.half()                               # a cast of the model leaves values and scales alone
    assert m.weight.dtype is E4M3 and m.scale.dtype is torch.float32 and m.bias.dtype is torch.float16
    again = conv.ConvLinearFP8(m.weight, m.scale, bias=m.bias, in_features=K)
    again.load_state_dict(m.state_dict())
    assert again.in_features == K and again.out_features == 200
    with pytest.raises(RuntimeError, match="B200 kernels"):
        m(torch.zeros(2, K))
    with pytest.raises(ValueError, match="power of 2"):
        conv.ConvLinearFP8.from_float(lin, rot_need=True, rot_size=100)
