"""Host side of the runtime's calls without a GPU: the library is a stub that
records what it is called with, the devices are stand-ins."""

import types

import pytest
import torch

from _pkg import load

rt = load("_b200_runtime")


@pytest.fixture
def lib(monkeypatch):
    """Two devices, 0 current and all tensors on 1; the library records (entry
    point, current device, arguments) and answers 0."""
    state = types.SimpleNamespace(current=0, calls=[])

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state.current = state.current, self.index

        def __exit__(self, *exc):
            state.current = self.before

    class Library:
        def __getattr__(self, name):
            def entry(*args):
                state.calls.append((name, state.current, args))
                return 0
            return entry

    library = Library()
    monkeypatch.setattr(rt, "B200_LIBRARY_LOADED", True)
    monkeypatch.setattr(rt.L, "lib", lambda: library)
    monkeypatch.setattr(rt, "_need_cuda", lambda what, *ts: None)
    monkeypatch.setattr(rt, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(rt, "_stream", lambda t: 0)
    monkeypatch.setattr(rt, "_num_sms", lambda device: 148)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1)
    monkeypatch.setattr(rt, "_current_device", lambda: state.current)
    monkeypatch.setattr(torch.cuda, "device", Device)
    rt._workspace.cache_clear()
    yield state
    rt._workspace.cache_clear()


def half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


ATTENTION_SIDE = {
    "qk_norm_rope": lambda: rt.qk_norm_rope(half(1, 2, 4, 64), half(1, 2, 4, 64)),
    "cross_attention": lambda: rt.cross_attention(half(1, 2, 4, 64), k=half(1, 3, 4, 64), v=half(1, 3, 4, 64)),
    "cross_attention, by name": lambda: rt.cross_attention(v=half(1, 3, 4, 64), scale=1.0, k=half(1, 3, 4, 64), q=half(1, 2, 4, 64)),
    "lora_batched": lambda: rt.lora_batched(half(4, 64), half(2, 8, 64), half(2, 32, 8), torch.zeros(4, dtype=torch.int32)),
}


def int8(*shape):
    return torch.zeros(*shape, dtype=torch.int8)


def packed(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


QUANTISED = {
    "prep_quantize": lambda: rt.prep_quantize(half(4, 64)),
    "dynamic_quantize_activation": lambda: rt.dynamic_quantize_activation(half(4, 64)),
    "fused_rmsnorm_quantize": lambda: rt.fused_rmsnorm_quantize(half(4, 64), torch.ones(64)),
    "gemm_a8": lambda: rt.gemm_a8(int8(4, 64), int8(32, 64), torch.ones(32), torch.ones(4), splits=1),
    "fused_int8_gemm_dequant": lambda: rt.fused_int8_gemm_dequant(int8(4, 64), int8(32, 64), torch.ones(32), torch.ones(4)),
    "int8_gemm_int8out": lambda: rt.int8_gemm_int8out(int8(4, 64), int8(32, 64), torch.ones(32), torch.ones(4)),
    "gemm_w4a16": lambda: rt.gemm_w4a16(half(4, 64), packed(32, 32), torch.ones(32, 1)),
    "lowrank_down": lambda: rt.lowrank_down(half(4, 64), half(8, 64)),
    "lowrank_add": lambda: rt.lowrank_add(half(4, 32), half(4, 8), half(32, 8), 1.0),
    "quantize_weight": lambda: rt.quantize_weight(torch.zeros(32, 64), 8),
    "lokr_add": lambda: rt.lokr_add(half(4, 32), half(4, 64), half(4, 8), half(8, 8), 1.0),
    "repack_int4": lambda: rt.repack_int4(packed(32, 32), 64, rt.L.IC_W_INT4R),
    "unpack_int4_to_int8": lambda: rt.unpack_int4_to_int8(packed(32, 32), 64),
    "unpack_int4_to_float16": lambda: rt.unpack_int4_to_float16(packed(32, 32), torch.ones(32, 1), 64),
}


@pytest.mark.parametrize("call", [*ATTENTION_SIDE, *QUANTISED])
def test_calls_run_on_the_tensors_device(lib, call):
    """Every entry point, the workspace sizes among them, is called with the
    tensors' device current; the caller's is back afterwards."""
    {**ATTENTION_SIDE, **QUANTISED}[call]()
    assert lib.calls and {device for _, device, _ in lib.calls} == {1}
    assert lib.current == 0


@pytest.mark.parametrize("call", ATTENTION_SIDE)
def test_the_current_device_is_not_switched(lib, monkeypatch, call):
    lib.current = 1
    monkeypatch.setattr(torch.cuda, "device", None)
    ATTENTION_SIDE[call]()
    assert {device for _, device, _ in lib.calls} == {1}


def test_the_device_is_back_after_a_refusal(lib):
    with pytest.raises(TypeError, match="float16/bfloat16"):
        rt.qk_norm_rope(torch.zeros(1, 2, 4, 64))
    assert lib.current == 0 and not lib.calls


def test_device_error_reads_the_device_it_is_asked_for(lib):
    rt.device_error(device=1)
    assert [(name, device) for name, device, _ in lib.calls] == [("ic_read_device_error", 1)]
    assert lib.current == 0


# ── index tensors ────────────────────────────────────────────────────────────

@pytest.mark.parametrize("dtype,values,want", [
    (torch.int64, [2**63 - 1, 2**32 + 1, 2**31, 2**31 - 1, 5, 0, -1, -2**32 + 3, -2**63],
     [2**31 - 1, 2**31 - 1, 2**31 - 1, 2**31 - 1, 5, 0, -1, -2**31, -2**31]),
    (torch.uint64, [2**63 + 1, 2**64 - 1, 2**32 + 1, 9], [2**31 - 1, 2**31 - 1, 2**31 - 1, 9]),
    (torch.uint32, [2**32 - 1, 2**31 + 1, 9], [2**31 - 1, 2**31 - 1, 9]),
    (torch.int16, [-3, 7], [-3, 7]), (torch.uint8, [255, 0], [255, 0]),
])
def test_index_tensors_saturate(dtype, values, want):
    """Narrowing keeps what is out of range out of range (2^32 + 1 is not 1)."""
    got = rt._index(torch.tensor(values, dtype=dtype))
    assert got.dtype == torch.int32 and got.tolist() == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bool, torch.complex64])
def test_index_tensors_hold_integers(dtype):
    with pytest.raises(TypeError, match="integers"):
        rt._index(torch.zeros(2, dtype=dtype))


# ── strides that say nothing ─────────────────────────────────────────────────

def one_sample(batch_stride, L=5, H=3, D=16):
    """[1, L, H, D] cut from a buffer whose samples are batch_stride apart."""
    return torch.zeros(2 * batch_stride, dtype=torch.float16).as_strided((2, L, H, D), (batch_stride, H * D, D, 1))[:1]


@pytest.mark.parametrize("call", ["qk_norm_rope", "cross_attention"])
def test_strides_of_dimensions_of_one_entry(lib, call):
    """A batch of one may have any batch stride: nothing is copied, and the
    library gets strides that it takes (multiples of 8)."""
    t, out = one_sample(5 * 3 * 16 + 1), one_sample(5 * 3 * 16 + 3)
    assert t.stride(0) % 8 and out.stride(0) % 8
    if call == "qk_norm_rope":
        y = rt.qk_norm_rope(t, q_out=out)
        (_, _, args), = [c for c in lib.calls if c[0] == "ic_qk_norm_rope"]
        tensors, strides = (args[0], args[1]), list(args[10])
    else:
        y = rt.cross_attention(t, t, t, out=out)
        (_, _, args), = [c for c in lib.calls if c[0] == "ic_cross_attention"]
        tensors, strides = (args[0], args[3]), list(args[11])
    assert y is out
    assert tensors == (t.data_ptr(), out.data_ptr())
    assert all(s % 8 == 0 for s in strides)
    assert strides[:3] == [0, 48, 16] and [0, 48, 16] in (strides[3:6], strides[9:])


def test_strides_that_need_a_copy(lib):
    """Rows at odd addresses are copied to a layout of their own, also where
    torch calls them contiguous; out is refused."""
    buf = torch.arange(2 + 5 * 3 * 16, dtype=torch.float16)
    buf = buf[1:] if buf.data_ptr() % 16 == 0 else buf
    odd = buf[:5 * 3 * 16].as_strided((1, 5, 3, 16), (7, 48, 16, 1))
    assert odd.is_contiguous() and odd.data_ptr() % 16
    got = rt._heads(odd)
    assert torch.equal(got, odd) and got.stride() == (240, 48, 16, 1) and got.data_ptr() % 16 == 0
    with pytest.raises(ValueError, match="out must have contiguous"):
        rt.qk_norm_rope(odd, q_out=odd)
    rows = torch.zeros(2, 5, 3, 17, dtype=torch.float16)[..., :16]
    assert rt._heads(rows).stride() == (240, 48, 16, 1)
    with pytest.raises(ValueError, match="out must have contiguous"):
        rt.qk_norm_rope(rows, q_out=rows)
    with pytest.raises(ValueError, match="out must have contiguous"):
        rt.qk_norm_rope(rows, q_out=torch.zeros(1, 5, 3, 16, dtype=torch.float16).expand(2, 5, 3, 16))


# ── empty sizes ──────────────────────────────────────────────────────────────

@pytest.mark.parametrize("lead,N", [((2, 3), 0), ((), 0), ((0, 3), 0), ((0, 3), 32), ((2, 0), 32)])
@pytest.mark.parametrize("with_base,with_out", [(False, False), (True, False), (True, True)])
def test_adapters_of_empty_sizes(lib, lead, N, with_base, with_out):
    """No rows or no columns: an empty result, nothing launched."""
    x, base, out = half(*lead, 64), half(*lead, N), half(*lead, N)
    rows = x.numel() // 64
    y = rt.lora_batched(x, half(2, 8, 64), half(2, N, 8), torch.zeros(rows, dtype=torch.int32),
                        base=base if with_base else None, out=out if with_out else None)
    assert y.shape == (*lead, N) and not lib.calls


@pytest.mark.parametrize("lead", [(), (6,), (2, 3), (1, 2, 3)])
def test_adapter_rows(lib, lead):
    """Leading dimensions fold into rows."""
    x = half(*lead, 64)
    rows = x.numel() // 64
    y = rt.lora_batched(x, half(2, 8, 64), half(2, 32, 8), torch.zeros(rows, dtype=torch.int32), base=half(*lead, 32))
    (_, _, args), = [c for c in lib.calls if c[0] == "ic_lora_batched"]
    assert y.shape == (*lead, 32) and args[2:5] == (rows, 64, 64) and args[0] == x.data_ptr()
