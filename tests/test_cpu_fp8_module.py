"""The e4m3 module's buffers on the host: moves, casts and state dicts."""

import pytest
import torch

from _pkg import load

conv = load("convlinear")
E4M3 = torch.float8_e4m3fn


def module(K, bias=True):
    torch.manual_seed(K)
    return conv.ConvLinearFP8.from_float(torch.nn.Linear(K, 200, bias=bias))


def same(a, b):
    return (torch.equal(a.weight.view(torch.uint8), b.weight.view(torch.uint8)) and torch.equal(a.scale, b.scale)
            and (a.bias is None) == (b.bias is None) and (a.bias is None or torch.equal(a.bias, b.bias)))


@pytest.mark.parametrize("K", [256, 300])
def test_deferred_loading(K):
    """Empty on the meta device, memory for it, then values."""
    m = module(K)
    state = {k: v.clone() for k, v in m.state_dict().items()}
    empty = module(K).to("meta")
    assert empty.weight.is_meta and empty.weight.dtype is E4M3 and empty.scale.dtype is torch.float32
    empty = empty.to_empty(device="cpu")
    assert empty.weight.shape == m.weight.shape and empty.weight.dtype is E4M3
    empty.load_state_dict(state)
    assert same(empty, m)


@pytest.mark.parametrize("cast", [
    lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.float16), lambda m: m.to("cpu", torch.bfloat16),
    lambda m: m.type(torch.float16), lambda m: torch.nn.Sequential(m).half()[0], lambda m: m.share_memory(),
])
def test_casts_leave_values_and_scales_alone(cast):
    m, want = module(300), module(300)
    got = cast(m)
    assert got.weight.dtype is E4M3 and got.scale.dtype is torch.float32
    want.bias = want.bias.to(got.bias.dtype)
    assert same(got, want)


def test_a_cast_makes_no_copies():
    """No cast of the weight that is thrown away, and no second copy of it."""
    m = module(300)
    at = m.weight.data_ptr(), m.scale.data_ptr()
    seen = []
    m._apply(lambda t: (seen.append((t.dtype, t.is_floating_point())), t.half() if t.is_floating_point() else t)[1])
    assert (m.weight.data_ptr(), m.scale.data_ptr()) == at
    assert sum(floating for _, floating in seen) == 1        # the bias


def test_a_failing_move_leaves_the_module_as_it_was():
    m = module(300)
    want = module(300)

    def fail(t):
        raise RuntimeError("no memory")

    with pytest.raises(RuntimeError, match="no memory"):
        m._apply(fail)
    assert m.weight.dtype is E4M3 and same(m, want)


@pytest.mark.parametrize("assign", [False, True])
@pytest.mark.parametrize("K", [1, 256, 300])
def test_state_dict_holds_the_weight_as_checkpoints_do(K, assign):
    m = module(K)
    state = {k: v.clone() for k, v in torch.nn.Sequential(m).state_dict().items()}
    assert state["0.weight"].shape == (200, K) and state["0.weight"].dtype is E4M3 and state["0.weight"].is_contiguous()
    before = dict(state)
    for deferred in (False, True):
        other = conv.ConvLinearFP8.from_float(torch.nn.Linear(K, 200))
        holder = torch.nn.Sequential(other.to("meta") if deferred and assign else other)
        assert not any(holder.load_state_dict(state, assign=assign))
        assert holder[0].weight.stride() == (-(-K // 16) * 16, 1) and same(holder[0], m)
    assert all(state[k] is before[k] for k in state)
    filled = dict(state)                       # as the module holds it
    filled["0.weight"] = m.weight
    other = conv.ConvLinearFP8.from_float(torch.nn.Linear(K, 200))
    torch.nn.Sequential(other).load_state_dict(filled, assign=assign)
    assert same(other, m)


def test_a_weight_of_another_shape_does_not_load():
    for shape in [(200, 299), (199, 300), (200, 300, 1)]:
        state = {**module(300).state_dict(), "weight": torch.zeros(shape, dtype=torch.uint8).view(E4M3)}
        with pytest.raises(RuntimeError, match="size mismatch"):
            module(300).load_state_dict(state)
