"""Outputs whose rows share elements are refused, by the runtime and at the C entry
point; those that lie between one another are not."""

import itertools

import pytest
import torch

from _pkg import load
from test_cpu_attention_runtime import lib  # noqa: F401  (the stub library on two devices)
from test_cpu_fp8_abi import norm, refused

rt = load("_b200_runtime")


def test_against_every_element():
    for B, L, C in [(1, 1, 3), (1, 4, 2), (5, 1, 2), (2, 5, 4), (3, 4, 2), (4, 3, 3), (6, 2, 5), (2, 2, 1)]:
        for far, near in itertools.product(range(0, 26), repeat=2):
            at = [b * far + l * near + c for b in range(B) for l in range(L) for c in range(C)]
            assert rt._overlap(B, far, L, near, C) == (len(set(at)) < len(at)), (B, L, C, far, near)


def strided(*strides):
    return torch.zeros(100000, dtype=torch.float16).as_strided((2, 5, 64), (*strides, 1))


@pytest.mark.parametrize("strides", [(64, 64), (320 - 8, 64), (128, 64), (160, 128), (64, 100), (63, 64 * 5), (136, 128)])
def test_runtime_refuses(lib, strides):  # noqa: F811
    with pytest.raises(ValueError, match="overlap"):
        rt.group_norm(torch.zeros(2, 5, 64, dtype=torch.float16), 4, out=strided(*strides))


@pytest.mark.parametrize("strides", [(320, 64), (64, 128), (1000, 71), (80, 200), (192, 128), (64 * 5, 128)])
def test_runtime_takes_what_lies_between(lib, strides):  # noqa: F811
    out = strided(*strides)
    assert rt.group_norm(torch.zeros(2, 5, 64, dtype=torch.float16), 4, out=out) is out
    (_, _, a), = [c for c in lib.calls if c[0] == "ic_group_norm"]
    assert tuple(a[8])[10:12] == strides


@pytest.mark.parametrize("change", [
    dict(y_batch=64), dict(y_batch=64 * 16 - 8), dict(y_batch=128), dict(y_batch=160, y_row=128), dict(y_batch=64, y_row=100),
    dict(B=1 << 10, L=1 << 10, y_batch=(1 << 62) + 5, y_row=1 << 62),        # strides whose multiples no int64 holds
])
def test_entry_point_refuses(change):
    refused(norm(**change), 1, "overlaps")
