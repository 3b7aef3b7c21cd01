"""Rotary parameters of several axes, on the CPU."""

from __future__ import annotations

import pytest
import torch

from plastic_infer import _native as N
from plastic_infer.kernel.rotary import rope_params

CPU = torch.device("cpu")


def test_sections_name_the_axis_of_each_pair():
    p = rope_params(16, sections=(2, 0, 6), device=CPU)
    assert p.axes.tolist() == [0, 0, 2, 2, 2, 2, 2, 2] and p.axes.dtype == torch.int32
    assert torch.equal(p.turns, rope_params(16, device=CPU).turns)
    assert rope_params(16, device=CPU).axes is None


@pytest.mark.parametrize("bad", [(), (4, 3), (9, -1), (8, 8)])
def test_sections_add_up_to_the_pairs(bad):
    with pytest.raises(ValueError, match="sections"):
        rope_params(16, sections=bad, device=CPU)


def test_the_library_refuses_before_any_launch():
    some = 1 << 20   # never dereferenced: every call below fails its checks first

    def call(num_axes, axes, pairs=2, heads=1):
        N.call("pia_rotary_axes", some, None, some, None, 8, 8, 0, 0, some, 1, axes, num_axes, some,
               pairs, 1.0, 0, 0, 4, heads, 0, 8, 0, None)

    for args in ((0, some), (-1, some), (2, None), (2, some, 5)):
        with pytest.raises(N.NativeError):
            call(*args)
