"""Sections of rotary positions are counts of pairs, on the CPU."""

from __future__ import annotations

import math

import pytest
import torch

from plastic_infer.kernel.rotary import rope_params

CPU = torch.device("cpu")


@pytest.mark.parametrize("bad", [(2.9, 3, 3), (2.5, 2.5, 3), (8.5,), (0.5, 8, 0), (math.nan, 8), (math.inf, 0),
                                 (8, -math.inf)])
def test_parts_of_a_pair_are_refused(bad):
    with pytest.raises(ValueError, match="sections must be counts"):
        rope_params(16, sections=bad, device=CPU)


@pytest.mark.parametrize("same", [(2, 3, 3), [2.0, 3.0, 3.0], torch.tensor([2, 3, 3])])
def test_whole_counts_of_any_type(same):
    assert rope_params(16, sections=same, device=CPU).axes.tolist() == [0, 0, 1, 1, 1, 2, 2, 2]
