"""Rotary scalings that lack something or make no frequencies are refused with a ValueError (CPU)."""

from __future__ import annotations

import math

import pytest
import torch

from plastic_infer.kernel.rotary import rope_params

YARN = {"type": "yarn", "factor": 2.0, "original_length": 4096}


@pytest.mark.parametrize("kw", [
    dict(scaling={"type": "linear"}), dict(scaling={"type": "ntk"}), dict(scaling={}),
    dict(scaling={"type": "yarn", "factor": 2.0}), dict(scaling={"type": "yarn", "original_length": 9}),
    dict(scaling={"type": "linear", "factor": math.inf}),
    dict(scaling={"type": "ntk", "factor": math.nan}), dict(base=math.inf), dict(base=math.nan),
    dict(scaling=YARN | {"beta_slow": 0}), dict(scaling=YARN | {"beta_slow": -1.0}),
    dict(scaling=YARN | {"beta_fast": 1, "beta_slow": 32}), dict(scaling=YARN | {"beta_fast": math.inf})])
def test_refused(kw):
    with pytest.raises(ValueError):
        rope_params(128, device=torch.device("cpu"), **kw)


def test_equal_betas_make_a_step():
    turns = rope_params(64, scaling=YARN | {"beta_fast": 4, "beta_slow": 4},
                        device=torch.device("cpu")).turns
    plain = rope_params(64, device=torch.device("cpu")).turns
    ratio = (plain / turns).tolist()
    assert ratio[0] == 1.0 and abs(ratio[-1] - 2.0) < 1e-12 and sorted(ratio) == ratio
