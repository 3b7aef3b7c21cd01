"""What a backward pass of the rotary map turns."""

from __future__ import annotations

import pytest
import torch

from plastic_infer.kernel import rotary as R
from plastic_infer.kernel.rotary import rope_params, rotary_embed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("needs", ["q", "k", "qk"])
def test_only_needed_gradients_are_turned(dev, needs, monkeypatch):
    q, k = torch.ones(4, 2, 16, device=dev), torch.ones(4, 1, 16, device=dev)
    q.requires_grad_("q" in needs)
    k.requires_grad_("k" in needs)
    pos = torch.arange(4, device=dev)
    qo, ko = rotary_embed(q, k, pos, rope_params(16, device=dev))
    turned, launch = [], R._launch

    def count(a, b, *args):
        turned.append((a is not None, b is not None))
        return launch(a, b, *args)

    monkeypatch.setattr(R, "_launch", count)
    (qo.sum() + ko.sum()).backward()
    assert turned == [("q" in needs, "k" in needs)]
    assert (q.grad is not None) == ("q" in needs) and (k.grad is not None) == ("k" in needs)
