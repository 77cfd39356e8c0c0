"""pack_adapters refuses scales that want a gradient, as it refuses a and b."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import nvjsel

B16 = torch.bfloat16


def _pack(scales):
    return nvjsel.pack_adapters(torch.zeros(2, 4, 8, dtype=B16), torch.zeros(2, 6, 4, dtype=B16), scales)


@pytest.mark.parametrize("scales", [torch.ones(2, requires_grad=True), torch.ones(2, requires_grad=True) * 2,
                                    [torch.ones((), requires_grad=True), torch.ones(())], (1.0, torch.ones((), requires_grad=True))],
                         ids=["leaf", "result", "list", "mixture"])
def test_refused(scales):
    with pytest.raises(ValueError, match="not differentiable"):
        _pack(scales)
    with torch.no_grad(), pytest.raises(ValueError, match="device tensors"):
        _pack(scales)


@pytest.mark.parametrize("scales", [torch.ones(2), [1.0, 2.0], (1, 2), np.ones(2), np.float32(2), 2.0, None])
def test_taken(scales):
    with pytest.raises(ValueError, match="device tensors"):
        _pack(scales)


def test_a_tangent_is_refused():
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        _pack(forward_ad.make_dual(torch.ones(2), torch.ones(2)))
