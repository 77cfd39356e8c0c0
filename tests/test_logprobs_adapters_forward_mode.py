"""Forward mode's tangents are refused by the entry points that would leave them behind, in any gradient mode."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import nvjsel

B16 = torch.bfloat16


def _calls():
    """Every entry point with each of its tensors that may carry a tangent, the others without."""
    t = torch.zeros(3, dtype=torch.int32)
    table = nvjsel.AdapterTable(torch.zeros(2, 512, dtype=B16), torch.zeros(2, 1024, dtype=B16), torch.zeros(2), 8, 6, 16)
    x, base = torch.zeros(3, 8), torch.zeros(3, 6)
    a, b = torch.zeros(2, 4, 8, dtype=B16), torch.zeros(2, 6, 4, dtype=B16)
    head, norm = torch.zeros(8, 6), torch.zeros(8)
    yield "logits", base, lambda d: nvjsel.token_logprobs(d, t)
    yield "logits with alternatives", base, lambda d: nvjsel.token_logprobs(d, t, num_top=2, entropy=True)
    yield "hidden", x, lambda d: nvjsel.lm_head_token_logprobs(d, head, t)
    yield "weight", head, lambda d: nvjsel.lm_head_token_logprobs(x, d, t)
    yield "norm weight", norm, lambda d: nvjsel.lm_head_token_logprobs(x, head, t, norm_weight=d)
    yield "x", x, lambda d: nvjsel.apply_adapters(d, base, table, t)
    yield "base", base, lambda d: nvjsel.apply_adapters(x, d, table, t)
    yield "out", base, lambda d: nvjsel.apply_adapters(x, base, table, t, out=d)
    yield "a", a, lambda d: nvjsel.pack_adapters(d, b)
    yield "b", b, lambda d: nvjsel.pack_adapters(list(a), list(d))


@pytest.mark.parametrize("name", [name for name, _, _ in _calls()])
@pytest.mark.parametrize("grad", [True, False])
def test_refused(name, grad):
    tensor, call = next((t, c) for n, t, c in _calls() if n == name)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(ValueError, match="forward-mode"):
            call(forward_ad.make_dual(tensor, torch.ones_like(tensor)))
        with pytest.raises(ValueError, match="device tensors"):  # within a level, without a tangent
            call(tensor)
    with pytest.raises(ValueError, match="device tensors"):
        call(tensor)


def test_refused_with_a_gradient_wanted():
    logits = torch.zeros(3, 6, requires_grad=True)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        nvjsel.token_logprobs(forward_ad.make_dual(logits, torch.ones(3, 6)), torch.zeros(3, dtype=torch.int64))


def test_refused_in_a_jacobian_vector_product():
    t = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda x: nvjsel.token_logprobs(x, t).logprobs, (torch.zeros(3, 6),), (torch.ones(3, 6),))
