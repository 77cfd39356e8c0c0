"""Log probabilities from the hidden states: the results' shapes, on both routes, with the launches
replaced; and the same on the GPU."""
from __future__ import annotations

import pytest
import torch

import nvjsel
from nvjsel import logprobs as module
from nvjsel._tensors import _HERE


@pytest.mark.parametrize("shape", [(), (1,), (3,), (2, 3)])
@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("entropy", [False, True])
def test_shapes(monkeypatch, shape, top, entropy):
    def results(x, w, tokens, *rest):
        assert x.shape == (tokens.numel(), 8) and tokens.ndim == 1
        n = tokens.numel()
        return [torch.zeros(n), torch.ones(n) if entropy else None, torch.zeros(n, top) if top else None,
                torch.zeros(n, top, dtype=torch.int32) if top else None]

    monkeypatch.setattr(module, "_require_cuda", lambda *ts: ts[0].device)
    monkeypatch.setattr(module, "_on_device", lambda device: _HERE)
    monkeypatch.setattr(module, "_scored", results)
    monkeypatch.setattr(module, "_scored_by_logits", results)
    r = nvjsel.lm_head_token_logprobs(torch.zeros(*shape, 8), torch.zeros(8, 30), torch.zeros(shape, dtype=torch.int64),
                                      num_top=top, entropy=entropy)
    assert r.logprobs.shape == shape and (r.entropy is None) == (not entropy)
    assert r.entropy is None or r.entropy.shape == shape
    assert (r.top_ids is None) == (top == 0) and (top == 0 or r.top_ids.shape == r.top_logprobs.shape == (*shape, top))


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [64, 72])  # without logits, by logits
def test_one_hidden_vector(hidden):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(hidden, generator=g).to(torch.bfloat16).cuda()
    w = (torch.randn(300, hidden, generator=g) / 8).to(torch.bfloat16).cuda()
    table = nvjsel.pack_adapters(torch.ones(1, 4, hidden, dtype=torch.bfloat16, device="cuda"),
                                 torch.ones(1, 300, 4, dtype=torch.bfloat16, device="cuda"))
    for kw in ({}, {"num_top": 3}, {"adapters": table, "adapter_ids": torch.zeros((), dtype=torch.int32, device="cuda")}):
        rows = {**kw, "adapter_ids": kw["adapter_ids"][None]} if "adapters" in kw else kw
        token = torch.tensor(17, device="cuda")
        one = nvjsel.lm_head_token_logprobs(x, w, token, weight_layout="vh", entropy=True, **kw)
        row = nvjsel.lm_head_token_logprobs(x[None], w, token[None], weight_layout="vh", entropy=True, **rows)
        assert one.logprobs.shape == one.entropy.shape == ()
        assert torch.equal(one.logprobs, row.logprobs[0]) and torch.equal(one.entropy, row.entropy[0])
        if "num_top" in kw:
            assert torch.equal(one.top_ids, row.top_ids[0]) and torch.equal(one.top_logprobs, row.top_logprobs[0])
