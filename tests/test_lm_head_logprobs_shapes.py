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


@pytest.mark.parametrize("vocab,rows", [(3, (1 << 20) + 5), (40, (1 << 20) + 5), (3, 100), (100_000, 3000)])
@pytest.mark.parametrize("adapted", [True, False])
def test_rows_of_a_step(monkeypatch, vocab, rows, adapted):
    """Logits are formed for as many rows at a time as every call on the way takes."""
    steps = []

    def logits(x, w, *, adapters, adapter_ids, **kw):
        assert (adapter_ids is not None) == adapted and (not adapted or adapter_ids.shape == x.shape[:1])
        steps.append(x.shape[0])
        return x

    def scored(logits, tokens, *, num_top, entropy):
        return nvjsel.TokenLogprobs(tokens.float(), None, None, None)

    monkeypatch.setattr(module, "lm_head_logits_hip", logits)
    monkeypatch.setattr(module, "token_logprobs", scored)
    tokens = torch.arange(rows)
    ids = torch.zeros(rows, dtype=torch.int32) if adapted else None
    r = module._scored_by_logits(torch.zeros(1, 2).expand(rows, 2), torch.zeros(2, vocab), tokens, 0, False, None, None,
                                 object() if adapted else None, ids)
    assert torch.equal(r[0], tokens.float()) and sum(steps) == rows
    assert max(steps) <= (1 << 20) and max(steps) * vocab * 4 <= max(1 << 28, 64 * vocab * 4)
    assert len(steps) == -(-rows // max(steps))


@pytest.mark.gpu
def test_more_rows_than_adapters_take():
    rows = (1 << 20) + 70
    g = torch.Generator().manual_seed(6)
    x = torch.randn(rows, 8, generator=g).to(torch.bfloat16)
    w = torch.randn(5, 8, generator=g).to(torch.bfloat16)
    a, b = torch.randn(1, 2, 8, generator=g).to(torch.bfloat16), torch.randn(1, 5, 2, generator=g).to(torch.bfloat16)
    t = torch.randint(0, 5, (rows,), generator=g)
    table = nvjsel.pack_adapters(a.cuda(), b.cuda())
    ids = (torch.arange(rows) % 2 - 1).to(torch.int32)
    r = nvjsel.lm_head_token_logprobs(x.cuda(), w.cuda(), t.cuda(), weight_layout="vh", reduce_cast=0, adapters=table,
                                      adapter_ids=ids.cuda())
    l = x.double() @ w.double().T + (ids == 0).double()[:, None] * ((x.double() @ a[0].double().T) @ b[0].double().T)
    want = torch.log_softmax(l, 1).gather(1, t[:, None])[:, 0]
    # fp32 sums of 8, 8 and 2 products (each addition 2^-23 of the magnitudes), y's terms 2^-21
    xs = x.double().abs()
    size = xs @ w.double().abs().T + (xs @ a[0].double().abs().T) @ b[0].double().abs().T
    off = size.amax(1) * 30 * 2.0 ** -23
    assert bool(((r.logprobs.double().cpu() - want).abs() <= 2 * off + 2.0 ** -19 + want.abs() * 2.0 ** -24).all())
