"""No log probability is above 0: a row with one token left, and tokens that are next to certain."""
from __future__ import annotations

import math

import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = math.inf


def _values(dtype):
    """Logits of one token left: a sixteenth apart, and any, far ones among them."""
    g = torch.Generator().manual_seed(3)
    far = [0.0, 1.0, -1.0, 100.0, -15000.0, 16000.0, 16384.0, 40000.0, -40000.0]
    return torch.cat([torch.arange(-600, 600) / 16, torch.randn(800, generator=g) * 20, torch.tensor(far)]).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("vocab,rows", [(1, None), (700, None), (50257, 6), (50257, 100)])
def test_one_token_left(dtype, top, vocab, rows):
    """Its log probability is 0, its entropy 0, and the gradients are 0."""
    v = _values(dtype)[slice(None) if rows is None else slice(0, None, 2009 // rows)]
    at = torch.arange(v.numel()) * 37 % vocab
    x = torch.full((v.numel(), vocab), -INF, dtype=v.dtype)
    x[torch.arange(v.numel()), at] = v
    leaf = x.cuda().requires_grad_()
    r = nvjsel.token_logprobs(leaf, at.cuda(), num_top=top, entropy=True)
    # S is at most 1 + 2^-19 (its tolerance), so the log probability at least -2^-19; at most 0
    assert bool((r.logprobs <= 0).all()) and bool((r.logprobs >= -(2.0 ** -19)).all())
    assert bool((r.entropy >= 0).all()) and bool((r.entropy <= 2.0 ** -18).all())
    if top:
        assert torch.equal(r.top_logprobs[:, 0], r.logprobs.detach())
        assert bool((r.top_logprobs[:, 1:] == -INF).all()) and torch.equal(r.top_ids[:, 0].cpu().long(), at)
    d, = torch.autograd.grad(r.logprobs.sum(), leaf)
    # g (1 - p) with p = exp(logprob), at least 1 - 2^-19, and its own rounding
    assert bool((d >= -(2.0 ** -22)).all()) and bool((d <= 2.0 ** -18).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("top", [0, 2])
def test_next_to_certain(dtype, top):
    """One logit 17 and more above a few others: 1 - p is below a rounding of 1."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(500, 40, generator=g)
    at = torch.randint(0, 40, (500,), generator=g)
    x[torch.arange(500), at] = 20 + 20 * torch.rand(500, generator=g)
    x = x.to(DT[dtype])
    r = nvjsel.token_logprobs(x.cuda(), at.cuda(), num_top=top)
    want = torch.log_softmax(x.double(), 1).gather(1, at[:, None])[:, 0]
    for got in [r.logprobs] + ([r.top_logprobs[:, 0]] if top else []):
        assert bool((got <= 0).all()) and bool(((got.double().cpu() - want).abs() <= 2.0 ** -19).all())


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
def test_scores(act):
    """From the hidden states: one row of the table far above the others."""
    g = torch.Generator().manual_seed(5)
    wt = torch.float16 if act == "f16" else torch.bfloat16
    w = (torch.randn(3000, 64, generator=g) * 0.02).to(wt)
    t = torch.randint(0, 3000, (300,), generator=g)
    x = (w[t].float() * 40 / (64 * 4e-4)).to(DT[act])
    for cast in (0, None):
        r = nvjsel.lm_head_token_logprobs(x.cuda(), w.cuda(), t.cuda(), weight_layout="vh", entropy=True, reduce_cast=cast)
        assert bool((r.logprobs <= 0).all()) and bool((r.entropy >= 0).all())
