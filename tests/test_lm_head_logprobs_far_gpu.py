"""Log probabilities from the hidden states: logits next to the largest numbers, whose differences from one
tile of the vocabulary to the next are beyond them once they are in units of log2 e."""
from __future__ import annotations

import math

import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cast", [0, None])
@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(3, 70001), (40, 70001), (130, 140003), (2100, 9001)])
def test_maxima_that_rise_by_almost_all(rows, vocab, act, cast):
    """One logit in a hundred is 1e38, the others -2e38: the entropy is ln of their number, to the tolerance of other
    rows; a row of one such logit has none."""
    g = torch.Generator().manual_seed(vocab)
    high = torch.rand(vocab, generator=g) < 0.01
    w = torch.zeros(vocab, 64)
    w[:, 0] = torch.where(high, 1e38, -2e38)
    w[:, 1] = -2e38
    w[vocab - 2, 1] = 1e38
    x = torch.zeros(rows, 64)
    x[:, 0] = 1.0
    x[rows // 2] = 0.0
    x[rows // 2, 1] = 1.0
    t = torch.full((rows,), int(high.nonzero()[7]))
    t[rows // 2] = vocab - 2
    dt = torch.bfloat16 if act == "bf16" else torch.float32
    r = nvjsel.lm_head_token_logprobs(x.to(dt).cuda(), w.to(torch.bfloat16).cuda(), t.cuda(), weight_layout="vh", entropy=True,
                                      reduce_cast=cast)
    n = torch.full((rows,), math.log(int(high.sum())), dtype=torch.float64)
    n[rows // 2] = 0.0
    assert bool(((r.logprobs.double().cpu() + n).abs() <= 2.0 ** -19 + n * 2.0 ** -24).all())
    tol = 2 * 2.0 ** -19 * (2 + 2 * math.log(vocab)) + n * 2.0 ** -24
    assert bool(((r.entropy.double().cpu() - n).abs() <= tol).all())
