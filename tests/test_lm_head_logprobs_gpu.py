"""Log probabilities of given tokens from the hidden states against a plain
64-bit form, on both routes: without logits and by logits of some rows at a
time."""
from __future__ import annotations

import math

import pytest
import torch

import nvjsel
from nvjsel import logprobs as module

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(rows, hidden, vocab, act="bf16", weight="bf16", seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed + rows * 13 + hidden + vocab)
    w = (torch.randn(vocab, hidden, generator=g) * 0.02).to(DT[weight])
    x = torch.randn(rows, hidden, generator=g) * (spread / (0.02 * math.sqrt(hidden)))
    t = torch.randint(0, vocab, (rows,), generator=g)
    x = x + (6.0 / (hidden * 4e-4)) * w[t].float() * (torch.arange(rows) % 2)[:, None]  # half of the tokens likely
    return x.to(DT[act]), w, t


def oracle(x, w, t, cast=None):
    """Results in 64 bits and what fp32 dots may be off by: H products added in any order, each addition 2^-23 of the sum of
    magnitudes (2^-24 rounded to nearest, twice that truncated); rounded logits (``cast``) besides may fall to the other side
    of a rounding."""
    l = x.double() @ w.double().T
    off = (x.double().abs() @ w.double().abs().T) * (x.shape[1] + 2) * 2.0 ** -23
    if cast is not None:
        l = l.to(cast).double()
        off = off + l.abs() * torch.finfo(cast).eps
    m = l.amax(1, keepdim=True)
    s = torch.log(torch.exp(l - m).sum(1, keepdim=True))
    lp = (l - m) - s
    p = torch.exp(lp)
    asked = (t >= 0) & (t < l.shape[1])
    at = t.clamp(0, l.shape[1] - 1)[:, None]
    mean_off = (p * off).sum(1)  # ln S moves by the mean of what its logits move by, as first order has it; twice that here
    lp_tol = off.gather(1, at)[:, 0] + 2 * mean_off
    # the entropy's derivative by l[v] is -p (ln p + entropy)
    ent = -(p * lp).sum(1)
    ent_tol = 2 * (p * off * (lp.abs() + ent[:, None])).sum(1)
    return torch.where(asked, lp.gather(1, at)[:, 0], 0.0), ent, torch.where(asked, lp_tol, 0.0), ent_tol


SUM = 2.0 ** -19  # of the sums of exponentials: the hardware's exp2, its argument and the additions, as for given logits


def check(x, w, t, cast=None, entropy=True, route="fused", **kw):
    xd = x.cuda()
    head = w.cuda()
    kw.setdefault("weight_layout", "vh")
    if kw["weight_layout"] == "hv":
        head = head.T.contiguous()
    calls = []
    keep = module._scored
    module._scored = lambda *a: calls.append(keep(*a)) or calls[-1]
    try:
        r = nvjsel.lm_head_token_logprobs(xd, head, t.to("cuda", torch.int32), entropy=entropy, **kw)
    finally:
        module._scored = keep
    if route is not None:
        assert (route == "fused") == (len(calls) == 1 and calls[0] is not None)
    lp, ent, lp_tol, ent_tol = oracle(x, w, t, cast)
    err, tol = (r.logprobs.double().cpu() - lp).abs(), lp_tol + SUM + lp.abs() * 2.0 ** -23
    assert bool((err <= tol).all()), (err / tol).max()
    if entropy:
        err, tol = (r.entropy.double().cpu() - ent).abs(), ent_tol + 2 * SUM * (2 + 2 * math.log(w.shape[0]))
        assert bool((err <= tol).all()), (err / tol).max()
    return r


@pytest.mark.parametrize("act,weight", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("rows", [1, 2, 31, 33, 64, 65, 127, 128, 129, 255, 257, 300, 385, 513])
def test_rows(rows, act, weight):
    check(*make(rows, 128, 1500, act, weight), reduce_cast=0, entropy=rows % 2 == 1)


@pytest.mark.parametrize("act,weight", [("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 255, 256, 257, 2048, 2055, 30001, 66001])
def test_vocabularies(vocab, act, weight):
    check(*make(70, 64, vocab, act, weight, seed=1), reduce_cast=0)
    check(*make(5, 192, vocab, act, weight, seed=2), reduce_cast=0)


@pytest.mark.parametrize("hidden", [64, 128, 192, 768, 1024, 2560])
def test_hidden_sizes(hidden):
    check(*make(150, hidden, 3000, seed=3), reduce_cast=0)


def test_many_row_blocks():
    check(*make(2048, 64, 5003, seed=4), reduce_cast=0)
    check(*make(2900, 64, 700, "f32", "bf16", seed=5), reduce_cast=0)
    check(*make(33 * 256 + 5, 64, 300, seed=6), reduce_cast=0)


@pytest.mark.parametrize("kind", ["f32w", "mixed", "odd_hidden", "hv", "cast", "unaligned"])
def test_other_calls_by_logits(kind):
    if kind == "f32w":
        check(*make(40, 96, 700, "f32", "f32"), route="logits")
    elif kind == "mixed":
        check(*make(40, 128, 700, "bf16", "f16"), route="logits", reduce_cast=0)
    elif kind == "odd_hidden":
        check(*make(40, 100, 700), route="logits", reduce_cast=0)
    elif kind == "cast":
        check(*make(40, 128, 700), cast=torch.float16, route="logits", reduce_cast=2)
    elif kind == "hv":
        check(*make(40, 128, 704), route="logits", reduce_cast=0, weight_layout="hv")
    else:
        x, w, t = make(9, 128, 700)
        buf = torch.zeros(700 * 128 + 1, dtype=w.dtype, device="cuda")
        head = buf[1:].view(700, 128)
        head.copy_(w)
        r = nvjsel.lm_head_token_logprobs(x.cuda(), head, t.cuda(), weight_layout="vh", reduce_cast=0)
        lp, _, tol, _ = oracle(x, w, t)
        assert bool(((r.logprobs.double().cpu() - lp).abs() <= tol + SUM + lp.abs() * 2.0 ** -23).all())


def test_logits_in_several_steps(monkeypatch):
    monkeypatch.setattr(module, "_LOGIT_BYTES", 1)  # 64 rows at a time
    x, w, t = make(200, 100, 333, seed=7)
    check(x, w, t, route="logits", reduce_cast=0)
    whole = nvjsel.token_logprobs(nvjsel.lm_head_logits_hip(x.cuda(), w.cuda(), weight_layout="vh"), t.cuda(), num_top=5)
    parts = nvjsel.lm_head_token_logprobs(x.cuda(), w.cuda(), t.cuda(), num_top=5, weight_layout="vh")
    assert torch.equal(whole.top_ids, parts.top_ids) and parts.top_logprobs.shape == (200, 5)


@pytest.mark.parametrize("act", ["bf16", "f16"])
def test_rounded_logits_by_default(act):
    """The reference's dot rounds to the operands' type: the same log probabilities as of those logits."""
    x, w, t = make(80, 128, 2000, act, act, seed=8)
    r = check(x, w, t, cast=DT[act], entropy=True)
    logits = nvjsel.lm_head_logits_hip(x.cuda(), w.cuda(), weight_layout="vh")
    s = nvjsel.token_logprobs(logits, t.cuda(), entropy=True)
    # the same rounded logits but for sums that lie next to a rounding's border
    assert bool(((r.logprobs - s.logprobs).abs() <= 2 * SUM + s.logprobs.abs() * 2.0 ** -23).float().mean() > 0.9)


@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_tokens_and_bad_values(act):
    x, w, t = make(70, 128, 900, act, "bf16", seed=9)
    t[3], t[4], t[5], t[69] = -1, 900, -(2 ** 31), -1
    r = check(x, w, t, reduce_cast=0)
    assert r.logprobs[3] == 0 and r.logprobs[69] == 0
    far = t.clone()
    far[0] = 2 ** 32 + 7
    got = nvjsel.lm_head_token_logprobs(x.cuda(), w.cuda(), far.cuda(), weight_layout="vh", reduce_cast=0)
    assert got.logprobs[0] == 0 and torch.equal(got.logprobs[1:], r.logprobs[1:])
    x[7, 5], x[8, 3], w[400] = math.nan, math.inf, w[399]
    got = nvjsel.lm_head_token_logprobs(x.cuda(), w.cuda(), t.cuda(), weight_layout="vh", reduce_cast=0, entropy=True)
    assert bool(torch.isnan(got.logprobs[7:9]).all()) and bool(torch.isnan(got.entropy[7:9]).all())
    keep = [i for i in range(70) if i not in (7, 8)]
    lp, ent, tol, _ = oracle(x[keep], w, t[keep])
    assert bool(((got.logprobs.double().cpu()[keep] - lp).abs() <= tol + SUM + lp.abs() * 2.0 ** -23).all())
    w[10] = math.nan  # a row of the table: every row's sum
    got = nvjsel.lm_head_token_logprobs(x.cuda(), w.cuda(), t.cuda(), weight_layout="vh", reduce_cast=0)
    assert bool(torch.isnan(got.logprobs[(t >= 0) & (t < 900)]).all()) and got.logprobs[3] == 0


def test_an_infinity_whose_logits_are_all_below():
    """f32 hidden: an infinity's terms hold a NaN; its logits are -inf here, and nothing is left."""
    g = torch.Generator().manual_seed(20)
    x = torch.randn(5, 64, generator=g)
    w = (torch.randn(301, 64, generator=g) * 0.02).to(torch.bfloat16)
    w[:, 9] = -w[:, 9].abs() - 0.01
    x[2, 9] = math.inf
    r = nvjsel.lm_head_token_logprobs(x.cuda(), w.cuda(), torch.tensor([1, 2, 3, -1, 300]).cuda(), weight_layout="vh", entropy=True)
    assert float(r.logprobs[2]) == -math.inf and float(r.entropy[2]) == 0.0
    keep = [0, 1, 3, 4]
    lp, _, tol, _ = oracle(x[keep], w, torch.tensor([1, 2, -1, 300]))
    assert bool(((r.logprobs.double().cpu()[keep] - lp).abs() <= tol + SUM + lp.abs() * 2.0 ** -23).all())


def test_far_logits():
    """Logits of thousands, and one far above the others: one token has all of the probability."""
    x, w, t = make(40, 64, 3000, "f32", "bf16", seed=10, spread=3.0)
    check(x * 300, w, t, reduce_cast=0)
    check(x * 1e-6, w, t, reduce_cast=0)
    check(x * 0, w, t, reduce_cast=0)


def test_views_shapes_norm_and_four_bits():
    x, w, t = make(24, 128, 600, seed=11)
    xd, wd, td = x.cuda(), w.cuda(), t.cuda()
    want = nvjsel.lm_head_token_logprobs(xd, wd, td, weight_layout="vh", entropy=True)
    tied = nvjsel.lm_head_token_logprobs(xd.reshape(2, 12, 128), wd.T, td.reshape(2, 12), entropy=True)
    assert tied.logprobs.shape == (2, 12) and torch.equal(tied.logprobs.reshape(-1), want.logprobs)
    assert torch.equal(tied.entropy.reshape(-1), want.entropy)
    wide = torch.zeros(24, 200, dtype=x.dtype, device="cuda")
    wide[:, 3:131] = xd
    assert torch.equal(nvjsel.lm_head_token_logprobs(wide[:, 3:131], wd.T, td).logprobs, want.logprobs)
    nw = torch.randn(128, device="cuda") * 0.1
    normed = nvjsel.rms_norm_hip(xd, nw, 1e-6, torch.bfloat16)
    assert torch.equal(nvjsel.lm_head_token_logprobs(xd, wd.T, td, norm_weight=nw, act_dtype=torch.bfloat16).logprobs,
                       nvjsel.lm_head_token_logprobs(normed, wd.T, td).logprobs)
    head = nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(wd.T, group_size=32))
    four = nvjsel.lm_head_token_logprobs(xd, head, td, num_top=3)
    by_logits = nvjsel.token_logprobs(nvjsel.lm_head_logits_hip(xd, head), td, num_top=3)
    assert torch.equal(four.logprobs, by_logits.logprobs) and torch.equal(four.top_ids, by_logits.top_ids)


def test_captured_and_again():
    x, w, t = make(300, 128, 9001, seed=12)
    xd, wd, td = x.cuda(), w.cuda(), t.cuda()
    call = lambda: nvjsel.lm_head_token_logprobs(xd, wd, td, weight_layout="vh", entropy=True)  # noqa: E731
    want = call()
    for _ in range(10):
        got = call()
        assert torch.equal(got.logprobs, want.logprobs) and torch.equal(got.entropy, want.entropy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        td.copy_(td.roll(k + 1))
        xd.mul_(0.75)
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out.logprobs, eager.logprobs) and torch.equal(out.entropy, eager.entropy)


def test_hundreds_of_row_blocks():
    check(*make((1 << 17) + 3, 64, 130, seed=7), reduce_cast=0)
    check(*make((1 << 15) + 33, 64, 130, "f32", "bf16", seed=8), reduce_cast=0, entropy=False)


@pytest.mark.parametrize("rows,hidden", [(33, 64), (64, 16384), (65, 16384), (40, 16448), (100, 16448)])
def test_f32_rows_as_terms_and_as_they_lie(rows, hidden):
    """More than 32 f32 rows are split beforehand up to 16,384 hidden values, as they are staged beyond."""
    check(*make(rows, hidden, 300, "f32", "bf16", seed=21), reduce_cast=0)


def test_f32_terms_of_an_infinity_and_captured():
    g = torch.Generator().manual_seed(22)
    x = torch.randn(150, 64, generator=g)
    w = (torch.randn(301, 64, generator=g) * 0.02).to(torch.bfloat16)
    w[:, 9] = -w[:, 9].abs() - 0.01
    x[[2, 70, 149], 9] = math.inf
    t = torch.randint(0, 301, (150,), generator=g)
    xd, wd, td = x.cuda(), w.cuda(), t.cuda()
    call = lambda: nvjsel.lm_head_token_logprobs(xd, wd, td, weight_layout="vh", entropy=True)  # noqa: E731
    r = call()
    bad = torch.zeros(150, dtype=torch.bool)
    bad[[2, 70, 149]] = True
    assert bool((r.logprobs.cpu()[bad] == -math.inf).all()) and bool((r.entropy.cpu()[bad] == 0.0).all())
    lp, _, tol, _ = oracle(x[~bad], w, t[~bad])
    assert bool(((r.logprobs.double().cpu()[~bad] - lp).abs() <= tol + SUM + lp.abs() * 2.0 ** -23).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        xd.mul_(0.5)
        td.copy_(td.roll(k + 1))
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out.logprobs, eager.logprobs) and torch.equal(out.entropy, eager.entropy)
