"""Log probabilities of given tokens, entropies, top alternatives and their
gradient against plain 64-bit forms, at the sizes and masks where they can go
wrong."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = math.inf


def make(rows, vocab, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + vocab)
    x = torch.empty(rows, vocab).exponential_(1.0, generator=g) + spread * torch.randn(rows, vocab, generator=g)
    return x.to(DT[dtype]), torch.randint(0, vocab, (rows,), generator=g)


def oracle(x, tokens, top=0):
    """Row by row in 64 bits on the CPU, as documented."""
    lps, ents, vals, ids = [], [], [], []
    for row, t in zip(x.double(), tokens.tolist()):
        v = row.numel()
        asked = 0 <= t < v
        if bool(torch.isnan(row).any()) or bool((row == INF).any()):
            lps.append(math.nan if asked else 0.0)
            ents.append(math.nan)
            n = min(top, v)
            vals.append([math.nan] * n + [-INF] * (top - n))
            ids.append(list(range(n)) + [-1] * (top - n))
            continue
        left = row[row > -INF]
        if left.numel() == 0:
            lps.append(-INF if asked else 0.0)
            ents.append(0.0)
            vals.append([-INF] * top)
            ids.append([-1] * top)
            continue
        m = left.max()  # differences first: a row of the lowest f32 values swallows ln S
        log_sum = torch.log(torch.exp(left - m).sum())
        lps.append(float((row[t] - m) - log_sum) if asked else 0.0)
        lp = (left - m) - log_sum
        ents.append(float(-(lp.exp() * torch.where(lp > -1e6, lp, 0.0)).sum()))
        value, order = torch.sort(row, descending=True, stable=True)
        n = min(top, left.numel())
        vals.append([float((u - m) - log_sum) for u in value[:n]] + [-INF] * (top - n))
        ids.append(order[:n].tolist() + [-1] * (top - n))
    return (torch.tensor(lps, dtype=torch.float64), torch.tensor(ents, dtype=torch.float64),
            torch.tensor(vals, dtype=torch.float64).reshape(len(lps), top),
            torch.tensor(ids, dtype=torch.int64).reshape(len(lps), top))


# The sum of exponentials is within 2^-19 (relative) of the exact one: the hardware's exp2
# is within 1 ulp (2^-23), its argument l log2 e - ref rounds once (2^-24 of at most 25 where the
# term counts, times ln 2: 2^-20), log2 e itself (2^-26 of it, alike), the tree five times (2^-24 each).
# Its logarithm is off by as much, the difference to it rounds to f32 once: half of 2^-23 of the result.
SUM = 2.0 ** -19


def near_logprobs(got, want):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = torch.isnan(want) | torch.isinf(want)
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    got, want = got[~same], want[~same]
    err, tol = (got - want).abs(), SUM + want.abs() * 2.0 ** -24
    assert bool((err <= tol).all()), (err / tol).max()


def near_entropy(got, want, vocab):
    """ln S - T / S: T's terms t y err as S's do, times |y|, whose mean is at most ln V + entropy (natural units), and
    their products round once more; twice for T / S and S."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    tol = 2 * SUM * (2.0 + 2.0 * math.log(vocab)) + want[ok].abs() * 2.0 ** -24
    err = (got[ok] - want[ok]).abs()
    assert bool((err <= tol).all()), (err / tol).max()


def check(x, tokens, top=0, entropy=True, device="cuda", token_dtype=torch.int32):
    xd = x.to(device) if x.device.type == "cpu" else x
    r = nvjsel.token_logprobs(xd, tokens.to(device, token_dtype), num_top=top, entropy=entropy)
    lp, ent, vals, ids = oracle(x.cpu(), tokens, top)
    near_logprobs(r.logprobs, lp)
    assert (r.entropy is None) == (not entropy) and (r.top_ids is None) == (top == 0)
    if entropy:
        near_entropy(r.entropy, ent, x.shape[1])
    if top:
        assert torch.equal(r.top_ids.cpu().long(), ids)
        near_logprobs(r.top_logprobs, vals)
    return r


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 63, 255, 1023, 1024, 1025, 2047, 2049, 8191, 16385, 50257])
def test_vocabularies(vocab, dtype):
    x, t = make(3, vocab, dtype)
    check(x, t)
    check(x, t, top=5, entropy=vocab % 2 == 0)


@pytest.mark.parametrize("rows,vocab", [(1, 248320), (2, 131075), (17, 30001), (70, 9000), (300, 2051), (1030, 777),
                                        (4097, 130), (5000, 33)])
@pytest.mark.parametrize("top", [0, 20])
def test_rows(rows, vocab, top):
    x, t = make(rows, vocab, "bf16", seed=1)
    check(x, t, top=top)


@pytest.mark.parametrize("top", [1, 2, 24, 25, 32, 33, 64])
@pytest.mark.parametrize("rows,vocab", [(1, 40), (5, 20011), (600, 5003)])
def test_tops(rows, vocab, top):
    x, t = make(rows, vocab, "f16", seed=2)  # many equal logits
    check(x, t, top=top, entropy=False)


def test_more_rows_than_one_scan_takes():
    x, t = make(8192 + 77, 40, "f32", seed=3)
    check(x, t, top=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("top", [0, 10])
def test_masks(dtype, top):
    x, t = make(12, 5000, dtype, seed=4)
    low = torch.finfo(DT[dtype]).min
    x[0] = -INF                      # nothing left
    x[1, 1:] = -INF                  # one left, and it is asked for
    t[1] = 0
    x[2, :] = -INF                   # few left, the last one among them
    x[2, [5, 77, 4999]] = torch.tensor([1.0, 3.0, 2.0], dtype=x.dtype)
    t[2] = 9                         # a masked token
    x[3, ::2] = low                  # the type's lowest value
    x[4] = low                       # all of them
    x[5, 100] = math.nan
    x[6, 4998] = INF
    x[7] = 1.5                       # all equal
    x[8, 17] = torch.finfo(DT[dtype]).max
    x[9, ::3] = -INF
    t[9] = 1
    x[10, 3] = math.nan              # and a row that asks for nothing
    t[10] = -1
    t[11] = 5000                     # just outside
    check(x, t, top=top)
    check(x[:1].clone(), t[:1], top=top)  # alone: one launch
    check(x[5:6].clone(), t[5:6], top=top)


@pytest.mark.parametrize("dtype,scale", [("f32", 3e4), ("f32", 1e30), ("f16", 2e4), ("bf16", 1e5), ("f32", 1e-30)])
@pytest.mark.parametrize("offset", [0.0, 1.0, -1.0])
@pytest.mark.parametrize("top", [0, 4])
def test_far_values(dtype, scale, offset, top):
    x, t = make(4, 3001, "f32", seed=5)
    x = ((x / x.abs().amax() + offset) * scale).to(DT[dtype])
    check(x, t, top=top)


def test_far_values_close_together():
    """Around 2e4 in steps of f32's last place there: differences count, not the values."""
    x, t = make(3, 9000, "f32", seed=6)
    check(x + 2e4, t, top=3)
    check(x - 2e4, t, top=3)
    check(x + 16384.0, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_large_logit_in_a_long_row(dtype):
    x = torch.full((2, 200003), -3.0).to(DT[dtype])
    x[0, 199999] = 9.5
    x[1, 0] = 20.0
    check(x, torch.tensor([199999, 5]), top=2)


def test_strides_shapes_and_token_types():
    x, t = make(30, 1003, "bf16", seed=7)
    wide = torch.zeros(30, 1100, dtype=x.dtype, device="cuda")
    wide[:, 33:1036] = x.cuda()
    check(wide[:, 33:1036], t, top=3)                      # rows further apart than V, at odd addresses
    check(x.cuda().T.contiguous().T, t, top=3)             # columns not contiguous
    check(x[:1].expand(30, 1003).cuda(), t)                # one row, asked for 30 tokens
    check(x[:1].cuda().expand(30, 1003), t, top=2)
    lp, ent, vals, ids = oracle(x, t, 3)
    r = nvjsel.token_logprobs(x.cuda().reshape(5, 6, 1003), t.cuda().reshape(5, 6), num_top=3, entropy=True)
    assert r.logprobs.shape == (5, 6) and r.top_ids.shape == (5, 6, 3) and r.entropy.shape == (5, 6)
    near_logprobs(r.logprobs.reshape(-1), lp)
    assert torch.equal(r.top_ids.cpu().long().reshape(30, 3), ids)
    one = nvjsel.token_logprobs(x[0].cuda(), t[0].cuda())
    assert one.logprobs.shape == ()
    near_logprobs(one.logprobs.reshape(1), lp[:1])
    far = t.clone()
    far[3], far[4], far[5] = 2 ** 32 + 5, -2 ** 33, 1003   # int64: nothing wraps into the vocabulary
    check(x, far, token_dtype=torch.int64)
    check(x, torch.arange(60)[::2], token_dtype=torch.int64)
    every = torch.arange(60, dtype=torch.int32, device="cuda")[::2]  # a strided view of tokens
    near_logprobs(nvjsel.token_logprobs(x.cuda(), every).logprobs, oracle(x, torch.arange(60)[::2])[0])


def test_same_results_however_often_and_beside_others():
    x, t = make(9, 60000, "bf16", seed=8)
    xd, td = x.cuda(), t.cuda()
    first = nvjsel.token_logprobs(xd, td, num_top=8, entropy=True)
    plain = nvjsel.token_logprobs(xd, td, entropy=True)
    for _ in range(20):
        for want, top in ((first, 8), (plain, 0)):
            got = nvjsel.token_logprobs(xd, td, num_top=top, entropy=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)


def test_streams_threads_and_devices_workspaces():
    """Two threads on one stream, and calls on streams of their own, at once."""
    work = [make(r, v, "bf16", seed=9) for r, v in ((1, 70001), (40, 9001), (3, 30011), (513, 2050))]
    dev = [(x.cuda(), t.cuda()) for x, t in work]
    want = [nvjsel.token_logprobs(x, t, num_top=6, entropy=True) for x, t in dev]
    torch.cuda.synchronize()
    bad = []

    def go(stream, offset):
        with torch.cuda.stream(stream):
            for i in range(24):
                j = (i + offset) % len(dev)
                got = nvjsel.token_logprobs(*dev[j], num_top=6 if i % 3 else 0, entropy=True)
                pairs = zip(got, want[j])
                if not all(a is None or torch.equal(a, b) or (a.dtype == torch.float32 and not i % 3
                                                              and torch.allclose(a, b, rtol=0, atol=1e-5))
                           for a, b in pairs):
                    bad.append((offset, i))
            stream.synchronize()

    shared = torch.cuda.Stream()
    for streams in ((shared, shared), (torch.cuda.Stream(), torch.cuda.Stream())):
        threads = [threading.Thread(target=go, args=(s, k)) for k, s in enumerate(streams)]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
    assert not bad


@pytest.mark.parametrize("top", [0, 7])
def test_captured_calls_share_nothing(top):
    """Two graphs captured on one stream, replayed in turn with eager calls between them."""
    xs = [make(r, v, "bf16", seed=10) for r, v in ((2, 90001), (20, 12000))]
    dev = [(x.cuda(), t.cuda()) for x, t in xs]
    for x, t in dev:
        nvjsel.token_logprobs(x, t, num_top=top, entropy=True)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, t in dev:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(nvjsel.token_logprobs(x, t, num_top=top, entropy=True))
        graphs.append(g)
    for k in range(5):
        for (x, t), g, out in zip(dev, graphs, outs):
            x.copy_(x.roll(k + 1, 1))
            g.replay()
            want = nvjsel.token_logprobs(x, t, num_top=top, entropy=True)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want) if a is not None)


# ---------------------------------------------------------------- the gradient


def formula(x, tokens, g, h):
    """dl of sum_n g_n logprob_n + h_n entropy_n in 64 bits, with what its parts may err by in f32."""
    l = x.double()
    d, tol = torch.zeros_like(l), torch.zeros_like(l)
    for i, t in enumerate(tokens.tolist()):
        row, v = l[i], l.shape[1]
        gi = float(g[i]) if g is not None and 0 <= t < v else 0.0
        hi = float(h[i]) if h is not None else 0.0
        if bool((row == -INF).all()) or (gi == 0.0 and hi == 0.0):
            continue
        m = row.max()
        s = torch.log(torch.exp(row - m).sum())
        lp = row - m - s
        p = torch.exp(lp)
        lp = torch.where(p == 0.0, 0.0, lp)
        ent = -(p * lp).sum()
        d[i] = -gi * p - hi * p * (lp + ent)
        # ln p in f32: two differences and the stored ln S round (2^-24 each of |l - m|, ln S and |ln p|), ln S is
        # within SUM, exp2 and its argument add 2^-23 and 2^-24 |ln p|: relative to p; then a few products
        rel = SUM + 2.0 ** -22 * (2.0 + lp.abs() + s.abs())
        tol[i] = p * rel * (abs(gi) + abs(hi) * (1.0 + lp.abs() + ent))
        tol[i] += abs(hi) * p * 2 * SUM * (2.0 + 2.0 * math.log(v + 1.0))  # the entropy's own error
        if 0 <= t < v:
            d[i, t] += gi
            tol[i, t] += abs(gi) * 2.0 ** -23
    return d, tol


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 7), (5, 1023), (2, 4097), (2, 16385), (40, 2051), (1030, 130)])
@pytest.mark.parametrize("which", ["g", "h", "gh"])
def test_gradient(rows, vocab, dtype, which):
    x, t = make(rows, vocab, dtype, seed=11)
    gen = torch.Generator().manual_seed(5)
    g = torch.randn(rows, generator=gen) if "g" in which else None
    h = torch.randn(rows, generator=gen) if "h" in which else None
    if rows > 2:
        t[1] = -1
        if g is not None:
            g[2] = 0.0
    xd = x.cuda().requires_grad_()
    r = nvjsel.token_logprobs(xd, t.cuda(), entropy="h" in which)
    outs = [o for o, k in ((r.logprobs, g), (r.entropy, h)) if k is not None]
    grads = [k.cuda() for k in (g, h) if k is not None]
    got, = torch.autograd.grad(outs, xd, grads)
    assert got.dtype == x.dtype and got.shape == x.shape
    want, tol = formula(x, t, g, h)
    eps = torch.finfo(x.dtype)
    tol = tol + want.abs() * (eps.eps / 2) * (1 + 2 ** -8) + eps.tiny * eps.eps
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max()


def test_gradient_against_differences():
    x, t = make(3, 17, "f32", seed=12)
    g, h = torch.tensor([1.0, -2.0, 0.5]), torch.tensor([0.3, 0.0, -1.0])

    def loss(x64):
        total = 0.0
        for i in range(3):
            lp = torch.log_softmax(x64[i], 0)
            total = total + g[i].double() * lp[t[i]] - h[i].double() * (lp.exp() * lp).sum()
        return total

    xd = x.cuda().requires_grad_()
    r = nvjsel.token_logprobs(xd, t.cuda(), entropy=True)
    ((r.logprobs * g.cuda()).sum() + (r.entropy * h.cuda()).sum()).backward()
    step = 2.0 ** -12
    for i in range(3):
        for v in range(17):
            e = torch.zeros(3, 17, dtype=torch.float64)
            e[i, v] = step
            diff = float((loss(x.double() + e) - loss(x.double() - e)) / (2 * step))
            # central differences: step^2 / 6 times a third derivative, below 20 here; f32's own rounding below
            assert abs(float(xd.grad[i, v]) - diff) <= 20 * step ** 2 / 6 + 2.0 ** -18


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gradient_of_masked_rows(dtype):
    x, t = make(7, 3000, dtype, seed=13)
    x[0] = -INF
    x[1, ::2] = torch.finfo(DT[dtype]).min
    x[2, ::3] = -INF
    t[2] = 3        # a masked token is asked for: the others' gradient stands
    x[3, 50] = math.nan
    x[4, 7] = math.nan
    t[4] = -1       # padding with anything in it
    x[5] = torch.finfo(DT[dtype]).min
    g = torch.randn(7, generator=torch.Generator().manual_seed(1))
    xd = x.cuda().requires_grad_()
    lp = nvjsel.token_logprobs(xd, t.cuda()).logprobs
    got, = torch.autograd.grad(lp, xd, g.cuda())
    got = got.double().cpu()
    assert bool(torch.isnan(got[3]).all()) and bool((got[4] == 0).all()) and bool((got[0] == 0).all())
    keep = [0, 1, 2, 5, 6]
    want, tol = formula(x[keep], t[keep], g[keep], None)
    eps = torch.finfo(x.dtype)
    tol = tol + want.abs() * (eps.eps / 2) * (1 + 2 ** -8) + eps.tiny * eps.eps
    assert bool(((got[keep] - want).abs() <= tol).all())


def test_gradient_through_views_and_alternatives():
    """Shared and broadcast logits sum their rows' gradients; alternatives carry none."""
    x, t = make(1, 901, "f32", seed=14)
    t = torch.tensor([3, 3, 900, -1])
    xd = x.cuda().requires_grad_()
    r = nvjsel.token_logprobs(xd.expand(4, 901), t.cuda(), num_top=3, entropy=True)
    assert not r.top_logprobs.requires_grad and not r.top_ids.requires_grad
    (r.logprobs.sum() + 0.5 * r.entropy.sum()).backward()
    want, tol = formula(x.expand(4, 901), t, torch.ones(4), torch.full((4,), 0.5))
    err = (xd.grad.double().cpu() - want.sum(0, keepdim=True)).abs()
    # the four rows' sum rounds three times in f32
    assert bool((err <= tol.sum(0) + 3 * 2.0 ** -24 * want.abs().sum(0)).all())
    big = torch.zeros(2, 3, 700, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    nvjsel.token_logprobs(big[:, :-1], torch.zeros(2, 2, dtype=torch.int64, device="cuda")).logprobs.sum().backward()
    assert bool((big.grad[:, -1] == 0).all()) and bool((big.grad[:, :-1, 0] > 0.99).all())


def test_no_gradient_is_kept_where_none_is_asked():
    x, t = make(2, 50, "f32", seed=15)
    xd = x.cuda().requires_grad_()
    with torch.no_grad():
        assert not nvjsel.token_logprobs(xd, t.cuda()).logprobs.requires_grad
    r = nvjsel.token_logprobs(xd, t.cuda())
    with pytest.raises(RuntimeError):  # once differentiable
        d, = torch.autograd.grad(r.logprobs.sum(), xd, create_graph=True)
        d.sum().backward()


def test_captured_training_pass():
    """Forward and gradient captured, replayed with eager passes between the replays."""
    x, t = make(6, 4001, "bf16", seed=16)
    xd, td = x.cuda(), t.cuda()
    g = torch.randn(6, device="cuda")

    def step():
        leaf = xd.detach().requires_grad_()
        r = nvjsel.token_logprobs(leaf, td, entropy=True)
        d, = torch.autograd.grad([r.logprobs, r.entropy], leaf, [g, g])
        return r.logprobs.detach(), r.entropy.detach(), d

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        xd.copy_(xd.roll(k + 1, 1))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_most_rows():
    """2^23 rows, the most of a call: results, alternatives and gradient."""
    rows, vocab = 1 << 23, 3
    g = torch.Generator().manual_seed(23)
    x = torch.randn(rows, vocab, generator=g)
    t = torch.randint(-1, vocab, (rows,), generator=g)
    asked = t >= 0
    lp = torch.log_softmax(x.double(), 1)
    want = torch.where(asked, lp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    leaf = x.cuda().requires_grad_()
    r = nvjsel.token_logprobs(leaf, t.cuda())
    plain = nvjsel.token_logprobs(leaf.detach(), t.cuda(), num_top=1)
    for got in (r.logprobs.detach(), plain.logprobs):
        assert bool(((got.cpu().double() - want).abs() <= SUM + want.abs() * 2.0 ** -23).all())
    best = lp.max(1)  # torch.randn's values differ within a row
    assert torch.equal(plain.top_ids.cpu().long()[:, 0], best.indices)
    assert bool(((plain.top_logprobs[:, 0].cpu().double() - best.values).abs() <= SUM + best.values.abs() * 2.0 ** -23).all())
    d, = torch.autograd.grad(r.logprobs, leaf, torch.ones(rows, device="cuda"))
    p = lp.exp()
    exact = torch.where(asked[:, None], torch.zeros_like(lp).scatter_(1, t.clamp(min=0)[:, None], 1.0) - p, 0.0)
    tol = p * (SUM + 2.0 ** -22 * (2.0 + lp.abs() + (x.amax(1, keepdim=True) - x.double().logsumexp(1, keepdim=True)).abs()))
    assert bool(((d.cpu().double() - exact).abs() <= tol + 2.0 ** -23).all())
