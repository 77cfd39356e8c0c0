"""Log probabilities and adapters as a server and a trainer run them: launches
kept together, made on their tensors' device, calls of all kinds at once, and
calls that the documentation allows at the edges."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import nvjsel
from nvjsel import _lib, adapters, logprobs, selection, w4
from tests.launch_recorder import launches

AT = 0x1000
TOP = (f"('nvjsel_token_logprobs', [P, I, L, I, L, P, I, I, P, P, P, P, P, P, Z, P], "
       f"[{AT}, 1, {{0}}, 50000, 50000, {AT}, 4, {{1}}, {AT}, {AT}, {AT}, {AT}, None, {AT}, 1 << 40, None])")
ADAPTERS = (f"('nvjsel_apply_adapters', [P, I, L, P, I, L, P, P, I, P, I, I, I, I, P, L, P, L, P, Z, P], "
            f"[{AT}, 1, 64, {AT}, 1, 500, {AT}, {AT}, 1, {AT}, 3, 16, 64, 500, {AT}, {{0}}, {2 * AT}, 500, {AT}, 1 << 40, None])")
SCORE = (f"('nvjsel_lm_head_token_logprobs', [P, I, P, I, I, L, I, I, I, P, I, P, P, P, Z, P], "
         f"[{AT}, 1, {AT}, 1, 0, {{0}}, 64, 9000, 0, {AT}, 4, {AT}, None, {AT}, 1 << 40, None])")


@pytest.mark.parametrize("first,other,several", [
    (TOP.format(64, 20), TOP.format(1, 5), 2),
    (TOP.format(9000, 3), TOP.format(64, 0), 4),
    (ADAPTERS.format(40), ADAPTERS.format(3), 2),
    (SCORE.format(300), SCORE.format(20), 4),
    (SCORE.format(20), TOP.format(64, 20), 2),
], ids=["top-one", "tops-sums", "adapters-adapters", "score-score", "score-top"])
def test_a_call_keeps_its_launches_together(tmp_path, first, other, several):
    order = [thread for thread, _ in launches(tmp_path, first, other)]
    n = order.count("first")
    assert n == several and order == ["first"] * n + ["other"] * (len(order) - n)


class Here:
    """In place of the context that makes a device the current one."""

    inside = 0

    def __enter__(self):
        Here.inside += 1

    def __exit__(self, *_):
        Here.inside -= 1


def _head(rows=6, hidden=128, vocab=501, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(vocab, hidden, generator=g) * 0.1).to(torch.bfloat16).cuda()
    x = torch.randn(rows, hidden, generator=g).to(torch.bfloat16).cuda()
    a = (torch.randn(2, 16, hidden, generator=g) * 0.1).to(torch.bfloat16).cuda()
    b = (torch.randn(2, vocab, 16, generator=g) * 0.1).to(torch.bfloat16).cuda()
    tokens = torch.randint(0, vocab, (rows,), generator=g).cuda()
    ids = (torch.arange(rows) % 3 - 1).to(torch.int32).cuda()
    return w, x, a, b, tokens, ids


@pytest.mark.gpu
def test_launches_are_made_on_their_tensors_device(monkeypatch):
    w, x, a, b, tokens, ids = _head()
    launched, outside = [], []
    real = _lib.call

    def call(name, *args):
        launched.append(name)
        if not Here.inside:
            outside.append(name)
        return real(name, *args)

    for module in (adapters, logprobs, selection, w4):
        monkeypatch.setattr(module, "_on_device", lambda device: Here())
    monkeypatch.setattr(_lib, "call", call)
    table = nvjsel.pack_adapters(a, b)
    norm = torch.zeros(128, device="cuda")
    temps, keys = torch.ones(6, device="cuda"), torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    four = nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(w.T))
    for head in (w.T, four):
        logits = nvjsel.lm_head_logits_hip(x, head, adapters=table, adapter_ids=ids)
        nvjsel.lm_head_sample_token_ids(x, head, temperatures=temps, rng_keys=keys, norm_weight=norm,
                                        act_dtype=torch.bfloat16, adapters=table, adapter_ids=ids)
        nvjsel.lm_head_token_ids_and_topk(x, head, top_k=2, adapters=table, adapter_ids=ids)
        for top in (0, 3):
            nvjsel.lm_head_token_logprobs(x, head, tokens, num_top=top, norm_weight=norm, act_dtype=torch.bfloat16)
    leaf = logits.detach().requires_grad_()
    r = nvjsel.token_logprobs(leaf, tokens, num_top=3, entropy=True)
    (r.logprobs.sum() + r.entropy.sum()).backward()
    nvjsel.apply_adapters(x, logits, table, ids)
    torch.cuda.synchronize()
    assert {"nvjsel_token_logprobs", "nvjsel_token_logprobs_grad", "nvjsel_lm_head_token_logprobs", "nvjsel_apply_adapters",
            "nvjsel_adapters_pack", "nvjsel_lm_head_logits", "nvjsel_lm_head_w4_logits", "nvjsel_sample", "nvjsel_topk",
            "nvjsel_rms_norm"} <= set(launched)
    assert not outside, outside


@pytest.mark.gpu
def test_two_threads_queue_calls_of_all_kinds():
    w, x, a, b, tokens, ids = _head(150, 128, 9001, 1)
    table = nvjsel.pack_adapters(a, b)
    logits = nvjsel.lm_head_logits_hip(x, w.T)
    calls = [
        [lambda: nvjsel.token_logprobs(logits, tokens, num_top=9).top_logprobs,
         lambda: nvjsel.apply_adapters(x, logits, table, ids),
         lambda: nvjsel.token_logprobs(logits[:3], tokens[:3], entropy=True).entropy,
         lambda: nvjsel.lm_head_token_logprobs(x, w.T, tokens).logprobs],
        [lambda: nvjsel.apply_adapters(x[:9], logits[:9], table, ids[:9]),
         lambda: nvjsel.token_logprobs(logits[:2], tokens[:2], num_top=64).top_logprobs,
         lambda: nvjsel.lm_head_token_logprobs(x[:40], w.T, tokens[:40], entropy=True).entropy,
         lambda: nvjsel.token_logprobs(logits, tokens).logprobs],
    ]
    want = [[call().clone() for call in mine] for mine in calls]
    torch.cuda.synchronize()
    got = [[], []]
    start = threading.Barrier(2)

    def queue(at):
        start.wait()
        for i in range(80):
            got[at].append(calls[at][i % 4]())

    threads = [threading.Thread(target=queue, args=(at,)) for at in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for at in range(2):
        assert len(got[at]) == 80 and all(torch.equal(out, want[at][i % 4]) for i, out in enumerate(got[at]))


@pytest.mark.gpu
def test_a_captured_servers_step():
    """LM head with adapters, sampler, log probabilities and alternatives in one graph, replayed with new hidden states
    and eager steps between."""
    w, x, a, b, tokens, ids = _head(5, 128, 3001, 2)
    table = nvjsel.pack_adapters(a, b, torch.tensor([0.5, 2.0]))
    temps, keys = torch.ones(5, device="cuda"), torch.arange(10, dtype=torch.int32, device="cuda").reshape(5, 2)

    def step():
        logits = nvjsel.lm_head_logits_hip(x, w.T, adapters=table, adapter_ids=ids)
        chosen = nvjsel.lm_head_sample_token_ids(x, w.T, temperatures=temps, rng_keys=keys, adapters=table, adapter_ids=ids)
        return (chosen, *nvjsel.token_logprobs(logits, chosen, num_top=5, entropy=True),
                nvjsel.lm_head_token_logprobs(x, w.T, chosen).logprobs)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(5):
        x.copy_(torch.roll(x, k + 1, 1))
        ids.copy_(ids.roll(1))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.gpu
def test_outputs_over_inputs_that_are_read_before():
    """A square projection whose result goes over its own input, and a token list that is overwritten behind the call."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(37, 96, generator=g).to(torch.bfloat16).cuda()
    base = torch.randn(37, 96, generator=g).to(torch.bfloat16).cuda()
    table = nvjsel.pack_adapters((torch.randn(2, 8, 96, generator=g) / 10).to(torch.bfloat16).cuda(),
                                 torch.randn(2, 96, 8, generator=g).to(torch.bfloat16).cuda())
    ids = (torch.arange(37) % 3).to(torch.int32).cuda()
    want = nvjsel.apply_adapters(x, base, table, ids)
    got = nvjsel.apply_adapters(x, base, table, ids, out=x)
    assert got is x and torch.equal(x, want)
    tokens = torch.arange(37, device="cuda")
    first = nvjsel.token_logprobs(base, tokens, num_top=2)
    tokens.zero_()
    again = nvjsel.token_logprobs(base, torch.arange(37, device="cuda"), num_top=2)
    assert torch.equal(first.logprobs, again.logprobs)


@pytest.mark.gpu
def test_a_trained_leaf_that_is_changed_is_refused():
    x = torch.randn(3, 50, device="cuda")
    leaf = x.clone().requires_grad_()
    logits = leaf * 1.0
    r = nvjsel.token_logprobs(logits, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with torch.no_grad():
        logits.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logprobs.sum().backward()


@pytest.mark.gpu
def test_gradient_once_with_create_graph():
    """create_graph alone is allowed, what needs a second derivative is not; one of two gradients may be missing."""
    x = torch.randn(3, 50, device="cuda", requires_grad=True)
    t = torch.tensor([1, 2, 3], device="cuda")
    r = nvjsel.token_logprobs(x, t, entropy=True)
    d, = torch.autograd.grad(r.entropy.sum(), x, create_graph=True)
    r = nvjsel.token_logprobs(x, t, entropy=True)
    e, = torch.autograd.grad(r.entropy.sum(), x)
    assert torch.equal(d, e)
    p = torch.softmax(x.detach().double(), 1)
    want = -(p * (p.log() + -(p * p.log()).sum(1, keepdim=True)))
    assert bool(((e.double() - want).abs() <= 2.0 ** -18 * math.log(50) * 4 * p + 2.0 ** -24).all())
    unused = nvjsel.token_logprobs(x, t)
    (x * 0).sum().backward()
    assert unused.logprobs.requires_grad


@pytest.mark.gpu
def test_the_largest_offsets():
    """Rows whose first element lies behind 2^31, with alternatives and without, and their gradient."""
    rows, vocab = 9, 1 << 28
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    buf = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")  # 4.8 GB: rows of 2^28 elements, 5000 of them used
    part = buf[:, 7:5007]
    g = torch.Generator().manual_seed(5)
    x = torch.randn(rows, 5000, generator=g).to(torch.bfloat16)
    part.copy_(x)
    t = torch.randint(0, 5000, (rows,), generator=g)
    lp = torch.log_softmax(x.double(), 1)
    want = lp.gather(1, t[:, None])[:, 0]
    leaf = part.detach().requires_grad_()
    r = nvjsel.token_logprobs(leaf, t.cuda(), num_top=3)
    assert bool(((r.logprobs.detach().double().cpu() - want).abs() <= 2.0 ** -19 + want.abs() * 2.0 ** -24).all())
    d, = torch.autograd.grad(r.logprobs, leaf, torch.ones(rows, device="cuda"))
    exact = torch.zeros_like(lp).scatter_(1, t[:, None], 1.0) - lp.exp()
    assert bool(((d.double().cpu() - exact).abs() <= lp.exp() * 2.0 ** -17 + 2.0 ** -23 + exact.abs() * 2.0 ** -8).all())
    plain = nvjsel.token_logprobs(part, t.cuda())
    assert bool(((plain.logprobs.double().cpu() - want).abs() <= 2.0 ** -19 + want.abs() * 2.0 ** -24).all())
    table = nvjsel.pack_adapters(torch.zeros(1, 8, 64, dtype=torch.bfloat16, device="cuda"),
                                 torch.zeros(1, 5000, 8, dtype=torch.bfloat16, device="cuda"))
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ids[4] = -1
    nvjsel.apply_adapters(torch.ones(rows, 64, dtype=torch.bfloat16, device="cuda"), part, table, ids, out=part)
    assert torch.equal(part.cpu(), x)
