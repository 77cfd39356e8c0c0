"""GPU: beam selection, state reordering and the step that joins them, against
plain forms in 64 bits.

Tolerances: a selected score is within half an fp32 step of its value plus 2^-20,
the fp32 sum of exponentials' share (about 256 additions per lane whose roundings
of 2^-24 are independent: 16 of them, and a few for the exponentials).  Two
candidates of one beam keep their logits' order exactly; two beams' candidates
may change places where they are closer than the two sums' errors."""
import math
import threading

import numpy as np
import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SUM = 2.0 ** -20
NINF = float("-inf")


def plain(logits, scores, k, finished=None, end=0):
    """(scores, places) of the K best of one request, in 64 bits; place -1: none."""
    w, v = logits.shape
    l = logits.double().numpy()
    total = np.full((w, v), -math.inf)
    for i in range(w):
        s = float(scores[i])
        if s == -math.inf:
            continue
        bad = math.isnan(s) or s == math.inf
        if finished is not None and finished[i]:
            total[i, end] = math.nan if bad else s
            continue
        m = l[i].max()
        if bad or np.isnan(l[i]).any() or m == math.inf:
            total[i] = math.nan
        elif m > -math.inf:
            total[i] = s + ((l[i] - m) - math.log(np.exp(l[i] - m).sum()))
    flat = total.reshape(-1)
    key = np.where(np.isnan(flat), math.inf, flat)  # no score is +inf
    # equal scores by beam, then token; a beam's own logits decide between them where
    # 64 bits do not: 1e-30 and 2e-30 less log n are one number
    live = np.isfinite(flat) & ~np.repeat(np.zeros(w, bool) if finished is None else finished.numpy().astype(bool), v)
    logit = np.where(live, l.reshape(-1), 0.0)
    order = np.lexsort((np.arange(w * v), -logit, np.arange(w * v) // v, -key))[:k]
    value = np.full(k, -math.inf)
    value[:len(order)] = flat[order]
    place = np.full(k, -1, np.int64)
    place[:len(order)] = np.where(flat[order] == -math.inf, -1, order)
    return value, place, flat


def check(logits, scores, k, finished=None, end=None, given=None):
    fin = None if finished is None else finished.cuda()
    got = nvjsel.beam_search_select(logits.cuda() if given is None else given, scores.cuda(), num_candidates=k,
                                    finished=fin, end_token=end)
    s, p, t = (x.cpu().numpy() for x in got)
    b, w, v = logits.shape
    assert s.shape == p.shape == t.shape == (b, k) and s.dtype == np.float32 and p.dtype == t.dtype == np.int32
    for i in range(b):
        value, place, flat = plain(logits[i], scores[i], k, None if finished is None else finished[i], end)
        nan = np.isnan(value)
        assert np.array_equal(np.isnan(s[i]), nan), i
        none = place < 0
        assert np.array_equal(p[i] < 0, none) and np.array_equal(t[i] < 0, none), (i, p[i], place)
        assert bool((s[i][none] == -math.inf).all())
        fine = ~nan & ~none
        tol = SUM + 2.0 ** -24 * np.abs(value)
        assert bool((np.abs(s[i] - value)[fine] <= tol[fine]).all()), (i, s[i], value)
        at = np.where(none, -1, p[i].astype(np.int64) * v + t[i])
        for j in np.nonzero(at != place)[0]:
            assert not nan[j] and not none[j] and at[j] // v != place[j] // v, (i, j, at, place)
            assert abs(flat[at[j]] - flat[place[j]]) <= 2 * SUM, (i, j, at, place)
        assert len(set(at[~none])) == (~none).sum()


def make(b, w, v, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.empty(b, w, v).exponential_(1.0, generator=g) * 1.2 + torch.randn(b, w, v, generator=g)
    return x.to(DT[dtype]), -torch.rand(b, w, generator=g).cumsum(1) * 2


@pytest.mark.parametrize("b,w,v,k,dtype", [
    (1, 1, 1, 1, "f32"), (1, 1, 5, 8, "bf16"), (2, 4, 7, 4, "f16"), (3, 3, 513, 6, "bf16"), (1, 4, 4096, 8, "bf16"),
    (1, 4, 4097, 8, "f32"), (5, 5, 50257, 10, "f32"), (2, 8, 32000, 16, "f16"), (1, 2, 248320, 64, "bf16"),
    (1, 64, 3001, 64, "f32"), (2, 33, 1000, 40, "bf16"), (17, 16, 2049, 32, "bf16"), (70, 10, 1003, 20, "f16"),
    (1, 1, 700001, 3, "bf16"),
])
def test_select(b, w, v, k, dtype):
    logits, scores = make(b, w, v, dtype, 1000 + v + k)
    check(logits, scores, k)


@pytest.mark.parametrize("b,w,v,k,dtype", [(18, 8, 2332, 16, "f16"), (16, 16, 2000, 16, "bf16"), (2, 16, 2000, 32, "f32"),
                                           (2, 64, 2000, 64, "f16"), (40, 64, 2100, 64, "bf16"), (5, 3, 5000, 64, "f32")])
def test_few_parts_many_candidates(b, w, v, k, dtype):
    """Fewer parts than candidates, or not many more: one bound from the parts is not enough."""
    logits, scores = make(b, w, v, dtype, 77 + v + w)
    check(logits, scores, k)
    finished = torch.zeros(b, w, dtype=torch.bool)
    finished[:, w // 2:] = True
    check(logits, scores, k, finished, 7)
    scores[:, ::2] = NINF
    check(logits, scores, k)
    if w <= 16:  # equal logits: more than are ranked
        check(logits.to(DT["bf16"]).round().to(DT[dtype]), torch.zeros_like(scores), k)


def test_first_step_and_ended_beams():
    logits, scores = make(4, 4, 5003, "bf16", 3)
    scores[:, 1:] = NINF
    logits[0, 1:] = float("nan")  # not looked at
    check(logits, scores, 8)
    logits, scores = make(4, 4, 5003, "f32", 4)
    finished = torch.tensor([[0, 1, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0], [1, 0, 1, 0]], dtype=torch.bool)
    scores[0, 1] = 5.0
    logits[1] = float("nan")
    logits[3, 0] = float("inf")
    check(logits, scores, 6, finished, 2)
    check(logits, scores, 6, finished.to(torch.uint8), 5002)
    scores[1, 2] = NINF  # an ended beam that is not live
    check(logits, scores, 4, finished, 0)


def test_masks():
    """-inf, the types' lowest values, and rows that a mask leaves empty."""
    for dtype in ("f32", "bf16", "f16"):
        logits, scores = make(3, 3, 9001, dtype, 6)
        low = torch.finfo(DT[dtype]).min
        logits[0, 0] = NINF
        logits[0, 1, :] = low
        logits[0, 2, 5:] = low
        logits[1, :, :8000] = NINF
        logits[1, 0, :] = NINF
        logits[1, 0, 8999] = -300.0  # one token alone, far below the others' maximum
        logits[2] = NINF  # nothing at all
        check(logits, scores, 6)
        logits[2, 1, 4] = low
        check(logits, scores, 6)
        few = torch.full((1, 2, 4100), NINF, dtype=DT[dtype])
        few[0, 0, 4099] = 1.0
        few[0, 1, 0] = 1.0
        few[0, 1, 4097] = -1.0
        check(few, torch.tensor([[-1.0, -2.0]]), 5)


def test_not_finite():
    logits, scores = make(6, 3, 2500, "f32", 8)
    logits[0, 1, 2400] = float("nan")
    logits[1, 2, 0] = float("inf")
    logits[2, 0, 7] = float("nan")
    logits[2, 2, 7] = float("inf")
    scores[3, 1] = float("nan")
    scores[4, 0] = float("inf")
    finished = torch.zeros(6, 3, dtype=torch.bool)
    finished[5, 1] = True
    scores[5, 1] = float("nan")
    check(logits, scores, 6, finished, 11)
    check(logits[:, :, :3].contiguous(), scores, 6, finished, 1)  # fewer tokens than candidates


def test_ties_go_to_the_lowest_place():
    """Equal logits, equal beams, zeros of both signs, and many at the border."""
    scores = torch.tensor([[-1.0, -1.0, -2.0]])
    for dtype in ("f32", "bf16", "f16"):
        same = torch.zeros(1, 3, 6001, dtype=DT[dtype])
        check(same, scores, 9)
        same[0, :, 1::2] = -0.0
        check(same, scores, 9)
        rows, _ = make(1, 1, 6001, dtype, 12)
        rows = (rows * 2).round().to(DT[dtype]).expand(1, 3, 6001).contiguous()
        check(rows, scores, 32)
        rows[0, :, 100:] = torch.minimum(rows[0, :, 100:], torch.zeros((), dtype=DT[dtype]))
        check(rows, scores, 64)


def test_large_and_small_logits():
    """Far from zero, spread wide, and next to each other."""
    for dtype, scale in (("f32", 1e30), ("bf16", 1e30), ("f16", 6e4), ("f32", 1e-30), ("f32", 50.0)):
        g = torch.Generator().manual_seed(5)
        logits = (torch.rand(2, 3, 5001, generator=g) * 2 - 1).mul(scale).to(DT[dtype])
        check(logits, torch.tensor([[0.0, -3.0, -500.0], [-1e6, -1e6 - 1, 0.0]]), 8)
    logits, scores = make(2, 2, 4500, "f32", 9)
    check(logits + 3e4, scores, 8)


def test_strides_and_views():
    for dtype in ("bf16", "f32"):
        logits, scores = make(3, 4, 1001, dtype, 14)
        wide = torch.zeros(3, 5, 1100, dtype=DT[dtype], device="cuda")
        view = wide[:, 1:, 3:1004]
        view.copy_(logits)
        check(logits, scores, 8, given=view)  # rows from any element
        turned = torch.empty(4, 3, 1001, dtype=DT[dtype], device="cuda").transpose(0, 1)
        turned.copy_(logits)
        check(logits, scores, 8, given=turned)
        inner = torch.empty(3, 4, 2002, dtype=DT[dtype], device="cuda")[:, :, ::2]
        inner.copy_(logits)
        check(logits, scores, 8, given=inner)
        one = logits[:, :1].expand(3, 4, 1001)
        check(one.contiguous(), scores, 8, given=logits[:, :1].cuda().expand(3, 4, 1001))


def test_select_twice_at_once_and_captured():
    """Two streams at a time, and a replayed graph with eager calls between."""
    data = [make(4, 4, 20011, "bf16", 40 + i) for i in range(3)]
    dev = [(l.cuda(), s.cuda()) for l, s in data]
    want = [nvjsel.beam_search_select(l, s, num_candidates=8) for l, s in dev]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for (l, s), st in zip(dev, streams):
        with torch.cuda.stream(st):
            got.append(nvjsel.beam_search_select(l, s, num_candidates=8))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    l, s = dev[0][0].clone(), dev[0][1].clone()
    state = torch.arange(16, device="cuda", dtype=torch.float32)[:, None].repeat(1, 33)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nvjsel.beam_search_select(l, s, num_candidates=8)
        nvjsel.reorder_beam_states(state, out[1][:, :4])
    for rep in range(4):
        l.copy_(dev[rep % 3][0])
        s.copy_(dev[rep % 3][1])
        state.copy_(torch.arange(16, device="cuda", dtype=torch.float32)[:, None].expand(16, 33))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want[rep % 3]))
        rows = torch.arange(4, device="cuda")[:, None] * 4 + want[rep % 3][1][:, :4]
        assert torch.equal(state[:, 5], rows.reshape(-1).float())
        assert torch.equal(nvjsel.beam_search_select(*dev[rep % 3], num_candidates=8)[2], want[rep % 3][2])


# ---------------------------------------------------------------- reordering


def moved(states, parents, slots=None, lengths=None, dim=None):
    b, w = parents.shape
    out = []
    for t in states:
        new = t.clone()
        for i in range(b):
            for j in range(w):
                p = int(parents[i, j])
                if not 0 <= p < w:
                    continue
                to, fr = (i * w + j, i * w + p) if slots is None else (int(slots[i, j]), int(slots[i, p]))
                if not (0 <= to < t.shape[0] and 0 <= fr < t.shape[0]):
                    continue
                if lengths is None:
                    new[to] = t[fr]
                else:
                    n = min(max(int(lengths[i]), 0), t.shape[dim])
                    new[to].narrow(dim - 1, 0, n).copy_(t[fr].narrow(dim - 1, 0, n))
        out.append(new)
    return out


def state(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    if dtype.is_floating_point:
        return torch.randn(shape, generator=g).to(dtype)
    return torch.randint(0, 100, shape, generator=g).to(dtype)


@pytest.mark.parametrize("b,w", [(1, 1), (1, 2), (3, 4), (2, 7), (2, 8), (2, 13), (1, 16), (2, 17), (1, 64)])
@pytest.mark.parametrize("row,dtype", [((8, 64), torch.float32), ((3, 5, 7), torch.bfloat16), ((1,), torch.uint8),
                                       ((257, 9), torch.int8), ((), torch.int64), ((2, 600), torch.float16)])
def test_reorder(b, w, row, dtype):
    s = state((b * w, *row), dtype, w + len(row))
    parents = torch.randint(-1, w + 1, (b, w), generator=torch.Generator().manual_seed(b + w), dtype=torch.int32)
    want = moved([s], parents)
    got = s.cuda()
    nvjsel.reorder_beam_states(got, parents.cuda())
    assert torch.equal(got.cpu(), want[0])


def test_reorder_long_and_many_pieces_together():
    """One state in a few long pieces beside one in many short ones."""
    lengths = torch.tensor([5, 70001], dtype=torch.int32)
    parents = torch.tensor([[1, 0, 0], [2, 2, 1]], dtype=torch.int32)
    states = [state((6, 1, 70001), torch.float32, 1), state((6, 3001, 9), torch.float16, 2), state((7, 2, 40), torch.uint8, 3)]
    got = [s.cuda() for s in states]
    nvjsel.reorder_beam_states(got, parents.cuda(), lengths=lengths.cuda(), length_dim=2)
    for a, b in zip(got, moved(states, parents, None, lengths, 2)):
        assert torch.equal(a.cpu(), b)
    with pytest.raises(ValueError, match="twice"):
        nvjsel.reorder_beam_states([got[0], got[1], got[0]], parents.cuda())


@pytest.mark.parametrize("w", [3, 16, 30])
def test_reorder_cycles_and_copies(w):
    """Every beam from the next one, all from one, and pairs that change places."""
    for parents in (torch.arange(w).roll(-1), torch.full((w,), w - 1), torch.arange(w).flip(0)):
        s = state((w, 1030), torch.float32, w)
        got = s.cuda()
        p = parents.to(torch.int32)[None]
        nvjsel.reorder_beam_states([got], p.cuda())
        assert torch.equal(got.cpu(), s[parents])


def test_reorder_slots_lengths_and_layouts():
    b, w = 4, 3
    g = torch.Generator().manual_seed(2)
    slots = torch.randperm(20, generator=g)[:b * w].reshape(b, w).to(torch.int32)
    slots[3, 1] = -1  # a row of padding
    slots[2, 0] = 20  # not in the table
    parents = torch.randint(0, w, (b, w), generator=g, dtype=torch.int32)
    lengths = torch.tensor([0, 1, 37, 500], dtype=torch.int32)
    shapes = [((20, 2, 40, 24), torch.bfloat16, 2), ((20, 40), torch.int32, 1), ((20, 40, 5), torch.uint8, 1),
              ((20, 3, 2, 40), torch.float16, 3)]
    for shape, dt, dim in shapes:
        s = state(shape, dt, dim)
        for ln in (None, lengths):
            want = moved([s], parents, slots, ln, dim)
            got = s.cuda()
            nvjsel.reorder_beam_states([got], parents.cuda(), slots=slots.cuda(),
                                       lengths=None if ln is None else ln.cuda(), length_dim=None if ln is None else dim)
            assert torch.equal(got.cpu(), want[0]), (shape, ln)
            if ln is not None:  # counted from the end
                again = s.cuda()
                nvjsel.reorder_beam_states([again], parents.cuda(), slots=slots.cuda(), lengths=ln.cuda(),
                                           length_dim=dim - len(shape))
                assert torch.equal(got, again)
    # many tensors of different sizes, rows apart and from any element, wider parents
    tensors, views = [], []
    for i in range(29):
        base = state((12, 3 + i, 11), torch.bfloat16, i)
        tensors.append(base)
        if i % 3 == 0:
            views.append(base.cuda())
        elif i % 3 == 1:
            room = torch.zeros(12, (3 + i) * 11 + 13, dtype=torch.bfloat16, device="cuda")
            views.append(room[:, 1:1 + (3 + i) * 11].unflatten(1, (3 + i, 11)))
            views[-1].copy_(base)
        else:
            flat = torch.zeros(12 * (3 + i) * 11 + 1, dtype=torch.bfloat16, device="cuda")
            views.append(flat[1:].reshape(12, 3 + i, 11))
            views[-1].copy_(base)
    wide = torch.zeros(b, 7, dtype=torch.int32, device="cuda")
    wide[:, :w] = parents.cuda()
    nvjsel.reorder_beam_states(views, wide[:, :w])
    for v, t in zip(views, moved(tensors, parents)):
        assert torch.equal(v.cpu(), t)


def test_reorder_large_offsets():
    """Rows behind the 4 GB mark of a state table."""
    s = torch.zeros(5, 1 << 30, dtype=torch.uint8, device="cuda")
    s[:, ::4099] = torch.arange(1, 6, dtype=torch.uint8, device="cuda")[:, None]
    slots = torch.tensor([[4, 0, 3]], dtype=torch.int32, device="cuda")
    nvjsel.reorder_beam_states(s, torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda"), slots=slots)
    for row, value in ((4, 4), (0, 5), (3, 1), (1, 2), (2, 3)):
        assert bool((s[row, ::4099] == value).all()) and int((s[row] != 0).sum()) == len(range(0, 1 << 30, 4099))


# ---------------------------------------------------------------- the whole step


@pytest.mark.parametrize("packed", [False, True])
def test_step(packed):
    """Several decode steps of two requests: the LM head (4-bit or bf16), the selection
    and the caches, against the same steps in 64 bits on the kernels' logits."""
    g = torch.Generator().manual_seed(77)
    b, w, h, v, steps, end = 2, 4, 256, 3003, 5, 17
    weight = (torch.randn(v, h, generator=g) * 0.05).to(torch.bfloat16).cuda()
    head = nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(weight.T, group_size=64)) if packed else weight.T
    norm = (0.1 * torch.randn(h, generator=g)).cuda()
    scores = torch.full((b, w), NINF)
    scores[:, 0] = 0.0
    finished = torch.zeros(b, w, dtype=torch.bool)
    cache = torch.zeros(b * w, 2, steps, 8)
    tokens = torch.full((b * w, steps), -1, dtype=torch.int32)
    d_scores, d_finished, d_cache, d_tokens = scores.cuda(), finished.cuda(), cache.cuda(), tokens.cuda()
    for step in range(steps):
        hidden = torch.randn(b, w, h, generator=g).to(torch.bfloat16).cuda()
        entry = torch.randn(b * w, 2, 8, generator=g)
        cache[:, :, step] = entry
        d_cache[:, :, step] = entry.cuda()
        lengths = torch.full((b,), step + 1, dtype=torch.int32, device="cuda")
        logits = nvjsel.lm_head_logits_hip(
            nvjsel.rms_norm_hip(hidden.reshape(b * w, h), norm, act_dtype=torch.bfloat16), head).reshape(b, w, v)
        new, parents, ids = nvjsel.lm_head_beam_search_step(
            hidden, head, d_scores, finished=d_finished, end_token=end, states=[d_cache], lengths=lengths, length_dim=2,
            norm_weight=norm, act_dtype=torch.bfloat16)
        nvjsel.reorder_beam_states(d_tokens, parents)
        for i in range(b):
            value, place, _ = plain(logits[i].cpu(), d_scores[i].cpu(), w, finished[i], end)
            assert np.abs(new[i].cpu().numpy() - value).max() <= SUM + 2.0 ** -24 * np.abs(value).max()
            assert np.array_equal(parents[i].cpu().numpy() * v + ids[i].cpu().numpy(), place)
        rows = (torch.arange(b)[:, None] * w + parents.cpu()).reshape(-1)
        cache = cache[rows]
        tokens = tokens[rows]
        tokens[:, step] = ids.cpu().reshape(-1)
        d_tokens[:, step] = ids.reshape(-1)
        finished = finished.reshape(-1)[rows].reshape(b, w) | (ids.cpu() == end)
        if step == 2:
            finished[0, 1] = True  # an end by length
        d_finished, d_scores = finished.cuda(), new
        assert torch.equal(d_cache.cpu(), cache) and torch.equal(d_tokens.cpu(), tokens)


def test_captured_step():
    """A whole step as a graph, replayed with new inputs and eager calls between."""
    g = torch.Generator().manual_seed(5)
    b, w, h, v = 3, 4, 256, 5003
    weight = (torch.randn(v, h, generator=g) * 0.05).to(torch.bfloat16).cuda()
    head = nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(weight.T))
    inputs = [(torch.randn(b, w, h, generator=g).to(torch.bfloat16).cuda(), torch.randn(b, w, generator=g).cuda(),
               torch.randn(b * w, 6, 33, generator=g).cuda()) for _ in range(3)]

    def step(hidden, scores, cache):
        return nvjsel.lm_head_beam_search_step(hidden, head, scores, states=[cache])

    want = []
    for hidden, scores, cache in inputs:
        moved_cache = cache.clone()
        want.append((*(x.clone() for x in step(hidden, scores, moved_cache)), moved_cache))
    fixed = tuple(x.clone() for x in inputs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*fixed)
    for rep in range(5):
        for to, x in zip(fixed, inputs[rep % 3]):
            to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((*out, fixed[2]), want[rep % 3]):
            assert torch.equal(x, y)
        assert torch.equal(step(*(x.clone() for x in inputs[1]))[2], want[1][2])


def test_threads_share_a_stream():
    """Two threads on one stream: selections in one launch and in two, and ids beside them."""
    small, large = [make(2, 4, 9001, "bf16", 60)], [make(24, 8, 20011, "f16", 61)]
    data = [(l.cuda(), s.cuda()) for l, s in small + large]
    want = [nvjsel.beam_search_select(l, s, num_candidates=8) for l, s in data]
    weight = (torch.randn(3001, 128, generator=torch.Generator().manual_seed(1)) * 0.1).to(torch.bfloat16).cuda()
    head = nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(weight.T))
    x = torch.randn(5, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    ids = nvjsel.lm_head_greedy_top1_hip(x, head)
    torch.cuda.synchronize()
    wrong = []

    def run(first):
        for i in range(40):
            at = (first + i) % 2
            got = nvjsel.beam_search_select(*data[at], num_candidates=8)
            same = torch.equal(nvjsel.lm_head_greedy_top1_hip(x, head), ids)
            if not same or not all(torch.equal(a, b) for a, b in zip(got, want[at])):
                wrong.append((first, i))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
