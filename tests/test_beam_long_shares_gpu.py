"""GPU: selections of so many rows that a wave walks 3 to 122 chunks of its row (2048
logits of 16 bits, 1024 of f32), against the definition in 64 bits on the device.

Tolerance of a beam's normaliser, for any length of a row and any values: the error of
log(sum) is at most the largest relative error of the sum's terms and of its additions.
A term's argument (x - m) log2 e is rounded once, by 2^-21 ln 2 below 16 and 2^-20 ln 2
below 32 (0.69 of 2^-20); terms beyond weigh less than 2^26 2^-32.  log2 e as an fp32
number is off by 1.4e-8 of itself, 17 x 0.69 x 1.4e-8 = 0.17 of 2^-20 for terms 2^-17
of the largest (V of them count as much as it).  The exponential: 1 ulp, 2^-23,
0.13 of 2^-20.  The additions of a chunk: at most 8 roundings of 2^-24 in a row, 0.5 of
2^-20; chunks, lanes and waves meet in fp64.  Together 1.5 of 2^-20, below 2^-19.  The
score adds its own rounding, half a step of fp32."""
import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SUM = 2.0 ** -19
NINF = float("-inf")


def rows_of(kind, b, w, v, dtype, seed):
    """Logits [b, w, v] on the device, made request by request."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty(b, w, v, dtype=DT[dtype], device="cuda")
    at = torch.arange(v, device="cuda")
    for i in range(b):
        x = torch.empty(w, v, device="cuda").exponential_(1.0, generator=g) * 1.2
        x += torch.randn(w, v, device="cuda", generator=g)
        if kind == "ascending":  # every chunk holds a new maximum of every lane
            x = at * (20.0 / v) + x * 1e-3
        elif kind == "descending":
            x = -at * (20.0 / v) + x * 1e-3
        elif kind == "equal":  # more pieces reach the bound than are set aside
            x = torch.zeros(w, v, device="cuda")
            x[:, v // 2] = 1.0
        elif kind == "steps":  # few values, many of them at the border
            x = (x * 2).round()
        elif kind == "masked":
            x[:, : v - 3000] = NINF
            x[:, ::7] = torch.finfo(DT[dtype]).min
            x[w - 1] = NINF
        out[i] = x.to(DT[dtype])
    return out, -torch.rand(b, w, device="cuda", generator=g).cumsum(1)


def check(logits, scores, k):
    """Each beam's tokens in its logits' own order, and scores and beams as the definition has them."""
    b, w, v = logits.shape
    got_s, got_p, got_t = nvjsel.beam_search_select(logits, scores, num_candidates=k)
    for i in range(b):
        l = logits[i].double() + 0.0  # one zero
        m = l.amax(1, keepdim=True)
        live = (m > NINF).squeeze(1)
        norm = torch.where(live[:, None], m + (l - m).exp().sum(1, keepdim=True).log(), torch.zeros_like(m))
        # the k largest logits of every beam, equal ones by token
        value, order = l.sort(dim=1, descending=True, stable=True)
        value, order = value[:, :k], order[:, :k]
        total = (scores[i].double()[:, None] + (value - norm)).cpu()
        order, parents, tokens = order.cpu(), got_p[i].cpu(), got_t[i].cpu()
        want = total.reshape(-1).sort(descending=True).values[:k]
        there = want > NINF
        assert torch.equal(parents >= 0, there) and torch.equal(tokens >= 0, there), i
        s = got_s[i].double().cpu()
        assert bool((s[~there] == NINF).all())
        tol = SUM + 2.0 ** -24 * want[there].abs()
        assert bool(((s[there] - want[there]).abs() <= tol).all()), (i, (s - want)[there].abs().max())
        for beam in range(w):
            mine = parents == beam
            n = int(mine.sum())
            assert torch.equal(tokens[mine].long(), order[beam, :n]), (i, beam)
            assert bool(((s[mine] - total[beam, :n]).abs() <= SUM + 2.0 ** -24 * total[beam, :n].abs()).all()), (i, beam)


@pytest.mark.parametrize("b,w,v,k,dtype,kind", [
    (32, 8, 98001, 16, "bf16", "random"),      # 3 chunks, the last one short
    (32, 8, 248321, 16, "bf16", "random"),     # 8
    (64, 4, 147003, 8, "f32", "random"),       # 9, two to a kept maximum
    (128, 16, 100003, 32, "bf16", "random"),   # 25, four
    (129, 16, 90007, 40, "f16", "random"),     # 44, six
    (48, 64, 40011, 64, "f32", "random"),      # 40, five
    (37, 60, 248321, 12, "bf16", "random"),    # 122, sixteen
    (32, 8, 248321, 16, "bf16", "ascending"),
    (40, 64, 60001, 24, "f16", "ascending"),
    (40, 64, 30011, 25, "f32", "ascending"),
    (40, 64, 60001, 8, "bf16", "descending"),
    (32, 8, 248321, 16, "bf16", "equal"),
    (40, 64, 60001, 30, "bf16", "equal"),
    (40, 64, 30011, 64, "f32", "equal"),
    (32, 8, 147003, 16, "f32", "steps"),
    (40, 64, 60001, 64, "f16", "steps"),
    (32, 8, 248321, 16, "bf16", "masked"),
    (40, 64, 60001, 8, "f16", "masked"),
    (40, 64, 30011, 8, "f32", "masked"),
])
def test_many_chunks(b, w, v, k, dtype, kind):
    check(*rows_of(kind, b, w, v, dtype, v + k), k)


@pytest.mark.parametrize("b,w,v,dtype", [(32, 8, 248320, "bf16"), (33, 64, 248320, "bf16"), (33, 64, 100003, "f32"),
                                         (33, 64, 100003, "f16")])
def test_rows_of_few_values(b, w, v, dtype):
    """Rows whose sums round the same way at every step: one larger value per lane and chunk's
    worth of the first logits, the rest equal, and rows that climb by a little in every chunk."""
    n = b * w
    at = torch.arange(v, device="cuda")
    logits = torch.empty(n, v, dtype=DT[dtype], device="cuda")
    low = torch.linspace(-9.0, -0.05, n, device="cuda")
    for r in range(n):
        if r % 2:
            x = torch.where(at < 512, 0.0, low[r])
        else:
            x = (at // 1024) * (low[r].abs() / 128) - 3.0
        logits[r] = x.to(DT[dtype])
    scores = torch.zeros(b, w, device="cuda")
    got, parents, tokens = (x.cpu() for x in nvjsel.beam_search_select(logits.reshape(b, w, v), scores))
    for i in range(b):
        l = logits.reshape(b, w, v)[i].double()
        norm = l.logsumexp(1)
        for j in range(w):
            p, t = int(parents[i, j]), int(tokens[i, j])
            want = float(l[p, t] - norm[p])
            assert abs(float(got[i, j]) - want) <= SUM + 2.0 ** -24 * abs(want), (i, j, p, float(got[i, j]) - want)
