"""Low-rank adapters beside a shared projection against a plain 64-bit form, and a
server's step that runs them with the LM head, the sampler and the log
probabilities."""
from __future__ import annotations

import math

import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(rows, hidden, width, ranks, act="bf16", table="bf16", base=None, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * rows + hidden + width)
    x = torch.randn(rows, hidden, generator=g).to(DT[act])
    y = torch.randn(rows, width, generator=g).to(DT[base or act])
    a = [(torch.randn(r, hidden, generator=g) / math.sqrt(hidden)).to(DT[table]) for r in ranks]
    b = [(torch.randn(width, r, generator=g) / math.sqrt(r)).to(DT[table]) for r in ranks]
    s = 0.5 + torch.rand(len(ranks), generator=g)
    ids = torch.randint(-1, len(ranks), (rows,), generator=g).to(torch.int32)
    return x, y, a, b, s, ids


def oracle(x, base, a, b, s, ids):
    """Result in 64 bits, and what fp32 sums in any order may be off by.

    y: H products sum in fp32 (each addition 2^-23 of the sum of magnitudes so far, whichever way it rounds), times
    the scale (2^-24).  Its terms keep 24 bits (bf16) or 22 (f16: 2^-22 of y and 2^-38 of the row's largest).  The second
    product sums 3 R terms likewise; the sum with base rounds in fp32 and once to its type, half a step each."""
    out, tol = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64)
    for n, k in enumerate(ids.tolist()):
        if not 0 <= k < len(a):
            continue
        A, B, xs = a[k].double(), b[k].double(), x[n].double()
        y = (A * xs).sum(1) * float(s[k])
        y_tol = ((A * xs).abs().sum(1) * (A.shape[1] + 4) * 2.0 ** -23) * float(s[k]) + y.abs() * 2.0 ** -21 + y.abs().max() * 2.0 ** -38
        delta = (B * y).sum(1)
        out[n] += delta
        size = (B.abs() * y.abs()).sum(1)
        tol[n] = (B.abs() * y_tol).sum(1) + size * (3 * A.shape[0] + 4) * 2.0 ** -23
        tol[n] += (base[n].double().abs() + delta.abs()) * 2.0 ** -24
        info = torch.finfo(base.dtype)
        tol[n] += out[n].abs() * (info.eps / 2) * (1 + 2.0 ** -6) + info.tiny * info.eps
    return out, tol


def check(x, base, a, b, s, ids, in_place=False):
    table = nvjsel.pack_adapters([t.cuda() for t in a], [t.cuda() for t in b], s)
    xd, bd, idd = x.cuda(), base.cuda(), ids.cuda()
    got = nvjsel.apply_adapters(xd, bd, table, idd, out=bd if in_place else None)
    assert got.dtype == base.dtype and got.shape == base.shape
    if in_place:
        assert got is bd
    else:
        assert torch.equal(bd.cpu(), base)
    want, tol = oracle(x, base, a, b, s, ids)
    got = got.cpu()
    none = (ids < 0) | (ids >= len(a))
    assert torch.equal(got[none].view(torch.int16 if base.element_size() == 2 else torch.int32),
                       base[none].view(torch.int16 if base.element_size() == 2 else torch.int32))
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (err / tol.clamp(min=1e-300)).max()


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("table", ["bf16", "f16"])
@pytest.mark.parametrize("base", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rank", [4, 16, 40])
def test_types(act, table, base, rank):
    check(*make(21, 200, 333, [rank] * 3, act, table, base))


@pytest.mark.parametrize("rank", [1, 7, 8, 9, 16, 17, 31, 32, 33, 64, 65, 128, 200, 512])
@pytest.mark.parametrize("table", ["bf16", "f16"])
def test_ranks(rank, table):
    check(*make(35, 96, 130, [rank] * 2, "f32" if rank % 2 else table, table, "f32", seed=1))


@pytest.mark.parametrize("hidden", [1, 2, 7, 8, 31, 32, 33, 100, 255, 1000, 2560])
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_hidden_sizes(hidden, act):
    check(*make(5, hidden, 70, [16, 3], act, "bf16", seed=2))


@pytest.mark.parametrize("width", [1, 2, 15, 16, 17, 63, 64, 65, 255, 257, 1000, 4099])
@pytest.mark.parametrize("base", ["bf16", "f32"])
def test_widths(width, base):
    check(*make(18, 64, width, [8, 16, 33], "bf16", "bf16", base, seed=3))


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100, 257, 1025])
def test_rows(rows):
    check(*make(rows, 128, 200, [16] * 5, seed=4))
    check(*make(rows, 128, 200, [32] * 70, "f16", "f16", seed=5), in_place=True)


def test_mixtures():
    x, y, a, b, s, _ = make(70, 256, 300, [5, 16, 24, 64], seed=6)
    for ids in (torch.full((70,), -1), torch.full((70,), 2), torch.arange(70) % 4, torch.arange(70) // 20,
                torch.where(torch.arange(70) == 69, 1, -1), torch.full((70,), 4), torch.full((70,), 2 ** 31 - 1),
                torch.full((70,), -2 ** 31)):
        check(x, y, a, b, s, ids.to(torch.int32))
        check(x, y, a, b, s, ids.to(torch.int32), in_place=True)


def test_large_and_small_values():
    """Far from 1 in both directions; f16 tables scale y's terms by the row's largest."""
    for table in ("bf16", "f16"):
        x, y, a, b, s, ids = make(20, 64, 90, [16, 16], "f32", table, "f32", seed=7)
        for scale in (1e20, 1e-20, 1e-30):
            check(x * scale, y * 0, a, b, s, ids)
        check(x * torch.logspace(-10, 10, 20)[:, None], y, a, b, s, ids)
        a[0][3] = 0
        a[0][5] *= 1e-3
        check(x, y, a, b, s, ids)
        check(x * 0, y, a, b, s, ids)


@pytest.mark.parametrize("table", ["bf16", "f16"])
@pytest.mark.parametrize("rank", [8, 16, 64])
def test_bad_values_stay_in_their_rows(table, rank):
    x, y, a, b, s, _ = make(40, 96, 200, [rank] * 3, table, table, seed=8)
    ids = (torch.arange(40) % 4 - 1).to(torch.int32)
    clean = nvjsel.apply_adapters(x.cuda(), y.cuda(), nvjsel.pack_adapters([t.cuda() for t in a], [t.cuda() for t in b], s),
                                  ids.cuda()).cpu()
    x[5, 7] = math.inf   # ids 0
    x[6, 1] = math.nan   # ids 1
    x[4, 3] = math.nan   # none
    b[2][17] = math.nan  # one column of adapter 2
    b[2][18, 0] = math.inf
    table_ = nvjsel.pack_adapters([t.cuda() for t in a], [t.cuda() for t in b], s)
    got = nvjsel.apply_adapters(x.cuda(), y.cuda(), table_, ids.cuda()).cpu()
    assert bool(torch.isnan(got[5]).all()) and bool(torch.isnan(got[6]).all())
    of2 = ids == 2
    assert bool(torch.isnan(got[of2][:, 17]).all()) and not bool(torch.isfinite(got[of2][:, 18]).any())
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[5] = keep[6] = False
    keep[of2, 17] = keep[of2, 18] = False
    assert torch.equal(got[keep], clean[keep])
    a[1][0, 0] = math.inf  # an adapter's own: its rows alone
    table_ = nvjsel.pack_adapters([t.cuda() for t in a], [t.cuda() for t in b], s)
    got = nvjsel.apply_adapters(x.cuda(), y.cuda(), table_, ids.cuda()).cpu()
    keep &= (ids != 1)[:, None]
    assert torch.equal(got[keep], clean[keep]) and bool(torch.isnan(got[ids == 1]).all())


def test_strides_and_shapes():
    x, y, a, b, s, ids = make(24, 100, 77, [16, 8], seed=9)
    table = nvjsel.pack_adapters([t.cuda() for t in a], [t.cuda() for t in b], s)
    want, tol = oracle(x, y, a, b, s, ids)

    def near(got):
        return bool(((got.double().cpu().reshape(24, 77) - want).abs() <= tol).all())

    wide = torch.zeros(24, 300, dtype=x.dtype, device="cuda")
    wide[:, 1:101] = x.cuda()
    wide[:, 101:178] = y.cuda()
    assert near(nvjsel.apply_adapters(wide[:, 1:101], wide[:, 101:178], table, ids.cuda()))
    before = wide.clone()
    assert near(nvjsel.apply_adapters(wide[:, 1:101], wide[:, 101:178], table, ids.cuda(), out=wide[:, 180:257]))
    assert torch.equal(wide[:, :180], before[:, :180]) and bool((wide[:, 257:] == 0).all())
    assert near(nvjsel.apply_adapters(x.cuda().T.contiguous().T, y.cuda().T.contiguous().T, table, ids.cuda()))
    r = nvjsel.apply_adapters(x.cuda().reshape(2, 12, 100), y.cuda().reshape(2, 12, 77), table, ids.cuda().reshape(2, 12))
    assert r.shape == (2, 12, 77) and near(r)
    shared = nvjsel.apply_adapters(x.cuda(), y[:1].cuda().expand(24, 77), table, ids.cuda())
    want, tol = oracle(x, y[:1].expand(24, 77), a, b, s, ids)
    assert near(shared)
    one = nvjsel.apply_adapters(x[0].cuda(), y[0].cuda(), table, ids[0].cuda())
    assert one.shape == (77,)


def test_deterministic_captured_and_on_other_streams():
    x, y, a, b, s, ids = make(50, 512, 3000, [16] * 6, seed=10)
    table = nvjsel.pack_adapters([t.cuda() for t in a], [t.cuda() for t in b], s)
    xd, yd, idd = x.cuda(), y.cuda(), ids.cuda()
    want = nvjsel.apply_adapters(xd, yd, table, idd)
    for _ in range(10):
        assert torch.equal(nvjsel.apply_adapters(xd, yd, table, idd), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = nvjsel.apply_adapters(xd, yd, table, idd)
    stream.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nvjsel.apply_adapters(xd, yd, table, idd)
    for k in range(4):
        idd.copy_(idd.roll(k + 1))
        graph.replay()
        eager = nvjsel.apply_adapters(xd, yd, table, idd)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("kind", ["bf16", "f32", "w4"])
def test_a_servers_step(kind):
    """LM head with adapters, sampled tokens, their log probabilities and alternatives, and the same scored from the
    hidden states: one result."""
    g = torch.Generator().manual_seed(11)
    rows, hidden, vocab = 13, 256, 3001
    weight = (torch.randn(vocab, hidden, generator=g) * 0.02).to(torch.bfloat16)
    x = (torch.randn(rows, hidden, generator=g) * 6).to(torch.float32 if kind == "f32" else torch.bfloat16).cuda()
    a = torch.randn(3, 16, hidden, generator=g).to(torch.bfloat16) / 16
    b = torch.randn(3, vocab, 16, generator=g).to(torch.bfloat16) / 8
    table = nvjsel.pack_adapters(a.cuda(), b.cuda(), [0.5, 1.0, 2.0])
    ids = (torch.arange(rows) % 4 - 1).to(torch.int32).cuda()
    head = weight.cuda().T if kind != "w4" else nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(weight.cuda().T))
    plain = nvjsel.lm_head_logits_hip(x, head)
    logits = nvjsel.lm_head_logits_hip(x, head, adapters=table, adapter_ids=ids)
    assert torch.equal(logits, nvjsel.apply_adapters(x, plain, table, ids))
    assert torch.equal(logits[ids < 0], plain[ids < 0]) and not torch.equal(logits[ids >= 0], plain[ids >= 0])
    temps = torch.full((rows,), 0.8, device="cuda")
    temps[2] = 0.0
    keys = torch.arange(2 * rows, dtype=torch.int32, device="cuda").reshape(rows, 2)
    tokens = nvjsel.lm_head_sample_token_ids(x, head, temperatures=temps, rng_keys=keys, adapters=table, adapter_ids=ids)
    assert torch.equal(tokens, nvjsel.sample_token_ids(logits, temps, keys))
    best, values, top = nvjsel.lm_head_token_ids_and_topk(x, head, top_k=4, adapters=table, adapter_ids=ids)
    again, _, _ = nvjsel.lm_head_token_ids_and_topk(x, head, adapters=table, adapter_ids=ids.reshape(rows, 1))
    assert torch.equal(best, again) and int(best[2]) == int(tokens[2])
    r = nvjsel.token_logprobs(logits, tokens, num_top=4, entropy=True)
    assert torch.equal(r.top_ids, top[:, 0])
    want = torch.log_softmax(logits.double().cpu(), 1)
    lp = want.gather(1, tokens.cpu().long()[:, None])[:, 0]
    assert bool(((r.logprobs.double().cpu() - lp).abs() <= 2.0 ** -19 + lp.abs() * 2.0 ** -24).all())
    scored = nvjsel.lm_head_token_logprobs(x, head, tokens, num_top=4, entropy=True, adapters=table, adapter_ids=ids)
    assert all(torch.equal(p, q) for p, q in zip(r, scored))


@pytest.mark.parametrize("rank", [16, 64, 512])
def test_most_rows(rank):
    """2^20 rows; 1000 of them have an adapter, the first and last ones too."""
    rows, hidden, width = 1 << 20, 8, 3
    g = torch.Generator().manual_seed(rank)
    x = torch.randn(rows, hidden, generator=g).to(torch.bfloat16)
    base = torch.randn(rows, width, generator=g).to(torch.bfloat16)
    a = [(torch.randn(rank, hidden, generator=g) / math.sqrt(hidden)).to(torch.bfloat16) for _ in range(2)]
    b = [(torch.randn(width, rank, generator=g) / math.sqrt(rank)).to(torch.bfloat16) for _ in range(2)]
    some = torch.randperm(rows, generator=g)[:998].tolist() + [0, rows - 1]
    ids = torch.full((rows,), -1, dtype=torch.int32)
    ids[some] = torch.randint(0, 2, (1000,), generator=g).to(torch.int32)
    s = torch.tensor([0.5, 1.5])
    table = nvjsel.pack_adapters([t.cuda() for t in a], [t.cuda() for t in b], s)
    got = nvjsel.apply_adapters(x.cuda(), base.cuda(), table, ids.cuda()).cpu()
    assert torch.equal(got[ids < 0], base[ids < 0])
    want, tol = oracle(x[some], base[some], a, b, s, ids[some])
    assert bool(((got[some].double() - want).abs() <= tol).all())
