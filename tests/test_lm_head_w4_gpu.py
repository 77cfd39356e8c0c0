"""GPU: the LM head with 4-bit weights and group scales against a plain product
in 64 bits.

Tolerance of an fp32 logit: four roundings (2^-24 each) of the sum of the
magnitudes that a group adds up, sum_G s_G (sum_k |x_k| (16 + q_k) + (16 + z) |sum_k
x_k|); a group's partial sums are about sqrt(group) smaller than that, so it
stands for some forty of their roundings.  One wrong code is off by s |x|, some
hundred times more.  A 16-bit logit adds half a step of its type."""
import numpy as np
import pytest
import torch

import nvjsel
from nvjsel import _lib

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(vocab, hidden, group, scale_dtype, zeros, seed):
    rng = np.random.default_rng(seed)
    codes = torch.from_numpy(rng.integers(0, 16, (vocab, hidden)).astype(np.uint8))
    scales = torch.from_numpy((0.002 + 0.01 * rng.random((vocab, hidden // group))).astype(np.float32)).to(scale_dtype)
    z = torch.from_numpy(rng.integers(0, 16, (vocab, hidden // group)).astype(np.uint8)) if zeros else None
    q = codes[:, 0::2] | (codes[:, 1::2] << 4)
    return codes, q.contiguous(), scales, z


def exact(codes, scales, zeros, group, x):
    """Logits in 64 bits, and the tolerance's magnitudes."""
    v, h = codes.shape
    q = codes.double().reshape(v, h // group, group)
    z = torch.full((v, h // group), 8.0, dtype=torch.float64) if zeros is None else zeros.double()
    s = scales.double()
    w = ((q - z[:, :, None]) * s[:, :, None]).reshape(v, h)
    x = x.double()
    logits = x @ w.T
    mag = x.abs() @ ((q + 16) * s[:, :, None]).reshape(v, h).T
    mag += x.reshape(-1, h // group, group).sum(2).abs() @ (s * (16 + z)).T
    return logits, mag


def tolerance(logits, mag, dtype):
    tol = 4 * 2.0 ** -24 * mag
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (logits.abs() + tol) + torch.finfo(dtype).smallest_normal
    return tol


def hidden_rows(rows, hidden, dtype, seed):
    return (torch.randn(rows, hidden, generator=torch.Generator().manual_seed(seed)) * 2).to(dtype)


@pytest.mark.parametrize("rows,vocab,hidden,group,act,scale,zeros", [
    (1, 1, 32, 32, "bf16", "bf16", False),
    (1, 17, 128, 128, "f32", "f16", True),
    (2, 15, 96, 32, "f16", "f16", False),
    (3, 1003, 160, 32, "bf16", "f16", True),
    (5, 300, 192, 64, "f32", "bf16", False),
    (1, 5000, 1024, 128, "bf16", "bf16", False),
    (8, 4099, 2560, 64, "f16", "f16", True),
    (16, 70001, 512, 128, "bf16", "bf16", False),  # several rounds of every wave
    (16, 515, 1024, 64, "f32", "f16", True),
    (17, 515, 768, 64, "bf16", "bf16", True),
    (32, 333, 768, 32, "f32", "bf16", False),
    (33, 300, 2048, 128, "f16", "f16", False),
    (48, 2000, 1024, 32, "bf16", "bf16", True),
    (64, 2000, 1024, 128, "bf16", "f16", False),
    (64, 600, 4096, 128, "f16", "f16", True),  # the hidden rows in parts
    (24, 600, 4096, 64, "f32", "bf16", False),
    (12, 40, 16384, 128, "bf16", "bf16", False),
    (131, 257, 256, 128, "bf16", "bf16", True),  # several passes
    (67, 99, 128, 32, "f32", "f16", False),
])
def test_logits_and_greedy(rows, vocab, hidden, group, act, scale, zeros):
    codes, q, scales, z = make(vocab, hidden, group, DT[scale], zeros, rows * 7919 + vocab)
    x = hidden_rows(rows, hidden, DT[act], vocab)
    head = nvjsel.pack_lm_head_w4(q.cuda(), scales.cuda(), None if z is None else z.cuda())
    want, mag = exact(codes, scales, z, group, x)
    xd = x.cuda().reshape(rows, 1, hidden)
    got = nvjsel.lm_head_logits_hip(xd, head)
    assert got.dtype == DT[act] and got.shape == (rows, vocab)
    assert bool(((got.double().cpu() - want).abs() <= tolerance(want, mag, DT[act])).all())
    fp32 = nvjsel.lm_head_logits_hip(xd, head, reduce_cast=0)
    assert fp32.dtype == torch.float32
    assert bool(((fp32.double().cpu() - want).abs() <= tolerance(want, mag, torch.float32)).all())
    # greedy is the first maximum of the same logits, rounded or not
    for rc, logits in ((None, got), (0, fp32)):
        ids, best = nvjsel.lm_head_greedy_top1_hip(xd, head, reduce_cast=rc, return_best=True)
        assert ids.shape == (rows, 1) and ids.dtype == torch.int32
        l = logits.float().cpu().numpy()
        assert np.array_equal(ids.cpu().numpy()[:, 0], l.argmax(1))
        assert np.array_equal(best.cpu().numpy(), l.max(1))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,vocab", [(3, 300), (16, 1000), (5, 40000), (16, 40000), (33, 40000)])
def test_f32_terms_do_not_round_each_other(rows, vocab, zeros):
    """Activations hi + lo, hi an integer of 8 bits and lo a multiple of 2^-11 below one:
    over 128 of them, each part's sum with codes below 32 fits 24 bits (255 x 31 x 128 <
    2^20; 2^11 x 31 x 128 < 2^23), both together need 31.  Kept apart they meet in at
    most two roundings, each of at most the result and lo's part (31 x 128 x 2^-8 < 16
    of the last term); the scale is a power of two."""
    rng = np.random.default_rng(rows + vocab)
    hi = rng.integers(128, 256, (rows, 128)) * rng.choice([-1, 1], (rows, 128))
    x = hi + np.sign(hi) * rng.integers(0, 2048, (rows, 128)) / 2048.0
    x = torch.from_numpy(x.astype(np.float32))
    codes, q, scales, z = make(vocab, 128, 128, torch.float16, zeros, 3)
    scales.fill_(0.125)
    head = nvjsel.pack_lm_head_w4(q.cuda(), scales.cuda(), None if z is None else z.cuda())
    want, _ = exact(codes, scales, z, 128, x)
    got = nvjsel.lm_head_logits_hip(x.cuda(), head).double().cpu()
    assert bool(((got - want).abs() <= 2.0 ** -24 * (2 * want.abs() + 2)).all())


@pytest.mark.parametrize("rows,vocab,hidden,group,act,zeros", [
    (16, 40000, 1024, 128, "f32", True),    # terms apart, hidden in LDS
    (16, 9000, 1664, 64, "f32", False),     # rows in fours: four groups of blocks
    (31, 70000, 2048, 128, "f32", False),   # terms apart, hidden in parts
    (64, 9000, 2048, 32, "bf16", True),     # four groups of 16 rows
    (40, 33000, 1024, 128, "f16", False),   # two groups of 32, the second with 8
    (48, 9000, 1024, 128, "bf16", False),   # three groups: blocks not a power of two
    (64, 70000, 1024, 64, "f16", True),     # one tile of 64
    (64, 70000, 8192, 128, "bf16", False),  # in parts
    (32, 66000, 5120, 64, "bf16", True),    # one tile of 32, in parts
    (16, 40000, 8192, 32, "f16", True),     # one of 16, in parts
    (4, 3001, 20480, 32, "bf16", True),     # rows in eights, in parts
    (4, 3001, 5120, 64, "f32", True),
    (7, 3001, 5120, 32, "f32", False),
    (9, 2000, 1024, 128, "f16", False),     # two groups of eight
    (256, 9000, 1024, 64, "bf16", True),    # sixteen groups
    (200, 40000, 2048, 128, "f16", False),
    (300, 2000, 640, 128, "f32", False),    # several launches
])
def test_tile_shapes(rows, vocab, hidden, group, act, zeros):
    """Sizes at which each shape of tiles is taken; a sample of the vocabulary is compared."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    q = torch.randint(0, 256, (vocab, hidden // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.002 + 0.01 * torch.rand(vocab, hidden // group, generator=g, device="cuda")).to(DT["f16"])
    z = torch.randint(0, 16, (vocab, hidden // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    x = hidden_rows(rows, hidden, DT[act], 4)
    head = nvjsel.pack_lm_head_w4(q, scales, z)
    logits = nvjsel.lm_head_logits_hip(x.cuda(), head, reduce_cast=0)
    pick = torch.cat([torch.arange(0, vocab, 37), torch.arange(vocab - 70, vocab)])
    qp = q[pick.cuda()].cpu()
    codes = torch.stack([qp & 15, qp >> 4], 2).reshape(len(pick), hidden)
    want, mag = exact(codes, scales[pick.cuda()].cpu(), None if z is None else z[pick.cuda()].cpu(), group, x)
    assert bool(((logits[:, pick.cuda()].double().cpu() - want).abs() <= tolerance(want, mag, torch.float32)).all())
    ids, best = nvjsel.lm_head_greedy_top1_hip(x.cuda().reshape(rows, 1, hidden), head, reduce_cast=0, return_best=True)
    l = logits.cpu().numpy()
    assert np.array_equal(ids.cpu().numpy()[:, 0], l.argmax(1))
    assert np.array_equal(best.cpu().numpy(), l.max(1))


def test_other_routes_take_the_weight():
    """Sampling, top-k, the prenorm input and the MTP route are those of the dense logits."""
    codes, q, scales, z = make(3001, 512, 64, torch.bfloat16, True, 5)
    head = nvjsel.pack_lm_head_w4(q.cuda(), scales.cuda(), z.cuda())
    x = hidden_rows(6, 512, torch.bfloat16, 9).cuda()
    logits = nvjsel.lm_head_logits_hip(x, head)
    keys = nvjsel.derive_rng_keys(torch.arange(6, device="cuda", dtype=torch.int32),
                                  torch.arange(6, device="cuda", dtype=torch.int32))[0]
    temps = torch.tensor([0.0, 0.7, 1.0, 0.9, 1.3, 0.5], device="cuda")
    top_k = torch.tensor([0, 5, 0, 20, 0, 0], device="cuda", dtype=torch.int32)
    for kw in ({}, {"top_k": top_k}):
        a = nvjsel.lm_head_sample_token_ids(x, head, temperatures=temps, rng_keys=keys, **kw)
        assert torch.equal(a, nvjsel.sample_token_ids(logits, temps, keys, **kw))
    ids, values, indices = nvjsel.lm_head_token_ids_and_topk(x.reshape(2, 3, 512), head, top_k=7)
    v, i = nvjsel.topk_hip(logits, 7)
    assert torch.equal(values.reshape(6, 7), v) and torch.equal(indices.reshape(6, 7), i)
    assert torch.equal(ids.reshape(6), i[:, 0])
    assert torch.equal(nvjsel.lm_head_token_ids_and_topk(x.reshape(2, 3, 512), head)[0].reshape(6), i[:, 0])
    assert torch.equal(nvjsel.mtp_greedy_top1_token_ids(x.reshape(2, 3, 512), head).reshape(6), i[:, 0])
    nw = 0.1 * torch.randn(512, device="cuda")
    normed = nvjsel.rms_norm_hip(x, nw, act_dtype=torch.bfloat16)
    assert torch.equal(nvjsel.lm_head_greedy_top1_hip(x, head, norm_weight=nw, act_dtype=torch.bfloat16),
                       nvjsel.lm_head_greedy_top1_hip(normed, head))


def test_views_strides_and_padding():
    """Hidden rows from any element and stride; logits rows apart by more than the vocabulary."""
    codes, q, scales, z = make(777, 256, 32, torch.float16, True, 3)
    head = nvjsel.pack_lm_head_w4(q.cuda(), scales.cuda(), z.cuda())
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        x = hidden_rows(5, 256, dt, 1)
        want = nvjsel.lm_head_logits_hip(x.cuda(), head)
        odd = torch.empty(5 * 256 + 1, dtype=dt, device="cuda")[1:].reshape(5, 256)
        odd.copy_(x)
        wide = torch.zeros(5, 300, dtype=dt, device="cuda")
        wide[:, 7:263] = x.cuda()
        assert torch.equal(nvjsel.lm_head_logits_hip(odd, head), want)
        assert torch.equal(nvjsel.lm_head_logits_hip(wide[:, 7:263], head), want)
        out = torch.full((5, 781), 7.0, dtype=dt, device="cuda")
        code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dt]
        _lib.call("nvjsel_lm_head_w4_logits", x.cuda().data_ptr(), code, head.packed.data_ptr(), head.packed.numel(),
                  _lib.F16, 1, 32, 5, 256, 777, code, out.data_ptr(), code, 781,
                  torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out[:, :777], want) and bool((out[:, 777:] == 7.0).all())


@pytest.mark.parametrize("act", ["bf16", "f16", "f32"])
def test_non_finite_rows_and_scales(act):
    """A NaN or an infinity makes its row NaN and no other; large finite values stay."""
    codes, q, scales, z = make(130, 128, 32, torch.bfloat16, False, 8)
    x = hidden_rows(4, 128, DT[act], 2)
    x[0, 3] = float("nan")
    x[1, 77] = float("inf")
    x[2] *= 1000.0
    scales[7] = 0.0
    head = nvjsel.pack_lm_head_w4(q.cuda(), scales.cuda())
    got = nvjsel.lm_head_logits_hip(x.cuda(), head, reduce_cast=0).cpu()
    assert bool(got[:2].isnan().all())
    want, mag = exact(codes, scales, None, 32, x[2:])
    assert bool(((got[2:].double() - want).abs() <= tolerance(want, mag, torch.float32)).all())
    assert bool((got[2:, 7] == 0).all())
    ids, best = nvjsel.lm_head_greedy_top1_hip(x.cuda(), head, return_best=True)
    assert ids[:2].flatten().tolist() == [0, 0] and bool(best[:2].isnan().all())  # the first NaN


@pytest.mark.parametrize("dtype,group,symmetric,layout,scale", [
    ("f32", 128, True, "vh", None), ("bf16", 64, False, None, None), ("f16", 32, True, "hv", torch.bfloat16),
    ("f32", 32, False, "vh", torch.float16),
])
def test_quantize(dtype, group, symmetric, layout, scale):
    g = torch.Generator().manual_seed(11)
    w = (torch.randn(203, 256, generator=g) * 0.02).to(DT[dtype])
    w[5, :group] = 0.0
    w[6] = w[6].abs()
    given = w.cuda() if layout == "vh" else w.cuda().T if layout is None else w.T.contiguous().cuda()
    q, s, z = nvjsel.quantize_lm_head_w4(given, group_size=group, symmetric=symmetric, scale_dtype=scale,
                                         weight_layout=layout)
    sdt = scale or (torch.bfloat16 if dtype == "f32" else DT[dtype])
    f = w.float().reshape(203, 256 // group, group)
    lo, hi = f.amin(2).clamp(max=0), f.amax(2).clamp(min=0)
    want_s = ((hi - lo) / 15 if not symmetric else torch.maximum(hi, -lo) / 7).to(sdt)
    assert torch.equal(s.cpu(), want_s)
    sf = want_s.float()
    some = sf > 0
    div = torch.where(some, sf, torch.ones(()))
    zero = torch.full_like(sf, 8.0) if symmetric else torch.where(some, torch.round(-lo / div).clamp(0, 15), torch.zeros(()))
    codes = torch.where(some[:, :, None], (torch.round(f / div[:, :, None]) + zero[:, :, None]).clamp(0, 15),
                        zero[:, :, None]).reshape(203, 256).to(torch.uint8)
    assert torch.equal(q.cpu(), codes[:, 0::2] | (codes[:, 1::2] << 4))
    assert (z is None) == symmetric and (symmetric or torch.equal(z.cpu(), zero.to(torch.uint8)))
    x = hidden_rows(3, 256, torch.bfloat16, 4)
    got = nvjsel.lm_head_logits_hip(x.cuda(), nvjsel.pack_lm_head_w4(q, s, z), reduce_cast=0).cpu()
    want, mag = exact(codes, want_s, None if symmetric else zero.to(torch.uint8), group, x)
    assert bool(((got.double() - want).abs() <= tolerance(want, mag, torch.float32)).all())


def test_captured_calls_keep_their_own_workspaces():
    """Two graphs captured on one stream, replayed at the same time on two others,
    with eager calls between; every replay against the eager ids."""
    codes, q, scales, z = make(20011, 512, 128, torch.bfloat16, False, 21)
    head = nvjsel.pack_lm_head_w4(q.cuda(), scales.cuda())
    xs = [hidden_rows(9, 512, torch.bfloat16, 30 + i).cuda() for i in range(4)]
    want = [nvjsel.lm_head_greedy_top1_hip(x, head).clone() for x in xs]
    side, graphs, inputs, outs = torch.cuda.Stream(), [], [], []
    for i in range(2):
        x = xs[i].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = nvjsel.lm_head_greedy_top1_hip(x, head)
        graphs.append(graph), inputs.append(x), outs.append(out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for i in range(2):
            inputs[i].copy_(xs[(rep + i) % 4])
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[(rep + i) % 4])
        assert torch.equal(nvjsel.lm_head_greedy_top1_hip(xs[rep], head), want[rep])


def test_large_packed_weight():
    """Offsets past 32 bits: 4.3 GB of packed weight, its last rows against the plain product."""
    vocab, hidden = 1 << 21, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randint(0, 256, (vocab, hidden // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.full((vocab, hidden // 128), 0.01, dtype=torch.bfloat16, device="cuda")
    head = nvjsel.pack_lm_head_w4(q, scales)
    assert head.packed.numel() > 1 << 32
    x = hidden_rows(2, hidden, torch.bfloat16, 6)
    got = nvjsel.lm_head_logits_hip(x.cuda(), head, reduce_cast=0)
    tail = q[-64:].cpu()
    codes = torch.stack((tail & 15, tail >> 4), 2).reshape(64, hidden)
    want, mag = exact(codes, scales[-64:].cpu(), None, 128, x)
    assert bool(((got[:, -64:].double().cpu() - want).abs() <= tolerance(want, mag, torch.float32)).all())
    ids = nvjsel.lm_head_greedy_top1_hip(x.cuda(), head, reduce_cast=0)
    assert torch.equal(ids[:, 0].long(), got.argmax(1))
