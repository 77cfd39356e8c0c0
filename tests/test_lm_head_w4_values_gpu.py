"""GPU: weights, scales and activations at the ends of their types through the 4-bit LM head."""
import pytest
import torch

import nvjsel
from nvjsel import _lib, _tensors
from tests.test_lm_head_w4_gpu import exact, tolerance

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def dequantized(q, s, z, group):
    codes = torch.stack((q & 15, q >> 4), 2).reshape(q.shape[0], -1).cpu().double()
    v, h = codes.shape
    zero = torch.full((v, h // group, 1), 8.0, dtype=torch.float64) if z is None else z.cpu().double()[:, :, None]
    return ((codes.reshape(v, h // group, group) - zero) * s.cpu().double()[:, :, None]).reshape(v, h)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype,group,scale", [("f32", 32, "bf16"), ("f32", 128, "f16"), ("bf16", 64, "bf16"),
                                               ("f16", 32, "f16"), ("bf16", 128, "f16")])
def test_weights_that_are_not_finite(dtype, group, scale, symmetric):
    """A group with a NaN or an infinity has a NaN scale: its row's logits are NaN, as with the
    weight itself, and nothing else changes."""
    w = (torch.randn(40, 256, generator=torch.Generator().manual_seed(group)) * 0.02).to(DT[dtype])
    kw = dict(group_size=group, symmetric=symmetric, scale_dtype=DT[scale], weight_layout="vh")
    q0, s0, z0 = nvjsel.quantize_lm_head_w4(w.cuda(), **kw)
    bad = {(3, 0): float("nan"), (7, 255): float("inf"), (8, group - 1): -float("inf"), (39, 131): float("nan")}
    for (v, k), x in bad.items():
        w[v, k] = x
    w[39] = float("nan")
    q, s, z = nvjsel.quantize_lm_head_w4(w.cuda(), **kw)
    at = torch.zeros(40, 256 // group, dtype=torch.bool)
    for v, k in bad:
        at[v, k // group] = True
    at[39] = True
    assert torch.equal(s.cpu().isnan(), at)
    assert torch.equal(s.cpu()[~at], s0.cpu()[~at])
    same = ~at.repeat_interleave(group // 2, 1)
    assert torch.equal(q.cpu()[same], q0.cpu()[same])
    assert symmetric or (torch.equal(z.cpu()[~at], z0.cpu()[~at]) and int(z.max()) <= 15)
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    logits = nvjsel.lm_head_logits_hip(x, nvjsel.pack_lm_head_w4(q, s, z), reduce_cast=0).cpu()
    want = nvjsel.lm_head_logits_hip(x, nvjsel.pack_lm_head_w4(q0, s0, z0), reduce_cast=0).cpu()
    rows = at.any(1)
    assert bool(logits[:, rows].isnan().all()) and torch.equal(logits[:, ~rows], want[:, ~rows])


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype,scale,size", [("f32", "f16", 1e6), ("bf16", "f16", 3e7), ("f32", "f16", 3e38),
                                              ("f32", "bf16", 3.3e38), ("bf16", "bf16", 3.3e38)])
def test_scales_beyond_their_type(dtype, scale, size, symmetric):
    """Finite weights whose scale does not fit its type: the largest scale, codes that end at
    0 and 15, and finite logits.  A code is the nearest one that there is: the value it
    stands for is off by half a scale at most, or ends at the codes' end."""
    w = torch.randn(17, 128, generator=torch.Generator().manual_seed(3)).clamp(-1, 1)
    w[5] *= 1e-3
    w[9] = 1.0
    w[10, ::2], w[10, 1::2] = 1.0, -1.0
    w = (w * size).to(DT[dtype])
    q, s, z = nvjsel.quantize_lm_head_w4(w.cuda(), group_size=32, symmetric=symmetric, scale_dtype=DT[scale],
                                         weight_layout="vh")
    assert bool(s.isfinite().all()) and bool((s > 0).all())
    wide = w.double().reshape(17, 4, 32)
    lo, hi = wide.amin(2).clamp(max=0), wide.amax(2).clamp(min=0)
    want = torch.maximum(hi, -lo) / 7 if symmetric else (hi - lo) / 15
    most = torch.finfo(DT[scale]).max
    step = torch.finfo(DT[scale]).eps / 2 + 2.0 ** -22  # the scale's rounding, and those of the f32 steps to it
    assert bool(((s.double().cpu() - want.clamp(max=most)).abs() <= step * want).all())
    assert bool((s.double().cpu()[want > most] == most).all())
    zero = torch.full((17, 4), 8.0, dtype=torch.float64) if symmetric else z.cpu().double()
    sd = s.cpu().double()
    bottom, top = -zero * sd, (15 - zero) * sd  # what the codes reach
    back = dequantized(q, s, z, 32).reshape(17, 4, 32)
    near = torch.minimum(torch.maximum(wide, bottom[:, :, None]), top[:, :, None])
    assert bool(((back - near).abs() <= sd[:, :, None] * (0.5 + 2.0 ** -18)).all())
    x = torch.randn(2, 128, generator=torch.Generator().manual_seed(2)) * 1e-6
    logits = nvjsel.lm_head_logits_hip(x.cuda(), nvjsel.pack_lm_head_w4(q, s, z))
    assert bool(logits.isfinite().all())


def test_zero_points_are_0_to_15():
    q = torch.randint(0, 256, (33, 64), dtype=torch.uint8, device="cuda")
    s = torch.full((33, 4), 0.01, dtype=torch.float16, device="cuda")
    z = torch.randint(0, 16, (33, 4), dtype=torch.uint8, device="cuda")
    head = nvjsel.pack_lm_head_w4(q, s, z)
    for bad in (16, 240, 255):
        wrong = z.clone()
        wrong[32, 3] = bad
        with pytest.raises(ValueError, match="0..15"):
            nvjsel.pack_lm_head_w4(q, s, wrong)
    # by the C ABI, which does not wait: the low four bits count
    packed, high = torch.empty_like(head.packed), z + 240
    _lib.call("nvjsel_w4_pack", q.data_ptr(), s.data_ptr(), high.data_ptr(), 33, 128, 32, packed.data_ptr(),
              packed.numel(), torch.cuda.current_stream().cuda_stream)
    x = torch.randn(3, 128, device="cuda")
    other = nvjsel.W4Weight(packed, 33, 128, 32, torch.float16, True)
    assert torch.equal(nvjsel.lm_head_logits_hip(x, other), nvjsel.lm_head_logits_hip(x, head))


@pytest.mark.parametrize("rows,vocab,hidden,group,act,zeros", [
    (1, 300, 1024, 128, "bf16", False), (16, 300, 512, 64, "bf16", True), (64, 70000, 2048, 128, "bf16", False),
    (3, 300, 1024, 128, "f32", True), (16, 40000, 1024, 128, "f32", False), (31, 70000, 2048, 32, "f32", True),
    (5, 300, 1024, 128, "f16", True)])
def test_largest_activations(rows, vocab, hidden, group, act, zeros):
    """Values of 2^115 (f16: its largest) whose offsets, partial sums and products add up the most."""
    size = torch.finfo(torch.float16).max if act == "f16" else 2.0 ** 115
    g = torch.Generator().manual_seed(rows)
    codes = torch.randint(0, 16, (vocab, hidden), generator=g, dtype=torch.uint8)
    codes[0], codes[1] = 15, 0
    scales = torch.full((vocab, hidden // group), 2.0 ** -10, dtype=torch.bfloat16)
    z = torch.randint(0, 16, (vocab, hidden // group), generator=g, dtype=torch.uint8) if zeros else None
    if zeros:
        z[0], z[1] = 0, 15
    x = (torch.randint(0, 2, (rows, hidden), generator=g) * 2 - 1) * size
    x[0] = size
    x[-1, hidden // 2:] = -size
    x = x.to(DT[act])
    q = codes[:, 0::2] | codes[:, 1::2] << 4
    head = nvjsel.pack_lm_head_w4(q.cuda(), scales.cuda(), None if z is None else z.cuda())
    got = nvjsel.lm_head_logits_hip(x.cuda(), head, reduce_cast=0)[:, :300].cpu()
    want, mag = exact(codes[:300], scales[:300], None if z is None else z[:300], group, x)
    assert bool(((got.double() - want).abs() <= tolerance(want, mag, torch.float32)).all())


def test_captured_routes_keep_their_own_workspaces(monkeypatch):
    """Every route of a 4-bit weight, captured: none takes the stream's workspace, and replays with
    eager calls between them give the eager results."""
    weight = (torch.randn(20011, 256, generator=torch.Generator().manual_seed(6)) * 0.1).to(torch.bfloat16).cuda()
    head = nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(weight.T))
    xs = [(torch.randn(9, 1, 256, generator=torch.Generator().manual_seed(i)) * 2).to(torch.bfloat16).cuda() for i in range(3)]
    keys = nvjsel.derive_rng_keys(torch.arange(9, device="cuda", dtype=torch.int32),
                                  torch.ones(9, device="cuda", dtype=torch.int32))[0]
    temps = torch.full((9,), 0.9, device="cuda")
    top_k = torch.full((9,), 12, device="cuda", dtype=torch.int32)
    norm = 0.1 * torch.randn(256, generator=torch.Generator().manual_seed(9)).cuda()
    scores = torch.zeros(3, 3, device="cuda")

    def routes(x):
        return [nvjsel.lm_head_greedy_top1_hip(x, head), nvjsel.lm_head_logits_hip(x, head),
                nvjsel.lm_head_sample_token_ids(x, head, temperatures=temps, rng_keys=keys),
                nvjsel.lm_head_sample_token_ids(x, head, temperatures=temps, rng_keys=keys, top_k=top_k, norm_weight=norm,
                                                act_dtype=torch.bfloat16),
                *nvjsel.lm_head_token_ids_and_topk(x.reshape(3, 3, 256), head, top_k=5),
                nvjsel.mtp_greedy_top1_token_ids(x.reshape(3, 3, 256), head),
                *nvjsel.lm_head_beam_search_step(x.reshape(3, 3, 256), head, scores)]

    want = [[t.clone() for t in routes(x)] for x in xs]
    fixed = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with monkeypatch.context() as m:
        m.setattr(type(_tensors._WS), "get", lambda *a: pytest.fail("a captured call took the stream's workspace"))
        with torch.cuda.graph(graph):
            out = routes(fixed)
    for rep in range(4):
        fixed.copy_(xs[rep % 3])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[rep % 3]))
        assert all(torch.equal(a, b) for a, b in zip(routes(xs[1]), want[1]))
