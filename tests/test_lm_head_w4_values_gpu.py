"""GPU: weights, scales and activations at the ends of their types through the 4-bit LM head."""
import pytest
import torch

import nvjsel

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
