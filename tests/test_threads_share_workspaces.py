"""Two threads on one stream, which share its workspaces: a call of several launches
keeps its launches together.  By the order of the launches on the CPU, and on the GPU by the
results of many calls that two threads queue without waiting for any."""
import threading

import pytest
import torch

import nvjsel
from tests.launch_recorder import launches

AT = 0x1000
SAMPLE = f"('nvjsel_sample', [P, I, I, I, L, P, P, P, P, P, P, P, Z, P], [{AT}, 1, {{0}}, {{1}}, {{1}}, {AT}, {{2}}, None, {AT}, None, {AT}, {AT}, 1 << 40, None])"
TOPK = f"('nvjsel_topk', [P, I, I, I, L, I, P, P, P, Z, P], [{AT}, 1, {{0}}, {{1}}, {{1}}, 8, {AT}, {AT}, {AT}, 1 << 40, None])"
PRENORM = (f"('nvjsel_lm_head_top1_prenorm', [P, I, P, I, F, I, P, I, I, I, I, I, I, P, P, P, Z, P], "
           f"[{AT}, 1, {AT}, 1, 1e-6, 1, {AT}, 1, 1, {{0}}, 1024, 248320, 1, {AT}, None, {AT}, 1 << 40, None])")
GREEDY = (f"('nvjsel_lm_head_top1', [P, I, P, I, I, I, I, I, I, P, P, P, Z, P], "
          f"[{AT}, 1, {AT}, 1, 1, 8, 1024, 248320, 1, {AT}, None, {AT}, 1 << 40, None])")
W4 = (f"('nvjsel_lm_head_w4_top1', [P, I, P, Z, I, I, I, I, I, I, I, P, P, P, Z, P], "
      f"[{AT}, 1, {AT}, 1 << 40, 1, 0, 128, 200, 1024, 32000, 1, {AT}, None, {AT}, 1 << 40, None])")


@pytest.mark.parametrize("first,other,several", [
    (SAMPLE.format(64, 248320, AT), SAMPLE.format(2, 9000, None), 4),
    (SAMPLE.format(64, 248320, AT), TOPK.format(8, 32000), 4),
    (TOPK.format(8, 32000), SAMPLE.format(2, 9000, None), 2),
    (TOPK.format(8, 32000), SAMPLE.format(64, 248320, AT), 2),
    (PRENORM.format(256), W4, 3),
    (PRENORM.format(256), GREEDY, 3),
], ids=["sample-sample", "sample-topk", "topk-sample", "topk-samples", "prenorm-w4", "prenorm-greedy"])
def test_a_call_keeps_its_launches_together(tmp_path, first, other, several):
    order = [thread for thread, _ in launches(tmp_path, first, other)]
    n = order.count("first")
    assert n == several and order == ["first"] * n + ["other"] * (len(order) - n)


@pytest.mark.gpu
def test_two_threads_queue_calls_of_all_kinds():
    g = torch.Generator().manual_seed(4)
    logits = (torch.randn(48, 50257, generator=g) * 2).to(torch.bfloat16).cuda()
    temps = torch.full((48,), 0.8, device="cuda")
    keys = nvjsel.derive_rng_keys(torch.arange(48, device="cuda", dtype=torch.int32),
                                  torch.zeros(48, device="cuda", dtype=torch.int32))[0]
    top_k = torch.full((48,), 20, device="cuda", dtype=torch.int32)
    weight = (torch.randn(9001, 256, generator=g) * 0.1).to(torch.bfloat16).cuda()
    head = nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(weight.T))
    norm = 0.1 * torch.randn(256, generator=g).cuda()
    x = torch.randn(150, 256, generator=g).to(torch.bfloat16).cuda()
    calls = [
        [lambda: nvjsel.sample_token_ids(logits, temps, keys, top_k=top_k),
         lambda: nvjsel.lm_head_greedy_top1_hip(x, weight.T, norm_weight=norm, act_dtype=torch.bfloat16),
         lambda: nvjsel.lm_head_greedy_top1_hip(x[:3], head)],
        [lambda: nvjsel.topk_hip(logits[:5], 9)[1],
         lambda: nvjsel.lm_head_greedy_top1_hip(x, head),
         lambda: nvjsel.lm_head_greedy_top1_hip(x[:9].float(), weight.T, norm_weight=norm, act_dtype=torch.float32),
         lambda: nvjsel.sample_token_ids(logits[:2], temps[:2], keys[:2])],
    ]
    want = [[call().clone() for call in mine] for mine in calls]
    torch.cuda.synchronize()
    got = [[], []]
    start = threading.Barrier(2)

    def queue(at):
        start.wait()
        for i in range(120):
            got[at].append(calls[at][i % len(calls[at])]())

    threads = [threading.Thread(target=queue, args=(at,)) for at in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for at in range(2):
        assert len(got[at]) == 120
        assert all(torch.equal(out, want[at][i % len(want[at])]) for i, out in enumerate(got[at]))
