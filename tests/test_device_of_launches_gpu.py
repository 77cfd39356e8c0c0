"""GPU: every launch of the 4-bit head's and of beam search's routes is made with its tensors'
device as the current one."""
import pytest
import torch

import nvjsel
from nvjsel import _lib, beam, selection, w4

pytestmark = pytest.mark.gpu


class Here:
    """In place of the context that makes a device the current one."""

    inside = 0

    def __enter__(self):
        Here.inside += 1

    def __exit__(self, *_):
        Here.inside -= 1


def test_launches_are_made_on_their_tensors_device(monkeypatch):
    weight = (torch.randn(501, 128) * 0.1).to(torch.bfloat16).cuda()
    x = torch.randn(4, 128, device="cuda").to(torch.bfloat16)
    norm = torch.zeros(128, device="cuda")
    keys = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    temps = torch.ones(4, device="cuda")
    top_k = torch.full((4,), 3, dtype=torch.int32, device="cuda")
    state = torch.zeros(4, 8, device="cuda")
    launched, outside = [], []
    real = _lib.call

    def call(name, *args):
        launched.append(name)
        if not Here.inside:
            outside.append(name)
        return real(name, *args)

    for module in (beam, selection, w4):
        monkeypatch.setattr(module, "_on_device", lambda device: Here(), raising=False)
    monkeypatch.setattr(_lib, "call", call)
    head = nvjsel.pack_lm_head_w4(*nvjsel.quantize_lm_head_w4(weight.T))
    nvjsel.lm_head_greedy_top1_hip(x, head, norm_weight=norm)
    nvjsel.lm_head_logits_hip(x, head)
    nvjsel.lm_head_sample_token_ids(x, head, temperatures=temps, rng_keys=keys)
    nvjsel.lm_head_sample_token_ids(x, head, temperatures=temps, rng_keys=keys, top_k=top_k)
    nvjsel.lm_head_token_ids_and_topk(x, head, top_k=2, norm_weight=norm)
    nvjsel.mtp_greedy_top1_token_ids(x[None], head)
    for output_weight in (head, weight.T):
        nvjsel.lm_head_beam_search_step(x[None], output_weight, torch.zeros(1, 4, device="cuda"), states=[state],
                                        norm_weight=norm, act_dtype=torch.bfloat16)
    torch.cuda.synchronize()
    assert {"nvjsel_w4_quantize", "nvjsel_w4_pack", "nvjsel_lm_head_w4_top1", "nvjsel_lm_head_w4_logits", "nvjsel_sample",
            "nvjsel_topk", "nvjsel_rms_norm", "nvjsel_lm_head_logits", "nvjsel_beam_select",
            "nvjsel_reorder_states"} == set(launched)
    assert not outside, outside
