"""Log probabilities from the hidden states: refusals, before anything is
launched."""
from __future__ import annotations

import pytest
import torch

import nvjsel


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


I32 = torch.int32


@pytest.mark.parametrize("x,w,t,kw,what", [
    (_t(2, 64), _t(64, 5), _t(3, dtype=I32), {}, "one token for every row"),
    (_t(0, 64), _t(64, 5), _t(0, dtype=I32), {}, "non-empty"),
    (_t(2, 64), _t(64, 5), _t(2, dtype=I32), {"num_top": 65}, "num_top"),
    (_t(2, 64), _t(64, 5), _t(2, dtype=torch.uint8), {}, "int32 or int64"),
    (_t(2, 64).requires_grad_(), _t(64, 5), _t(2, dtype=I32), {}, "not differentiable"),
    (_t(2, 64), _t(64, 5).requires_grad_(), _t(2, dtype=I32), {}, "not differentiable"),
    (_t(2, 64), _t(64, 5), _t(2, dtype=I32), {}, "device tensors"),
    (_t(1, 1).expand((1 << 23) + 1, 1), _t(1, 5), _t(1, dtype=I32).expand((1 << 23) + 1), {}, "at most"),
])
def test_refusals(x, w, t, kw, what):
    with pytest.raises(ValueError, match=what):
        nvjsel.lm_head_token_logprobs(x, w, t, **kw)


P = 1 << 20  # an address that nothing reads: every call here is refused


@pytest.mark.parametrize("change,code,what", [
    ({"x": None}, -1, "null"), ({"w": None}, -1, "null"), ({"t": None}, -1, "null"), ({"out": None}, -1, "null"),
    ({"xd": 4}, -1, "dtype"), ({"wd": 4}, -1, "dtype"), ({"layout": 2}, -1, "layout"), ({"rows": 0}, -1, "non-empty"),
    ({"h": 0}, -1, "non-empty"), ({"v": 0}, -1, "non-empty"), ({"rc": 3}, -1, "reduce_cast"), ({"tb": 2}, -1, "tokens"),
    ({"t": P + 2}, -1, "tokens"), ({"rows": (1 << 23) + 1}, -1, "at most"), ({"layout": 1}, -2, "takes"),
    ({"rc": 2}, -2, "reduce_cast"), ({"wd": 0}, -2, "takes"), ({"xd": 2}, -2, "takes"), ({"h": 96}, -2, "takes"), ({"x": P + 2}, -2, "aligned"),
    ({"w": P + 8}, -2, "aligned"), ({"ws": None}, -3, "workspace"), ({"wsb": 64}, -3, "workspace"), ({"ws": P + 8}, -3, "workspace"),
])
def test_c_refusals(change, code, what):
    a = {"x": P, "xd": 1, "w": P, "wd": 1, "layout": 0, "rows": 5, "h": 128, "v": 1000, "rc": 0, "t": P, "tb": 4, "out": P,
         "ent": None, "ws": P, "wsb": 1 << 40, "stream": None}
    a.update(change)
    lib = nvjsel.load()
    assert lib.nvjsel_lm_head_token_logprobs(*a.values()) == code and what in lib.nvjsel_last_error().decode()


def test_workspace_query():
    size = nvjsel.load().nvjsel_lm_head_token_logprobs_workspace_size
    assert size(1, 1, 0, 5, 128, 1000) > 0 and size(0, 1, 0, 5, 128, 1000) > 0 and size(2, 2, 0, 5, 128, 1000) > 0
    assert size(1, 2, 0, 5, 128, 1000) == 0 and size(1, 1, 1, 5, 128, 1000) == 0 and size(1, 1, 0, 5, 100, 1000) == 0
