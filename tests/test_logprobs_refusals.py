"""Log probabilities: what the entry points refuse, before anything is launched."""
from __future__ import annotations

import pytest
import torch

import nvjsel


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("logits,tokens,kw,what", [
    (_x(2, 5), _x(3, dtype=torch.int32), {}, "one token for every row"),
    (_x(2, 5), _x(2, 1, dtype=torch.int32), {}, "one token for every row"),
    (_x(0, 5), _x(0, dtype=torch.int32), {}, "non-empty"),
    (_x(2, 0), _x(2, dtype=torch.int32), {}, "non-empty"),
    (_x(2, 5), _x(2, dtype=torch.int32), {"num_top": 65}, "num_top"),
    (_x(2, 5), _x(2, dtype=torch.int32), {"num_top": -1}, "num_top"),
    (_x(2, 5, dtype=torch.float64), _x(2, dtype=torch.int32), {}, "unsupported logits dtype"),
    (_x(2, 5, dtype=torch.int32), _x(2, dtype=torch.int32), {}, "unsupported logits dtype"),
    (_x(2, 5), _x(2, dtype=torch.int16), {}, "int32 or int64"),
    (_x(2, 5), _x(2), {}, "int32 or int64"),
    (_x(2, 5), _x(2, dtype=torch.int32), {}, "device tensors"),
    (_x(1, 1).expand(1, (1 << 26) + 1), _x(1, dtype=torch.int32), {}, "at most"),
    (_x(1, 1).expand((1 << 23) + 1, 1), _x(1, dtype=torch.int32).expand((1 << 23) + 1), {}, "at most"),
])
def test_refusals(logits, tokens, kw, what):
    with pytest.raises(ValueError, match=what):
        nvjsel.token_logprobs(logits, tokens, **kw)


def _call(name, *args):
    lib = nvjsel.load()
    return getattr(lib, name)(*args), lib.nvjsel_last_error().decode()


P = 1 << 20  # an address that nothing reads: every call here is refused


@pytest.mark.parametrize("change,what", [
    ({"logits": None}, "null pointer"), ({"tokens": None}, "null pointer"), ({"dtype": 3}, "dtype"),
    ({"rows": 0}, "non-empty"), ({"vocab": 0}, "non-empty"), ({"vocab": (1 << 26) + 1}, "at most"),
    ({"rows": (1 << 23) + 1}, "at most"), ({"row_stride": -1}, "negative stride"), ({"token_bytes": 2}, "int32 or int64"),
    ({"num_top": 65}, "num_top"), ({"logits": P + 2}, "unaligned logits"), ({"tokens": P + 2}, "unaligned tokens"),
    ({"out": None}, "null output"), ({"num_top": 2}, "null output"), ({"ws_bytes": 100}, "workspace"), ({"ws": None}, "workspace"),
    ({"ws": P + 4}, "workspace"),
])
def test_c_refusals(change, what):
    a = {"logits": P, "dtype": 0, "rows": 3, "vocab": 10, "row_stride": 10, "tokens": P, "token_bytes": 4, "num_top": 0,
         "out": P, "entropy": None, "top": None, "ids": None, "stats": None, "ws": P, "ws_bytes": 1 << 40, "stream": None}
    a.update(change)
    rc, message = _call("nvjsel_token_logprobs", *a.values())
    assert rc < 0 and what in message


@pytest.mark.parametrize("change,what", [
    ({"stats": None}, "null pointer"), ({"out": None}, "null pointer"), ({"g": None}, "null pointer"),
    ({"out_stride": 9}, "stride < vocab"), ({"out": P + 1}, "unaligned gradient"), ({"dtype": 7}, "dtype"),
    ({"rows": 0}, "non-empty"), ({"logits": None}, "null pointer"), ({"token_bytes": 1}, "int32 or int64"),
])
def test_c_gradient_refusals(change, what):
    a = {"logits": P, "dtype": 1, "rows": 3, "vocab": 10, "row_stride": 10, "tokens": P, "token_bytes": 8, "stats": P, "g": P,
         "h": None, "out": P, "out_stride": 10, "stream": None}
    a.update(change)
    rc, message = _call("nvjsel_token_logprobs_grad", *a.values())
    assert rc < 0 and what in message


def test_workspaces_grow_with_the_call():
    lib = nvjsel.load()
    size = lib.nvjsel_token_logprobs_workspace_size
    assert size(1, 1, 248320, 0) > 16 * 1024 and size(1, 100000, 50, 0) == 16 * 1024
    assert size(1, 1, 248320, 20) > size(1, 1, 248320, 0)
    assert size(0, 0, 5, 0) == 0 and size(0, 5, 5, 65) == 0
