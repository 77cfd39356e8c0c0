"""Low-rank adapters: what the entry points refuse, before anything is launched."""
from __future__ import annotations

import pytest
import torch

import nvjsel
from nvjsel import adapters as module

B16 = torch.bfloat16


def _t(*shape, dtype=B16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("a,b,kw,what", [
    ([], [], {}, "at least one"),
    ([_t(4, 8)], [_t(6, 4), _t(6, 4)], {}, "at least one"),
    ([_t(4)], [_t(6, 4)], {}, "is a"),
    ([_t(4, 0)], [_t(6, 4)], {}, "non-empty"),
    ([_t(0, 8)], [_t(6, 0)], {}, "non-empty"),
    ([_t(4, 8), _t(4, 9)], [_t(6, 4)] * 2, {}, "one hidden size"),
    ([_t(4, 8)] * 2, [_t(6, 4), _t(7, 4)], {}, "one hidden size"),
    ([_t(4, 8)], [_t(6, 5)], {}, "ranks must match"),
    ([_t(4, 8, dtype=torch.float32)], [_t(6, 4, dtype=torch.float32)], {}, "bfloat16 or float16"),
    ([_t(4, 8)], [_t(6, 4, dtype=torch.float16)], {}, "bfloat16 or float16"),
    ([_t(513, 8)], [_t(6, 513)], {}, "at most 512"),
    ([_t(4, 8).requires_grad_()], [_t(6, 4)], {}, "not differentiable|device tensors"),
    ([_t(4, 8)], [_t(6, 4)], {}, "device tensors"),
])
def test_pack_refusals(a, b, kw, what):
    with pytest.raises(ValueError, match=what):
        nvjsel.pack_adapters(a, b, **kw)


def _table(hidden=8, width=6, rank=16, count=2):
    return nvjsel.AdapterTable(_t(count, rank * 32), _t(count, 64 * rank), _t(count, dtype=torch.float32), hidden, width, rank)


@pytest.mark.parametrize("change,what", [
    ({"x": _t(3, 8, 1)}, "one adapter id"), ({"ids": _t(4, dtype=torch.int32)}, "one adapter id"),
    ({"base": _t(2, 6)}, "one adapter id"), ({"x": _t(0, 8), "base": _t(0, 6), "ids": _t(0, dtype=torch.int32)}, "non-empty"),
    ({"x": _t(3, 9)}, "hidden 8 and width 6"), ({"base": _t(3, 7)}, "hidden 8 and width 6"),
    ({"x": _t(3, 8, dtype=torch.float64)}, "unsupported x"), ({"base": _t(3, 6, dtype=torch.int16)}, "unsupported base"),
    ({"ids": _t(3, dtype=torch.int64)}, "int32"),  ({"x": _t(3, 8).requires_grad_()}, "not differentiable"),
    ({"base": _t(3, 6).requires_grad_()}, "not differentiable"), ({}, "device tensors"),
    ({"x": _t(1, 8).expand((1 << 20) + 1, 8), "base": _t(1, 6).expand((1 << 20) + 1, 6),
      "ids": _t(1, dtype=torch.int32).expand((1 << 20) + 1)}, "at most"),
])
def test_apply_refusals(change, what):
    args = {"x": _t(3, 8), "base": _t(3, 6), "ids": _t(3, dtype=torch.int32), "out": None}
    args.update(change)
    with pytest.raises(ValueError, match=what):
        nvjsel.apply_adapters(args["x"], args["base"], _table(), args["ids"], out=args["out"])


def test_outputs_that_meet_the_base(monkeypatch):
    monkeypatch.setattr(module, "_require_cuda", lambda *ts: ts[0].device)
    buf = _t(10, 40)
    ids = _t(3, dtype=torch.int32)
    for out in (_t(3, 7), _t(3, 6, dtype=torch.float32)):
        with pytest.raises(ValueError, match="shape, type and device"):
            nvjsel.apply_adapters(_t(3, 8), _t(3, 6), _table(), ids, out=out)
    for base, out, what in ((buf[:3, :6], buf[1:4, :6], "share no memory"), (buf[:3, :6], buf[:3, 3:9], "share no memory"),
                            (buf[:3, :6], buf[0:6:2, :6], "share no memory"), (_t(3, 6), _t(1, 6).expand(3, 6), "must not overlap"),
                            (_t(3, 6), _t(6, 3).T, "contiguous")):
        with pytest.raises(ValueError, match=what):
            nvjsel.apply_adapters(_t(3, 8), base, _table(), ids, out=out)
    assert not module._meet(buf[:3, :6], buf[:3, 6:12]) and not module._meet(buf[:3, :6], buf[3:6, :6])
    assert module._meet(buf[:3, :6], buf[2:5, :6])
    assert not module._meet(buf[:3, 30:], buf[1:4, :10])


@pytest.mark.parametrize("fn", ["logits", "sample", "topk", "score"])
def test_the_lm_heads_entry_points_want_ids(fn):
    x, w = _t(3, 8), _t(8, 6)
    kw = {"adapters": _table(), "adapter_ids": None}
    with pytest.raises(ValueError, match="adapter_ids|device tensors"):
        if fn == "logits":
            nvjsel.lm_head_logits_hip(x, w, **kw)
        elif fn == "sample":
            nvjsel.lm_head_sample_token_ids(x, w, temperatures=_t(3), rng_keys=_t(3, 2), **kw)
        elif fn == "topk":
            nvjsel.lm_head_token_ids_and_topk(x, w, **kw)
        else:
            nvjsel.lm_head_token_logprobs(x, w, _t(3, dtype=torch.int32), **kw)


P = 1 << 20  # an address that nothing reads: every call here is refused


@pytest.mark.parametrize("change,what", [
    ({"x": None}, "null"), ({"base": None}, "null"), ({"a": None}, "null"), ({"b": None}, "null"), ({"scales": None}, "null"),
    ({"ids": None}, "null"), ({"out": None}, "null"), ({"xd": 5}, "dtype"), ({"od": -1}, "dtype"), ({"td": 0}, "dtype"),
    ({"count": 0}, "non-empty"), ({"rows": 0}, "non-empty"), ({"hidden": 0}, "non-empty"), ({"width": 0}, "non-empty"),
    ({"rank": 4}, "rank"), ({"rank": 24}, "rank"), ({"rank": 544}, "rank"), ({"rows": (1 << 20) + 1}, "rows"),
    ({"a": P + 8}, "unaligned tables"), ({"b": P + 2}, "unaligned tables"), ({"x": P + 1}, "unaligned rows"),
    ({"out": P + 1}, "unaligned rows"), ({"xs": -1}, "negative"), ({"bs": -4}, "negative"), ({"os": 5}, "stride < width"),
    ({"base": P, "out": P, "bs": 7, "os": 6}, "another stride"), ({"ws": None}, "workspace"), ({"wsb": 16}, "workspace"),
    ({"hidden": 7}, "below 8"), ({"rank": 8}, "rank"),
    ({"hidden": (1 << 24) + 1}, "too large"), ({"width": (1 << 28) + 1, "os": 1 << 30}, "too large"),
])
def test_c_refusals(change, what):
    a = {"x": P, "xd": 1, "xs": 8, "base": 2 * P, "od": 1, "bs": 6, "a": P, "b": P, "td": 1, "scales": P, "count": 2, "rank": 16,
         "hidden": 8, "width": 6, "ids": P, "rows": 3, "out": P, "os": 6, "ws": P, "wsb": 1 << 40, "stream": None}
    a.update(change)
    lib = nvjsel.load()
    assert lib.nvjsel_apply_adapters(*a.values()) < 0 and what in lib.nvjsel_last_error().decode()


@pytest.mark.parametrize("change,what", [
    ({"which": 2}, "which"), ({"count": 0}, "non-empty"), ({"rank": 0}, "non-empty"), ({"hidden": 0}, "non-empty"),
    ({"width": 0}, "non-empty"), ({"rank": 17}, "bad sizes"), ({"pad": 24}, "bad sizes"), ({"pad": 544, "rank": 530}, "bad sizes"),
    ({"plain": None}, "null"), ({"packed": None}, "null"), ({"plain": P + 1}, "unaligned"), ({"packed": P + 8}, "unaligned"),
    ({"cs": -1}, "negative"), ({"rs": -1}, "negative"), ({"bytes": 2 * 16 * 32 * 2 - 1}, "too small"),
    ({"width": 1 << 28, "which": 1, "bytes": 1 << 60, "pad": 512}, "too many"),
])
def test_c_pack_refusals(change, what):
    a = {"plain": P, "which": 0, "cs": 128, "rs": 8, "count": 2, "rank": 16, "hidden": 8, "width": 6, "pad": 16, "packed": P,
         "bytes": 1 << 20, "stream": None}
    a.update(change)
    lib = nvjsel.load()
    assert lib.nvjsel_adapters_pack(*a.values()) < 0 and what in lib.nvjsel_last_error().decode()


def test_workspace_sizes():
    size = nvjsel.load().nvjsel_adapters_workspace_size
    assert size(1, 3, 16) == 3 * 3 * 16 * 2 + 12 and size(2, 3, 16) == 3 * 2 * 16 * 2 + 12
    assert size(0, 3, 16) == 0 and size(1, 0, 16) == 0 and size(1, 3, 20) == 0
