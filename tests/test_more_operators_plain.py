"""The plain forms of perf/more_operators.py leave what they are given as it is: a second pass over the
same inputs gives the first one's results."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

_FILE = Path(__file__).resolve().parent.parent / "perf" / "more_operators.py"


def _module():
    spec = importlib.util.spec_from_file_location("more_operators", _FILE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _state(kind, dtype):
    g = torch.Generator().manual_seed(1)
    if kind == "adapters":
        return {"kind": kind, "x": torch.randn(5, 16, generator=g).to(dtype), "base": torch.randn(5, 12, generator=g).to(dtype),
                "a": torch.randn(2, 4, 16, generator=g).to(torch.bfloat16), "b": torch.randn(2, 12, 4, generator=g).to(torch.bfloat16),
                "scales": torch.tensor([0.5, 2.0]), "ids": torch.tensor([0, 1, -1, 1, 0], dtype=torch.int32)}
    tokens = torch.tensor([3, 0, -1, 29, 7])
    if kind == "score":
        return {"kind": kind, "hidden": torch.randn(5, 16, generator=g).to(dtype),
                "weight": torch.randn(30, 16, generator=g).to(torch.bfloat16), "tokens": tokens, "entropy": True}
    logits = torch.randn(5, 30, generator=g).to(dtype)
    logits[2] = -torch.inf
    return {"kind": "logprobs", "logits": logits, "tokens": tokens, "top": 0 if kind == "grad" else 3, "entropy": True,
            "grad": kind == "grad", "grad_logprobs": torch.randn(5, generator=g), "grad_entropy": torch.randn(5, generator=g)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["adapters", "score", "logprobs", "grad"])
def test_a_second_pass_gives_the_same(kind, dtype):
    module = _module()
    state = _state(kind, dtype)
    before = {k: v.clone() for k, v in state.items() if torch.is_tensor(v)}

    def run():
        out = module.run(state)
        return [t.clone() for t in (out if isinstance(out, list) else [out])]

    first, second = run(), run()
    assert all(torch.equal(state[k], v) for k, v in before.items())
    assert len(first) == len(second) and all(torch.equal(p, q) for p, q in zip(first, second))
