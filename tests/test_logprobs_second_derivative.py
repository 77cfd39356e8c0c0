"""token_logprobs is differentiable once: a second derivative is refused whatever stands beside it in the
loss.  Here with the launches replaced, and on the GPU."""
from __future__ import annotations

import pytest
import torch

import nvjsel
from nvjsel import _lib
from nvjsel import logprobs as module
from nvjsel._tensors import _HERE


def _replaced(monkeypatch):
    """Results in torch; the gradient's launch writes nothing."""
    def forward(logits, tokens, num_top, entropy, stats):
        lp = torch.log_softmax(logits.detach(), 1)
        return (lp.gather(1, tokens.long()[:, None])[:, 0], -(lp.exp() * lp).sum(1) if entropy else None, None, None,
                torch.zeros(logits.shape[0], 3))

    monkeypatch.setattr(module, "_require_cuda", lambda *ts: ts[0].device)
    monkeypatch.setattr(module, "_on_device", lambda device: _HERE)
    monkeypatch.setattr(module, "_stream_handle", lambda device: 0)
    monkeypatch.setattr(module, "_forward", forward)
    monkeypatch.setattr(_lib, "call", lambda *args: None)


def _second(device):
    x = torch.randn(3, 20, device=device, requires_grad=True)
    t = torch.tensor([1, 2, 3], device=device)
    for entropy in (False, True):
        for loss in (lambda r: r.logprobs.sum(), lambda r: (r.logprobs * torch.arange(3.0, device=device)).sum(),
                     lambda r: (r.logprobs + (r.entropy if entropy else 0)).pow(2).sum()):
            r = nvjsel.token_logprobs(x, t, entropy=entropy)
            d, = torch.autograd.grad(loss(r), x, create_graph=True)
            assert d.requires_grad
            with pytest.raises(RuntimeError, match="differentiable once"):
                (d.pow(2).sum() + (x * 2).sum()).backward()  # a penalty beside a loss of its own
            r = nvjsel.token_logprobs(x, t, entropy=entropy)
            d, = torch.autograd.grad(loss(r), x, create_graph=True)
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(d.sum(), x, allow_unused=True)
    z = x.detach().requires_grad_()
    nvjsel.token_logprobs(z, t).logprobs.sum().backward()
    assert not z.grad.requires_grad


def test_refused_whatever_stands_beside_it(monkeypatch):
    _replaced(monkeypatch)
    _second("cpu")


@pytest.mark.gpu
def test_refused_on_the_gpu():
    _second("cuda")


@pytest.mark.gpu
def test_the_gradient_in_the_graph_is_the_same():
    x = torch.randn(5, 301, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    t = torch.tensor([0, 300, -1, 7, 8], device="cuda")

    def gradient(create_graph):
        r = nvjsel.token_logprobs(x, t, entropy=True)
        return torch.autograd.grad([r.logprobs, r.entropy], x, [torch.ones(5, device="cuda"), torch.full((5,), 0.5, device="cuda")],
                                   create_graph=create_graph)[0]

    assert torch.equal(gradient(True).detach(), gradient(False))
