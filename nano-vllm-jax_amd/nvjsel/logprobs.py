"""Log probabilities of given tokens, with entropies and top alternatives, and
their gradient."""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from . import _lib
from ._tensors import _dtype_code, _on_device, _require_cuda, _stream_handle, _workspace

MAX_TOP = 64  # alternatives of a row
MAX_ROWS, MAX_VOCAB = 1 << 23, 1 << 26  # of a call
_AT_REST = 16 * 1024  # bytes of the workspace that are zero at rest


class TokenLogprobs(NamedTuple):
    """``token_logprobs``'s results; None where not asked for."""

    logprobs: torch.Tensor  # f32, the tokens' shape
    entropy: torch.Tensor | None  # f32, the tokens' shape
    top_logprobs: torch.Tensor | None  # f32, the tokens' shape and num_top
    top_ids: torch.Tensor | None  # int32, likewise


@lru_cache(maxsize=1024)
def _bytes(device: int, *shape: int) -> int:  # by device: its compute units count
    return _lib.load().nvjsel_token_logprobs_workspace_size(*shape)


def _row_stride(logits: torch.Tensor) -> int:
    return logits.stride(0) if logits.shape[0] > 1 else logits.shape[1]


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _forward(logits, tokens, num_top: int, entropy: bool, stats: bool):
    """Of ``logits [N, V]`` with unit token stride; and the rows' statistics for the gradient."""
    rows, vocab = logits.shape
    dev = logits.device
    logprobs = torch.empty((rows,), dtype=torch.float32, device=dev)
    ent = torch.empty_like(logprobs) if entropy else None
    kept = torch.empty((rows, 3), dtype=torch.float32, device=dev) if stats else None
    top = ids = None
    if num_top:
        top = torch.empty((rows, num_top), dtype=torch.float32, device=dev)
        ids = torch.empty((rows, num_top), dtype=torch.int32, device=dev)
    dt = _dtype_code(logits, "logits")
    with _on_device(dev):
        nbytes = _bytes(dev.index, dt, rows, vocab, num_top)
        stream = _stream_handle(dev)
        ws = _workspace(dev, stream, "logprobs", nbytes, _AT_REST)
        _lib.call("nvjsel_token_logprobs", logits.data_ptr(), dt, rows, vocab, _row_stride(logits), tokens.data_ptr(),
                  tokens.element_size(), num_top, logprobs.data_ptr(), _ptr(ent), _ptr(top), _ptr(ids), _ptr(kept),
                  ws.data_ptr(), nbytes, stream)
    return logprobs, ent, top, ids, kept


class _Differentiable(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, num_top, entropy):
        logprobs, ent, top, ids, stats = _forward(logits, tokens, num_top, entropy, True)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.set_materialize_grads(False)
        if top is not None:
            ctx.mark_non_differentiable(top, ids)
        return logprobs, ent, top, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprobs, grad_entropy, *_):
        if grad_logprobs is None and grad_entropy is None:
            return None, None, None, None
        logits, tokens, stats = ctx.saved_tensors
        rows, vocab = logits.shape
        g, h = (None if t is None else t.to(torch.float32).contiguous() for t in (grad_logprobs, grad_entropy))
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
        with _on_device(logits.device):
            _lib.call("nvjsel_token_logprobs_grad", logits.data_ptr(), _dtype_code(logits, "logits"), rows, vocab,
                      _row_stride(logits), tokens.data_ptr(), tokens.element_size(), stats.data_ptr(),
                      _ptr(g), _ptr(h), out.data_ptr(), vocab, _stream_handle(logits.device))
        return out, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, num_top: int = 0,
                   entropy: bool = False) -> TokenLogprobs:
    """``log_softmax(logits)`` at the given tokens, one of every row.

    ``logits [..., V]`` (f32, bf16 or f16), ``tokens`` int32 or int64 of the shape
    before V.  With ``entropy`` also ``-sum p ln p`` of every row; with ``num_top``
    (at most 64) the likeliest tokens and their log probabilities, the best first,
    equal ones by token.  Sums are taken in 32 and 64 bits, results are f32.

    A token outside 0..V-1 (the -1 of padding) asks for nothing: its log probability is
    0 and gives no gradient.  Logits of ``-inf`` (masked) have no probability and are no
    alternatives: where fewer than ``num_top`` are left the rest is ``-inf`` with
    token -1; a row with nothing left has log probability ``-inf`` and entropy 0.  A NaN or
    ``+inf`` in a row makes its results NaN, its alternatives the first tokens.

    Differentiable in ``logits`` through ``logprobs`` and ``entropy`` (once; the
    alternatives carry no gradient).  A row whose own two gradients are 0, or one
    with nothing left, gets a gradient of zeros."""
    if logits.ndim < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError("token_logprobs takes logits [..., V] and one token for every row")
    if logits.numel() == 0:
        raise ValueError("token_logprobs requires non-empty dimensions")
    vocab = logits.shape[-1]
    rows = logits.numel() // vocab
    num_top = int(num_top)
    if not 0 <= num_top <= MAX_TOP:
        raise ValueError(f"num_top must be in 0..{MAX_TOP} (got {num_top})")
    if rows > MAX_ROWS or vocab > MAX_VOCAB:
        raise ValueError(f"at most {MAX_ROWS} rows and {MAX_VOCAB} tokens (got {rows} and {vocab})")
    _dtype_code(logits, "logits")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tokens must be int32 or int64 (got {tokens.dtype})")
    _require_cuda(logits, tokens)
    shape = tokens.shape
    if logits.ndim != 2:
        logits = logits.reshape(rows, vocab)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    tokens = tokens.reshape(rows).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        lp, ent, top, ids = _Differentiable.apply(logits, tokens, num_top, bool(entropy))
    else:
        lp, ent, top, ids, _ = _forward(logits, tokens, num_top, bool(entropy), False)
    if len(shape) != 1:
        lp, ent = lp.reshape(shape), None if ent is None else ent.reshape(shape)
        if top is not None:
            top, ids = top.reshape(*shape, num_top), ids.reshape(*shape, num_top)
    return TokenLogprobs(lp, ent, top, ids)
