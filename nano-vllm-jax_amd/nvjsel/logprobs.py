"""Log probabilities of given tokens, with entropies and top alternatives: over
logits, with their gradient, and from the hidden states."""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from . import _lib
from .adapters import MAX_ROWS as _ADAPTER_ROWS, AdapterTable, _no_gradient, _no_tangent
from .selection import _adapter_ids, _normed, _weight_operand, lm_head_logits_hip, reference_reduce_cast
from .w4 import W4Weight
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
    logprobs = torch.empty_like(tokens, dtype=torch.float32)
    ent = torch.empty_like(logprobs) if entropy else None
    kept = logprobs.new_empty((rows, 3)) if stats else None
    top = ids = None
    if num_top:
        top = logprobs.new_empty((rows, num_top))
        ids = torch.empty_like(top, dtype=torch.int32)
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
    def backward(ctx, grad_logprobs, grad_entropy, *_):
        if grad_logprobs is None and grad_entropy is None:
            return None, None, None, None
        g = None if grad_logprobs is None else grad_logprobs.contiguous()  # f32, as their outputs
        h = None if grad_entropy is None else grad_entropy.contiguous()
        # with create_graph the gradient stands in the graph, between the logits and a refusal
        gradient = _Once.apply if torch.is_grad_enabled() else _gradient
        return gradient(*ctx.saved_tensors, g, h), None, None, None


def _gradient(logits, tokens, stats, g, h):
    rows, vocab = logits.shape
    out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    with _on_device(logits.device):
        _lib.call("nvjsel_token_logprobs_grad", logits.data_ptr(), _dtype_code(logits, "logits"), rows, vocab,
                  _row_stride(logits), tokens.data_ptr(), tokens.element_size(), stats.data_ptr(),
                  _ptr(g), _ptr(h), out.data_ptr(), vocab, _stream_handle(logits.device))
    return out


class _Once(torch.autograd.Function):
    """The gradient, whose own derivative is refused, not left out."""

    @staticmethod
    def forward(ctx, *operands):
        return _gradient(*operands)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("token_logprobs is differentiable once: a second derivative was asked for")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, num_top: int = 0,
                   entropy: bool = False) -> TokenLogprobs:
    """``log_softmax(logits)`` at the given tokens, one of every row.

    ``logits [..., V]`` (f32, bf16 or f16), ``tokens`` int32 or int64 of the shape
    before V.  With ``entropy`` also ``-sum p ln p`` of every row; with ``num_top``
    (at most 64) the likeliest tokens and their log probabilities, the best first,
    equal ones by token.  Sums are taken in 32 and 64 bits, results are f32, no
    log probability above 0.

    A token outside 0..V-1 (the -1 of padding) asks for nothing: its log probability is
    0 and gives no gradient.  Logits of ``-inf`` (masked) have no probability and are no
    alternatives: where fewer than ``num_top`` are left the rest is ``-inf`` with
    token -1; a row with nothing left has log probability ``-inf`` and entropy 0.  A NaN or
    ``+inf`` in a row makes its results NaN, its alternatives the first tokens.

    Differentiable in ``logits`` through ``logprobs`` and ``entropy`` (backward, once: forward mode and a second
    derivative raise; the alternatives carry no gradient).  A row whose own two gradients are 0, or one
    with nothing left, gets a gradient of zeros.  In a captured graph take the gradient of a
    leaf made within the capture (``logits.detach().requires_grad_()``, ``torch.autograd.grad``)."""
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
    _no_tangent("token_logprobs", logits)
    _require_cuda(logits, tokens)
    shape = tokens.shape
    if logits.ndim != 2:
        logits = logits.reshape(rows, vocab)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    if tokens.ndim != 1 or not tokens.is_contiguous():
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


_LOGIT_BYTES = 1 << 28  # of logits that are formed at a time


def lm_head_token_logprobs(hidden: torch.Tensor, output_weight, tokens: torch.Tensor, *, num_top: int = 0,
                           entropy: bool = False, weight_layout: str | None = None, reduce_cast: int | None = None,
                           norm_weight: torch.Tensor | None = None, rms_norm_eps: float = 1e-6,
                           act_dtype: torch.dtype = torch.float32, adapters: AdapterTable | None = None,
                           adapter_ids: torch.Tensor | None = None) -> TokenLogprobs:
    """``token_logprobs`` of the LM head's logits, from the hidden states: the score of a prompt or a draft.

    ``hidden [..., H]``, ``tokens`` int32 or int64 of the shape before H; ``output_weight``,
    ``weight_layout``, ``reduce_cast``, ``adapters`` and ``adapter_ids`` (one for every row) as in ``lm_head_logits_hip``, whose logits'
    log probabilities these are; ``norm_weight``: pre-norm hidden, as in ``lm_head_greedy_top1_hip``.
    Logits are not written for a 16-bit weight ``[V, H]`` (the tied table) with H a multiple of 64 and
    hidden of its type, or f32 beside bf16, without alternatives or adapters; other calls form them for some
    rows at a time.  Not differentiable."""
    if hidden.ndim < 1 or tokens.shape != hidden.shape[:-1]:
        raise ValueError("lm_head_token_logprobs takes hidden [..., H] and one token for every row")
    if hidden.numel() == 0:
        raise ValueError("LM-head log probabilities require non-empty dimensions")
    num_top = int(num_top)
    if not 0 <= num_top <= MAX_TOP:
        raise ValueError(f"num_top must be in 0..{MAX_TOP} (got {num_top})")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tokens must be int32 or int64 (got {tokens.dtype})")
    if tokens.numel() > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows (got {tokens.numel()})")
    weight = output_weight.packed if isinstance(output_weight, W4Weight) else output_weight
    _no_gradient("lm_head_token_logprobs", hidden, weight, norm_weight)
    shape, rows = tokens.shape, tokens.numel()
    x = hidden.reshape(rows, hidden.shape[-1])
    tokens = tokens.reshape(rows).contiguous()
    dev = _require_cuda(x, tokens)
    if adapters is not None:
        adapter_ids = _adapter_ids(adapter_ids, x)
    with _on_device(dev):
        if norm_weight is not None:
            x = _normed(x, norm_weight, rms_norm_eps, act_dtype)
        r = None
        if adapters is None and num_top == 0 and not isinstance(output_weight, W4Weight):
            r = _scored(x, output_weight, tokens, entropy, weight_layout, reduce_cast)
        if r is None:
            r = _scored_by_logits(x, output_weight, tokens, num_top, entropy, weight_layout, reduce_cast, adapters,
                                  adapter_ids)
    return TokenLogprobs(*(t if t is None else t.reshape((*shape, *t.shape[1:])) for t in r))


def _scored(x, output_weight, tokens, entropy, weight_layout, reduce_cast):
    """Without logits; None for a call that the kernel does not take."""
    w, layout, vocab = _weight_operand(output_weight, weight_layout, int(x.shape[1]))
    hd, wd = _dtype_code(x, "hidden"), _dtype_code(w, "weight")
    dev = _require_cuda(x, w)
    x = x.contiguous()
    if vocab == 0 or (x.data_ptr() | w.data_ptr()) & 15:
        return None
    nbytes = _score_bytes(dev.index, hd, wd, layout, int(x.shape[0]), int(x.shape[1]), vocab)
    if nbytes == 0:
        return None
    own = reference_reduce_cast(x.dtype, w.dtype)
    rc = own if reduce_cast is None else int(reduce_cast)
    if rc not in (0, own):
        return None
    logprobs = torch.empty_like(tokens, dtype=torch.float32)
    ent = torch.empty_like(logprobs) if entropy else None
    stream = _stream_handle(dev)
    ws = _workspace(dev, stream, "score", nbytes, 0)
    _lib.call("nvjsel_lm_head_token_logprobs", x.data_ptr(), hd, w.data_ptr(), wd, layout, x.shape[0], x.shape[1], vocab, rc,
              tokens.data_ptr(), tokens.element_size(), logprobs.data_ptr(), _ptr(ent), ws.data_ptr(), nbytes, stream)
    return logprobs, ent, None, None


@lru_cache(maxsize=1024)
def _score_bytes(device: int, *shape: int) -> int:
    return _lib.load().nvjsel_lm_head_token_logprobs_workspace_size(*shape)


def _scored_by_logits(x, output_weight, tokens, num_top, entropy, weight_layout, reduce_cast, adapters, adapter_ids):
    vocab = output_weight.vocab if isinstance(output_weight, W4Weight) else max(output_weight.shape)
    step = min(max(64, _LOGIT_BYTES // (4 * vocab) // 64 * 64), _ADAPTER_ROWS)
    parts = []
    for i in range(0, x.shape[0], step):
        ids = None if adapters is None else adapter_ids[i:i + step]
        logits = lm_head_logits_hip(x[i:i + step], output_weight, weight_layout=weight_layout, reduce_cast=reduce_cast,
                                    adapters=adapters, adapter_ids=ids)
        parts.append(token_logprobs(logits, tokens[i:i + step], num_top=num_top, entropy=entropy))
    return [None if p[0] is None else p[0] if len(parts) == 1 else torch.cat(p) for p in zip(*parts)]
