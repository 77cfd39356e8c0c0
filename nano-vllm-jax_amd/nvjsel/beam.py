"""Beam search: selection over beams and vocabulary, reordering of the beams'
states, and the decode step that joins them with the LM head."""
from __future__ import annotations

import math
from functools import lru_cache

import torch

from . import _lib
from ._tensors import _dtype_code, _on_device, _require_cuda, _stream_handle, _workspace
from .selection import lm_head_logits_hip, rms_norm_hip

MAX_BEAMS = 64  # beams and candidates of a request
MAX_REQUESTS, MAX_VOCAB = 65536, 1 << 26  # of a selection
_MAX_STATES = 4096  # descriptions of one call


@lru_cache(maxsize=1024)
def _select_bytes(device: int, *shape: int) -> int:  # by device: its compute units count
    return _lib.load().nvjsel_beam_select_workspace_size(*shape)


def beam_search_select(logits: torch.Tensor, scores: torch.Tensor, *, num_candidates: int | None = None,
                       finished: torch.Tensor | None = None, end_token: int | None = None):
    """The best continuations of every request's beams.

    ``logits [B, W, V]`` (f32, bf16 or f16; any strides with unit token stride),
    ``scores`` f32 ``[B, W]`` the beams' cumulative log-probabilities.  The
    candidates of request ``b`` are ``scores[b, w] + log_softmax(logits[b, w])[v]``;
    the ``num_candidates`` (default W, at most 64) best ones come back as
    ``(scores f32[B, K], parents int32[B, K], tokens int32[B, K])``, the best first, equal
    ones by beam; within a beam the larger logit first, equal ones by token.

    A beam whose score is ``-inf`` is not live (the first step has one live beam): it
    has no candidates and its logits are not looked at.  A beam with ``finished`` set (bool
    or uint8 ``[B, W]``) stays as it is: one candidate, ``end_token`` at its own score.
    Tokens masked with ``-inf`` are no candidates; where fewer than K are left the
    rest is ``-inf`` with parent and token -1.  A NaN or ``+inf`` among a live beam's
    logits, or as its score, makes its candidates NaN, which come first."""
    if logits.ndim != 3:
        raise ValueError("beam search takes logits [B, W, V]")
    batch, beams, vocab = logits.shape
    if batch == 0 or beams == 0 or vocab == 0:
        raise ValueError("beam search requires non-empty dimensions")
    k = beams if num_candidates is None else int(num_candidates)
    if beams > MAX_BEAMS or not 1 <= k <= MAX_BEAMS:
        raise ValueError(f"beams and num_candidates must be in 1..{MAX_BEAMS} (got {beams} and {k})")
    if batch > MAX_REQUESTS or vocab > MAX_VOCAB:
        raise ValueError(f"at most {MAX_REQUESTS} requests and {MAX_VOCAB} tokens (got {batch} and {vocab})")
    dt = _dtype_code(logits, "logits")
    if scores.shape != (batch, beams) or scores.dtype != torch.float32:
        raise ValueError("scores must be float32 [B, W]")
    if finished is not None:
        if finished.shape != (batch, beams) or finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError("finished must be bool or uint8 [B, W]")
        if end_token is None or not 0 <= end_token < vocab:
            raise ValueError("finished beams need an end_token of the vocabulary")
        finished = finished.contiguous()
    dev = _require_cuda(logits, scores, finished)
    if logits.stride(2) != 1 and vocab > 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    out, parents, tokens = scores.new_empty((3, batch, k), dtype=torch.int32).unbind(0)
    out_scores = out.view(torch.float32)
    with _on_device(dev):
        nbytes = _select_bytes(dev.index, dt, batch, beams, vocab, k)
        stream = _stream_handle(dev)
        ws = _workspace(dev, stream, "beam", nbytes, 4 * batch)  # at rest: the requests' tickets
        _lib.call("nvjsel_beam_select", logits.data_ptr(), dt, batch, beams, vocab, logits.stride(0), logits.stride(1),
                  scores.data_ptr(), None if finished is None else finished.data_ptr(), end_token or 0, k,
                  out_scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(), ws.data_ptr(), nbytes,
                  stream)
    return out_scores, parents, tokens


def _describe_state(t: torch.Tensor, rows: int | None, length_dim: int | None) -> tuple:
    """A nvjsel_state without its pointer."""
    shape = t.shape
    if t.ndim == 0 or (rows is not None and shape[0] < rows):
        raise ValueError("a state needs one row per beam along its first dimension")
    n = t.numel()
    if n == 0:
        raise ValueError("states must not be empty")
    row = n // shape[0]
    if not t.is_contiguous() and (not t[0].is_contiguous() or (shape[0] > 1 and t.stride(0) < row)):
        raise ValueError("a state's rows must be contiguous and must not overlap")
    size = t.element_size()
    outer, length = 1, 1
    if length_dim is not None:
        at = length_dim + t.ndim if length_dim < 0 else length_dim
        if not 1 <= at < t.ndim:
            raise ValueError(f"length_dim {length_dim} is not a dimension of a row of {tuple(shape)}")
        outer, length = math.prod(shape[1:at]), shape[at]
    if max(shape[0], outer) >= 1 << 31:
        raise ValueError("a state has less than 2^31 rows, and positions before length_dim")
    return (t.stride(0) if shape[0] > 1 else row) * size, length, row // (outer * length) * size, outer, shape[0]


def reorder_beam_states(states, parents: torch.Tensor, *, slots: torch.Tensor | None = None,
                        lengths: torch.Tensor | None = None, length_dim: int | None = None) -> None:
    """Give every beam its parent's state, in place, in one launch per 24 tensors.

    ``states``: a tensor or a sequence of tensors (caches, recurrent states, token
    histories; any types), one row per beam along the first dimension, each row
    contiguous, no two of them sharing memory.  Row ``b * W + w``, or ``slots[b, w]`` (int32 ``[B, W]``, distinct) of a
    state table, receives what the row of beam ``parents[b, w]`` held.  With ``lengths``
    (int32 ``[B]``) only the first ``lengths[b]`` positions along ``length_dim`` move and
    the rest stays as it is.  ``parents`` is int32 ``[B, W]``, e.g. the first W columns of
    ``beam_search_select``'s.  A beam whose parent is itself or not in 0..W-1 (the -1
    of a missing candidate), or whose own or parent's slot is not in the table, stays as
    it is."""
    if torch.is_tensor(states):
        states = (states,)
    if parents.ndim != 2 or parents.dtype != torch.int32 or parents.numel() == 0:
        raise ValueError("parents must be a non-empty int32 [B, W]")
    batch, beams = parents.shape
    if beams > MAX_BEAMS or batch > 65535:
        raise ValueError(f"at most {MAX_BEAMS} beams and 65535 requests (got {beams} and {batch})")
    if parents.stride(1) != 1 and beams > 1:
        parents = parents.contiguous()
    if slots is not None:
        if slots.shape != parents.shape or slots.dtype != torch.int32:
            raise ValueError("slots must be int32 [B, W]")
        slots = slots.contiguous()
    if (lengths is None) != (length_dim is None):
        raise ValueError("lengths and length_dim go together")
    if lengths is not None:
        if lengths.shape != (batch,) or lengths.dtype != torch.int32:
            raise ValueError("lengths must be int32 [B]")
        lengths = lengths.contiguous()
    count = len(states)
    if not 1 <= count <= _MAX_STATES:
        raise ValueError(f"reorder_beam_states takes 1..{_MAX_STATES} states")
    dev = _require_cuda(parents, slots, lengths, *states)
    table, last = [], None
    for t in states:
        form = (t.shape, t.stride(), t.dtype)
        if form != last:  # the layers of a cache are alike
            described, last = _describe_state(t, None if slots is not None else batch * beams, length_dim), form
        table.append(t.data_ptr())
        table += described
    if len(set(table[::6])) != count:
        raise ValueError("a state is given twice")
    with _on_device(dev):
        _lib.call("nvjsel_reorder_states", _lib.states(table), count, parents.data_ptr(), parents.stride(0),
                  None if slots is None else slots.data_ptr(), None if lengths is None else lengths.data_ptr(), batch,
                  beams, _stream_handle(dev))


def lm_head_beam_search_step(hidden: torch.Tensor, output_weight, scores: torch.Tensor, *,
                             finished: torch.Tensor | None = None, end_token: int | None = None, states=None,
                             slots: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                             length_dim: int | None = None, norm_weight: torch.Tensor | None = None,
                             rms_norm_eps: float = 1e-6, act_dtype: torch.dtype = torch.float32,
                             weight_layout: str | None = None, reduce_cast: int | None = None):
    """One decode step of beam search from the hidden states ``[B, W, H]``.

    The LM head's logits (``output_weight`` as in ``lm_head_logits_hip``, a ``W4Weight``
    among them; ``norm_weight``: pre-norm hidden), the W best continuations of every
    request (``beam_search_select``), and, with ``states``, their beams' states moved
    to the new order (``reorder_beam_states``).  Returns
    ``(scores f32[B, W], parents int32[B, W], tokens int32[B, W])``."""
    if hidden.ndim != 3:
        raise ValueError("hidden must be [B, W, H]")
    batch, beams, hidden_dim = hidden.shape
    flat = hidden.reshape(batch * beams, hidden_dim)
    with _on_device(_require_cuda(flat)):
        if norm_weight is not None:
            flat = rms_norm_hip(flat, norm_weight, rms_norm_eps, act_dtype)
        logits = lm_head_logits_hip(flat, output_weight, weight_layout=weight_layout, reduce_cast=reduce_cast)
    new_scores, parents, tokens = beam_search_select(logits.reshape(batch, beams, -1), scores, finished=finished,
                                                     end_token=end_token)
    if states is not None:
        reorder_beam_states(states, parents, slots=slots, lengths=lengths, length_dim=length_dim)
    return new_scores, parents, tokens
