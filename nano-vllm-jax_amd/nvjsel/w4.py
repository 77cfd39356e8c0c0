"""The LM head's weight in 4 bits with group scales.

``w[v, k] = scale[v, G] * (q[v, k] - zero[v, G])`` with ``G = k // group``, ``q``
in 0..15 and ``zero = 8`` where there are no zero points.  The plain form is
``qweight`` uint8 ``[V, H / 2]`` (even ``k`` in the low nibble), ``scales``
bf16 / f16 ``[V, H / group]`` and ``zeros`` uint8 ``[V, H / group]`` or None.
``pack_lm_head_w4`` lays it out for the kernels once, when a checkpoint is
loaded; the ``W4Weight`` it returns stands in for the weight tensor in
``lm_head_greedy_top1_hip``, ``lm_head_logits_hip``, ``lm_head_sample_token_ids``,
``lm_head_token_ids_and_topk``, ``mtp_greedy_top1_token_ids`` and
``lm_head_beam_search_step``.

The weight's values are not of a 16-bit type, so results round (``reduce_cast``
None) to the activations' type alone: bf16 activations give bf16 logits, f16
f16, f32 f32.  A hidden row holding a NaN or an infinity gets NaN for every
logit; bf16 and f32 values above 2^115 (4e34) in magnitude may take a group's sums out of
fp32 and make its logits NaN or infinite too.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from ._tensors import _TORCH_DTYPES, _dtype_code, _on_device, _require_cuda, _stream_handle, _workspace

GROUP_SIZES = (32, 64, 128)
_SCALE_DTYPES = (torch.bfloat16, torch.float16)
_CAST = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_OUT = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}


@dataclass(frozen=True)
class W4Weight:
    """A packed 4-bit weight: ``vocab`` rows of ``hidden`` values."""

    packed: torch.Tensor
    vocab: int
    hidden: int
    group_size: int
    scale_dtype: torch.dtype
    has_zeros: bool


def _check_group(hidden: int, group: int) -> None:
    if group not in GROUP_SIZES:
        raise ValueError(f"group size must be one of {GROUP_SIZES} (got {group})")
    if hidden % group:
        raise ValueError(f"hidden {hidden} is not a multiple of the group size {group}")


def quantize_lm_head_w4(weight: torch.Tensor, *, group_size: int = 128, symmetric: bool = True,
                        scale_dtype: torch.dtype | None = None, weight_layout: str | None = None):
    """Round an LM-head weight to 4 bits by groups of ``group_size`` along H.

    ``weight`` as the LM-head entry points take it: ``[H, V]`` (``E.T`` of the
    tied table in place) or, with ``weight_layout="vh"``, ``[V, H]``; f32, bf16 or
    f16, any strides.  ``symmetric``: ``scale = max|w| / 7`` and codes around 8, zeros
    None; else ``scale = (max - min) / 15`` over the values and 0, and zero points.
    Scales are of ``scale_dtype`` (the weight's own 16-bit type, bf16 for f32), and
    the codes are rounded against them as stored.  A group that holds a NaN or an
    infinity gets a NaN scale: its row's logits are NaN.  A scale beyond its type is the
    type's largest, and weights that its codes do not reach end at the last one.  Returns the plain form
    ``(qweight, scales, zeros)``."""
    if weight.ndim != 2:
        raise ValueError("the LM-head weight must be [H, V] (or [V, H] with weight_layout='vh')")
    if weight_layout not in (None, "hv", "vh"):
        raise ValueError(f"weight_layout must be None, 'hv' or 'vh' (got {weight_layout!r})")
    table = weight if weight_layout == "vh" else weight.T
    vocab, hidden = (int(d) for d in table.shape)
    if vocab == 0 or hidden == 0:
        raise ValueError("LM-head quantization requires non-empty dimensions")
    wd = _dtype_code(table, "weight")
    _check_group(hidden, group_size)
    sdt = (weight.dtype if weight.dtype in _SCALE_DTYPES else torch.bfloat16) if scale_dtype is None else scale_dtype
    if sdt not in _SCALE_DTYPES:
        raise ValueError(f"scale dtype must be bfloat16 or float16 (got {sdt})")
    dev = _require_cuda(table)
    if min(table.stride()) < 1:  # an expanded dimension
        table = table.contiguous()
    q = torch.empty((vocab, hidden // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((vocab, hidden // group_size), dtype=sdt, device=dev)
    zeros = None if symmetric else torch.empty((vocab, hidden // group_size), dtype=torch.uint8, device=dev)
    with _on_device(dev):
        _lib.call("nvjsel_w4_quantize", table.data_ptr(), wd, table.stride(0), table.stride(1), vocab, hidden,
                  group_size, _TORCH_DTYPES[sdt], q.data_ptr(), scales.data_ptr(),
                  None if zeros is None else zeros.data_ptr(), _stream_handle(dev))
    return q, scales, zeros


def pack_lm_head_w4(qweight: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None) -> W4Weight:
    """Lay the plain form out for the kernels (a copy; the plain form may go).

    The group size is ``H / scales.shape[1]``: 32, 64 or 128.  ``zeros`` hold 0..15:
    larger ones are refused, which waits for the device once (under graph capture, where
    nothing can be waited for, their low four bits count)."""
    if qweight.ndim != 2 or qweight.dtype != torch.uint8:
        raise ValueError("qweight must be uint8 [V, H / 2]")
    vocab, hidden = int(qweight.shape[0]), 2 * int(qweight.shape[1])
    if vocab == 0 or hidden == 0:
        raise ValueError("pack_lm_head_w4 requires non-empty dimensions")
    if scales.ndim != 2 or int(scales.shape[0]) != vocab or scales.shape[1] == 0 or hidden % int(scales.shape[1]):
        raise ValueError("scales must be [V, H / group]")
    if scales.dtype not in _SCALE_DTYPES:
        raise ValueError(f"scales must be bfloat16 or float16 (got {scales.dtype})")
    group = hidden // int(scales.shape[1])
    _check_group(hidden, group)
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError("zeros must be uint8 [V, H / group]")
    dev = _require_cuda(qweight, scales, zeros)
    qweight, scales = qweight.contiguous(), scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    lib = _lib.load()
    packed = torch.empty((lib.nvjsel_w4_packed_size(vocab, hidden, group, zeros is not None),), dtype=torch.uint8,
                         device=dev)
    with _on_device(dev):
        if zeros is not None and not torch.cuda.is_current_stream_capturing() and int(zeros.max()) > 15:
            raise ValueError("zeros must be 0..15")
        _lib.call("nvjsel_w4_pack", qweight.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
                  vocab, hidden, group, packed.data_ptr(), packed.numel(), _stream_handle(dev))
    return W4Weight(packed, vocab, hidden, group, scales.dtype, zeros is not None)


def _operands(x: torch.Tensor, weight: W4Weight, weight_layout, reduce_cast):
    """Checks and the arguments that the two products share."""
    if weight_layout is not None:
        raise ValueError("a 4-bit weight has its own layout: weight_layout must be None")
    if int(x.shape[0]) == 0:
        raise ValueError("LM-head products require non-empty dimensions")
    if int(x.shape[1]) != weight.hidden:
        raise ValueError("hidden dimension must match output weight rows")
    hd = _dtype_code(x, "hidden")
    rc = _CAST[x.dtype] if reduce_cast is None else int(reduce_cast)
    if rc not in _OUT:
        raise ValueError("reduce_cast must be 0, 1 or 2")
    dev = _require_cuda(x, weight.packed)
    x = x.contiguous()
    return x, rc, dev, (x.data_ptr(), hd, weight.packed.data_ptr(), weight.packed.numel(),
                        _TORCH_DTYPES[weight.scale_dtype], int(weight.has_zeros), weight.group_size, int(x.shape[0]),
                        weight.hidden, weight.vocab, rc)


def w4_logits(x: torch.Tensor, weight: W4Weight, weight_layout=None, reduce_cast=None) -> torch.Tensor:
    x, rc, dev, args = _operands(x, weight, weight_layout, reduce_cast)
    out = torch.empty((int(x.shape[0]), weight.vocab), dtype=_OUT[rc], device=dev)
    with _on_device(dev):
        _lib.call("nvjsel_lm_head_w4_logits", *args, out.data_ptr(), _TORCH_DTYPES[_OUT[rc]], weight.vocab,
                  _stream_handle(dev))
    return out


def w4_greedy(x: torch.Tensor, weight: W4Weight, weight_layout=None, reduce_cast=None, return_best=False):
    x, rc, dev, args = _operands(x, weight, weight_layout, reduce_cast)
    batch = int(x.shape[0])
    out = torch.empty((batch, 1), dtype=torch.int32, device=dev)
    best = torch.empty((batch,), dtype=torch.float32, device=dev) if return_best else None
    nbytes = _lib.load().nvjsel_lm_head_workspace_size(batch)
    with _on_device(dev):
        stream = _stream_handle(dev)
        ws = _workspace(dev, stream, "lm_head", nbytes, nbytes)
        _lib.call("nvjsel_lm_head_w4_top1", *args, out.data_ptr(), best.data_ptr() if return_best else None,
                  ws.data_ptr(), ws.numel(), stream)
    return (out, best) if return_best else out
