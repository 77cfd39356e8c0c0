"""Low-rank adapters of many requests at once beside a shared projection.

``out[n] = base[n] + scales[a] * (x[n] @ A[a].T) @ B[a].T`` with ``a = adapter_ids[n]``, and
``base[n]`` alone where that names no adapter.  ``pack_adapters`` lays the adapters out once,
when they are loaded; the ``AdapterTable`` it returns is also taken by
``lm_head_logits_hip``, ``lm_head_sample_token_ids``, ``lm_head_token_ids_and_topk`` and
``lm_head_token_logprobs``, where the projection is the LM head.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from ._tensors import _TORCH_DTYPES, _dtype_code, _on_device, _require_cuda, _stream_handle, _workspace

MAX_RANK = 512
MAX_ROWS = 1 << 20
_MIN_HIDDEN = 8
_TABLE_DTYPES = (torch.bfloat16, torch.float16)


@dataclass(frozen=True)
class AdapterTable:
    """Adapters laid out for the kernels."""

    a: torch.Tensor  # [count, rank * hidden], both rounded up
    b: torch.Tensor  # [count, width * rank], likewise
    scales: torch.Tensor  # f32 [count]
    hidden: int
    width: int
    rank: int  # rounded up to 16 or a multiple of 32

    @property
    def count(self) -> int:
        return int(self.a.shape[0])


def _no_tangent(who: str, *ts) -> None:
    """Refuses forward mode's dual tensors, whose tangents the launches would leave behind."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    if any(torch.is_tensor(t) and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ValueError(f"{who} has no forward-mode derivative: call it on tensors without a tangent")


def _no_gradient(who: str, *ts) -> None:
    _no_tangent(who, *ts)
    if not torch.is_grad_enabled():
        return
    if any(t is not None and t.requires_grad for t in ts):
        raise ValueError(f"{who} is not differentiable: call it under torch.no_grad() or on detached tensors")


def pack_adapters(a, b, scales=None) -> AdapterTable:
    """Lay out ``a`` (``[L, R, H]``, or one ``[R_i, H]`` per adapter) and ``b`` (``[L, D, R]``, or one
    ``[D, R_i]`` each) of bf16 or f16 for the kernels: a copy; the plain form may go.

    ``scales`` (f32 ``[L]`` or numbers; 1 where None) multiply the adapters' parts, ``alpha / R`` as
    a rule.  Ranks may differ, up to 512 (a table's ranks are laid out as its largest, rounded up to 16 or a
    multiple of 32).  Not differentiable: tensors that want a gradient, scales too, are refused."""
    if torch.is_tensor(a) and torch.is_tensor(b) and a.ndim == b.ndim == 3 and a.shape[0] == b.shape[0]:
        plain = [(a, b)]  # all of one rank: one launch each
    else:
        plain = [(s[None], t[None]) for s, t in zip(a, b)]
    a, b = list(a), list(b)
    if not a or len(a) != len(b):
        raise ValueError("pack_adapters takes one a and one b for every adapter, at least one")
    if any(t.ndim != 2 for t in a + b):
        raise ValueError("an adapter is a [R, H] and b [D, R]")
    hidden, width = int(a[0].shape[1]), int(b[0].shape[0])
    if hidden == 0 or width == 0 or any(t.shape[0] == 0 for t in a):
        raise ValueError("pack_adapters requires non-empty dimensions")
    if any(t.shape[1] != hidden for t in a) or any(t.shape[0] != width for t in b):
        raise ValueError("all adapters of a table have one hidden size and one width")
    if any(s.shape[0] != t.shape[1] for s, t in zip(a, b)):
        raise ValueError("a's and b's ranks must match")
    dtype = a[0].dtype
    if dtype not in _TABLE_DTYPES or any(t.dtype != dtype for t in a + b):
        raise ValueError("adapters must be bfloat16 or float16, a and b alike")
    given = scales if isinstance(scales, (list, tuple)) else [scales]
    _no_gradient("pack_adapters", *a, *b, *(t for t in given if torch.is_tensor(t)))
    most = max(int(t.shape[0]) for t in a)
    if most > MAX_RANK:
        raise ValueError(f"ranks must be at most {MAX_RANK} (got {most})")
    if hidden > 1 << 24 or width > 1 << 28:
        raise ValueError("hidden must be at most 2^24 and width 2^28")
    dev = _require_cuda(*a, *b)
    rank = 16 if most <= 16 else (most + 31) // 32 * 32
    pa = torch.empty((len(a), rank * ((hidden + 31) // 32 * 32)), dtype=dtype, device=dev)
    pb = torch.empty((len(a), rank * ((width + 63) // 64 * 64)), dtype=dtype, device=dev)
    if scales is None:
        ps = torch.ones((len(a),), dtype=torch.float32, device=dev)
    else:
        ps = torch.as_tensor(scales, dtype=torch.float32, device=dev).detach().reshape(-1).clone()
        if ps.numel() != len(a):
            raise ValueError("scales must have one value for every adapter")
    with _on_device(dev):
        at = 0
        for s, t in plain:
            n, own = int(s.shape[0]), int(s.shape[1])
            for which, (p, to) in enumerate(((s, pa[at:]), (t, pb[at:]))):
                if p.stride(2) != 1 and p.shape[2] > 1:
                    p = p.contiguous()
                _lib.call("nvjsel_adapters_pack", p.data_ptr(), which, p.stride(0) if n > 1 else 0,
                          p.stride(1) if p.shape[1] > 1 else 0, n, own, hidden, width, rank, to.data_ptr(),
                          to.numel() * to.element_size(), _stream_handle(dev))
            at += n
    return AdapterTable(pa, pb, ps, hidden, width, rank)


@lru_cache(maxsize=1024)
def _bytes(*shape: int) -> int:
    return _lib.load().nvjsel_adapters_workspace_size(*shape)


def _rows(t: torch.Tensor, rows: int) -> torch.Tensor:
    """``[rows, D]`` with unit column stride, a copy where a view cannot be."""
    t = t if t.ndim == 2 else t.reshape(rows, t.shape[-1])
    return t.contiguous() if t.stride(1) != 1 and t.shape[1] > 1 else t


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _meet(s: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether two [rows, D] tensors may share memory."""
    size = s.element_size()
    first, other = sorted((s, t), key=lambda u: u.data_ptr())
    apart = other.data_ptr() - first.data_ptr()
    pitch, width = _stride(first) * size, first.shape[1] * size
    if apart >= (first.shape[0] - 1) * pitch + width:
        return False
    side_by_side = pitch == _stride(other) * size and pitch > 0
    return not (side_by_side and width <= apart % pitch <= pitch - width)


def apply_adapters(x: torch.Tensor, base: torch.Tensor, adapters: AdapterTable, adapter_ids: torch.Tensor, *,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """``base`` with every row's own adapter added: ``base + scale (x A^T) B^T``.

    ``x [..., H]`` are the projection's inputs and ``base [..., D]`` its outputs (f32, bf16 or
    f16 each, rows with unit stride as they lie), ``adapter_ids`` int32 of the shape before H, one
    outside 0..L-1 (the -1 of a row without an adapter) leaves its row as it is.  Any order and
    mixture of adapters.  Sums are fp32; the result, of ``base``'s type, is rounded once.
    ``out`` receives it (``base`` itself for in place), a new tensor where None.  A NaN or an infinity
    in a row of ``x``, or in its own adapter's A or scale, makes that row's results NaN; one in row ``v`` of B leaves
    column ``v`` of that adapter's rows NaN or infinite; neither reaches other values.
    Not differentiable."""
    rows_shape, hidden, width = adapter_ids.shape, adapters.hidden, adapters.width
    if x.ndim < 1 or base.ndim < 1 or x.shape[:-1] != rows_shape or base.shape[:-1] != rows_shape:
        raise ValueError("apply_adapters takes x [..., H], base [..., D] and one adapter id for every row")
    rows = adapter_ids.numel()
    if rows == 0:
        raise ValueError("apply_adapters requires non-empty dimensions")
    if x.shape[-1] != hidden or base.shape[-1] != width:
        raise ValueError(f"the adapters are of hidden {hidden} and width {width} (got {x.shape[-1]} and {base.shape[-1]})")
    xd, od = _dtype_code(x, "x"), _dtype_code(base, "base")
    if adapter_ids.dtype != torch.int32:
        raise ValueError(f"adapter_ids must be int32 (got {adapter_ids.dtype})")
    if rows > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows (got {rows})")
    _no_gradient("apply_adapters", x, base, out)
    a = adapters.a
    dev = _require_cuda(x, base, a, adapter_ids)
    if out is None:
        result = flat = torch.empty_like(base, memory_format=torch.contiguous_format)
    else:
        if out.shape != base.shape or out.dtype != base.dtype or out.device != dev:
            raise ValueError("out must have base's shape, type and device")
        result, flat = out, out
    if x.ndim != 2:
        try:
            flat = result.view(rows, width)
        except RuntimeError:
            raise ValueError("out's rows must be apart by one stride") from None
    if out is not None and ((flat.stride(1) != 1 and width > 1) or _stride(flat) < width):
        raise ValueError("out's rows must be contiguous and must not overlap")
    x, base = _rows(x, rows), _rows(base, rows)
    ids = adapter_ids if adapter_ids.ndim == 1 and adapter_ids.is_contiguous() else adapter_ids.reshape(rows).contiguous()
    if out is not None and (base.data_ptr(), _stride(base)) != (flat.data_ptr(), _stride(flat)) and _meet(base, flat):
        raise ValueError("out must be base itself or share no memory with it")
    if hidden < _MIN_HIDDEN:  # zeros beside the table's zeros
        x = torch.nn.functional.pad(x, (0, _MIN_HIDDEN - hidden))
        hidden = _MIN_HIDDEN
    with _on_device(dev):
        td = _TORCH_DTYPES[a.dtype]
        nbytes = _bytes(td, rows, adapters.rank)
        stream = _stream_handle(dev)
        ws = _workspace(dev, stream, "adapters", nbytes, 0)
        _lib.call("nvjsel_apply_adapters", x.data_ptr(), xd, _stride(x), base.data_ptr(), od, _stride(base), a.data_ptr(),
                  adapters.b.data_ptr(), td, adapters.scales.data_ptr(), a.shape[0], adapters.rank, hidden, width,
                  ids.data_ptr(), rows, flat.data_ptr(), _stride(flat), ws.data_ptr(), nbytes, stream)
    if out is not None:
        increment_version(out)  # a backward pass that saved it is to notice
    return result
