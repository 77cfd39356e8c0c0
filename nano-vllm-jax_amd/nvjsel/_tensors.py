"""What the entry points share: dtype codes, device checks, the stream and the
zero-filled workspaces."""
from __future__ import annotations

import threading
from contextlib import nullcontext

import torch

from . import _lib

_TORCH_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _dtype_code(t: torch.Tensor, what: str) -> int:
    try:
        return _TORCH_DTYPES[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported {what} dtype: {t.dtype}") from None


def _require_cuda(*ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    if dev.type != "cuda":
        raise ValueError("nvjsel kernels take device tensors (got a CPU tensor)")
    for t in ts:
        if t is not None and t.device != dev:
            if t.device.type != "cuda":
                raise ValueError("nvjsel kernels take device tensors (got a CPU tensor)")
            raise ValueError("all tensors must live on one device")
    return dev


# The current stream's handle without a torch.cuda.Stream object around it: 0.1 us
# a call against 1.9.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_handle(device: torch.device) -> int:
    if _raw_stream is None or device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return _raw_stream(device.index)


class _WorkspacePool:
    """Zero-filled scratch buffers per (device, stream, kind).

    Each entry point leaves its workspace zero-filled when it returns, so a
    buffer is zeroed once at allocation and reused in stream order.  A captured call may hold
    a buffer for as long as its graph lives, so a larger one does not replace it but comes
    beside it, at twice its size; those that no captured call takes go."""

    UNCAPTURED = ("beam", "logprobs", "score", "adapters")

    def __init__(self):
        self._bufs: dict = {}
        self._held: list = []
        self._lock = threading.Lock()

    def get(self, device: torch.device, stream: int, kind: str, nbytes: int) -> torch.Tensor:
        key = (device.index, stream, kind)
        buf = self._bufs.get(key)
        if buf is not None and buf.numel() >= nbytes:
            return buf
        with self._lock:
            buf = self._bufs.get(key)
            if buf is None or buf.numel() < nbytes:
                size = max(nbytes, 4096)
                if buf is not None and kind not in self.UNCAPTURED:
                    self._held.append(buf)
                    size = max(size, 2 * buf.numel())
                buf = torch.zeros(size, dtype=torch.uint8, device=device)
                self._bufs[key] = buf
            return buf


_WS = _WorkspacePool()


def _workspace(device: torch.device, stream: int, kind: str, nbytes: int, at_rest: int) -> torch.Tensor:
    """The stream's workspace, or, under capture, one of the graph's own: graphs captured on
    one stream may be replayed at the same time.  Every replay zeroes its first ``at_rest``
    bytes again.  For a call with ``device`` the current one."""
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        ws[:at_rest].zero_()
        return ws
    return _WS.get(device, stream, kind, nbytes)


_HERE = nullcontext()
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _on_device(device: torch.device):
    """Makes ``device`` the current one for a launch, where it is not already."""
    return _HERE if _current_device() == device.index else torch.cuda.device(device)
