"""Device plumbing for the host layer: dtype codes, pointers, streams and the scratch workspace.

torch is used for device memory and streams only; every computation happens inside
libhidet_b200q.so.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Tuple

import torch

from . import ffi, native

FLOAT_CODES = {torch.float16: ffi.F16, torch.bfloat16: ffi.BF16, torch.float32: ffi.F32}
QUANT_CODES = {torch.int8: ffi.I8, torch.int16: ffi.I16}
QUANT_NAMES = {'int8': torch.int8, 'i8': torch.int8, 'int16': torch.int16, 'i16': torch.int16}


def require_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError('{} must be a torch.Tensor, got {}'.format(name, type(t).__name__))
    if not t.is_cuda:
        raise ffi.BackendException(
            '{} lives on {}: hidet_b200 runs on CUDA devices only and has no CPU implementation'.format(name, t.device)
        )


def current_stream_ptr(device: torch.device) -> int:
    """The stream kernels are launched on: torch's current stream, as in the reference, whose runtime
    asks torch for it through a callback (src/hidet/runtime/cuda/context.cpp:78-88)."""
    return torch.cuda.current_stream(device).cuda_stream


class _Workspaces:
    """Grow-only, zero-initialised scratch per (device, stream), the role request_cuda_workspace
    plays in the reference (src/hidet/runtime/cuda/context.cpp:31-49,90-104).  The library keeps the
    part that must be zero (its tile counters) zero between calls, so a buffer is cleared only when it
    is created.

    A buffer that is made while a graph is captured is cleared by a node of that graph, so it is nobody else's: not
    another graph's, which may be replayed first, nor that of calls outside.  One that is replaced by a larger one is kept,
    since a graph may have been captured with it; sizes double, so that all of them are no more than the last."""

    def __init__(self):
        self._buffers: Dict[Tuple[int, int], torch.Tensor] = {}
        self._replaced: List[torch.Tensor] = []

    def get(self, device: torch.device, nbytes: int) -> Tuple[int, int]:
        if nbytes == 0:
            return 0, 0
        index = device.index if device.index is not None else torch.cuda.current_device()
        key = (index, current_stream_ptr(device))
        buf, capture = self._buffers.get(key), self._capture(key[1])
        made_by = self._made_by(buf)
        if buf is None or buf.numel() < nbytes or made_by not in (0, capture):
            size = 1 << max(20, (nbytes - 1).bit_length())
            if buf is not None and made_by == 0:
                self._replaced.append(buf)
            if capture:
                buf = self._allocate(torch.empty, index, size)
                buf[:ffi.WORKSPACE_HEAD].zero_()  # with every replay
                buf.made_by = capture
            else:
                buf = self._allocate(torch.zeros, index, size)
            self._buffers[key] = buf
        self._tell(key)  # the native host path, which may be younger than the buffer
        return buf.data_ptr(), buf.numel()

    @staticmethod
    def _capture(stream: int) -> int:
        """The capture that the current stream is in, or 0."""
        return ffi.func('b200q_capture_id')(stream) if torch.cuda.is_current_stream_capturing() else 0

    @staticmethod
    def _allocate(how, index: int, size: int) -> torch.Tensor:
        return how(size, dtype=torch.uint8, device=torch.device('cuda', index))

    @staticmethod
    def _made_by(buffer: Optional[torch.Tensor]) -> int:
        """The capture that made a buffer, or 0.  It stands with the buffer, which may leave its place and come back (swap)."""
        return getattr(buffer, 'made_by', 0)

    def _tell(self, key: Tuple[int, int]) -> None:
        buf = self._buffers.get(key)
        if buf is None or self._made_by(buf):
            native.set_scratch(*key, 0, 0)  # the native host path does not know of captures
        else:
            native.set_scratch(*key, buf.data_ptr(), buf.numel())

    def clear(self) -> None:
        self._buffers.clear()
        self._replaced.clear()
        native.clear_scratch()

    def swap(self, device: torch.device, stream: int, buffer: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        """Puts `buffer` (None: nothing, a new one is made when it is needed) in the place of a stream's scratch and
        returns what was there.  A captured graph takes the buffer its launches were recorded with into its own keeping
        this way: streams come from a small pool, so a later graph or eager call may run on the same one, and must neither
        share the buffer nor replace it by a larger one while the graph still writes to it."""
        index = device.index if device.index is not None else torch.cuda.current_device()
        before = self._buffers.pop((index, stream), None)
        if buffer is not None:
            self._buffers[(index, stream)] = buffer
        self._tell((index, stream))
        return before


workspaces = _Workspaces()
