"""Device plumbing for the host layer: dtype codes, pointers, streams and the scratch workspace.

torch is used for device memory and streams only; every computation happens inside
libhidet_b200q.so.
"""
from __future__ import annotations

from typing import Dict, Optional, Set, Tuple

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

    A graph has scratch of its own: what its capture makes is cleared by a node of the graph and is nobody else's, neither another graph's, which
    may be replayed first or at the same time, nor that of calls outside, which have theirs again when the capture is over.  So no graph holds what calls
    outside outgrow.  CudaGraph instead captures with the buffer that its own warm-up made and takes that away (swap, exclusive)."""

    def __init__(self):
        # A buffer that a capture made stands in front of the one of calls outside, which it keeps as `outside`.
        self._buffers: Dict[Tuple[int, int], torch.Tensor] = {}
        self._exclusive: Set[Tuple[int, int]] = set()

    def get(self, device: torch.device, nbytes: int) -> Tuple[int, int]:
        if nbytes == 0:
            return 0, 0
        index = device.index if device.index is not None else torch.cuda.current_device()
        key = (index, current_stream_ptr(device))
        last, capture = self._buffers.get(key), self._capture(key[1])
        outside = self.outside(last)
        if capture and self._made_by(last) == capture:
            buf = last
        else:
            buf = outside if not capture or key in self._exclusive else None
        if buf is None or buf.numel() < nbytes:
            size = 1 << max(20, (nbytes - 1).bit_length())
            if capture:
                buf = self._allocate(torch.empty, index, size)
                buf[:ffi.WORKSPACE_HEAD].zero_()  # with every replay
                buf.made_by, buf.outside = capture, outside
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

    def outside(self, buffer: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        """What calls outside captures have of a stream's scratch: the buffer, or the one behind it."""
        return buffer.outside if self._made_by(buffer) else buffer

    def _tell(self, key: Tuple[int, int]) -> None:
        """The native host path takes what calls outside have; it leaves a capture's calls to this one."""
        buf = self.outside(self._buffers.get(key))
        native.set_scratch(*key, *((buf.data_ptr(), buf.numel()) if buf is not None else (0, 0)))

    def clear(self) -> None:
        self._buffers.clear()
        native.clear_scratch()

    def swap(self, device: torch.device, stream: int, buffer: Optional[torch.Tensor], exclusive: bool = False) -> Optional[torch.Tensor]:
        """Puts `buffer` (None: nothing, a new one is made when it is needed) in the place of a stream's scratch and
        returns what was there.  A captured graph takes the buffer its launches were recorded with into its own keeping
        this way: streams come from a small pool, so a later graph or eager call may run on the same one, and must neither
        share the buffer nor replace it by a larger one while the graph still writes to it.  exclusive: until the next swap a capture
        may use what calls outside made, since its owner takes it away."""
        index = device.index if device.index is not None else torch.cuda.current_device()
        key = (index, stream)
        before = self._buffers.pop(key, None)
        (self._exclusive.add if exclusive else self._exclusive.discard)(key)
        if buffer is not None:
            self._buffers[key] = buffer
        self._tell(key)
        return before


workspaces = _Workspaces()
