"""Addresses that the ctypes calls take, of tensors and of streams, and where a call's results are allocated."""
from __future__ import annotations

import functools

try:
    import torch
except ImportError:  # pragma: no cover - the host API needs torch for device memory
    torch = None


def address(t):
    """A tensor's data pointer (None: NULL)."""
    return None if t is None else t.data_ptr()


def stream_address(stream, device: int) -> int:
    """A cudaStream_t: of a torch stream, of an address, or (None) of the device's current stream."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device)  # torch.cuda.current_stream().cuda_stream takes 3 us
    return stream if isinstance(stream, int) else stream.cuda_stream


def stream_scope(stream, device: int):
    """Makes `stream` (as above; None: no change) current.  Memory allocated on another stream may still be written or
    read by what is pending there, which the call's own stream does not wait for."""
    if stream is not None and not isinstance(stream, torch.cuda.Stream):
        at = stream_address(stream, device)  # 0 and 1: the legacy default stream
        stream = torch.cuda.ExternalStream(at, device=device) if at > 1 else torch.cuda.default_stream(device)
    return torch.cuda.stream(stream)


def on_its_stream(method):
    """A method whose results belong to the stream that the call names."""
    @functools.wraps(method)
    def call(self, *args, stream=None, **options):
        if stream is None or stream_address(stream, self.device) == stream_address(None, self.device):
            return method(self, *args, stream=stream, **options)
        with stream_scope(stream, self.device):
            return method(self, *args, stream=stream, **options)
    return call
