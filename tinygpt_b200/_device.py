"""Addresses that the ctypes calls take: of tensors and of streams."""
from __future__ import annotations

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
