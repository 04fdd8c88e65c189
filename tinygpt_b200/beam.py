"""Beam search's selection over beams and vocabulary (tg_beam_select).

`BeamSearch.select` takes a step's logits of all beams and returns the next beams:
parents, tokens, scores (sums of log-probabilities), finished flags and, given histories,
the reordered histories.  `PagedCache.fork` reorders the caches by the parents.  The
reference decodes by sampling only; it has no beam search.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

from . import _lib
from ._device import address, on_its_stream, stream_address
from ._lib import check
from .sampler import _dtype_code

try:
    import torch
except ImportError:  # pragma: no cover - the host API needs torch for device memory
    torch = None


class Beams(NamedTuple):
    """The next beams, best first: int32 parents, tokens, finished and float32 scores [batch, beams]; with
    histories also int32 history [batch * beams, stride] and history_len [batch * beams]."""
    parents: "torch.Tensor"
    tokens: "torch.Tensor"
    scores: "torch.Tensor"
    finished: "torch.Tensor"
    history: "torch.Tensor | None"
    history_len: "torch.Tensor | None"


class BeamSearch:
    """A tg_beam handle on one CUDA device (one per device and stream)."""

    def __init__(self, vocab: int, beams: int, max_batch: int, device: int = 0):
        self._L = _lib.load()
        self._h = None
        self.vocab, self.beams, self.max_batch, self.device = int(vocab), int(beams), int(max_batch), int(device)
        h = ctypes.c_void_p()
        check(self._L.tg_beam_create(self.device, self.vocab, self.beams, self.max_batch, ctypes.byref(h)))
        self._h = h

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._L.tg_beam_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001
            pass

    def device_status(self) -> int:
        """Status bits since the last call (synchronizes; see tgsample.h)."""
        bits = ctypes.c_uint32(0)
        check(self._L.tg_beam_device_status(self._h, ctypes.byref(bits)))
        return bits.value

    def _of(self, t, name, dtype, shape):
        if t is not None and (t.dtype is not dtype or t.shape != shape or t.get_device() != self.device or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on CUDA device {self.device}")

    @on_its_stream
    def select(self, logits, scores, *, finished=None, eos_id: int = -1, pad_id: int = 0, mask_table=None, state_id=None,
               history=None, history_len=None, stream=None) -> Beams:
        """logits [batch * beams, vocab or more] fp32/bf16, scores float32 [batch, beams] (-inf: a beam that does not
        take part, as all but the first at the start), finished int32 [batch, beams], mask_table and state_id as
        Sampler.sample, history int32 [batch * beams, stride] with history_len [batch * beams].  With `stream` given the
        results are allocated for it, and inputs have to be ready on it."""
        B, W = scores.shape
        rows = B * W
        if W != self.beams or logits.dim() != 2 or logits.shape[0] != rows or logits.shape[1] < self.vocab:
            raise ValueError(f"logits must be [batch * {self.beams}, at least {self.vocab}] and scores [batch, {self.beams}]")
        if logits.stride(1) != 1 and self.vocab > 1:
            raise ValueError("logits rows must be contiguous")
        if logits.get_device() != self.device:
            raise ValueError(f"logits must be on device {self.device}")
        self._of(scores, "scores", torch.float32, (B, W))
        self._of(finished, "finished", torch.int32, (B, W))
        self._of(state_id, "state_id", torch.int32, (rows,))
        num_states = 0
        if state_id is not None:
            words = (self.vocab + 31) // 32
            if mask_table is None or mask_table.dim() != 2 or mask_table.shape[1] != words or mask_table.element_size() != 4 or \
                    not mask_table.is_contiguous() or mask_table.get_device() != self.device:
                raise ValueError(f"mask_table must be a contiguous 32-bit tensor [states, {words}] on device {self.device}")
            num_states = mask_table.shape[0]
        ints = torch.empty_like(scores, dtype=torch.int32) if finished is None else torch.empty_like(finished)
        parents, tokens, done = ints, torch.empty_like(ints), torch.empty_like(ints)
        best = torch.empty_like(scores)
        new_history = new_len = None
        stride = 0
        if history is not None:
            stride = history.shape[1]
            self._of(history, "history", torch.int32, (rows, stride))
            if history_len is None:
                raise ValueError("history given without history_len")
            self._of(history_len, "history_len", torch.int32, (rows,))
            new_history, new_len = torch.empty_like(history), torch.empty_like(history_len)
        check(self._L.tg_beam_select(self._h, logits.data_ptr(), _dtype_code(logits), logits.stride(0) if rows > 1 else logits.shape[1], B,
                                     scores.data_ptr(), address(finished), address(mask_table), num_states, address(state_id), eos_id, pad_id,
                                     address(history), address(history_len), stride, parents.data_ptr(), tokens.data_ptr(), best.data_ptr(),
                                     done.data_ptr(), address(new_history), address(new_len), stream_address(stream, self.device)))
        return Beams(parents, tokens, best, done, new_history, new_len)
