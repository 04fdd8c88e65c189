"""Paged key/value cache and the attention of drafted trees over it (tg_cache_*, tg_tree_*).

What a decoder keeps between the calls of the sampler: `PagedCache` holds the keys
and values of many sequences in pages that beams share, and all of its
bookkeeping lives on the device, so a step whose lengths are decided there (a tree's
accepted path) needs no round trip to the host.  The reference keeps one
sequence's contiguous cache per layer; it has no counterpart of pages, forks or trees.

A speculative step:  extend -> tree_attention (every layer) -> Sampler.sample over the
nodes' logits -> accept.  A beam step:  BeamSearch.select -> fork -> extend ->
tree_attention (every layer, one node) -> commit.

Device arrays are torch CUDA tensors; every call goes through libtgsample.so on the
current stream (or `stream`: results are allocated for it, inputs have to be ready on it
and to be kept until it has run the call).
"""
from __future__ import annotations

import ctypes
import math

from . import _lib
from ._device import address, on_its_stream, stream_address, stream_scope
from ._lib import check

try:
    import torch
except ImportError:  # pragma: no cover - the host API needs torch for device memory
    torch = None


class _Handle:
    """Destroys a tg_cache when the cache and every view of its state are gone."""

    def __init__(self, lib, ptr):
        self.lib, self.ptr = lib, ptr

    def __del__(self):
        try:
            self.lib.tg_cache_destroy(self.ptr)
        except Exception:  # noqa: BLE001
            pass


class _DeviceInts:
    """An int32 array that a handle owns, for torch.as_tensor: the tensor keeps the handle alive."""

    def __init__(self, handle: _Handle, ptr: int, shape):
        self.handle = handle
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<i4", "data": (ptr, False), "version": 2}


def _rows(t, name: str, n: int | None, device: int) -> int:
    """The length of an int32 contiguous vector on the device, n entries if given (None: not given, 0)."""
    if t is None:
        return 0
    shape = t.shape
    if t.dtype is not torch.int32 or len(shape) != 1 or t.get_device() != device or not t.is_contiguous() or (n is not None and shape[0] != n):
        raise ValueError(f"{name} must be a contiguous int32 vector{'' if n is None else f' of {n} entries'} on CUDA device {device}")
    return shape[0]


def _dense(t, name: str, shape, device: int, dtype):
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on CUDA device {device}")
    return t


def tree_masks(parents, n_nodes=None, *, out=None, stream=None):
    """tg_tree_masks: int64 [n, nodes] bit sets (a node and its ancestors) from int32 parents [n, nodes]."""
    n, nodes = parents.shape
    dev = parents.get_device()
    if dev < 0:
        raise ValueError("parents must be a CUDA tensor")
    _dense(parents, "parents", (n, nodes), dev, torch.int32)
    _rows(n_nodes, "n_nodes", n, dev)
    with torch.cuda.device(dev), stream_scope(stream, dev):
        if out is None:
            out = torch.empty((n, nodes), dtype=torch.int64, device=parents.device)
        _dense(out, "out", (n, nodes), dev, torch.int64)
        check(_lib.load().tg_tree_masks(n, nodes, address(n_nodes), address(parents), address(out), stream_address(stream, dev)))
    return out


class PagedCache:
    """A tg_cache handle and its pools k, v [layers, pages, kv_heads, page_size, head_dim].

    lens, counts, tables and refs are views of the handle's device state, to read:
    lengths and page counts by slot, page ids by slot (-1 past the count), holders by page.
    """

    def __init__(self, layers: int, kv_heads: int, head_dim: int, page_size: int, num_pages: int, max_seqs: int,
                 max_pages_per_seq: int, *, dtype=None, device: int = 0, k=None, v=None):
        dtype = torch.bfloat16 if dtype is None else dtype
        code = {torch.bfloat16: _lib.TG_DTYPE_BF16, torch.float16: _lib.TG_DTYPE_F16}.get(dtype)
        if code is None:
            raise TypeError(f"a cache holds bfloat16 or float16, got {dtype}")
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self._L = _lib.load()
        self._h = None
        self.device = int(device)
        self.dtype = dtype
        self.layers, self.kv_heads, self.head_dim, self.page_size = int(layers), int(kv_heads), int(head_dim), int(page_size)
        self.num_pages, self.max_seqs, self.max_pages_per_seq = int(num_pages), int(max_seqs), int(max_pages_per_seq)
        self._scale = 1.0 / math.sqrt(self.head_dim) if self.head_dim > 0 else 0.0
        if min(shape) <= 0:
            raise ValueError(f"the pools' shape {shape} must be positive")
        self._where = where = torch.device("cuda", self.device)
        self.k = torch.empty(shape, dtype=dtype, device=where) if k is None else k
        self.v = torch.empty(shape, dtype=dtype, device=where) if v is None else v
        for name, t in (("k", self.k), ("v", self.v)):
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous() or t.device != where:
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {where}")
        cfg = _lib.CacheConfig(self.layers, self.kv_heads, self.head_dim, self.page_size, self.num_pages, self.max_seqs,
                               self.max_pages_per_seq, code)
        h = ctypes.c_void_p()
        check(self._L.tg_cache_create(self.device, ctypes.byref(cfg), address(self.k), address(self.v), ctypes.byref(h)))
        self._owner, self._h = _Handle(self._L, h), h
        st = _lib.CacheState()
        check(self._L.tg_cache_get_state(self._h, ctypes.byref(st)))
        view = lambda p, *dims: torch.as_tensor(_DeviceInts(self._owner, p, dims), device=where)  # noqa: E731
        self.lens = view(st.lens, self.max_seqs)
        self.counts = view(st.counts, self.max_seqs)
        self.tables = view(st.tables, self.max_seqs, self.max_pages_per_seq)
        self.refs = view(st.refs, self.num_pages)

    @property
    def handle(self):
        return self._h

    def close(self) -> None:
        """Lets go of the handle and the pools; views of the state that the caller holds keep the handle."""
        self._h = self._owner = self.k = self.v = self.lens = self.counts = self.tables = self.refs = None

    def device_status(self) -> int:
        """Status bits since the last call (synchronizes; see tgsample.h)."""
        bits = ctypes.c_uint32(0)
        check(self._L.tg_cache_device_status(self._h, ctypes.byref(bits)))
        return bits.value

    def extend(self, seqs, counts, *, stream=None) -> None:
        """Pages for counts[i] tokens past slot seqs[i]'s length; a shared last page is copied first."""
        n = _rows(seqs, "seqs", None, self.device)
        _rows(counts, "counts", n, self.device)
        check(self._L.tg_cache_extend(self._h, n, seqs.data_ptr(), counts.data_ptr(), stream_address(stream, self.device)))

    def fork(self, src, dst, *, stream=None) -> None:
        """Slots dst[i] become copies of slots src[i] (-1: empty), all at once, sharing pages."""
        n = _rows(src, "src", None, self.device)
        _rows(dst, "dst", n, self.device)
        check(self._L.tg_cache_fork(self._h, n, src.data_ptr(), dst.data_ptr(), stream_address(stream, self.device)))

    def truncate(self, seqs, lens, *, stream=None) -> None:
        """Sets lengths back to lens[i]; pages past them are freed."""
        n = _rows(seqs, "seqs", None, self.device)
        _rows(lens, "lens", n, self.device)
        check(self._L.tg_cache_truncate(self._h, n, seqs.data_ptr(), lens.data_ptr(), stream_address(stream, self.device)))

    def free(self, seqs, *, stream=None) -> None:
        """Empties slots."""
        n = _rows(seqs, "seqs", None, self.device)
        check(self._L.tg_cache_truncate(self._h, n, seqs.data_ptr(), None, stream_address(stream, self.device)))

    def commit(self, seqs, counts, *, stream=None) -> None:
        """Advances lengths by counts[i] stored tokens."""
        n = _rows(seqs, "seqs", None, self.device)
        _rows(counts, "counts", n, self.device)
        check(self._L.tg_cache_commit(self._h, n, seqs.data_ptr(), counts.data_ptr(), stream_address(stream, self.device)))

    def _strides(self, t, name: str, shape):
        st = t.stride()
        if t.dtype is not self.dtype or t.shape != shape or t.get_device() != self.device or (st[3] != 1 and shape[3] != 1):
            raise ValueError(f"{name} must be a {self.dtype} tensor of shape {shape} on CUDA device {self.device}, its last dimension contiguous")
        return st

    def append(self, layer: int, seqs, k, v, counts=None, *, stream=None) -> None:
        """Stores keys and values [n, tokens, kv_heads, head_dim] of one layer past the lengths (reserve with
        extend, advance with commit)."""
        n = _rows(seqs, "seqs", None, self.device)
        if k.dim() != 4:
            raise ValueError("k must be [n, tokens, kv_heads, head_dim]")
        shape = (n, k.shape[1], self.kv_heads, self.head_dim)
        ks, vs = self._strides(k, "k", shape), self._strides(v, "v", shape)
        _rows(counts, "counts", n, self.device)
        check(self._L.tg_cache_append(self._h, layer, n, seqs.data_ptr(), address(counts), shape[1], k.data_ptr(), ks[0], ks[1], ks[2],
                                      v.data_ptr(), vs[0], vs[1], vs[2], stream_address(stream, self.device)))

    @on_its_stream
    def tree_attention(self, layer: int, seqs, q, k, v, masks=None, *, n_nodes=None, scale: float | None = None, out=None,
                       want_lse: bool = False, lse=None, stream=None):
        """tg_tree_attention: q [n, nodes, q_heads, head_dim] over the slots' cached tokens and the nodes' own k, v
        [n, nodes, kv_heads, head_dim], which are also stored past the lengths.  masks: int64 [n, nodes] bit sets
        (tree_masks; None: a chain).  Returns out, or (out, lse) with want_lse or lse given."""
        device, dim = self.device, self.head_dim
        n = _rows(seqs, "seqs", None, device)
        if q.dim() != 4:
            raise ValueError("q must be [n, nodes, q_heads, head_dim]")
        _, nodes, heads, _ = q.shape
        shape, kv = (n, nodes, heads, dim), (n, nodes, self.kv_heads, dim)
        qs, ks, vs = self._strides(q, "q", shape), self._strides(k, "k", kv), self._strides(v, "v", kv)
        if masks is not None:
            _dense(masks, "masks", (n, nodes), device, torch.int64)
        _rows(n_nodes, "n_nodes", n, device)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            _dense(out, "out", shape, device, self.dtype)
        if lse is not None:
            _dense(lse, "lse", shape[:3], device, torch.float32)
        elif want_lse:
            lse = q.new_empty(shape[:3], dtype=torch.float32)
        check(self._L.tg_tree_attention(self._h, layer, n, seqs.data_ptr(), nodes, address(n_nodes), address(masks), heads,
                                        q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2],
                                        self._scale if scale is None else scale, out.data_ptr(), address(lse),
                                        stream_address(stream, device)))
        return out if lse is None else (out, lse)

    @on_its_stream
    def accept(self, seqs, parents, tokens, ids, *, n_nodes=None, out_ids=None, out_n=None, stream=None):
        """tg_cache_accept: walks each tree (parents, drafted tokens [n, nodes]) with the target's ids [n, nodes] and
        keeps the accepted path in the cache.  Returns (out_ids int32 [n, nodes], out_n int32 [n])."""
        device = self.device
        n = _rows(seqs, "seqs", None, device)
        shape = (n, parents.shape[1])
        for name, t in (("parents", parents), ("tokens", tokens), ("ids", ids)):
            _dense(t, name, shape, device, torch.int32)
        _rows(n_nodes, "n_nodes", n, device)
        if out_ids is None:
            out_ids = torch.empty_like(ids)
        else:
            _dense(out_ids, "out_ids", shape, device, torch.int32)
        if out_n is None:
            out_n = torch.empty_like(seqs)
        else:
            _rows(out_n, "out_n", n, device)
        check(self._L.tg_cache_accept(self._h, n, seqs.data_ptr(), shape[1], address(n_nodes), parents.data_ptr(), tokens.data_ptr(),
                                      ids.data_ptr(), out_ids.data_ptr(), out_n.data_ptr(), stream_address(stream, device)))
        return out_ids, out_n
