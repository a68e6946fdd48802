"""A paged K/V cache on the device and attention over it, behind the C ABI.

The reference has no K/V cache: its generation loop re-runs the whole sequence for
every token (examples/demo_inference.py:131-144).  ``PagedKVCache`` holds keys and values
of many sequences in pages of a pool of torch tensors (layout and rules:
include/moe_sm100.h, "paged K/V cache"), so a decode step costs one token per sequence:

    cache = PagedKVCache.allocate(layers=2, pages=512, page_size=64, kv_heads=8,
                                  head_dim=128, sequences=64, max_blocks=64)
    cache.reserve(seqs, counts)                 # room for the step's new tokens
    for layer in range(2):
        cache.append(k, v, seqs, starts, layer=layer)
        out = cache.attend(q, seqs, starts, layer=layer)

``seqs`` (int32 [n]) names the sequences of the step, ``starts`` (int32 [n + 1]) the
offsets of their rows in ``q`` / ``k`` / ``v``: sequence ``seqs[i]`` brings rows
``starts[i] .. starts[i + 1] - 1``, its last tokens.  Index arguments are CUDA tensors
(or lists, copied to the device), so a step can be captured in a CUDA graph; errors
in their values are found on the device and raised by ``status()``.  Every call takes
``stream=`` (default: the current stream of the cache's device).
"""
from __future__ import annotations

import functools
import math
from ctypes import byref, c_int64, c_void_p
from typing import Any

from . import _lib
from ._lib import check, lib
from .layer import _stream_handle, _torch

_PAIR = c_int64 * 2


def _strides(t: Any) -> list[int]:
    """Element strides; a dimension of one entry gets 0 (torch leaves it arbitrary)."""
    return [st if n > 1 else 0 for n, st in zip(t.shape, t.stride())]


def _on_stream(method: Any) -> Any:
    """With ``stream=`` the call runs as if that stream were current, so that the buffers
    it allocates belong to that stream too."""
    @functools.wraps(method)
    def call(self: Any, *args: Any, stream: Any = None, **kw: Any) -> Any:
        if stream is None:
            return method(self, *args, **kw)
        torch = _torch()
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(_stream_handle(stream), device=self.device)
        with torch.cuda.stream(stream):
            return method(self, *args, **kw)
    return call


class PagedKVCache:
    """Handle of one cache over the caller's tensors; all calls are stream-ordered."""

    def __init__(self, k: Any, v: Any, block_table: Any, lengths: Any, refs: Any) -> None:
        """``k``, ``v``: CUDA f16 / bf16 ``[layers, pages, kv_heads, page_size, head_dim]``
        (strided views are fine); ``block_table`` int32 ``[sequences, max_blocks]``,
        ``lengths`` int32 ``[sequences]``, ``refs`` int32 ``[pages]``."""
        torch = _torch()
        self._h = c_void_p()
        for name, t in (("k", k), ("v", v)):
            if not (isinstance(t, torch.Tensor) and t.is_cuda
                    and t.dtype in (torch.float16, torch.bfloat16) and t.dim() == 5):
                raise TypeError(f"{name} must be a 5-D CUDA float16 or bfloat16 tensor")
            if t.stride(4) != 1 and t.shape[4] > 1:
                raise ValueError(f"the last dimension of {name} must be contiguous")
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must have the same shape and dtype")
        layers, pages, kv_heads, page_size, head_dim = k.shape
        for name, t, shape in (("block_table", block_table, None), ("lengths", lengths, None),
                               ("refs", refs, (pages,))):
            if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.int32
                    and t.is_contiguous()):
                raise TypeError(f"{name} must be a contiguous CUDA int32 tensor")
            if shape is not None and tuple(t.shape) != shape:
                raise ValueError(f"{name} must have shape {shape}")
        if block_table.dim() != 2 or tuple(lengths.shape) != (block_table.shape[0],):
            raise ValueError("block_table must be [sequences, max_blocks], lengths [sequences]")
        if len({t.device for t in (k, v, block_table, lengths, refs)}) != 1:
            raise ValueError("all tensors of a cache must be on one device")
        self.k, self.v = k, v
        self.block_table, self.lengths, self.refs = block_table, lengths, refs
        self.device = k.device
        self.dtype = k.dtype
        self.kv_heads, self.page_size, self.head_dim = kv_heads, page_size, head_dim
        cfg = _lib.MoeKvConfigC(
            k=k.data_ptr(), v=v.data_ptr(), k_strides=(c_int64 * 4)(*_strides(k)[:4]),
            v_strides=(c_int64 * 4)(*_strides(v)[:4]), block_table=block_table.data_ptr(),
            lengths=lengths.data_ptr(), refs=refs.data_ptr(),
            dtype=_lib.MOE_KV_BF16 if k.dtype == torch.bfloat16 else _lib.MOE_KV_F16,
            layers=layers, pages=pages, kv_heads=kv_heads, page_size=page_size, head_dim=head_dim,
            sequences=block_table.shape[0], max_blocks=block_table.shape[1],
            device=k.device.index)
        self._scratch = torch.zeros(max(int(lib().moe_kv_scratch_bytes(byref(cfg))), 4) // 4,
                                    dtype=torch.int32, device=k.device)
        cfg.scratch = self._scratch.data_ptr()
        check(lib().moe_kv_create(byref(cfg), byref(self._h)))

    @classmethod
    def allocate(cls, *, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 sequences: int, max_blocks: int, dtype: Any = None,
                 device: Any = None) -> "PagedKVCache":
        """An empty cache; its pool takes 4 * layers * pages * kv_heads * page_size *
        head_dim bytes of HBM."""
        torch = _torch()
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else \
            torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        dtype = torch.float16 if dtype is None else dtype
        shape = (layers, pages, kv_heads, page_size, head_dim)
        i32 = dict(dtype=torch.int32, device=dev)
        return cls(torch.zeros(shape, dtype=dtype, device=dev),
                   torch.zeros(shape, dtype=dtype, device=dev),
                   torch.full((sequences, max_blocks), -1, **i32),
                   torch.zeros(sequences, **i32), torch.zeros(pages, **i32))

    # -- lifetime ---------------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            lib().moe_kv_destroy(self._h)
            self._h = c_void_p()

    def __del__(self) -> None:  # pragma: no cover - interpreter shutdown order
        try:
            self.close()
        except Exception:
            pass

    # -- arguments ----------------------------------------------------------------
    def _index(self, name: str, t: Any) -> Any:
        torch = _torch()
        if not isinstance(t, torch.Tensor):
            t = torch.tensor(list(t), dtype=torch.int32).to(self.device)
        if t.dtype != torch.int32 or t.dim() != 1 or t.device != self.device:
            raise TypeError(f"{name} must be a 1-D int32 tensor on {self.device}")
        return t if t.is_contiguous() else t.contiguous()

    def _indices(self, a: str, x: Any, b: str, y: Any) -> tuple[Any, Any]:
        x, y = self._index(a, x), self._index(b, y)
        if x.shape[0] != y.shape[0]:
            raise ValueError(f"{a} and {b} must have one entry each")
        return x, y

    def _batch(self, seqs: Any, starts: Any) -> tuple[Any, Any]:
        seqs, starts = self._index("seqs", seqs), self._index("starts", starts)
        if starts.shape[0] != seqs.shape[0] + 1:
            raise ValueError("starts must have one entry more than seqs")
        return seqs, starts

    def _rows(self, name: str, t: Any) -> Any:
        torch = _torch()
        if not (isinstance(t, torch.Tensor) and t.dtype == self.dtype and t.device == self.device):
            raise TypeError(f"{name} must be a {self.dtype} tensor on {self.device}")
        if t.dim() != 3 or t.shape[2] != self.head_dim or (t.stride(2) != 1 and t.numel()):
            raise ValueError(f"{name} must be [rows, heads, {self.head_dim}], the last dimension "
                             "contiguous")
        return t

    def _stream(self) -> int:
        return _torch().cuda.current_stream(self.device).cuda_stream

    # -- pages --------------------------------------------------------------------
    @_on_stream
    def reserve(self, seqs: Any, counts: Any) -> None:
        """Lengthen ``seqs[i]`` by ``counts[i]`` tokens, with pages for them."""
        seqs, counts = self._indices("seqs", seqs, "counts", counts)
        check(lib().moe_kv_reserve(self._h, seqs.data_ptr(), counts.data_ptr(), seqs.shape[0],
                                   self._stream()))

    @_on_stream
    def fork(self, parents: Any, children: Any) -> None:
        """Make the empty sequence ``children[i]`` a copy of ``parents[i]`` that shares
        its pages; a page is copied when one of its holders next writes to it."""
        parents, children = self._indices("parents", parents, "children", children)
        check(lib().moe_kv_fork(self._h, parents.data_ptr(), children.data_ptr(),
                                parents.shape[0], self._stream()))

    @_on_stream
    def truncate(self, seqs: Any, lengths: Any) -> None:
        """Shorten ``seqs[i]`` to ``lengths[i]`` tokens and let its other pages go."""
        seqs, lengths = self._indices("seqs", seqs, "lengths", lengths)
        check(lib().moe_kv_truncate(self._h, seqs.data_ptr(), lengths.data_ptr(), seqs.shape[0],
                                    self._stream()))

    @_on_stream
    def free(self, seqs: Any) -> None:
        """Empty the sequences: ``truncate`` to no tokens."""
        seqs = self._index("seqs", seqs)
        self.truncate(seqs, _torch().zeros_like(seqs))

    @_on_stream
    def copy_pages(self, src: Any, dst: Any) -> None:
        """Copy pages ``src[i]`` to ``dst[i]`` in every layer; tables and refs stay."""
        src, dst = self._indices("src", src, "dst", dst)
        check(lib().moe_kv_copy_pages(self._h, src.data_ptr(), dst.data_ptr(), src.shape[0],
                                      self._stream()))

    @_on_stream
    def compact(self, into: "PagedKVCache | None" = None) -> None:
        """Move the live pages to the lowest numbers, or, dense and in order, ``into``
        another cache (whose sequences are overwritten): how a pool changes its size."""
        check(lib().moe_kv_compact(self._h, into._h if into is not None else None,
                                   self._stream()))

    # -- tokens -------------------------------------------------------------------
    @_on_stream
    def append(self, k: Any, v: Any, seqs: Any, starts: Any, layer: int = 0) -> None:
        """Write the batch's keys and values ``[rows, kv_heads, head_dim]`` to the last
        places of their sequences (after ``reserve``)."""
        seqs, starts = self._batch(seqs, starts)
        k, v = self._rows("k", k), self._rows("v", v)
        if k.shape != v.shape or k.shape[1] != self.kv_heads:
            raise ValueError(f"k and v must both be [rows, {self.kv_heads}, {self.head_dim}]")
        check(lib().moe_kv_append(self._h, layer, k.data_ptr(), v.data_ptr(),
                                  _PAIR(*_strides(k)[:2]), _PAIR(*_strides(v)[:2]),
                                  seqs.data_ptr(), starts.data_ptr(), seqs.shape[0], k.shape[0],
                                  self._stream()))

    @_on_stream
    def attend(self, q: Any, seqs: Any, starts: Any, layer: int = 0, scale: float | None = None,
               out: Any = None, lse: Any = None) -> Any:
        """Causal attention of the batch's rows ``q`` ``[rows, heads, head_dim]`` over all
        tokens of their sequences; returns ``out``, shaped as ``q``.  ``lse``: an fp32
        ``[rows, heads]`` tensor that receives the log of the sum of the exponentials."""
        torch = _torch()
        seqs, starts = self._batch(seqs, starts)
        q = self._rows("q", q)
        heads = q.shape[1]
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"heads must be a multiple of {self.kv_heads}")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        elif self._rows("out", out).shape != q.shape:
            raise ValueError("out must have the shape of q")
        if lse is not None and (lse.dtype != torch.float32 or lse.device != self.device
                                or lse.shape != q.shape[:2]):
            raise ValueError("lse must be a float32 [rows, heads] tensor on the cache's device")
        rows, n = q.shape[0], seqs.shape[0]
        if rows == 0 or n == 0:
            return out
        args = _lib.MoeKvAttendArgsC(
            q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(),
            _PAIR(*_strides(q)[:2]), _PAIR(*_strides(out)[:2]),
            _PAIR() if lse is None else _PAIR(*_strides(lse)), seqs.data_ptr(), starts.data_ptr(),
            n, rows, heads, layer,
            1.0 / math.sqrt(self.head_dim) if scale is None else scale)
        # the scratch of one call: torch's allocator keeps it apart from other streams' and
        # graphs' scratch
        need = lib().moe_kv_attend_workspace_bytes(self._h, heads, rows, n)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        check(lib().moe_kv_attend(self._h, byref(args), ws.data_ptr(), need, self._stream()))
        return out

    @_on_stream
    def status(self) -> None:
        """Wait for the stream and raise what the cache's kernels reported, if anything."""
        check(lib().moe_kv_status(self._h, self._stream()))
