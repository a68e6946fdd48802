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

Calls on one cache are to run in order (attention calls may overlap each other).  A new
handle may be used on any stream, and may be dropped while torch's streams still work on
it; work on a stream given by its handle, and graphs, have to be over by then.
"""
from __future__ import annotations

import math
import struct
from ctypes import byref, c_int64, c_void_p
from typing import Any

from . import _lib
from ._lib import check, lib
from .layer import _stream_handle, _torch


# MoeKvAttendArgs as bytes: cheaper to fill on every call than a ctypes structure
_ATTEND_ARGS = struct.Struct("@QQQqqqqqqQQiiiif4x")


def _strides(t: Any) -> list[int]:
    """Element strides; a dimension of one entry gets 0 (torch leaves it arbitrary)."""
    return [st if n > 1 else 0 for n, st in zip(t.shape, t.stride())]


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
        self._dev = k.get_device()
        self._lib = lib()
        self._i32, self._f32, self._u8 = torch.int32, torch.float32, torch.uint8
        self._empty = torch.empty
        # the handle of the current stream without a Stream object around it
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
        self._scale = 1.0 / math.sqrt(head_dim)
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
        self._used_on: set[int] = set()  # streams that the tensors are recorded on
        # the scratch is zero before another stream uses it
        with torch.cuda.device(self.device):
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()

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
    # A decode step makes these calls once a layer, and its kernels take some
    # microseconds: the checks read the tensors as little as they can.
    def _index(self, name: str, t: Any) -> tuple[Any, int]:
        """``t`` as a contiguous 1-D int32 tensor on the cache's device, and its length."""
        try:
            if t.dtype is self._i32 and t.get_device() == self._dev:
                n, = t.shape
                return (t if t.is_contiguous() else t.contiguous()), n
        except AttributeError:  # not a tensor
            t = _torch().tensor(list(t), dtype=self._i32).to(self.device)
            return t, t.shape[0]
        except ValueError:      # not 1-D
            pass
        raise TypeError(f"{name} must be a 1-D int32 tensor on {self.device}")

    def _indices(self, a: str, x: Any, b: str, y: Any) -> tuple[int, int, int, Any]:
        """Two index arrays of one length: their addresses, the length, what keeps them alive."""
        x, n = self._index(a, x)
        y, m = self._index(b, y)
        if n != m:
            raise ValueError(f"{a} and {b} must have one entry each")
        return x.data_ptr(), y.data_ptr(), n, (x, y)

    def _batch(self, seqs: Any, starts: Any) -> tuple[Any, Any, int]:
        seqs, n = self._index("seqs", seqs)
        starts, m = self._index("starts", starts)
        if m != n + 1:
            raise ValueError("starts must have one entry more than seqs")
        return seqs, starts, n

    def _rows(self, name: str, t: Any) -> tuple[int, int, int, int]:
        """Rows and heads of ``t`` and their strides."""
        if not hasattr(t, "data_ptr") or t.dtype is not self.dtype or t.get_device() != self._dev:
            raise TypeError(f"{name} must be a {self.dtype} tensor on {self.device}")
        shape = t.shape
        if len(shape) != 3 or shape[2] != self.head_dim:
            raise ValueError(f"{name} must be [rows, heads, {self.head_dim}]")
        rows, heads, _ = shape
        token, head, dim = t.stride()
        if dim != 1 and rows and heads:
            raise ValueError(f"the last dimension of {name} must be contiguous")
        return rows, heads, token if rows > 1 else 0, head if heads > 1 else 0

    def _stream(self) -> int:
        """The current stream's handle, for a call that is about to use it."""
        raw = self._raw_stream(self._dev)
        if raw not in self._used_on:
            self._first_use(raw)
        return raw

    def _first_use(self, raw: int) -> None:
        """Tell torch's allocator, so that memory let go with the cache waits for the stream.
        Not of streams made elsewhere: those may be gone by then, and the allocator would
        still ask them (and their handles may come again)."""
        stream = _torch().cuda.current_stream(self.device)
        if stream.stream_id == 0 or stream.stream_id & 1:  # torch's own are odd, or the default
            for t in (self.k, self.v, self.block_table, self.lengths, self.refs, self._scratch):
                t.record_stream(stream)
            self._used_on.add(raw)

    def _on(self, stream: Any, method: Any, *args: Any) -> Any:
        """The call as if ``stream`` were current, so that the buffers it allocates belong
        to that stream too."""
        torch = _torch()
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(_stream_handle(stream), device=self.device)
        with torch.cuda.stream(stream):
            return method(*args)

    # -- pages --------------------------------------------------------------------
    def reserve(self, seqs: Any, counts: Any, stream: Any = None) -> None:
        """Lengthen ``seqs[i]`` by ``counts[i]`` tokens, with pages for them."""
        if stream is not None:
            return self._on(stream, self.reserve, seqs, counts)
        x, y, n, _keep = self._indices("seqs", seqs, "counts", counts)
        check(self._lib.moe_kv_reserve(self._h, x, y, n, self._stream()))

    def fork(self, parents: Any, children: Any, stream: Any = None) -> None:
        """Make the empty sequence ``children[i]`` a copy of ``parents[i]`` that shares
        its pages; a page is copied when one of its holders next writes to it."""
        if stream is not None:
            return self._on(stream, self.fork, parents, children)
        x, y, n, _keep = self._indices("parents", parents, "children", children)
        check(self._lib.moe_kv_fork(self._h, x, y, n, self._stream()))

    def truncate(self, seqs: Any, lengths: Any, stream: Any = None) -> None:
        """Shorten ``seqs[i]`` to ``lengths[i]`` tokens and let its other pages go."""
        if stream is not None:
            return self._on(stream, self.truncate, seqs, lengths)
        x, y, n, _keep = self._indices("seqs", seqs, "lengths", lengths)
        check(self._lib.moe_kv_truncate(self._h, x, y, n, self._stream()))

    def free(self, seqs: Any, stream: Any = None) -> None:
        """Empty the sequences: ``truncate`` to no tokens."""
        if stream is not None:
            return self._on(stream, self.free, seqs)
        seqs, _n = self._index("seqs", seqs)
        self.truncate(seqs, _torch().zeros_like(seqs))

    def copy_pages(self, src: Any, dst: Any, stream: Any = None) -> None:
        """Copy pages ``src[i]`` to ``dst[i]`` in every layer; tables and refs stay."""
        if stream is not None:
            return self._on(stream, self.copy_pages, src, dst)
        x, y, n, _keep = self._indices("src", src, "dst", dst)
        check(self._lib.moe_kv_copy_pages(self._h, x, y, n, self._stream()))

    def compact(self, into: "PagedKVCache | None" = None, stream: Any = None) -> None:
        """Move the live pages to the lowest numbers, or, dense and in order, ``into``
        another cache (whose sequences are overwritten): how a pool changes its size."""
        if stream is not None:
            return self._on(stream, self.compact, into)
        if into is not None:
            if not into._h.value:  # null would mean: in place
                raise ValueError("into is closed")
            into._stream()  # its tensors are used too
        check(self._lib.moe_kv_compact(self._h, None if into is None else into._h, self._stream()))

    # -- tokens -------------------------------------------------------------------
    def append(self, k: Any, v: Any, seqs: Any, starts: Any, layer: int = 0,
               stream: Any = None) -> None:
        """Write the batch's keys and values ``[rows, kv_heads, head_dim]`` to the last
        places of their sequences (after ``reserve``).  A batch with wrong ``starts``, or with
        rows of one sequence in two entries, writes nothing (see ``status``)."""
        if stream is not None:
            return self._on(stream, self.append, k, v, seqs, starts, layer)
        seqs, starts, n = self._batch(seqs, starts)
        rows, heads, kt, kh = self._rows("k", k)
        vrows, vheads, vt, vh = self._rows("v", v)
        if heads != self.kv_heads or vheads != heads or vrows != rows:
            raise ValueError(f"k and v must both be [rows, {self.kv_heads}, {self.head_dim}]")
        check(self._lib.moe_kv_append(self._h, layer, k.data_ptr(), v.data_ptr(), kt, kh, vt, vh,
                                      seqs.data_ptr(), starts.data_ptr(), n, rows, self._stream()))

    def attend(self, q: Any, seqs: Any, starts: Any, layer: int = 0, scale: float | None = None,
               out: Any = None, lse: Any = None, stream: Any = None) -> Any:
        """Causal attention of the batch's rows ``q`` ``[rows, heads, head_dim]`` over all
        tokens of their sequences; returns ``out``, shaped as ``q``.  ``lse``: an fp32
        ``[rows, heads]`` tensor that receives the log of the sum of the exponentials."""
        if stream is not None:
            return self._on(stream, self.attend, q, seqs, starts, layer, scale, out, lse)
        seqs, starts, n = self._batch(seqs, starts)
        rows, heads, qt, qh = self._rows("q", q)
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"heads must be a multiple of {self.kv_heads}")
        if out is None:
            out = self._empty((rows, heads, self.head_dim), dtype=self.dtype, device=self.device)
            ot, oh = heads * self.head_dim, self.head_dim
        else:
            orows, oheads, ot, oh = self._rows("out", out)
            if orows != rows or oheads != heads:
                raise ValueError("out must have the shape of q")
        lp, lt, lh = 0, 0, 0
        if lse is not None:
            if lse.dtype is not self._f32 or lse.get_device() != self._dev or lse.shape != q.shape[:2]:
                raise ValueError("lse must be a float32 [rows, heads] tensor on the cache's device")
            lp, (lt, lh) = lse.data_ptr(), _strides(lse)
        if rows == 0 or n == 0:
            return out
        # the scratch of one call: torch's allocator keeps it apart from other streams' and
        # graphs' scratch
        need = self._lib.moe_kv_attend_workspace_bytes(self._h, heads, rows, n)
        ws = self._empty(need, dtype=self._u8, device=self.device)
        args = _ATTEND_ARGS.pack(q.data_ptr(), out.data_ptr(), lp, qt, qh, ot, oh, lt, lh,
                                 seqs.data_ptr(), starts.data_ptr(), n, rows, heads, layer,
                                 self._scale if scale is None else scale)
        check(self._lib.moe_kv_attend(self._h, args, ws.data_ptr(), need, self._stream()))
        return out

    def status(self, stream: Any = None) -> None:
        """Wait for the stream and raise what the cache's kernels reported, if anything."""
        if stream is not None:
            return self._on(stream, self.status)
        check(self._lib.moe_kv_status(self._h, self._stream()))
