"""The paged 4-bit key/value cache of a serving step, over the mq_b200 C ABI.

A step over ragged requests, as the batched forward runs it:

* ``PlanPages`` (``mq_pages_plan``) once: new pages, slots and positions of the step's rows;
* for each layer ``Kv4Cache.store`` (``mq_kv4_store``) of its key and value rows, then
  ``Kv4Cache.attention`` (``mq_kv4_attention``) of its query rows;
* ``ReleasePages`` (``mq_pages_release``) for the requests that ended.

Lengths, offsets, slots and tables are int32 tensors on the cache's device and are read when the
kernels run, so that a step can be captured in a CUDA graph. Wrong arguments raise ``ValueError``
or ``RuntimeError`` before anything is launched.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import NamedTuple

from . import _lib
from ._lib import check, lib


def _torch():
    import torch  # plumbing only: device memory and streams

    return torch


def _stream_on(torch, device: int, stream) -> int:
    """The handle of `stream`, or of the current stream of `device`."""
    if stream is None:
        return torch.cuda.current_stream(device).cuda_stream
    if stream.device.index != device:
        raise ValueError(f"the stream is of device {stream.device.index}, the call's of device {device}")
    return stream.cuda_stream


def _allocating_on(torch, stream):
    """The allocator reuses memory in the order of the stream that it was allocated on: the launch's."""
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _ints(torch, name: str, t, device: int, shape: tuple | None = None) -> int:
    """The address of an int32 tensor on `device` with `shape` (None: any number of elements)."""
    if t.dtype is not torch.int32 or not t.is_cuda or t.get_device() != device:
        raise RuntimeError(f"{name}: an int32 tensor on cuda:{device} is needed, not {t.dtype} on {t.device}")
    if not t.is_contiguous() or (shape is not None and t.shape != shape):
        raise RuntimeError(f"{name}: shape mismatch (contiguous {shape} is needed, not {tuple(t.shape)})")
    return t.data_ptr()


def _ok(rc: int, what: str) -> None:
    if rc == _lib.MQ_ERR_INVALID:
        raise ValueError(f"{what}: {_lib.last_error()}")
    check(rc, what)


class PagePlan(NamedTuple):
    """What ``PlanPages`` writes: row offsets ``[n + 1]`` and lengths ``[n]`` of the requests, slots and
    positions ``[rows]`` (-1 behind the last request), the free pages left and the requests refused ``[1]``."""

    offsets: object
    seq_lens: object
    slots: object
    positions: object
    n_free: object
    refused: object

    @classmethod
    def empty(cls, n_seqs: int, rows: int, device: int = 0) -> "PagePlan":
        torch = _torch()
        at = torch.device("cuda", device)
        return cls(*(torch.empty(n, dtype=torch.int32, device=at) for n in (n_seqs + 1, n_seqs, rows, rows, 1, 1)))


def PlanPages(ctx_lens, new_lens, block_tables, free_pages, n_free, page_size: int, rows: int | None = None,
              out: PagePlan | None = None, stream=None) -> PagePlan:
    """Gives the requests the pages that their new rows need and maps the rows to slots (mq_pages_plan).

    ``block_tables`` ``[n, max_pages]`` is updated in place. ``rows`` is the capacity of the row arrays; with
    ``out`` (whose ``seq_lens`` may be ``ctx_lens`` and whose ``n_free`` may be ``n_free``) it is theirs.
    """
    torch = _torch()
    if block_tables.dim() != 2:
        raise RuntimeError("block_tables: shape mismatch ([requests, pages] is needed)")
    n, width = block_tables.shape
    device = block_tables.get_device()
    if out is None:
        if rows is None:
            raise ValueError("PlanPages needs rows (the row arrays' capacity) or out")
        out = PagePlan.empty(n, rows, max(device, 0))
    elif rows is None:
        rows = out.slots.shape[0]
    _ok(lib().mq_pages_plan(
        device, _ints(torch, "ctx_lens", ctx_lens, device, (n,)), _ints(torch, "new_lens", new_lens, device, (n,)), n,
        page_size, _ints(torch, "block_tables", block_tables, device), width,
        _ints(torch, "free_pages", free_pages, device), free_pages.numel(),
        _ints(torch, "n_free", n_free, device, (1,)), rows, _ints(torch, "offsets", out.offsets, device, (n + 1,)),
        _ints(torch, "seq_lens", out.seq_lens, device, (n,)), _ints(torch, "slots", out.slots, device, (rows,)),
        _ints(torch, "positions", out.positions, device, (rows,)), _ints(torch, "n_free", out.n_free, device, (1,)),
        _ints(torch, "refused", out.refused, device, (1,)), _stream_on(torch, device, stream)), "PlanPages")
    return out


def ReleasePages(requests, seq_lens, block_tables, free_pages, n_free, page_size: int, stream=None) -> None:
    """Ends the requests of these rows of ``block_tables``: their pages go back to the stack and their lengths
    become 0, all in place (mq_pages_release)."""
    torch = _torch()
    if block_tables.dim() != 2:
        raise RuntimeError("block_tables: shape mismatch ([requests, pages] is needed)")
    n, width = block_tables.shape
    device = block_tables.get_device()
    _ok(lib().mq_pages_release(
        device, _ints(torch, "requests", requests, device), requests.numel(), n, page_size,
        _ints(torch, "seq_lens", seq_lens, device, (n,)), _ints(torch, "block_tables", block_tables, device), width,
        _ints(torch, "free_pages", free_pages, device), free_pages.numel(),
        _ints(torch, "n_free", n_free, device, (1,)), _stream_on(torch, device, stream)), "ReleasePages")


class Kv4Cache:
    """A paged key/value cache in 4-bit blocks on one GPU (mq_kv4_create), all zeros at first.

    Its memory is torch's: after use on other streams than the one it was made on, drop it only once they are done.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, device: int = 0,
                 stream=None):
        torch = _torch()
        self.handle = None
        need = lib().mq_kv4_bytes(layers, pages, page_size, kv_heads, head_dim)
        if not need:
            raise ValueError(f"Kv4Cache: {_lib.last_error()}")
        sh = _stream_on(torch, device, stream)
        with _allocating_on(torch, stream):
            self.memory = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", device))
        handle = C.c_void_p()
        _ok(lib().mq_kv4_create(device, layers, pages, page_size, kv_heads, head_dim, self.memory.data_ptr(), need, sh,
                                C.byref(handle)), "Kv4Cache")
        self.handle = handle
        self.device, self.layers, self.pages, self.page_size = device, layers, pages, page_size
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self._workspace = {}  # bytes by (heads, max_new)

    @property
    def device_bytes(self) -> int:
        n = C.c_size_t()
        check(lib().mq_kv4_info(self.handle, None, None, None, None, None, None, C.byref(n)))
        return n.value

    def _rows(self, torch, name: str, t, heads: int | None):
        """``t`` ``[rows, heads, head_dim]``, checked."""
        if t.dtype is not torch.float32 or not t.is_cuda or t.get_device() != self.device:
            raise RuntimeError(f"{name}: F32 rows on the cache's device are needed, not {t.dtype} on {t.device}")
        if t.dim() != 3 or t.shape[2] != self.head_dim or (heads is not None and t.shape[1] != heads):
            raise RuntimeError(f"{name}: shape mismatch ([rows, {heads or 'heads'}, {self.head_dim}] is needed, not "
                               f"{tuple(t.shape)})")
        if t.stride(2) != 1:
            raise RuntimeError(f"{name}: the elements of a head must be contiguous")
        return t

    def store(self, layer: int, k, v, slots, stream=None) -> None:
        """Packs ``k`` and ``v`` ``[rows, kv_heads, head_dim]`` into ``layer`` at ``slots`` (mq_kv4_store)."""
        torch = _torch()
        k, v = self._rows(torch, "keys", k, self.kv_heads), self._rows(torch, "values", v, self.kv_heads)
        rows = k.shape[0]
        if v.shape[0] != rows:
            raise RuntimeError(f"values: shape mismatch ({v.shape[0]} rows, {rows} of keys)")
        _ok(lib().mq_kv4_store(self.handle, layer, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                               v.stride(1), _ints(torch, "slots", slots, self.device, (rows,)), rows,
                               _stream_on(torch, self.device, stream)), "Kv4Cache.store")

    def load(self, layer: int, slots, stream=None):
        """The values that ``layer`` holds at ``slots``: ``(k, v)``, ``[rows, kv_heads, head_dim]`` (mq_kv4_load)."""
        torch = _torch()
        at = _ints(torch, "slots", slots, self.device)
        rows = slots.numel()
        handle = _stream_on(torch, self.device, stream)
        with _allocating_on(torch, stream):
            k, v = torch.empty((2, rows, self.kv_heads, self.head_dim), dtype=torch.float32, device=slots.device)
        _ok(lib().mq_kv4_load(self.handle, layer, at, rows, k.data_ptr(), v.data_ptr(), handle), "Kv4Cache.load")
        return k, v

    def attention(self, layer: int, q, offsets, seq_lens, block_tables, max_new: int | None = None,
                  scale: float | None = None, out=None, stream=None):
        """Causal attention of ``q`` ``[rows, heads, head_dim]`` over ``layer`` (mq_kv4_attention).

        ``offsets`` ``[n + 1]`` and ``seq_lens`` ``[n]`` as ``PlanPages`` gives them, ``block_tables``
        ``[n, max_pages]``. ``max_new`` is the most rows that a request brings (None: unknown). Rows past
        ``offsets[n]`` of ``out`` stay as they are; without ``out`` they are 0. ``scale`` defaults to
        1 / sqrt(head_dim).
        """
        torch = _torch()
        q = self._rows(torch, "queries", q, None)
        rows, heads = q.shape[0], q.shape[1]
        if block_tables.dim() != 2:
            raise RuntimeError("block_tables: shape mismatch ([requests, pages] is needed)")
        n, width = block_tables.shape
        handle = _stream_on(torch, self.device, stream)
        if out is not None and self._rows(torch, "output", out, heads).shape[0] < rows:
            raise RuntimeError(f"output: shape mismatch ({out.shape[0]} rows, {rows} of queries)")
        if max_new is None:
            max_new = rows
        need = self._workspace.get((heads, max_new))
        if need is None:
            need = lib().mq_kv4_attention_workspace(self.handle, heads, max_new)
            self._workspace[heads, max_new] = need
        with _allocating_on(torch, stream):
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            if out is None:
                out = torch.zeros((rows, heads, self.head_dim), dtype=torch.float32, device=q.device)
        _ok(lib().mq_kv4_attention(
            self.handle, layer, q.data_ptr(), q.stride(0), q.stride(1), rows, heads,
            _ints(torch, "offsets", offsets, self.device, (n + 1,)),
            _ints(torch, "seq_lens", seq_lens, self.device, (n,)),
            _ints(torch, "block_tables", block_tables, self.device), n, width, max_new,
            1.0 / math.sqrt(self.head_dim) if scale is None else scale, out.data_ptr(), out.stride(0), out.stride(1),
            ws.data_ptr(), need, handle), "Kv4Cache.attention")
        return out

    def close(self) -> None:
        if getattr(self, "handle", None):
            lib().mq_kv4_destroy(self.handle)
            self.handle = self.memory = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


__all__ = ["Kv4Cache", "PagePlan", "PlanPages", "ReleasePages"]
