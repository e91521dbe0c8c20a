"""The paged 4-bit key/value cache of a serving step, over the mq_b200 C ABI.

A step over ragged requests, as the batched forward runs it:

* ``PlanPages`` (``mq_pages_plan``) once: new pages, slots and positions of the step's rows;
* for each layer ``Kv4Cache.store`` (``mq_kv4_store``) of its key and value rows, then
  ``Kv4Cache.attention`` (``mq_kv4_attention``) of its query rows;
* ``ReleasePages`` (``mq_pages_release``) for the requests that ended.

Lengths, offsets, slots and tables are int32 tensors on the cache's device and are read when the
kernels run, so that a step can be captured in a CUDA graph. Wrong arguments raise ``ValueError``
or ``RuntimeError`` before anything is launched.

A decode step's kernels take a few microseconds each, so the calls do little else: arguments are
checked by single comparisons, and spelled out only once one fails.
"""
from __future__ import annotations

import ctypes as C
import math

from . import _lib
from ._lib import check, lib


def _torch():
    global _current
    import torch  # plumbing only: device memory and streams

    if _current is False:  # the handle itself, without a Stream object around it (1.5 us)
        _current = getattr(torch._C, "_cuda_getCurrentRawStream", None) if torch.cuda.is_available() else None
    return torch


_current = False


def _stream_on(torch, device: int, stream) -> int:
    """The handle of `stream`, or of the current stream of `device`."""
    if stream is None:
        return _current(device) if _current else torch.cuda.current_stream(device).cuda_stream
    if stream.device.index != device:
        raise ValueError(f"the stream is of device {stream.device.index}, the call's of device {device}")
    return stream.cuda_stream


def _empty(torch, shape, dtype, device, stream):
    """Memory for a call on `stream`: the allocator reuses it in the order of the stream it was allocated on."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


_MOST = 1 << 31  # counts are 32-bit in C: those that would wrap on their way there are refused here


def _ints(torch, name: str, t, device: int, n: int, most: int = _MOST) -> int:
    """The address of `n` contiguous int32 values on `device`."""
    if t.dtype is torch.int32 and t.get_device() == device and t.numel() == n < most and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not torch.int32 or t.get_device() != device:
        raise RuntimeError(f"{name}: an int32 tensor on cuda:{device} is needed, not {t.dtype} on {t.device}")
    if n >= most:
        raise RuntimeError(f"{name}: shape mismatch ({n} values: they must stay below 2^31)")
    raise RuntimeError(f"{name}: shape mismatch ({n} contiguous values are needed, not {tuple(t.shape)})")


def _table(torch, t):
    """(device, requests, pages, address) of block tables."""
    if t.dim() != 2:
        raise RuntimeError("block_tables: shape mismatch ([requests, pages] is needed)")
    device = t.get_device()
    n, width = t.shape
    if max(n, width) >= _MOST:
        raise RuntimeError("block_tables: shape mismatch (requests and pages must stay below 2^31)")
    return device, n, width, _ints(torch, "block_tables", t, max(device, 0), n * width, n * width + 1)


def _page(page_size: int) -> int:
    if not 0 < page_size <= 1024:  # (a size of more bits would wrap on its way into C)
        raise ValueError(f"page size {page_size}: a multiple of 16 up to 1024 is needed")
    return page_size


def _ok(rc: int, what: str) -> None:
    if rc == _lib.MQ_ERR_INVALID:
        raise ValueError(f"{what}: {_lib.last_error()}")
    check(rc, what)


class PagePlan:
    """What ``PlanPages`` writes: row offsets ``[n + 1]`` and lengths ``[n]`` of the requests, slots and
    positions ``[rows]`` (-1 behind the last request), the free pages left and the requests refused ``[1]``.

    The tensors are checked here once and stay the plan's for its life: they cannot be replaced.
    """

    __slots__ = ("offsets", "seq_lens", "slots", "positions", "n_free", "refused", "device", "_sizes", "_addresses")

    def __init__(self, offsets, seq_lens, slots, positions, n_free, refused):
        torch = _torch()
        device = max(offsets.get_device(), 0)
        n, rows = seq_lens.numel(), slots.numel()
        tensors = (("offsets", offsets, n + 1), ("seq_lens", seq_lens, n), ("slots", slots, rows),
                   ("positions", positions, rows), ("n_free", n_free, 1), ("refused", refused, 1))
        addresses = tuple(_ints(torch, name, t, device, size) for name, t, size in tensors)
        for name, t, _ in tensors:
            object.__setattr__(self, name, t)
        for name, value in (("device", device), ("_sizes", (n, rows)), ("_addresses", addresses)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"PagePlan.{name} stays what the plan was made with")

    def __delattr__(self, name):
        raise AttributeError(f"PagePlan.{name} stays what the plan was made with")

    def __reduce__(self):  # a copy has its own tensors' addresses
        return PagePlan, (self.offsets, self.seq_lens, self.slots, self.positions, self.n_free, self.refused)

    @classmethod
    def empty(cls, n_seqs: int, rows: int, device: int = 0, seq_lens=None, n_free=None, stream=None) -> "PagePlan":
        """A plan of its own memory; with ``seq_lens`` or ``n_free`` those, as a step that advances the lengths and
        the stack in place wants it."""
        torch = _torch()
        make = lambda n: _empty(torch, n, torch.int32, torch.device("cuda", device), stream)  # noqa: E731
        return cls(make(n_seqs + 1), make(n_seqs) if seq_lens is None else seq_lens, make(rows), make(rows),
                   make(1) if n_free is None else n_free, make(1))


def PlanPages(ctx_lens, new_lens, block_tables, free_pages, n_free, page_size: int, rows: int | None = None,
              out: PagePlan | None = None, stream=None) -> PagePlan:
    """Gives the requests the pages that their new rows need and maps the rows to slots (mq_pages_plan).

    ``block_tables`` ``[n, max_pages]`` is updated in place. ``rows`` is the capacity of the row arrays; with
    ``out`` (whose ``seq_lens`` may be ``ctx_lens`` and whose ``n_free`` may be ``n_free``) it is theirs. What the
    attention answers for the rows of a refused request means nothing; their slots and positions are -1.
    """
    torch = _torch()
    if out is None and rows is None:
        raise ValueError("PlanPages needs rows (the row arrays' capacity) or out")
    device, n, width, tables = _table(torch, block_tables)
    if out is None:
        out = PagePlan.empty(n, rows, device, stream=stream)
    if out._sizes[0] != n or out.device != device or (rows is not None and rows != out._sizes[1]):
        raise RuntimeError(f"out: shape mismatch (a plan of {n} requests on cuda:{device} is needed)")
    offsets, seq_lens, slots, positions, n_free_out, refused = out._addresses
    free = free_pages.numel()
    _ok(lib().mq_pages_plan(
        device, _ints(torch, "ctx_lens", ctx_lens, device, n), _ints(torch, "new_lens", new_lens, device, n), n,
        _page(page_size), tables, width, _ints(torch, "free_pages", free_pages, device, free), free,
        _ints(torch, "n_free", n_free, device, 1), out._sizes[1], offsets, seq_lens, slots, positions, n_free_out,
        refused, _stream_on(torch, device, stream)), "PlanPages")
    return out


def ReleasePages(requests, seq_lens, block_tables, free_pages, n_free, page_size: int, stream=None) -> None:
    """Ends the requests of these rows of ``block_tables``: their pages go back to the stack and their lengths
    become 0, all in place (mq_pages_release)."""
    torch = _torch()
    device, n, width, tables = _table(torch, block_tables)
    count, free = requests.numel(), free_pages.numel()
    _ok(lib().mq_pages_release(
        device, _ints(torch, "requests", requests, device, count), count, n, _page(page_size),
        _ints(torch, "seq_lens", seq_lens, device, n), tables, width,
        _ints(torch, "free_pages", free_pages, device, free), free, _ints(torch, "n_free", n_free, device, 1),
        _stream_on(torch, device, stream)), "ReleasePages")


class Kv4Cache:
    """A paged key/value cache in 4-bit blocks on one GPU (mq_kv4_create), all zeros at first.

    Its memory is torch's: after use on other streams than the one it was made on, drop it only once they are done.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, device: int = 0,
                 stream=None):
        torch = _torch()
        self.handle = None
        sizes = (layers, pages, page_size, kv_heads, head_dim)
        if max(sizes) >= _MOST or min(sizes) < -_MOST:
            raise ValueError("Kv4Cache: cache size overflow")
        need = lib().mq_kv4_bytes(layers, pages, page_size, kv_heads, head_dim)
        if not need:
            raise ValueError(f"Kv4Cache: {_lib.last_error()}")
        if not torch.cuda.is_available():
            raise RuntimeError("Kv4Cache needs a GPU")
        sh = _stream_on(torch, device, stream)
        self.memory = _empty(torch, need, torch.uint8, torch.device("cuda", device), stream)
        handle = C.c_void_p()
        _ok(lib().mq_kv4_create(device, layers, pages, page_size, kv_heads, head_dim, self.memory.data_ptr(), need, sh,
                                C.byref(handle)), "Kv4Cache")
        self.handle = handle
        self.device, self.layers, self.pages, self.page_size = device, layers, pages, page_size
        self.kv_heads, self.head_dim = kv_heads, head_dim

    @property
    def device_bytes(self) -> int:
        n = C.c_size_t()
        check(lib().mq_kv4_info(self.handle, None, None, None, None, None, None, C.byref(n)))
        return n.value

    def _layer(self, layer: int) -> int:
        if 0 <= layer < self.layers:
            return layer
        raise ValueError(f"layer {layer} of {self.layers}")

    def _rows(self, torch, name: str, t, rows: int | None, heads: int | None):
        """(shape, strides) of F32 `t` [rows, heads, head_dim] whose heads are contiguous."""
        shape = t.shape
        if (t.dtype is torch.float32 and t.get_device() == self.device and len(shape) == 3
                and shape[2] == self.head_dim and (heads is None or shape[1] == heads)
                and (rows is None or shape[0] == rows) and shape[0] < _MOST and shape[1] < _MOST):
            strides = t.stride()
            if strides[2] == 1:
                return shape, strides
            raise RuntimeError(f"{name}: the elements of a head must be contiguous")
        if t.dtype is not torch.float32 or t.get_device() != self.device:
            raise RuntimeError(f"{name}: F32 rows on the cache's device are needed, not {t.dtype} on {t.device}")
        raise RuntimeError(f"{name}: shape mismatch ([{'rows' if rows is None else rows}, {heads or 'heads'}, "
                           f"{self.head_dim}] is needed, not {tuple(shape)})")

    def store(self, layer: int, k, v, slots, stream=None) -> None:
        """Packs ``k`` and ``v`` ``[rows, kv_heads, head_dim]`` into ``layer`` at ``slots`` (mq_kv4_store)."""
        torch = _torch()
        (rows, _, _), (ld_k, hs_k, _) = self._rows(torch, "keys", k, None, self.kv_heads)
        _, (ld_v, hs_v, _) = self._rows(torch, "values", v, rows, self.kv_heads)
        _ok(lib().mq_kv4_store(self.handle, self._layer(layer), k.data_ptr(), ld_k, hs_k, v.data_ptr(), ld_v, hs_v,
                               _ints(torch, "slots", slots, self.device, rows), rows,
                               _stream_on(torch, self.device, stream)), "Kv4Cache.store")

    def load(self, layer: int, slots, stream=None):
        """The values that ``layer`` holds at ``slots``: ``(k, v)``, ``[rows, kv_heads, head_dim]`` (mq_kv4_load)."""
        torch = _torch()
        rows = slots.numel()
        at = _ints(torch, "slots", slots, self.device, rows)
        sh = _stream_on(torch, self.device, stream)
        shape = (rows, self.kv_heads, self.head_dim)
        if stream is None:
            k, v = slots.new_empty(shape, dtype=torch.float32), slots.new_empty(shape, dtype=torch.float32)
        else:
            k, v = (_empty(torch, shape, torch.float32, slots.device, stream) for _ in range(2))
        _ok(lib().mq_kv4_load(self.handle, self._layer(layer), at, rows, k.data_ptr(), v.data_ptr(), sh), "Kv4Cache.load")
        return k, v

    def attention(self, layer: int, q, offsets, seq_lens, block_tables, max_new: int | None = None,
                  scale: float | None = None, out=None, stream=None):
        """Causal attention of ``q`` ``[rows, heads, head_dim]`` over ``layer`` (mq_kv4_attention).

        ``offsets`` ``[n + 1]`` and ``seq_lens`` ``[n]`` as ``PlanPages`` gives them, ``block_tables``
        ``[n, max_pages]``. ``max_new`` is the most rows that a request brings (None: unknown). Rows past
        ``offsets[n]`` of ``out`` stay as they are; without ``out`` they are 0. ``scale`` defaults to
        1 / sqrt(head_dim). ``MQError`` (``MQ_ERR_TIMEOUT``): a wait of an earlier launch on the device ran out, and
        rows of its output are NaN.
        """
        torch = _torch()
        device = self.device
        (rows, heads, _), (ld_q, hs_q, _) = self._rows(torch, "queries", q, None, None)
        on, n, width, tables = _table(torch, block_tables)
        if on != device:
            raise RuntimeError(f"block_tables: an int32 tensor on cuda:{device} is needed")
        sh = _stream_on(torch, device, stream)
        if out is None:
            out = _empty(torch, (rows, heads, self.head_dim), torch.float32, q.device, stream)
            if stream is None:
                out.zero_()
            else:
                with torch.cuda.stream(stream):
                    out.zero_()
        (out_rows, _, _), (ld_o, hs_o, _) = self._rows(torch, "output", out, None, heads)
        if out_rows < rows:
            raise RuntimeError(f"output: shape mismatch ({out_rows} rows, {rows} of queries)")
        if max_new is None or max_new > rows:
            max_new = rows
        elif max_new < 0:
            max_new = -1  # (refused, however many bits it has)
        need = lib().mq_kv4_attention_workspace(self.handle, heads, max_new)
        ws = _empty(torch, need, torch.uint8, q.device, stream)
        _ok(lib().mq_kv4_attention(
            self.handle, self._layer(layer), q.data_ptr(), ld_q, hs_q, rows, heads, _ints(torch, "offsets", offsets, device, n + 1),
            _ints(torch, "seq_lens", seq_lens, device, n), tables, n, width, max_new,
            1.0 / math.sqrt(self.head_dim) if scale is None else scale, out.data_ptr(), ld_o, hs_o, ws.data_ptr(),
            need, sh), "Kv4Cache.attention")
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
