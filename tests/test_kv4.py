"""The paged 4-bit key/value cache on the CPU side: argument checks, which come before any launch."""
from __future__ import annotations

import ctypes as C

import pytest

BUF = (C.c_int * 64)()
INTS = C.addressof(BUF)


def _create(mq, **kw):
    a = dict(device=0, layers=1, pages=4, page=16, kv=2, hd=64) | kw
    out = C.c_void_p()
    rc = mq.lib().mq_kv4_create(a["device"], a["layers"], a["pages"], a["page"], a["kv"], a["hd"], a.get("memory"),
                                a.get("bytes", 0), None, C.byref(out))
    assert not out.value
    return rc


@pytest.mark.parametrize("kw", [dict(layers=0), dict(pages=0), dict(kv=0), dict(pages=-1), dict(page=0), dict(page=8),
                                dict(page=24), dict(page=1040), dict(hd=0), dict(hd=16), dict(hd=48), dict(hd=160),
                                dict(pages=1 << 28), dict(layers=1 << 30, pages=1 << 27, kv=1 << 30)],
                         ids=lambda kw: "-".join(f"{k}{v}" for k, v in kw.items()))
def test_create_refuses(mq, kw):
    assert _create(mq, **kw) == mq._lib.MQ_ERR_INVALID
    assert mq._lib.last_error()


def test_create_refuses_null_output(mq):
    assert mq.lib().mq_kv4_create(0, 1, 1, 16, 1, 32, None, 0, None, None) == mq._lib.MQ_ERR_INVALID


def test_cache_bytes(mq):
    size = mq.lib().mq_kv4_bytes
    assert size(3, 5, 32, 4, 96) == 3 * 5 * 32 * 4 * 96 * 9 // 8
    assert size(80, 2 ** 20, 64, 8, 128) == 80 * 2 ** 26 * 8 * 144
    assert size(1, 1, 16, 1, 16) == 0 and "head size" in mq._lib.last_error()
    assert _create(mq, memory=1 << 20, bytes=size(1, 4, 16, 2, 64) - 1) == mq._lib.MQ_ERR_SIZE
    assert _create(mq, memory=(1 << 20) + 8, bytes=1 << 20) == mq._lib.MQ_ERR_INVALID
    with pytest.raises(ValueError, match="page size"):
        mq.Kv4Cache(1, 4, 8, 2, 64)


def test_null_handles(mq):
    lib, bad = mq.lib(), mq._lib.MQ_ERR_INVALID
    lib.mq_kv4_destroy(None)
    assert lib.mq_kv4_info(None, None, None, None, None, None, None, None) == bad
    assert lib.mq_kv4_store(None, 0, INTS, 32, 32, INTS, 32, 32, INTS, 1, None) == bad
    assert lib.mq_kv4_load(None, 0, INTS, 1, INTS, INTS, None) == bad
    assert lib.mq_kv4_attention_workspace(None, 1, 1) == 0
    assert lib.mq_kv4_attention(None, 0, INTS, 32, 32, 1, 1, INTS, INTS, INTS, 1, 1, 1, 1.0, INTS, 32, 32, INTS, 16,
                                None) == bad
    assert b"null cache" in lib.mq_last_error()


PLAN = dict(device=0, ctx=INTS, new=INTS + 32, n=2, page=16, tables=INTS, width=4, free=INTS, cap=8, n_free=INTS,
            rows=8, offsets=INTS, lens=INTS, slots=INTS, positions=INTS, n_free_out=INTS, refused=INTS)


@pytest.mark.parametrize("kw", [dict(n=-1), dict(n=8193), dict(rows=-1), dict(page=0), dict(page=20), dict(width=0),
                                dict(width=1 << 30), dict(cap=-1), dict(ctx=None), dict(new=None), dict(tables=None),
                                dict(free=None), dict(n_free=None), dict(offsets=None), dict(lens=None),
                                dict(slots=None), dict(positions=None), dict(n_free_out=None), dict(refused=None),
                                dict(lens=INTS + 32)],
                         ids=lambda kw: "-".join(f"{k}{v}" for k, v in kw.items()).replace(str(INTS + 32), "new"))
def test_plan_refuses(mq, kw):
    assert mq.lib().mq_pages_plan(*(PLAN | kw).values(), None) == mq._lib.MQ_ERR_INVALID
    assert mq._lib.last_error()


@pytest.mark.parametrize("kw", [dict(n=-1), dict(n_seqs=-1), dict(page=12), dict(width=0), dict(cap=-1),
                                dict(requests=None), dict(lens=None), dict(tables=None), dict(free=None),
                                dict(n_free=None)], ids=lambda kw: "-".join(f"{k}{v}" for k, v in kw.items()))
def test_release_refuses(mq, kw):
    a = dict(device=0, requests=INTS, n=1, n_seqs=2, page=16, lens=INTS, tables=INTS, width=4, free=INTS, cap=8,
             n_free=INTS) | kw
    assert mq.lib().mq_pages_release(*a.values(), None) == mq._lib.MQ_ERR_INVALID


def test_python_refuses_host_tensors(mq):
    import torch

    i = torch.zeros(2, dtype=torch.int32)
    tables = torch.zeros((2, 4), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="int32 tensor on cuda"):
        mq.PagePlan(torch.zeros(3, dtype=torch.int32), i, i, i, i[:1], i[:1])
    with pytest.raises(RuntimeError, match="int32 tensor on cuda"):
        mq.PlanPages(i, i, tables, i, i[:1], 16, rows=4)
    with pytest.raises(ValueError, match="rows"):
        mq.PlanPages(i, i, tables, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="shape"):
        mq.PlanPages(i, i, i, i, i[:1], 16, rows=4)
    with pytest.raises(RuntimeError, match="int32 tensor on cuda"):
        mq.ReleasePages(i, i, tables, i, i[:1], 16)


class _Ints:
    """An int32 tensor on cuda:0, as far as the argument checks look at it."""

    def __init__(self, n, device=0, at=0x1000):
        import torch

        self.dtype, self.device, self.shape, self._n, self._device, self._at = torch.int32, "cuda:0", (n,), n, device, at

    def get_device(self):
        return self._device

    def numel(self):
        return self._n

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self._at


def test_a_plan_keeps_its_tensors(mq):
    """The plan's addresses are taken once, so its tensors can be neither replaced nor dropped."""
    plan = mq.PagePlan(_Ints(3), _Ints(2), _Ints(8), _Ints(8), _Ints(1), _Ints(1))
    for name in ("offsets", "seq_lens", "slots", "positions", "n_free", "refused", "device"):
        held = getattr(plan, name)
        with pytest.raises(AttributeError, match="PagePlan"):
            setattr(plan, name, _Ints(8))
        with pytest.raises(AttributeError, match="PagePlan"):
            delattr(plan, name)
        assert getattr(plan, name) is held


def test_a_copied_plan_has_its_own_addresses(mq):
    import copy

    plan = mq.PagePlan(_Ints(3), _Ints(2), _Ints(8), _Ints(8), _Ints(1), _Ints(1))
    same = copy.copy(plan)
    assert same.slots is plan.slots and same._addresses == plan._addresses
    moved = [copy.copy(t) for t in (plan.offsets, plan.seq_lens, plan.slots, plan.positions, plan.n_free, plan.refused)]
    for i, t in enumerate(moved):
        t._at += 0x100 * (i + 1)
    memo = {id(a): b for a, b in zip((plan.offsets, plan.seq_lens, plan.slots, plan.positions, plan.n_free, plan.refused), moved)}
    other = copy.deepcopy(plan, memo)
    assert other.slots is moved[2] and other._addresses == tuple(t._at for t in moved)


class _Table(_Ints):
    def __init__(self, n, width):
        super().__init__(n * width)
        self.shape = (n, width)

    def dim(self):
        return 2


class _Rows:
    """F32 rows on cuda:0, all at one address."""

    def __init__(self, rows, heads, hd):
        import torch

        self.dtype, self.device, self.shape = torch.float32, "cuda:0", (rows, heads, hd)

    def get_device(self):
        return 0

    def stride(self):
        return 0, self.shape[2], 1

    def data_ptr(self):
        return 0x1000


def test_python_refuses_sizes_that_would_wrap(mq):
    """Counts are 32-bit in C: larger ones are refused, not taken modulo 2^32."""
    one, big = _Ints(1), (1 << 32) + 1
    for n in (1 << 31, big):
        with pytest.raises(RuntimeError, match="shape"):
            mq.PagePlan(_Ints(2), one, _Ints(n), _Ints(n), one, one)
        with pytest.raises(RuntimeError, match="shape"):
            mq.ReleasePages(_Ints(n), one, _Table(1, 2), one, one, 16)
        with pytest.raises(RuntimeError, match="shape"):
            mq.ReleasePages(one, one, _Table(1, 2), _Ints(n), one, 16)
        with pytest.raises(RuntimeError, match="shape"):
            mq.ReleasePages(one, one, _Table(1, n), one, one, 16)
    plan = mq.PagePlan(_Ints(2), one, _Ints(8), _Ints(8), one, one)
    for page in (-(1 << 32) + 16, -(1 << 31) - 16, -16, 0):
        with pytest.raises(ValueError, match="page size"):
            mq.PlanPages(one, one, _Table(1, 2), one, one, page, out=plan, stream=_Stream())
    with pytest.raises(ValueError, match="overflow"):
        mq.Kv4Cache(1, -(1 << 32) + 4, 16, 2, 64)
    cache = object.__new__(mq.Kv4Cache)
    cache.handle, cache.device, cache.layers, cache.kv_heads, cache.head_dim = None, 0, 1, 1, 32
    for n in (1 << 31, big):
        with pytest.raises(RuntimeError, match="shape"):
            cache.store(0, _Rows(n, 1, 32), _Rows(n, 1, 32), _Ints(n), stream=_Stream())
        with pytest.raises(RuntimeError, match="shape"):
            cache.attention(0, _Rows(n, 1, 32), _Ints(2), one, _Table(1, 2), out=_Rows(n, 1, 32), stream=_Stream())
        with pytest.raises(RuntimeError, match="shape"):
            cache.load(0, _Ints(n), stream=_Stream())


class _Stream:
    cuda_stream = 0

    class device:
        index = 0
