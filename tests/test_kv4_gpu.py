"""The paged 4-bit key/value cache on a B200: packing, block tables and attention against 64-bit references.

Packing and tables are exact. Attention: with u = 2^-24, every score's error is at most
    ds = scale * (2^-22 + 44 * 2^-23) * sum_e |q_e k_e|
(q enters as fp16 hi + lo, off by 2^-22 of it; at most 44 additions in a row, a tensor core's truncating ones off by
2^-23 each), exp2 and the weight's own hi + lo split add 2^-22 each, and the weighted sum and the sum of the weights
at most 256 additions in a row. A weight off by a relative e moves an output by at most 2 e * sum p |v| / sum p.
Weights far below the largest lose that relative precision: the lo part of a pair is an fp16 number, off by at most
2^-25 where it is subnormal, in units in which the largest weight is 2^8 or more (the reference is set 8 below a
score that the row has, and later only raised with the scores). A weight is therefore off by at most 2^-33 of the
largest weight p_max beside its relative error, and an output by at most 2^-33 * p_max * sum |v|. With sum p = 1:
    |d out| <= (2 * (max ds + 2^-21) + 256 * 2^-23) * sum p |v| + 2^-33 * p_max * sum |v|.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


# ------------------------------------------------------------------ references
def ref_blocks(x: np.ndarray) -> np.ndarray:
    """What the cache holds for x [..., hd], in float64."""
    b = x.astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    out = np.zeros_like(b)
    for i in np.ndindex(b.shape[:-1]):
        e = b[i]
        if not np.all(np.isfinite(e)):
            out[i] = np.nan
            continue
        d = e[np.argmax(np.abs(e))] / -8
        if d != 0:
            m, p = math.frexp(d)
            d = math.ldexp(np.rint(m * 256), p - 8)
        if abs(d) > 8160:
            out[i] = np.nan
            continue
        d = float(np.float16(d))
        if d != 0:
            out[i] = np.clip(np.rint(e / d), -8, 7) * d
    return out.reshape(x.shape)


def ref_plan(ctx, new, tables, free, n_free, page, rows):
    n, width = tables.shape
    tables, lens = tables.copy(), ctx.copy()
    offsets, slots, positions = [0], np.full(rows, -1), np.full(rows, -1)
    upto = taken = refused = 0
    for r in range(n):
        c, m = int(ctx[r]), int(new[r])
        offsets.append(offsets[-1] + max(m, 0))
        fits = c >= 0 and m >= 0 and c + m <= width * page and offsets[-1] <= rows
        more = -(-(c + m) // page) - -(-c // page) if fits else 0
        if not fits or (more and upto + more > n_free):
            refused += 1
            upto += more
            continue
        held = -(-c // page)
        for i in range(more):
            tables[r, held + i] = free[n_free - 1 - upto - i]
        upto += more
        taken += more
        lens[r] = c + m
        for i in range(m):
            p = c + i
            positions[offsets[-2] + i] = p
            slots[offsets[-2] + i] = tables[r, p // page] * page + p % page
    return tables, lens, np.array(offsets), slots, positions, n_free - taken, refused


def ref_attention(torch, q, k, v, news, lens, scale):
    """out, and the tolerance of each of its elements. k, v: per request [len, kv, hd] float64 of the cache's values."""
    q = q.double()
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    row = 0
    for m, length, ks, vs in zip(news, lens, k, v):
        group = q.shape[1] // max(ks.shape[1], 1)
        for i in range(m):
            last = length - m + i
            if last >= 0:
                kk, vv = (x[:last + 1].repeat_interleave(group, 1) for x in (ks, vs))
                s = torch.einsum("hd,shd->hs", q[row + i], kk) * scale
                p = torch.softmax(s, -1)
                out[row + i] = torch.einsum("hs,shd->hd", p, vv)
                size = torch.einsum("hd,shd->hs", q[row + i].abs(), kk.abs()).amax(-1) * abs(scale)
                rel = 2 * (size * (2 ** -22 + 44 * 2 ** -23) + 2 ** -21) + 256 * 2 ** -23
                tol[row + i] = rel[:, None] * torch.einsum("hs,shd->hd", p, vv.abs())
                tol[row + i] += 2 ** -33 * p.amax(-1)[:, None] * vv.abs().sum(0)
        row += m
    return out, tol


def assert_attention(torch, out, want, tol):
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    off = torch.nan_to_num((out.double() - want).abs()) - torch.nan_to_num(tol)
    worst = int(off.argmax())
    assert float(off.max()) <= 1e-30, f"element {np.unravel_index(worst, out.shape)} off by {float(off.max()):.3e} more than allowed"


def ints(torch, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


class Batch:
    """Requests of given lengths in a cache of random pages, with their values."""

    def __init__(self, mq, torch, lens, kv, hd, page, seed, extra=2, poison=True, layers=1, layer=0, pages=None):
        rng = np.random.default_rng(seed)
        self.lens, self.page, self.layer = list(lens), page, layer
        need = [-(-n // page) for n in lens]
        total = sum(need) + extra if pages is None else pages
        self.cache = mq.Kv4Cache(layers, total, page, kv, hd)
        order = rng.permutation(total)[-max(sum(need), 1):] if pages is None else total - 1 - np.arange(sum(need))
        width = max(max(need, default=0), 1) + 1
        tables = np.full((len(lens), width), -1, dtype=np.int32)
        at = 0
        slots = []
        for r, n in enumerate(lens):
            tables[r, :need[r]] = order[at:at + need[r]]
            at += need[r]
            p = np.arange(n)
            slots.append(tables[r, p // page] * page + p % page)
        if poison and pages is None:  # what no request sees is NaN
            everything = np.arange(total * page)
            bad = np.setdiff1d(everything, np.concatenate(slots) if slots else [])
            x = torch.full((len(bad), kv, hd), math.nan, device="cuda")
            self.cache.store(layer, x, x, ints(torch, bad))
        g = torch.Generator().manual_seed(seed)
        self.k = [torch.randn(n, kv, hd, generator=g) * 2 for n in lens]
        self.v = [torch.randn(n, kv, hd, generator=g) + 0.25 for n in lens]
        self.tables, self.slots = ints(torch, tables), ints(torch, np.concatenate(slots) if slots else [])
        self.cache.store(layer, torch.cat(self.k).cuda(), torch.cat(self.v).cuda(), self.slots)
        self.hk, self.hv = ([torch.from_numpy(ref_blocks_fast(torch, y)).cuda() for y in x] for x in (self.k, self.v))


def ref_blocks_fast(torch, x):
    """ref_blocks for finite values of ordinary size (checked against it below)."""
    b = x.double().unflatten(-1, (-1, 32))
    s = b.gather(-1, b.abs().argmax(-1, keepdim=True)) / -8
    m, e = torch.frexp(s)
    d = torch.ldexp(torch.round(m * 256), e - 8)
    return (torch.round(b / d).clamp(-8, 7) * d).flatten(-2).numpy()


def run_attention(torch, b, heads, news, seed, max_new=None, scale=None, spare=2, q=None, **kw):
    hd = b.cache.head_dim
    if q is None:
        q = torch.randn(sum(news) + spare, heads, hd, generator=torch.Generator().manual_seed(seed)).cuda()
    out = torch.full((sum(news) + spare, heads, hd), 7.0, device="cuda")
    offsets = ints(torch, np.concatenate([[0], np.cumsum(news)]))
    b.cache.attention(b.layer, q, offsets, ints(torch, b.lens), b.tables, max_new=max_new, scale=scale, out=out, **kw)
    return q, out


# ------------------------------------------------------------------ packing
def _odd_rows(rng, rows, kv, hd):
    x = rng.standard_normal((rows, kv, hd)).astype(np.float32)
    f = x.reshape(-1, 32)
    n = len(f)
    f[0 % n] = 0
    f[1 % n] = np.float32(-0.0)
    f[2 % n, :] = 1.0  # ties of the largest: the first one counts
    f[2 % n, 5] = -1.0
    f[3 % n] *= 1e-9  # fp16 has no such scale: 0
    f[4 % n] *= 2e-6  # a subnormal scale
    f[5 % n, 7] = 65280.0  # the largest that is held
    f[6 % n, 7] = 65600.0  # rounds up to a scale of 8192: NaN
    f[7 % n, 31] = np.inf
    f[8 % n, 0] = np.nan
    f[9 % n, 3] = -np.inf
    d = np.float32(0.8125)  # halves: ties to even
    f[10 % n] = (np.arange(32) % 16 - 7.5).astype(np.float32) * d
    f[10 % n, 4] = -8 * d
    f[11 % n] *= 1e30
    f[12 % n, :] = np.float32(1e-45)
    return x


@pytest.mark.parametrize("kv,hd,page,rows", [(1, 32, 16, 1), (8, 128, 64, 33), (5, 96, 16, 50), (3, 64, 48, 100),
                                             (2, 128, 1024, 300)])
@pytest.mark.parametrize("layout", ["fused", "headmajor", "unaligned"])
def test_store_and_load(mq, torch, kv, hd, page, rows, layout):
    rng = np.random.default_rng(rows + hd)
    pages = -(-rows // page) + 2
    c = mq.Kv4Cache(2, pages, page, kv, hd)
    assert c.device_bytes == 2 * pages * page * kv * hd * 9 // 8
    k, v = _odd_rows(rng, rows, kv, hd), _odd_rows(rng, rows, kv, hd)[::-1].copy()
    if layout == "fused":
        both = torch.from_numpy(np.concatenate([k.reshape(rows, -1), v.reshape(rows, -1)], 1)).cuda()
        tk, tv = both[:, :kv * hd].view(rows, kv, hd), both[:, kv * hd:].view(rows, kv, hd)
    elif layout == "headmajor":
        tk, tv = (torch.from_numpy(x.transpose(1, 0, 2).copy()).cuda().transpose(0, 1) for x in (k, v))
    else:
        flat = torch.empty(2 * k.size + 1, device="cuda")
        tk, tv = flat[1:1 + k.size].view(rows, kv, hd), flat[1 + k.size:].view(rows, kv, hd)
        tk.copy_(torch.from_numpy(k)), tv.copy_(torch.from_numpy(v))
    slots = rng.permutation(pages * page)[:rows].astype(np.int32)
    given = slots.copy()
    if rows > 4:
        given[1], given[3] = -1, pages * page  # skipped
    c.store(1, tk, tv, ints(torch, given))
    want_k, want_v = ref_blocks(k), ref_blocks(v)
    want_k[given != slots] = 0
    want_v[given != slots] = 0
    got_k, got_v = c.load(1, ints(torch, slots))
    np.testing.assert_array_equal(got_k.cpu().numpy(), want_k)
    np.testing.assert_array_equal(got_v.cpu().numpy(), want_v)
    # the other slots, the other layer, and slots outside
    rest = np.setdiff1d(np.arange(pages * page), slots)
    outside = np.concatenate([rest, [-1, pages * page, -2 ** 31, 2 ** 31 - 1]])
    for layer, at in ((1, outside), (0, np.arange(pages * page))):
        for x in c.load(layer, ints(torch, at)):
            assert not x.any()
    # written again: the last call's rows
    c.store(1, tv, tk, ints(torch, slots))
    np.testing.assert_array_equal(c.load(1, ints(torch, slots))[0].cpu().numpy(), ref_blocks(v))


def test_cache_of_its_own_memory(mq, torch):
    import ctypes as C

    lib, h = mq.lib(), C.c_void_p()
    assert lib.mq_kv4_create(0, 1, 2, 16, 1, 32, None, 0, None, C.byref(h)) == 0
    x, at = torch.randn(2, 1, 32, device="cuda"), ints(torch, [3, 30])
    out = torch.empty(2, 2, 1, 32, device="cuda")
    torch.cuda.synchronize()
    assert lib.mq_kv4_store(h, 0, x.data_ptr(), 32, 32, x.data_ptr(), 32, 32, at.data_ptr(), 2, None) == 0
    assert lib.mq_kv4_load(h, 0, at.data_ptr(), 2, out[0].data_ptr(), out[1].data_ptr(), None) == 0
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out[1].cpu().numpy(), ref_blocks(x.cpu().numpy()))
    lib.mq_kv4_destroy(h)


def test_fast_reference(torch):
    x = torch.randn(9, 2, 64, generator=torch.Generator().manual_seed(1)) * 2
    np.testing.assert_array_equal(ref_blocks_fast(torch, x), ref_blocks(x.numpy()))


def test_load_to_unaligned_memory(mq, torch):
    c = mq.Kv4Cache(1, 1, 16, 2, 32)
    x = torch.randn(3, 2, 32, device="cuda")
    at = ints(torch, [0, 5, 15])
    c.store(0, x, -x, at)
    flat = torch.zeros(2 * x.numel() + 1, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    rc = mq.lib().mq_kv4_load(c.handle, 0, at.data_ptr(), 3, flat[1:].data_ptr(), flat[1 + x.numel():].data_ptr(), stream)
    assert rc == 0
    k, v = c.load(0, at)
    assert torch.equal(flat[1:], torch.cat([k.flatten(), v.flatten()]))


# ------------------------------------------------------------------ block tables
def _plan_case(rng, n, ctx_max, new_max, page, width=None, short=0):
    ctx, new = rng.integers(0, ctx_max + 1, n), rng.integers(0, new_max + 1, n)
    held, need = -(-ctx // page), -(-(ctx + new) // page)
    width = width or int(max(1, need.max(initial=0)))
    pages = int(need.sum()) + 5
    order = rng.permutation(pages).astype(np.int32)
    tables = np.full((n, width), -1, dtype=np.int32)
    at = 0
    for r in range(n):
        m = min(int(held[r]), width)
        tables[r, :m] = order[at:at + m]
        at += m
    free = order[at:].copy()
    return ctx.astype(np.int32), new.astype(np.int32), tables, free, max(0, len(free) - 5 - short)


def _check_plan(mq, torch, ctx, new, tables, free, n_free, page, rows, in_place=False):
    want = ref_plan(ctx, new, tables, free, n_free, page, rows)
    t, c, nf = ints(torch, tables), ints(torch, ctx), ints(torch, [n_free])
    out = None
    if in_place:
        out = mq.PagePlan.empty(len(ctx), rows, seq_lens=c, n_free=nf)
    p = mq.PlanPages(c, ints(torch, new), t, ints(torch, free), nf, page, rows=rows, out=out)
    got = (t, p.seq_lens, p.offsets, p.slots, p.positions, p.n_free, p.refused)
    for name, g, w in zip(("tables", "lens", "offsets", "slots", "positions", "n_free", "refused"), got, want):
        np.testing.assert_array_equal(g.cpu().numpy().reshape(np.shape(w)), w, err_msg=name)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,ctx_max,new_max,page,spare", [
    (0, 0, 0, 16, 0), (0, 0, 0, 16, 70), (1, 0, 1, 16, 0), (1, 100, 5000, 16, 3), (7, 50, 3, 16, 1), (33, 200, 40, 48, 64),
    (1023, 300, 1, 64, 0), (1025, 100, 9, 32, 7), (5000, 40, 4, 16, 11), (8192, 20, 2, 128, 0)])
def test_plan(mq, torch, n, ctx_max, new_max, page, spare, in_place):
    rng = np.random.default_rng(n + page)
    ctx, new, tables, free, n_free = _plan_case(rng, n, ctx_max, new_max, page)
    _check_plan(mq, torch, ctx, new, tables, free, n_free, page, int(new.sum()) + spare, in_place)


@pytest.mark.parametrize("why", ["pages", "width", "rows", "negative", "no pages", "garbage count"])
@pytest.mark.parametrize("n", [5, 1500])
def test_plan_refuses_requests(mq, torch, why, n):
    rng = np.random.default_rng(n)
    ctx, new, tables, free, n_free = _plan_case(rng, n, 60, 30, 16)
    rows = int(new.sum())
    if why == "pages":
        n_free //= 2
    elif why == "width":
        tables = tables[:, :3].copy()
    elif why == "rows":
        rows -= rows // 3
    elif why == "negative":
        ctx[n // 2], new[n // 3] = -1, -(2 ** 31)
        rows += 10
    elif why == "no pages":
        n_free = 0
    _check_plan(mq, torch, ctx, new, tables, free, n_free, 16, rows)
    if why == "garbage count":  # clamped to the stack's capacity
        t = ints(torch, tables)
        p = mq.PlanPages(ints(torch, ctx), ints(torch, new), t, ints(torch, free), ints(torch, [2 ** 31 - 1]), 16, rows=rows)
        w = ref_plan(ctx, new, tables, free, len(free), 16, rows)
        np.testing.assert_array_equal(t.cpu().numpy(), w[0])
        assert int(p.n_free) == w[5]


def test_plan_of_huge_lengths(mq, torch):
    """Lengths whose sums pass 32 bits are refused, not wrapped."""
    ctx, new = [2 ** 31 - 1, 0, 5], [2 ** 31 - 1, 2 ** 31 - 1, 3]
    _check_plan_tail = mq.PlanPages(ints(torch, ctx), ints(torch, new), ints(torch, np.full((3, 2), 1)),
                                    ints(torch, [4, 5, 6]), ints(torch, [3]), 16, rows=8)
    assert int(_check_plan_tail.refused) == 3 and int(_check_plan_tail.n_free) == 3
    assert _check_plan_tail.seq_lens.tolist() == ctx
    assert _check_plan_tail.slots.tolist() == [-1] * 8


@pytest.mark.parametrize("n,ended", [(1, [0]), (9, [3, 1, 3, -1, 9, 7, 1]), (3000, None)])
def test_release(mq, torch, n, ended):
    rng = np.random.default_rng(n)
    page = 16
    lens = rng.integers(0, 100, n).astype(np.int32)
    pages = -(-lens // page)
    order = rng.permutation(int(pages.sum()) + 6).astype(np.int32)
    tables = np.full((n, 8), -1, dtype=np.int32)
    at = 0
    for r in range(n):
        tables[r, :pages[r]] = order[at:at + pages[r]]
        at += pages[r]
    ended = list(rng.integers(-5, n + 5, 2500)) if ended is None else ended
    stack = np.full(len(order), -7, dtype=np.int32)
    stack[:6] = order[at:]
    want, left = list(stack[:6]), lens.copy()
    for r in ended:
        if 0 <= r < n:
            want += list(tables[r, :-(-left[r] // page)])
            left[r] = 0
    t_lens, t_stack, t_free = ints(torch, lens), ints(torch, stack), ints(torch, [6])
    mq.ReleasePages(ints(torch, ended), t_lens, ints(torch, tables), t_stack, t_free, page)
    assert t_lens.tolist() == left.tolist()
    assert int(t_free) == len(want) and t_stack.tolist()[:len(want)] == want


def test_release_never_overfills(mq, torch):
    stack, n_free, lens = ints(torch, [9, 9, 9, 9]), ints(torch, [3]), ints(torch, [40, 40])
    guarded = torch.cat([stack, ints(torch, [77])])
    mq.ReleasePages(ints(torch, [0, 1]), lens, ints(torch, [[1, 2, 3], [4, 5, 6]]), guarded[:4], n_free, 16)
    assert int(n_free) == 4 and guarded.tolist() == [9, 9, 9, 1, 77] and lens.tolist() == [0, 0]


# ------------------------------------------------------------------ attention
LENS = [0, 1, 15, 16, 17, 31, 33, 64, 127, 128, 129, 255, 300, 700]


@pytest.mark.parametrize("page", [16, 48, 64, 128])
@pytest.mark.parametrize("heads,kv,hd", [(4, 1, 32), (8, 8, 64), (6, 2, 96), (8, 2, 128), (28, 4, 128), (16, 1, 128),
                                         (25, 1, 64)])
def test_decode(mq, torch, heads, kv, hd, page):
    b = Batch(mq, torch, LENS, kv, hd, page, seed=heads + hd)
    news = [1] * len(LENS)
    q, out = run_attention(torch, b, heads, news, 5, max_new=1)
    want, tol = ref_attention(torch, q[:-2], b.hk, b.hv, news, LENS, hd ** -0.5)
    assert_attention(torch, out[:-2], want, tol)
    assert (out[-2:] == 7.0).all()


@pytest.mark.parametrize("max_new", [None, 1, 100000])
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 128, 16), (7, 1, 64, 64), (3, 3, 96, 128), (12, 4, 32, 48)])
def test_mixed_rows(mq, torch, heads, kv, hd, page, max_new):
    """Decode rows, chunks, whole prompts, requests without rows, and rows before the first token, in one batch."""
    lens = [5, 200, 64, 1, 0, 131, 40, 300, 3]
    news = [5, 1, 64, 1, 0, 37, 0, 290, 6]  # the last: three rows stand before the first token
    b = Batch(mq, torch, lens, kv, hd, page, seed=3)
    q, out = run_attention(torch, b, heads, news, 6, max_new=max_new)
    want, tol = ref_attention(torch, q[:-2], b.hk, b.hv, news, lens, hd ** -0.5)
    assert_attention(torch, out[:-2], want, tol)
    assert (out[-2:] == 7.0).all()
    assert not out[sum(news) - 6:sum(news) - 3].any()


@pytest.mark.parametrize("heads,kv,hd,lens,news", [
    (8, 8, 64, [9000], [1]), (16, 2, 128, [5000, 3], [1, 1]), (4, 1, 128, [4100], [9]), (8, 1, 128, [2500], [600]),
    (2, 2, 96, [1500, 1400], [1500, 700]), (4, 4, 32, [20000], [2])])
def test_long(mq, torch, heads, kv, hd, lens, news):
    """Contexts that are split over many CTAs, and prompts of many tiles."""
    b = Batch(mq, torch, lens, kv, hd, 64, seed=8)
    q, out = run_attention(torch, b, heads, news, 9, max_new=max(news))
    want, tol = ref_attention(torch, q[:-2], b.hk, b.hv, news, lens, hd ** -0.5)
    assert_attention(torch, out[:-2], want, tol)


@pytest.mark.parametrize("heads,kv,hd,lens,news", [
    (32, 8, 64, [1500], [1400]), (32, 8, 128, [700, 900, 300], [700, 333, 300]), (40, 20, 32, [500] * 12, [400] * 12)])
def test_many_items_a_cta(mq, torch, heads, kv, hd, lens, news):
    """Many items follow one another in every CTA: its roles stay in step over many segments and steps."""
    b = Batch(mq, torch, lens, kv, hd, 64, seed=15)
    for again in range(3):
        q, out = run_attention(torch, b, heads, news, 16, max_new=max(news))
        if again:
            assert torch.equal(out, first)
        first = out
    at = 0
    for r, m in enumerate(news):  # all rows of a request share one product
        group = heads // kv
        k, v = (x.repeat_interleave(group, 1) for x in (b.hk[r], b.hv[r]))
        qq = q[at:at + m].double()
        s = torch.einsum("ihd,shd->his", qq, k) * hd ** -0.5
        sees = torch.arange(lens[r], device="cuda") <= torch.arange(lens[r] - m, lens[r], device="cuda")[:, None]
        p = torch.softmax(torch.where(sees, s, -math.inf), -1)
        want = torch.einsum("his,shd->ihd", p, v)
        size = torch.where(sees, torch.einsum("ihd,shd->his", qq.abs(), k.abs()), 0).amax(-1) * hd ** -0.5
        rel = (2 * (size * (2 ** -22 + 44 * 2 ** -23) + 2 ** -21) + 256 * 2 ** -23).T
        tol = rel[..., None] * torch.einsum("his,shd->ihd", p, v.abs())
        tol += 2 ** -33 * p.amax(-1).T[..., None] * v.abs().sum(0)
        assert_attention(torch, out[at:at + m], want, tol)
        at += m


@pytest.mark.parametrize("page", [16, 1024])
def test_many_requests(mq, torch, page):
    """More requests than a kernel has threads, most with one row, some with none or many."""
    rng = np.random.default_rng(page)
    n = 1700 if page == 16 else 300
    lens = rng.integers(0, 40, n)
    news = np.where(rng.random(n) < 0.05, np.minimum(lens, 30), np.minimum(lens, rng.integers(0, 2, n)))
    b = Batch(mq, torch, [int(x) for x in lens], 1, 32, page, seed=page)
    news = [int(x) for x in news]
    q, out = run_attention(torch, b, 2, news, 1)
    want, tol = ref_attention(torch, q[:-2], b.hk, b.hv, news, b.lens, 32 ** -0.5)
    assert_attention(torch, out[:-2], want, tol)
    assert (out[-2:] == 7.0).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales_and_sizes(mq, torch, scale):
    """Score scales of either sign, flat and one-hot softmaxes, queries and values of extreme sizes."""
    for size in (1.0, 1e-12, 1e12):
        b = Batch(mq, torch, [77, 300], 2, 64, 16, seed=4)
        q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(2)).cuda() * size
        q, out = run_attention(torch, b, 4, [1, 1], 0, max_new=1, scale=scale / size, spare=0, q=q)
        want, tol = ref_attention(torch, q, b.hk, b.hv, [1, 1], b.lens, scale / size)
        assert_attention(torch, out, want, tol)


@pytest.mark.parametrize("max_new", [1, 40])
def test_uneven_value_scales(mq, torch, max_new):
    """Values and keys whose blocks differ by many powers of two keep their precision."""
    b = Batch(mq, torch, [400], 2, 128, 64, seed=14)
    f = torch.logspace(-4, 3, 8).repeat_interleave(32).view(2, 128)
    k, v = b.k[0] * f.flip(0), b.v[0] * f
    b.cache.store(0, k.cuda(), v.cuda(), b.slots)
    b.hk, b.hv = ([torch.from_numpy(ref_blocks(y.numpy())).cuda()] for y in (k, v))
    news = [max_new]
    q, out = run_attention(torch, b, 4, news, 1, max_new=max_new, scale=1e-3)
    want, tol = ref_attention(torch, q[:-2], b.hk, b.hv, news, b.lens, 1e-3)
    assert_attention(torch, out[:-2], want, tol)


@pytest.mark.parametrize("new", [1, 50])
def test_strides(mq, torch, new):
    """Rows of a fused projection, head-major rows, rows at an odd address, and the output in the query's place."""
    b = Batch(mq, torch, [90, 200], 2, 64, 32, seed=2)
    news, heads = [new, new], 6
    q0, out0 = run_attention(torch, b, heads, news, 3, spare=0)
    offsets, lens = ints(torch, [0, new, 2 * new]), ints(torch, b.lens)
    fused = torch.zeros(2 * new, (heads + 4) * 64, device="cuda")
    q1 = fused[:, :heads * 64].view(2 * new, heads, 64)
    q2 = torch.zeros(heads, 2 * new, 64, device="cuda").transpose(0, 1)
    q3 = torch.zeros(2 * new * heads * 64 + 1, device="cuda")[1:].view(2 * new, heads, 64)
    for q in (q1, q2, q3):
        q.copy_(q0)
        assert torch.equal(b.cache.attention(0, q, offsets, lens, b.tables), out0)
        o = torch.empty_like(q)
        assert torch.equal(b.cache.attention(0, q, offsets, lens, b.tables, out=o), out0)
        assert torch.equal(b.cache.attention(0, q, offsets, lens, b.tables, out=q), out0)
    assert not fused[:, heads * 64:].any()


@pytest.mark.parametrize("new", [1, 70])
def test_pages_outside_the_cache_are_not_seen(mq, torch, new):
    lens = [200, 90]
    b = Batch(mq, torch, lens, 2, 64, 16, seed=12)
    bad = b.tables.clone()
    bad[0, 2], bad[0, 7], bad[1, 0] = -1, b.cache.pages, 2 ** 31 - 1
    b.tables = bad
    news = [new, new]
    q, out = run_attention(torch, b, 4, news, 1)
    hidden = [[2, 7], [0]]
    row = 0
    for r, n in enumerate(lens):
        for i in range(new):
            last = n - new + i
            s = [p for p in range(last + 1) if p // 16 not in hidden[r]]
            want, tol = ref_attention(torch, q[row:row + 1], [b.hk[r][s]], [b.hv[r][s]], [1], [len(s)], 64 ** -0.5)
            assert_attention(torch, out[row:row + 1], want, tol)
            row += 1


@pytest.mark.parametrize("new", [1, 40])
def test_non_finite(mq, torch, new):
    """NaN in the cache reaches the rows and heads that see it; a non-finite query its own row and head."""
    lens, news = [100, 60], [new, new]
    b = Batch(mq, torch, lens, 2, 64, 16, seed=21)
    seen = 100 - new + new // 2  # by the last half of the first request's rows
    k, v = b.k[0][seen:seen + 1].clone(), b.v[0][seen:seen + 1].clone()
    k[0, 0, 3] = math.inf
    v[0, 1, 40] = math.nan
    b.cache.store(0, k.cuda(), v.cuda(), b.slots[seen:seen + 1].contiguous())
    q = torch.randn(2 * new, 4, 64, generator=torch.Generator().manual_seed(1)).cuda()
    q[2 * new - 1, 1, 9] = math.nan
    if new > 1:
        q[2 * new - 3, 2, 0] = math.inf
    _, out = run_attention(torch, b, 4, news, 0, spare=0, q=q)
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[new // 2:new, :2] = True  # the key's block: every element of the heads that share it
    nan[new // 2:new, 2:, 32:] = True  # the value's block only
    nan[2 * new - 1, 1] = True
    if new > 1:
        nan[2 * new - 3, 2] = True
    assert torch.equal(torch.isnan(out), nan)


def test_empty_batches(mq, torch):
    b = Batch(mq, torch, [10], 1, 32, 16, seed=0)
    out = b.cache.attention(0, torch.randn(3, 2, 32, device="cuda"), ints(torch, [0, 0]), ints(torch, [10]), b.tables)
    assert out.shape == (3, 2, 32) and not out.any()
    out = b.cache.attention(0, torch.randn(0, 2, 32, device="cuda"), ints(torch, [0, 0]), ints(torch, [10]), b.tables)
    assert out.shape == (0, 2, 32)
    none = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    out = b.cache.attention(0, torch.randn(3, 2, 32, device="cuda"), ints(torch, [0]), ints(torch, []), none)
    assert not out.any()
    b.cache.store(0, torch.empty(0, 1, 32, device="cuda"), torch.empty(0, 1, 32, device="cuda"), ints(torch, []))
    assert b.cache.load(0, ints(torch, []))[0].shape == (0, 1, 32)


def test_offsets_past_the_rows(mq, torch):
    """Offsets that name more rows than the buffers have: those rows are not touched, the others as ever (up to the
    order of sums: fewer rows are other work for the kernels to divide)."""
    b = Batch(mq, torch, [100, 50], 1, 32, 16, seed=5)
    q, _ = run_attention(torch, b, 2, [60, 40], 1, spare=0)
    want, tol = ref_attention(torch, q, b.hk, b.hv, [60, 40], b.lens, 32 ** -0.5)
    for rows in (30, 59, 61, 99):
        out = torch.full((100, 2, 32), 7.0, device="cuda")
        b.cache.attention(0, q[:rows], ints(torch, [0, 60, 100]), ints(torch, b.lens), b.tables, out=out)
        assert_attention(torch, out[:rows], want[:rows], tol[:rows])
        assert (out[rows:] == 7.0).all()


def test_lengths_past_the_tables(mq, torch):
    """A length that its table cannot hold counts as the table's."""
    b = Batch(mq, torch, [64, 33], 1, 32, 16, seed=6)
    tables = b.tables[:, :4].contiguous()
    q = torch.randn(2, 2, 32, device="cuda")
    offsets = ints(torch, [0, 1, 2])
    want = b.cache.attention(0, q, offsets, ints(torch, [64, 33]), tables)
    got = b.cache.attention(0, q, offsets, ints(torch, [2 ** 31 - 1, 33]), tables)
    assert torch.equal(got, want)
    got = b.cache.attention(0, q, offsets, ints(torch, [-5, 33]), tables)
    assert not got[0].any() and torch.equal(got[1], want[1])


@pytest.mark.parametrize("news", [[1], [700]])
def test_cache_past_4gib(mq, torch, news):
    """Page addresses past 32 bits: the last pages of the last layer of a 5 GiB cache."""
    b = Batch(mq, torch, [900], 8, 128, 64, seed=7, layers=3, layer=2, pages=25000)
    assert b.cache.device_bytes > 5 * 2 ** 30
    q, out = run_attention(torch, b, 8, news, 1)
    want, tol = ref_attention(torch, q[:-2], b.hk, b.hv, news, [900], 128 ** -0.5)
    assert_attention(torch, out[:-2], want, tol)
    k, _ = b.cache.load(2, b.slots)
    assert torch.equal(k.double(), b.hk[0])
    assert not b.cache.load(1, b.slots)[0].any()


def test_refusals(mq, torch):
    c = mq.Kv4Cache(2, 4, 16, 2, 64)
    x, at = torch.zeros(3, 2, 64, device="cuda"), ints(torch, [0, 1, 2])
    for layer in (-1, 2, 1 << 32):
        with pytest.raises(ValueError, match="layer"):
            c.store(layer, x, x, at)
        with pytest.raises(ValueError, match="layer"):
            c.load(layer, at)
    for k, v, s in ((x[:2], x, at), (x, x[:, :1], at), (x, x[..., :32], at), (x, x, at[:2]), (x.double(), x, at),
                    (x.cpu(), x, at), (x, x, at.long()), (x, x, at.cpu()),
                    (torch.zeros(3, 64, 2, device="cuda").transpose(1, 2), x, at)):
        with pytest.raises(RuntimeError):
            c.store(0, k, v, s)
    offsets, lens, tables = ints(torch, [0, 1, 3]), ints(torch, [1, 2]), ints(torch, [[0, 1], [2, 3]])
    q = torch.zeros(3, 4, 64, device="cuda")
    c.attention(0, q, offsets, lens, tables)
    for a in ((q[:, :3], offsets, lens, tables),):
        with pytest.raises(ValueError, match="evenly"):
            c.attention(0, *a)
    for a in ((q[..., :32], offsets, lens, tables), (q, offsets[:2], lens, tables), (q, offsets, lens[:1], tables),
              (q, offsets, lens, tables[0]), (q, offsets, lens, tables.T), (q.half(), offsets, lens, tables),
              (q, offsets.long(), lens, tables), (q, offsets, lens.float(), tables)):
        with pytest.raises(RuntimeError):
            c.attention(0, *a)
    for out in (q[:2], q[:, :2], q.half(), q.cpu()):
        with pytest.raises(RuntimeError):
            c.attention(0, q, offsets, lens, tables, out=out)
    for scale in (math.inf, math.nan):
        with pytest.raises(ValueError, match="finite"):
            c.attention(0, q, offsets, lens, tables, scale=scale)
    with pytest.raises(ValueError):
        c.attention(0, q, offsets, lens, tables, max_new=-1)
    assert torch.equal(c.attention(0, q, offsets, lens, tables, max_new=1 << 40), c.attention(0, q, offsets, lens, tables))
    with pytest.raises(ValueError, match="overflow"):
        mq.Kv4Cache(1, (1 << 32) + 4, 16, 2, 64)
    with pytest.raises(ValueError, match="page size"):
        mq.ReleasePages(at, lens, tables, at, at[:1], (1 << 32) + 16)
    lib, e = mq.lib(), mq._lib
    need = lib.mq_kv4_attention_workspace(c.handle, 4, 3)
    assert need > 0
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    good = dict(layer=0, q=q.data_ptr(), ldq=256, hsq=64, rows=3, heads=4, offsets=offsets.data_ptr(),
                lens=lens.data_ptr(), tables=tables.data_ptr(), n=2, width=2, new=3, scale=1.0, out=q.data_ptr(),
                ldo=256, hso=64, ws=ws.data_ptr(), bytes=need)
    call = lambda **kw: lib.mq_kv4_attention(c.handle, *(good | kw).values(), None)  # noqa: E731
    torch.cuda.synchronize()
    assert call() == e.MQ_OK
    for kw in (dict(rows=-1), dict(heads=0), dict(n=-1), dict(width=0), dict(q=None), dict(out=None), dict(offsets=None),
               dict(lens=None), dict(tables=None), dict(hsq=63), dict(hso=32), dict(ldq=-1), dict(ldo=0), dict(width=1 << 27), dict(q=q.data_ptr() + 2)):
        assert call(**kw) == e.MQ_ERR_INVALID, kw
    for kw in (dict(ws=None), dict(bytes=need - 1)):
        assert call(**kw) == e.MQ_ERR_SIZE, kw
    assert call(ws=ws.data_ptr() + 8) == e.MQ_ERR_INVALID
    torch.cuda.synchronize()


# ------------------------------------------------------------------ as a step runs them
class Server:
    """A few requests over one cache, driven as a serving loop drives it, with their values kept on the host."""

    def __init__(self, mq, torch, slots, page=16, kv=2, heads=4, hd=64, pages=40, layers=2):
        self.mq, self.torch, self.page, self.heads, self.kv, self.hd, self.layers = mq, torch, page, heads, kv, hd, layers
        self.cache = mq.Kv4Cache(layers, pages, page, kv, hd)
        self.lens, self.tables = ints(torch, [0] * slots), ints(torch, np.full((slots, 12), -1))
        self.free, self.n_free = ints(torch, np.arange(pages)), ints(torch, [pages])
        self.pages = pages
        self.k = [[torch.zeros(0, kv, hd) for _ in range(slots)] for _ in range(layers)]
        self.v = [[torch.zeros(0, kv, hd) for _ in range(slots)] for _ in range(layers)]

    def step(self, news, gen):
        torch, mq = self.torch, self.mq
        rows = sum(news) + 3
        plan = mq.PagePlan.empty(len(news), rows, seq_lens=self.lens, n_free=self.n_free)
        mq.PlanPages(self.lens, ints(torch, news), self.tables, self.free, self.n_free, self.page, out=plan)
        assert int(plan.refused) == 0
        for layer in range(self.layers):
            x = torch.randn(rows, (self.heads + 2 * self.kv) * self.hd, generator=gen)
            y = x.cuda()
            q, k, v = (z.reshape(rows, -1, self.hd) for z in
                       y.split([self.heads * self.hd, self.kv * self.hd, self.kv * self.hd], 1))
            self.cache.store(layer, k, v, plan.slots)
            out = self.cache.attention(layer, q, plan.offsets, plan.seq_lens, self.tables, max_new=max(news))
            at = 0
            for r, m in enumerate(news):
                for held, z in ((self.k, k), (self.v, v)):
                    held[layer][r] = torch.cat([held[layer][r], z[at:at + m].cpu()])
                at += m
            hk, hv = ([torch.from_numpy(ref_blocks_fast(torch, z)).cuda() if len(z) else z.double().cuda()
                       for z in held[layer]] for held in (self.k, self.v))
            lens = [len(z) for z in self.k[layer]]
            want, tol = ref_attention(torch, q[:sum(news)], hk, hv, news, lens, self.hd ** -0.5)
            assert_attention(torch, out[:sum(news)], want, tol)
            assert not out[sum(news):].any()
        assert self.lens.tolist() == lens

    def end(self, requests):
        self.mq.ReleasePages(ints(self.torch, requests), self.lens, self.tables, self.free, self.n_free, self.page)
        for held in (*self.k, *self.v):
            for r in requests:
                held[r] = held[r][:0]


def test_serving_loop(mq, torch):
    """Prompts, decode steps, ended requests whose pages others take over, idle requests: plan, store and attention."""
    s = Server(mq, torch, 4)
    gen = torch.Generator().manual_seed(11)
    s.step([40, 7, 0, 100], gen)
    for _ in range(3):
        s.step([1, 1, 0, 1], gen)
    s.end([3, 1])
    s.step([1, 90, 33, 0], gen)
    s.step([1, 1, 1, 150], gen)
    s.end([0, 1, 2, 3])
    assert int(s.n_free) == s.pages and sorted(s.free.tolist()) == list(range(s.pages))


def test_graph_of_a_step(mq, torch):
    """A decode step captured once serves the steps after it; the lengths advance in place."""
    lens = [100, 31, 16, 5]
    b = Batch(mq, torch, lens, 2, 64, 16, seed=31, extra=8, poison=False)
    used = set(b.tables.flatten().tolist())
    free = ints(torch, [p for p in range(b.cache.pages) if p not in used])
    n_free, ctx = ints(torch, [free.numel()]), ints(torch, lens)
    tables = torch.cat([b.tables, torch.full((4, 2), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    plan = mq.PagePlan.empty(4, 4, seq_lens=ctx, n_free=n_free)
    one = ints(torch, [1] * 4)
    x = torch.zeros(4, 8 * 64, device="cuda")
    q, k, v = (z.reshape(4, -1, 64) for z in x.split([4 * 64, 2 * 64, 2 * 64], 1))
    out = torch.zeros(4, 4, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mq.PlanPages(ctx, one, tables, free, n_free, 16, out=plan)
        b.cache.store(0, k, v, plan.slots)
        b.cache.attention(0, q, plan.offsets, plan.seq_lens, tables, max_new=1, out=out)
    hk, hv = list(b.hk), list(b.hv)
    gen = torch.Generator().manual_seed(1)
    for step in range(1, 20):
        x.copy_(torch.randn(4, 8 * 64, generator=gen))
        graph.replay()
        hk, hv = ([torch.cat([h, torch.from_numpy(ref_blocks_fast(torch, z[r:r + 1].cpu())).cuda()])
                   for r, h in enumerate(held)] for held, z in ((hk, k), (hv, v)))
        now = [n + step for n in lens]
        assert ctx.tolist() == now
        want, tol = ref_attention(torch, q, hk, hv, [1] * 4, now, 64 ** -0.5)
        assert_attention(torch, out, want, tol)


@pytest.mark.parametrize("news", [[1, 1], [80, 300]])
def test_two_graphs_at_once(mq, torch, news):
    """Graphs captured one after the other and replayed on two streams share nothing; equal inputs give equal bits."""
    a = Batch(mq, torch, [3000, 400], 2, 128, 64, seed=1)
    b = Batch(mq, torch, [2500, 900], 2, 128, 64, seed=2)
    side = [torch.cuda.Stream() for _ in range(2)]
    runs = []
    for i, c in enumerate((a, b)):
        q, want = run_attention(torch, c, 8, news, i, max_new=max(news))
        out, graph = torch.full_like(want, 7.0), torch.cuda.CUDAGraph()
        offsets, lens = ints(torch, [0, news[0], sum(news)]), ints(torch, c.lens)
        with torch.cuda.graph(graph):
            c.cache.attention(0, q, offsets, lens, c.tables, max_new=max(news), out=out)
        runs.append((graph, out, want, q, offsets, lens))
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, out, *_), s in zip(runs, side):
            with torch.cuda.stream(s):
                out.fill_(7.0)
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, *_ in runs:
            assert torch.equal(out, want)


def test_other_streams(mq, torch):
    """Calls given a stream run there, in its order, without the current stream."""
    b = Batch(mq, torch, [700, 20], 2, 64, 16, seed=3)
    q, want = run_attention(torch, b, 4, [1, 1], 1, spare=0)
    offsets, lens = ints(torch, [0, 1, 2]), ints(torch, b.lens)
    x = torch.cat(b.k).cuda(), torch.cat(b.v).cuda()
    fresh = mq.Kv4Cache(1, b.cache.pages, 16, 2, 64)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    fresh.store(0, *x, b.slots, stream=s)
    out = fresh.attention(0, q, offsets, lens, b.tables, stream=s)
    k, _ = fresh.load(0, b.slots, stream=s)
    s.synchronize()
    assert torch.equal(out, want) and torch.equal(k.double(), torch.cat(b.hk))


def test_other_device(mq, torch):
    """A cache on another device than the current one (needs two)."""
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    c = mq.Kv4Cache(1, 4, 16, 1, 32, device=1)
    x = torch.randn(5, 1, 32, device="cuda:1")
    at = torch.arange(5, dtype=torch.int32, device="cuda:1")
    c.store(0, x, x, at)
    k, _ = c.load(0, at)
    np.testing.assert_array_equal(k.cpu().numpy(), ref_blocks(x.cpu().numpy()))
    with pytest.raises(RuntimeError):
        c.load(0, at.to("cuda:0"))
    assert torch.cuda.current_device() == 0


# ------------------------------------------------------------------ limits
def test_plan_sizes_in_a_fresh_process():
    """Every request count plans in a process that has planned none larger (what a large plan allows its kernel stays
    allowed): the sizes around the 48 KB of shared memory that need no permission."""
    code = ("import numpy as np, torch, mini_ai_b200 as mq, test_kv4_gpu as t\n"
            "for n in (4070, 4074, 4075, 4085, 4095, 4096, 4100):\n"
            "    rng = np.random.default_rng(n)\n"
            "    ctx, new, tables, free, n_free = t._plan_case(rng, n, 60, 3, 16)\n"
            "    for in_place in (False, True):\n"
            "        t._check_plan(mq, torch, ctx, new, tables, free, n_free, 16, int(new.sum()), in_place)\n"
            "print('planned', n)\n")
    _run_child(code, "planned 4100")


def _run_child(code, last):
    import os
    import subprocess
    import sys
    from pathlib import Path

    here = Path(__file__).resolve().parent
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(here.parent), str(here), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.splitlines()[-1:] == [last], r.stdout + r.stderr


def test_errors_of_earlier_calls():
    """A call reports its own errors only: not that of a product before it that could not get its memory. (In a process
    of its own, which takes the error that the product leaves behind with it.)"""
    _run_child(EARLIER_ERRORS, "done")


EARLIER_ERRORS = """
import numpy as np, torch, mini_ai_b200 as mq
from test_kv4_gpu import ints
rng = np.random.default_rng(0)
w = mq.CudaWeight(mq.QuantizeTensor(rng.standard_normal((128, 256)).astype(np.float32), mq.QuantType.kQ40), device=0)
x = torch.zeros(1, 256, device="cuda")
c, at = mq.Kv4Cache(1, 1, 16, 1, 32), ints(torch, [3])
row = torch.randn(1, 1, 32, device="cuda")
lens, tables, stack, n_free = ints(torch, [5]), ints(torch, [[0]]), ints(torch, [7, 7]), ints(torch, [1])
torch.cuda.synchronize()


def fail():  # the gate product of these rows would take 8 TiB; nothing is launched
    rc = mq.lib().mq_linear_swiglu(w.handle, w.handle, x.data_ptr(), 1 << 20, 256, x.data_ptr(), 1 << 21, None)
    assert rc == mq._lib.MQ_ERR_CUDA and "memory" in mq._lib.last_error()


fail()
c.store(0, row, -row, at)
fail()
k, v = c.load(0, at)
assert torch.equal(k, -v) and k.any()
fail()
mq.ReleasePages(ints(torch, [0]), lens, tables, stack, n_free, 16)
assert n_free.tolist() == [2] and stack.tolist() == [7, 0]
fail()
q = torch.randn(1, 32, 32, device="cuda")
for max_new in (0, 1):
    c.attention(0, q, ints(torch, [0, 1]), ints(torch, [4]), tables, max_new=max_new)
plan = mq.PlanPages(lens, ints(torch, [1]), tables, stack, n_free, 16, rows=1)
assert plan.refused.tolist() == [0]
w.close()
print("done")
"""


WAITS = [  # heads, kv, head size, cached tokens, new rows: few rows whole and cut; many rows whole, cut, many items a CTA
    (8, 2, 64, [100, 33], [1, 1], 16), (16, 2, 128, [20000, 40], [1, 1], 64), (4, 4, 32, [70] * 600, [1] * 600, 16),
    (8, 1, 128, [2500], [600], 64), (2, 2, 96, [1500, 1400, 9], [1500, 700, 1], 64), (32, 8, 64, [1500], [1400], 64)]


@pytest.mark.parametrize("heads,kv,hd,lens,news,page", WAITS)
def test_waits_that_run_out(mq, torch, monkeypatch, heads, kv, hd, lens, news, page):
    """Copies that never complete: every row is NaN, whichever CTA had it; the next call says so, once."""
    monkeypatch.setenv("MQ_KV4_LOSE_COPIES", "1")
    monkeypatch.setenv("MQ_KV4_WAIT_NS", "2000000")
    b = Batch(mq, torch, lens, kv, hd, page, seed=1)
    monkeypatch.delenv("MQ_KV4_LOSE_COPIES")
    monkeypatch.delenv("MQ_KV4_WAIT_NS")
    good = Batch(mq, torch, lens, kv, hd, page, seed=1)
    q, want = run_attention(torch, good, heads, news, 2, max_new=max(news))
    torch.cuda.synchronize()
    launches = mq.lib().mq_kernel_launches()
    for again in range(2):
        _, out = run_attention(torch, b, heads, news, 2, max_new=max(news))
        torch.cuda.synchronize()
        assert torch.isnan(out[:-2]).all() and (out[-2:] == 7.0).all()
        before = mq.lib().mq_kernel_launches()
        with pytest.raises(mq.MQError, match="bounded wait") as info:
            run_attention(torch, b if again else good, heads, news, 2, max_new=max(news))
        assert info.value.code == mq._lib.MQ_ERR_TIMEOUT
        assert mq.lib().mq_kernel_launches() == before > launches
    _, out = run_attention(torch, good, heads, news, 2, max_new=max(news))
    assert torch.equal(out, want)


def test_wait_flag_of_the_device(mq, torch):
    """The device's flag, raised as any tensor-core kernel raises it, fails the next attention before its launch."""
    import ctypes as C

    from cuda.bindings import runtime as rt

    b = Batch(mq, torch, [50], 1, 32, 16, seed=1)
    _, want = run_attention(torch, b, 2, [1], 1, max_new=1)
    flag = C.c_void_p()
    assert mq.lib().mq_device_error_flag(0, C.byref(flag)) == 0
    assert int(rt.cudaMemset(flag.value, 1, 4)[0]) == 0
    torch.cuda.synchronize()
    with pytest.raises(mq.MQError) as info:
        run_attention(torch, b, 2, [1], 1, max_new=1)
    assert info.value.code == mq._lib.MQ_ERR_TIMEOUT
    assert torch.equal(run_attention(torch, b, 2, [1], 1, max_new=1)[1], want)


def _shared(mq, torch, n, length, kv, hd, k, v):
    """n requests over the same `length` cached tokens: (cache, tables)."""
    page = 1024
    pages = -(-length // page)
    c = mq.Kv4Cache(1, pages, page, kv, hd)
    c.store(0, k, v, torch.arange(length, dtype=torch.int32, device="cuda"))
    return c, torch.arange(pages, dtype=torch.int32, device="cuda").expand(n, pages).contiguous()


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_long_sums_of_values(mq, torch, hd):
    """Every CTA of the few-row kernel has 131072 tokens of its own and values of one sign: the sums' roundings must not
    add up. One item a CTA; all requests share the pages."""
    length, heads = 131072, 8
    n = 3 * torch.cuda.get_device_properties(0).multi_processor_count
    g = torch.Generator().manual_seed(hd)
    k, v = torch.randn(length, 1, hd, generator=g) * 2, 1 + 0.1 * torch.randn(length, 1, hd, generator=g)
    c, tables = _shared(mq, torch, n, length, 1, hd, k.cuda(), v.cuda())
    q = torch.randn(n, heads, hd, generator=g).cuda()
    scale = 0.05 / hd
    out = c.attention(0, q, ints(torch, np.arange(n + 1)), ints(torch, [length] * n), tables, max_new=1, scale=scale)
    hk, hv = (torch.from_numpy(ref_blocks_fast(torch, x)).cuda()[:, 0] for x in (k, v))
    for r in range(0, n, 37):
        qq = q[r:r + 37].double()
        p = torch.softmax(qq @ hk.T * scale, -1)
        size = (qq.abs() @ hk.abs().T).amax(-1) * scale
        rel = 2 * (size * (2 ** -22 + 44 * 2 ** -23) + 2 ** -21) + 256 * 2 ** -23
        tol = rel[..., None] * (p @ hv.abs()) + 2 ** -33 * p.amax(-1)[..., None] * hv.abs().sum(0)
        assert_attention(torch, out[r:r + 37], p @ hv, tol)


@pytest.mark.parametrize("new", [1, 64])
def test_long_sums_of_weights(mq, torch, new):
    """A few strong tokens, and behind them thousands of equal weights whose 24 bits fall between the sum's: added one by
    one, each 4096 of them round the sum up by 5.4e-5 of it. All values are 1, so every output is 1. One item a CTA.

    Both sums are of the same weights p, which enter the one over values as hi + lo, off by 2^-22 of it. Few rows: a
    thread adds 256 weights and a product 64 units between two that are kept, and 32 of these; many rows: 32 and 16
    additions a step, 128 steps. Tensor cores' additions are off by 2^-23, others by 2^-24 of the sum:
    (4 + 256 + 32 + 2 * 64 + 32 + 8) and (4 + 32 + 128 + 2 * 16 + 128 + 8) * 2^-24, 8 for the joins and the quotient."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    length, n, heads = (65536, 3 * sms, 8) if new == 1 else (16384, sms // 2, 4)
    hd, bits = 32, 3.997  # the weights' logarithm below the strong tokens'
    k, v = torch.zeros(length, 1, hd, device="cuda"), torch.ones(length, 1, hd, device="cuda")
    k[[0, 32, 64, 96]] = 1.0  # for each of the few-row kernel's warps
    c, tables = _shared(mq, torch, n, length, 1, hd, k, v)
    q = torch.ones(n * new, heads, hd, device="cuda")
    out = c.attention(0, q, ints(torch, np.arange(n + 1) * new), ints(torch, [length] * n), tables, max_new=new,
                      scale=bits * math.log(2) / hd)
    off = float((out.double() - 1).abs().max())
    assert off <= (460 if new == 1 else 332) * 2 ** -24, off


def test_output_layouts(mq, torch):
    """Outputs whose heads share memory are refused; every layout in which they do not is written."""
    b = Batch(mq, torch, [40, 30], 2, 64, 16, seed=2)
    for rows, heads in ((2, 4), (6, 4), (2, 2)):
        news = [rows // 2] * 2
        q, want = run_attention(torch, b, heads, news, 1, spare=0)
        offsets, lens = ints(torch, [0, news[0], rows]), ints(torch, b.lens)
        memory = torch.empty(200 * 64, device="cuda")
        taken = 0
        for ld in (0, 32, 64, 96, 128, 129, 192, 255, 256, 320, 448, 512):
            for hs in (64, 65, 96, 128, 192, 384, 512):
                at = [i * ld + h * hs for i in range(rows) for h in range(heads)]
                apart = all(abs(x - y) >= 64 for n, x in enumerate(at) for y in at[:n])
                out = memory.as_strided((rows, heads, 64), (ld, hs, 1))
                if apart:
                    memory.fill_(7.0)
                    b.cache.attention(0, q, offsets, lens, b.tables, out=out)
                    assert torch.equal(out, want), (ld, hs)
                    assert int((memory == 7.0).sum()) == memory.numel() - want.numel()
                    taken += 1
                else:
                    with pytest.raises(ValueError, match="overlap"):
                        b.cache.attention(0, q, offsets, lens, b.tables, out=out)
        assert taken > 5


@pytest.mark.parametrize("new", [2, 40])
def test_rows_of_a_refused_request(mq, torch, new):
    """The plan leaves a refused request's length as it was, so the attention takes its rows for its last cached ones (and
    for none where it has fewer): finite rows that mean nothing. The other requests' rows are as ever."""
    lens = [70, 50, 0, 33]
    b = Batch(mq, torch, lens, 2, 64, 16, seed=4, poison=False, extra=12)
    used = set(b.tables.flatten().tolist())
    free = ints(torch, [p for p in range(b.cache.pages) if p not in used])
    tables = torch.cat([b.tables, torch.full((4, 4), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    need = -(-(70 + new) // 16) - 5
    news = [new, new, new, 0]  # pages for the first request only
    plan = mq.PlanPages(ints(torch, lens), ints(torch, news), tables, free, ints(torch, [need]), 16, rows=3 * new + 3)
    assert plan.refused.tolist() == [1 if new == 2 else 2]
    served = [70 + new, 52 if new == 2 else 50, 0, 33]
    assert plan.seq_lens.tolist() == served and plan.n_free.tolist() == [0]
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(3 * new + 3, h, 64, generator=g).cuda() for h in (4, 2, 2))
    b.cache.store(0, k, v, plan.slots)
    out = b.cache.attention(0, q, plan.offsets, plan.seq_lens, tables, max_new=new)
    hk, hv = ([torch.cat([h, torch.from_numpy(ref_blocks_fast(torch, z[r * new:(r + 1) * new].cpu())).cuda()])
               if served[r] > lens[r] else h for r, h in enumerate(held)] for held, z in ((b.hk, k), (b.hv, v)))
    want, tol = ref_attention(torch, q[:3 * new], hk, hv, news, served, 64 ** -0.5)
    assert_attention(torch, out[:3 * new], want, tol)
    assert not out[2 * new:].any()


def test_scores_keep_the_low_parts(mq, torch):
    """Scores of 16 whose last bits are sums of the queries' lo parts: seven sums of just below 2^-19, the step of 32-bit
    numbers there, which one addition each to the score would lose. All operands are exact as hi + lo. What may be lost
    is a step where the score reaches 16, and one where it is rounded: 2 * 2^-19 of a score, half of that times the scale
    of the output, tanh of half the scores' difference. (2^-20 for weights, sums and quotient.)"""
    c = mq.Kv4Cache(1, 1, 16, 1, 128)
    k, v = torch.ones(2, 1, 128, device="cuda"), torch.ones(2, 1, 128, device="cuda")
    k[1, :, :112] = 0.0
    v[1] = -1.0
    c.store(0, k, v, ints(torch, [0, 1]))
    q = torch.ones(1, 32, 128, device="cuda")
    q[..., :112] = 2 ** -12 * (1 + 2 ** -11 * (1 - 2 ** -6))
    scale = 64 * math.log(2)
    out = c.attention(0, q, ints(torch, [0, 1]), ints(torch, [2]), ints(torch, [[0]]), max_new=1, scale=scale)
    want = math.tanh(float(q[0, 0, :112].double().sum()) * scale / 2)
    off = float((out.double() - want).abs().max())
    assert off <= 2 ** -19 * scale + 2 ** -20, off
