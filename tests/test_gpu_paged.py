"""kernels.paged on the GPU against the operators in 64 bits: appending to pages, attention over them in
full and over a window with sinks, and attention behind a shared prefix, at the lengths, masks and
layouts where they can go wrong, and a serving step of all of them together."""

import math

import pytest
import torch

from _paged import Pages, assert_within, attention64, rows_of
from kernels import paged
from kernels.attention import k_from_tiles, k_to_tiles, v_from_tiles, vt_to_tiles
from kernels.sample import token_logprobs

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def q_of(T, nq, hd, dtype, seed=0):
    g = torch.Generator().manual_seed(100 + seed)
    return (1.3 * torch.randn(T, nq, hd, generator=g)).to(dtype)


# ------------------------------------------------------------------------------------------ append
def rope64(x, pos, inv_freq):
    """x [n, heads, hd] (64 bits) turned by pos [n]."""
    a = pos.double()[:, None] * inv_freq.double()
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi = x.double().chunk(2, -1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1), lo.abs() + hi.abs()


def freqs(hd, theta=1e6):
    return 1.0 / (theta ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd))


def check_append(lens, news, nq, nkv, hd, page, dtype, rope_pos=None, rotate=True, cu=True, rows=None, in_place=False,
                 max_pages=None, room=None, seed=0):
    """Appends `news` tokens to sequences of `lens` positions (with them) and checks q, every written slot
    and that nothing else changed."""
    pg = Pages([max(0, n - m) for n, m in zip(lens, news)], nkv, hd, page, dtype, seed=seed, fill=3.0,
               room=room or [max(n, 0) for n in lens], max_pages=max_pages)
    starts = rows_of(news)
    T = rows or starts[-1]
    g = torch.Generator().manual_seed(seed + 50)
    qkv = torch.randn(T, (nq + 2 * nkv) * hd, generator=g).to(dtype)
    inv = freqs(hd) if rotate else None
    before_k, before_v = k_from_tiles(pg.k_pages.cpu()), v_from_tiles(pg.vt_pages.cpu())
    d_qkv = qkv.cuda()
    out = d_qkv.view(T, nq + 2 * nkv, hd)[:, :nq] if in_place else None
    q = paged.paged_append(d_qkv, i32(lens), pg.table, pg.k_pages, pg.vt_pages, None if inv is None else inv.cuda(), nq,
                           cu_seqlens=i32(starts) if cu else None,
                           rope_pos=None if rope_pos is None else rope_pos.cuda(), out=out)
    x = qkv.view(T, nq + 2 * nkv, hd)
    want_k, want_v = before_k.double(), before_v.double()
    slack = torch.zeros_like(want_k)
    half = torch.finfo(dtype).eps / 2
    q = q.cpu()
    for b, (n, m) in enumerate(zip(lens, news)):
        r = torch.arange(starts[b], starts[b + 1])
        p = torch.arange(n - m, n)
        if rotate:
            y, size = rope64(x[r, :nq + nkv], p if rope_pos is None else rope_pos[r], inv)
            size = torch.cat([size, size], -1)
        else:
            y, size = x[r, :nq + nkv].double(), torch.zeros(m, nq + nkv, hd, dtype=torch.float64)
        # one rounding of the result; cos and sin to 2^-22, two products and a sum in fp32
        tol = half * y.abs() + 2.0 ** -21 * size + (2.0 ** -25 if dtype == F16 and rotate else 0)
        assert ((q[r].double() - y[:, :nq]).abs() <= tol[:, :nq]).all(), f"q of sequence {b}"
        for i in range(m):
            t = int(p[i])
            if t < 0 or t >= pg.table.shape[1] * page:
                continue
            at = int(pg.table[b, t // page])
            if 0 <= at < want_k.shape[0]:
                want_k[at, :, t % page], slack[at, :, t % page] = y[i, nq:], tol[i, nq:]
                want_v[at, :, t % page] = x[r[i], nq + nkv:].double()
    got_k, got_v = k_from_tiles(pg.k_pages.cpu()).double(), v_from_tiles(pg.vt_pages.cpu()).double()
    assert ((got_k - want_k).abs() <= slack).all()
    assert torch.equal(got_v, want_v)
    if in_place:  # the k and v columns and the rows behind the batch keep their values
        assert torch.equal(d_qkv.view(T, nq + 2 * nkv, hd)[:, nq:].cpu(), x[:, nq:])
    return pg


@pytest.mark.parametrize("dtype,hd,nq,nkv,page", [(F16, 128, 12, 2, 64), (BF16, 128, 32, 8, 32), (F16, 64, 14, 2, 96),
                                                  (BF16, 64, 16, 16, 128), (F16, 128, 1, 1, 32)])
@pytest.mark.parametrize("lens", [[1], [33, 1, 64, 100], [500, 32, 31, 65, 7, 1, 90, 96, 97]])
def test_append_one_token(dtype, hd, nq, nkv, page, lens):
    check_append(lens, [1] * len(lens), nq, nkv, hd, page, dtype, cu=False)


@pytest.mark.parametrize("dtype,hd,nq,nkv,page", [(F16, 128, 12, 2, 64), (BF16, 64, 6, 2, 32)])
@pytest.mark.parametrize("lens,news", [([1], [1]), ([70], [70]), ([100, 40, 31, 200], [31, 40, 1, 64]),
                                       ([64, 0, 5, 97, 33], [32, 0, 5, 97, 2]), ([300, 129], [255, 128]),
                                       ([32] * 40, [1] * 40), ([63, 63], [31, 33])])
def test_append_ragged(dtype, hd, nq, nkv, page, lens, news):
    """Chunks that begin and end inside the new tokens, sequences without new tokens, whole chunks."""
    check_append(lens, news, nq, nkv, hd, page, dtype)


@pytest.mark.parametrize("cu", [False, True])
def test_append_positions_apart_from_the_cache(cu):
    """rope_pos far away (a 32-bit angle would be off by 0.06 radians at 10^6), and beyond 32 bits."""
    pos = torch.tensor([1_000_000, 0, 131_071, 2 ** 33 + 5])
    check_append([5, 40, 64, 65], [1, 1, 1, 1], 4, 2, 128, 32, F16, rope_pos=pos, cu=cu)


@pytest.mark.parametrize("cu", [False, True])
def test_append_without_rotation_is_a_copy(cu):
    check_append([5, 40, 64], [1, 1, 1], 4, 4, 64, 32, BF16, rotate=False, cu=cu)


@pytest.mark.parametrize("cu", [False, True])
def test_append_in_place(cu):
    check_append([5, 40, 64], [1, 1, 1], 8, 2, 128, 32, F16, cu=cu, in_place=True, rows=5)


@pytest.mark.parametrize("cu", [False, True])
def test_append_where_there_is_no_page(cu):
    """Positions below 0 (kv_lens below the new tokens), past the table, and on absent pages: q is turned,
    nothing is written."""
    check_append([0, 70, 40], [1, 1, 1], 4, 2, 128, 32, F16, cu=cu, room=[0, 64, 32], max_pages=2)
    if cu:
        check_append([10, 70, 40], [30, 50, 33], 4, 2, 128, 32, F16, room=[10, 64, 32], max_pages=2)


def test_append_page_ids_outside_the_pool():
    pg = Pages([40, 40], 2, 128, 32, F16, fill=3.0)
    pg.table[0, 1], pg.table[1, 1] = 10 ** 6, -7
    before = pg.k_pages.clone(), pg.vt_pages.clone()
    qkv = torch.randn(2, 8 * 128, device="cuda").half()
    paged.paged_append(qkv, i32([40, 40]), pg.table, pg.k_pages, pg.vt_pages, freqs(128).cuda(), 4)
    assert torch.equal(before[0], pg.k_pages) and torch.equal(before[1], pg.vt_pages)


def test_append_rows_behind_the_batch_and_strides():
    """A padded batch: rows behind the last sequence keep their values; qkv and out strided; pages of a
    pool that holds two layers."""
    nq, nkv, hd, page = 4, 2, 128, 32
    pool_k = torch.full((5, 2) + paged.k_pages_shape(1, nkv, page, hd)[1:], 3.0, dtype=F16, device="cuda")
    pool_v = torch.full((5, 2) + paged.vt_pages_shape(1, nkv, page, hd)[1:], 3.0, dtype=F16, device="cuda")
    wide = torch.randn(6, 2 * (nq + 2 * nkv) * hd, device="cuda").half()
    qkv = wide[:, :(nq + 2 * nkv) * hd]
    big = torch.full((6, nq + 3, hd), 9.0, dtype=F16, device="cuda")
    table = i32([[0], [3], [4]])
    for cu in (None, i32([0, 1, 2, 3])):
        big.fill_(9.0)
        q = paged.paged_append(qkv, i32([7, 8, 9]), table, pool_k[:, 1], pool_v[:, 1], freqs(hd).cuda(), nq,
                               cu_seqlens=cu, out=big[:, :nq])
        assert q.data_ptr() == big.data_ptr()
        assert (big[3:] == 9.0).all() and (big[:, nq:] == 9.0).all() and not (big[:3, :nq] == 9.0).any(-1).any()
        assert (pool_k[:, 0] == 3.0).all() and (pool_v[:, 0] == 3.0).all()
        assert torch.equal(v_from_tiles(pool_v[:, 1])[3, :, 7], qkv.view(6, -1)[1, (nq + nkv) * hd:].view(nkv, hd))


def test_append_past_four_gibibytes():
    """Pages whose offsets pass 32 bits, in bytes and in elements."""
    nq, nkv, hd, page = 2, 2, 128, 512
    pages = 20000  # 2.6e9 elements of K, 5.2 GB
    k = torch.empty(paged.k_pages_shape(pages, nkv, page, hd), dtype=F16, device="cuda")
    vt = torch.empty(paged.vt_pages_shape(pages, nkv, page, hd), dtype=F16, device="cuda")
    table = i32([[pages - 1], [17000], [3]])
    for t in (k, vt):
        t[table[:, 0].long()] = 0
    qkv = torch.randn(3, (nq + 2 * nkv) * hd, device="cuda").half()
    lens = i32([300, 2, 1])
    paged.paged_append(qkv, lens, table, k, vt, None, nq)
    v_new = qkv.view(3, -1, hd)[:, nq + nkv:]
    for b, n in enumerate([300, 2, 1]):
        page_id = int(table[b, 0])
        assert torch.equal(v_from_tiles(vt[page_id])[:, n - 1], v_new[b])
        assert torch.equal(k_from_tiles(k[page_id])[:, n - 1], qkv.view(3, -1, hd)[b, nq:nq + nkv])
    q = q_of(3, nq, hd, F16).cuda()
    one = paged.paged_attention(q, i32([1, 1, 1]), i32([[pages - 1], [17000], [3]]), k, vt, 0.1)
    first = torch.stack([v_from_tiles(vt[int(p)])[:, 0] for p in table[:, 0]])
    assert torch.equal(one, first)  # one position: its v


# --------------------------------------------------------------------------------------- attention
def check_attention(lens, news, nq, nkv, hd, page, dtype, window=0, sinks=0, cu=True, rows=None, max_q="given", seed=0,
                    prefix=0, fill=float("nan")):
    """lens: positions with the new tokens (past the prefix, where there is one)."""
    pg = Pages([max(n, 0) for n in lens], nkv, hd, page, dtype, seed=seed, fill=fill, prefix=prefix)
    starts = rows_of(news)
    T = rows or max(1, starts[-1])
    q = q_of(T, nq, hd, dtype, seed)
    scale = hd ** -0.5
    out = torch.full((T, nq, hd), 7.0, dtype=dtype, device="cuda")
    kw = dict(cu_seqlens=i32(starts) if cu else None, max_q=max(1, max(news)) if max_q == "given" else max_q, out=out)
    kv = i32([n + prefix for n in lens])
    if prefix:
        table = torch.cat([torch.full((len(lens), prefix // page), 10 ** 6, dtype=torch.int32, device="cuda"), pg.table], 1)
        got = paged.shared_prefix_attention(q.cuda(), kv, table, i32(pg.prefix_ids), prefix, pg.k_pages, pg.vt_pages, scale, **kw)
    else:
        got = paged.paged_attention(q.cuda(), kv, pg.table, pg.k_pages, pg.vt_pages, scale, window=window, sinks=sinks, **kw)
    assert got is out
    for b, (n, m) in enumerate(zip(lens, news)):
        r = slice(starts[b], starts[b + 1])
        k, v = pg.k[b], pg.v[b]
        if prefix:
            k, v = torch.cat([pg.pk, k]), torch.cat([pg.pv, v])
        ref, bound = attention64(q[r], k, v, scale, [prefix + n - m + i for i in range(m)], window, sinks)
        assert_within(got[r], ref, bound, f"sequence {b}")
    assert (out[starts[-1]:] == 7.0).all()


LAYOUTS = [(F16, 128, 12, 2, 64), (BF16, 128, 32, 8, 32), (F16, 64, 14, 2, 96), (BF16, 64, 16, 16, 128), (F16, 128, 20, 1, 32)]


@pytest.mark.parametrize("dtype,hd,nq,nkv,page", LAYOUTS)
@pytest.mark.parametrize("lens", [[1], [33, 1, 64, 0, 100], [700, 32, 31, 65, 7, 2000, 90], [5000]])
def test_attention_one_token(dtype, hd, nq, nkv, page, lens):
    check_attention(lens, [1] * len(lens), nq, nkv, hd, page, dtype, cu=False)


@pytest.mark.parametrize("dtype,hd,nq,nkv,page", LAYOUTS)
@pytest.mark.parametrize("lens,news", [([70], [70]), ([100, 40, 31, 200], [31, 40, 1, 64]),
                                       ([64, 0, 5, 97, 33, 12], [32, 0, 5, 97, 2, 0]), ([400], [3]), ([260, 900], [130, 140])])
def test_attention_ragged(dtype, hd, nq, nkv, page, lens, news):
    check_attention(lens, news, nq, nkv, hd, page, dtype)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 33), (100, 70), (5000, 9), (64, 1000), (0, 5)])
@pytest.mark.parametrize("dtype,hd,nq,nkv,page", LAYOUTS[:3])
def test_attention_window(dtype, hd, nq, nkv, page, window, sinks):
    check_attention([1, 300, 97, 640], [1] * 4, nq, nkv, hd, page, dtype, window, sinks, cu=False)
    check_attention([10, 300, 97, 640], [10, 70, 97, 5], nq, nkv, hd, page, dtype, window, sinks)


@pytest.mark.parametrize("window,sinks", [(1024, 0), (1024, 4), (1500, 40), (2000, 100)])
@pytest.mark.parametrize("dtype,hd,nq,nkv,page", LAYOUTS[:3])
def test_attention_window_over_ranges(dtype, hd, nq, nkv, page, window, sinks):
    """Windows whose chunks, with those of the sinks a gap before them, are cut into several ranges that a
    merge joins: one token per sequence, and a few; short sequences beside them."""
    lens = [6000, 300, 3100, 1, 4500]
    check_attention(lens, [1] * 5, nq, nkv, hd, page, dtype, window, sinks, cu=False)
    check_attention(lens, [3, 2, 1, 1, 2], nq, nkv, hd, page, dtype, window, sinks)


@pytest.mark.parametrize("window,sinks", [(2000, 40), (1300, 5)])
def test_attention_window_over_ranges_of_many_sequences(window, sinks):
    """The same where the ranges are found in a launch of their own."""
    lens = [(37 * i) % 90 + 1 for i in range(100)]
    lens[3], lens[50], lens[99] = 5000, 3300, 2500
    check_attention(lens, [1] * 100, 4, 2, 128, 32, F16, window, sinks, cu=False)
    check_attention(lens, [min(n, 1 + i % 3) for i, n in enumerate(lens)], 8, 2, 128, 32, BF16, window, sinks)


@pytest.mark.parametrize("new", [200, 600])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 3), (40, 100)])
@pytest.mark.parametrize("dtype,hd,nq,nkv,page", [(F16, 128, 4, 2, 64), (BF16, 64, 3, 1, 32)])
def test_attention_prompts(dtype, hd, nq, nkv, page, window, sinks, new):
    """Blocks of many rows whose masks begin and end inside them, behind cached positions and from 0."""
    check_attention([new, new + 333, 50], [new, new - 31, 50], nq, nkv, hd, page, dtype, window, sinks)


def test_attention_many_sequences():
    """More sequences than a wave has lanes, with empty ones among them."""
    lens = [(37 * i) % 300 for i in range(150)]
    check_attention(lens, [1] * 150, 4, 2, 64, 32, F16, cu=False)
    news = [min(n, i % 4) for i, n in enumerate(lens)]
    check_attention(lens, news, 4, 2, 64, 32, F16)


@pytest.mark.parametrize("prefix", [0, 128])
@pytest.mark.parametrize("count", [257, 1100])
def test_attention_ranges_of_very_many_sequences(count, prefix):
    """Ranges that one workgroup finds for the batch: short sequences, empty ones, and a few of many ranges."""
    lens = [(37 * i) % 90 for i in range(count)]
    lens[3] = lens[count // 2] = lens[-1] = 1500
    check_attention([max(n, 1) for n in lens], [1] * count, 4, 2, 64, 32, F16, cu=False, prefix=prefix)
    check_attention(lens, [min(n, i % 3) for i, n in enumerate(lens)], 4, 2, 64, 32, BF16, prefix=prefix)


@pytest.mark.parametrize("prefix", [0, 64])
def test_attention_long_contexts_beside_prompts(prefix):
    """A batch that decodes and prefills at once: one token after many positions beside whole prompts."""
    check_attention([9000, 300, 17000, 40], [1, 300, 2, 1], 4, 1, 64, 32, F16, prefix=prefix)


def test_attention_positions_below_zero():
    """kv_lens below the new tokens' count: the tokens at positions below 0 give zeros."""
    pg = Pages([10, 3], 2, 128, 32, F16)
    q = q_of(20, 4, 128, F16)
    for max_q in (12, None):
        got = paged.paged_attention(q.cuda(), i32([10, 3]), pg.table, pg.k_pages, pg.vt_pages, 0.1, cu_seqlens=i32([0, 12, 20]),
                                    max_q=max_q)
        for b, (lo, hi, n) in enumerate([(0, 12, 10), (12, 20, 3)]):
            ref, bound = attention64(q[lo:hi], pg.k[b], pg.v[b], 0.1, [n - (hi - lo) + i for i in range(hi - lo)])
            assert_within(got[lo:hi], ref, bound)
        assert (got[:2] == 0).all() and (got[12:17] == 0).all()


@pytest.mark.parametrize("news", [[1, 1, 1], [200, 3, 90]])
def test_attention_absent_pages(news):
    """Ids outside the pool hide their positions, as does a table shorter than the sequence."""
    pg = Pages([300, 100, 96], 2, 64, 32, BF16, max_pages=10)
    table = pg.table.clone()
    table[0, 2], table[0, 5], table[1, 3], table[2, :3] = -1, 10 ** 6, 2 ** 30, -5
    q = q_of(sum(news), 6, 64, BF16)
    cu = rows_of(news)
    for max_pages, lens in ((10, [300, 100, 96]), (4, [300, 100, 96])):
        got = paged.paged_attention(q.cuda(), i32(lens), table[:, :max_pages], pg.k_pages, pg.vt_pages, 0.125,
                                    cu_seqlens=None if max(news) == 1 else i32(cu), max_q=max(news))
        for b, n in enumerate(lens):
            at = torch.arange(n)
            ok = torch.zeros(n, dtype=torch.bool)
            for i in range(n):
                if i < max_pages * 32:
                    ok[i] = 0 <= int(table[b, i // 32]) < pg.k_pages.shape[0]
            ref, bound = attention64(q[cu[b]:cu[b + 1]], pg.k[b], pg.v[b], 0.125, (at[-news[b]:]).tolist(), present=ok)
            assert_within(got[cu[b]:cu[b + 1]], ref, bound, f"sequence {b}")
        assert (got[cu[2]:cu[3]] == 0).all()


def test_attention_max_q_bounds_what_is_computed():
    """Rows past max_q of a sequence are not computed, the others are."""
    pg = Pages([50, 60], 2, 64, 32, F16)
    q = q_of(24, 4, 64, F16)
    out = torch.full((24, 4, 64), 7.0, dtype=F16, device="cuda")
    paged.paged_attention(q.cuda(), i32([50, 60]), pg.table, pg.k_pages, pg.vt_pages, 0.125, cu_seqlens=i32([0, 20, 24]),
                          max_q=5, out=out)
    for b, lo, n, first in ((0, 0, 5, 30), (1, 20, 4, 56)):
        ref, bound = attention64(q[lo:lo + n], pg.k[b], pg.v[b], 0.125, [first + i for i in range(n)])
        assert_within(out[lo:lo + n], ref, bound)
    assert (out[5:20] == 7.0).all()


@pytest.mark.parametrize("news", [[1, 1], [150, 33]])
def test_attention_strides(news):
    """q a view of the projection's rows, out a view of wider rows, pages of a two-layer pool, a table that
    is a slice of a wider one."""
    nq, nkv, hd, page = 4, 2, 128, 32
    pg = Pages([200, 150], nkv, hd, page, F16)
    n = pg.k_pages.shape[0]
    pool_k = torch.full((n, 2) + tuple(pg.k_pages.shape[1:]), float("nan"), dtype=F16, device="cuda")
    pool_v = torch.full((n, 2) + tuple(pg.vt_pages.shape[1:]), float("nan"), dtype=F16, device="cuda")
    pool_k[:, 1], pool_v[:, 1] = pg.k_pages, pg.vt_pages
    T = sum(news)
    wide = q_of(T, nq + 4, hd, F16).cuda()
    out = torch.full((T, nq + 3, hd), 7.0, dtype=F16, device="cuda")
    table = torch.cat([pg.table, pg.table], 1)
    cu = rows_of(news)
    paged.paged_attention(wide[:, :nq], i32([200, 150]), table[:, :pg.table.shape[1]], pool_k[:, 1], pool_v[:, 1], 0.09,
                          cu_seqlens=None if max(news) == 1 else i32(cu), max_q=max(news), out=out[:, :nq])
    for b, L in enumerate([200, 150]):
        ref, bound = attention64(wide[cu[b]:cu[b + 1], :nq].cpu(), pg.k[b], pg.v[b], 0.09,
                                 list(range(L - news[b], L)))
        assert_within(out[cu[b]:cu[b + 1], :nq], ref, bound)
    assert (out[:, nq:] == 7.0).all()


@pytest.mark.parametrize("news", [[1], [40]])
def test_attention_large_scores(news):
    """Scores of both signs up to some hundreds: the maximum is subtracted before the exponential."""
    pg = Pages([400], 1, 64, 32, F16)
    q = 40 * q_of(news[0], 4, 64, F16)
    got = paged.paged_attention(q.cuda(), i32([400]), pg.table, pg.k_pages, pg.vt_pages, 0.125,
                                cu_seqlens=None if news == [1] else i32([0, news[0]]))
    ref, bound = attention64(q, pg.k[0], pg.v[0], 0.125, list(range(400 - news[0], 400)))
    assert_within(got, ref, bound)


def _one_pool(k, v, page):
    """Pages of one sequence's k, v [L, 1, hd] in order, and their table."""
    L, _, hd = k.shape
    k, v = (t.view(L // page, page, 1, hd).transpose(1, 2).contiguous() for t in (k, v))
    return k_to_tiles(k).cuda(), vt_to_tiles(v).cuda(), torch.arange(L // page, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64)])
def test_attention_of_equal_scores_far_from_zero(dtype, hd):
    """131072 positions of one score, 840, the first half of value 1 and the others of 0: every weight is the
    same, whatever the maximum's product with scale log2 e loses in rounding (here 2^-14 of an exponent, at each
    of a wave's 512 chunks). The result is a half: the fp32 sums of 512 chunks and 8 waves, each to half a step of
    2^-24 per term, and one rounding, of which a half of the type's step is 2^-1 eps / 2."""
    B, L, page = 170, 131072, 64
    k, v = torch.zeros(L, 1, hd, dtype=dtype), torch.zeros(L, 1, hd, dtype=dtype)
    k[:, 0, 0], v[:L // 2] = 112.0, 1.0
    k, v, table = _one_pool(k, v, page)
    q = torch.zeros(B, 1, hd, dtype=dtype, device="cuda")
    q[:, 0, 0] = 62.5  # 7000 exactly
    got = paged.paged_attention(q, i32([L] * B), table.expand(B, -1).contiguous(), k, v, 0.12)
    assert ((got.double() - 0.5).abs() <= torch.finfo(dtype).eps / 4 + (2 * 512 + 64) * 2.0 ** -24).all(), got.double().sub(0.5).abs().max()


@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("prefix", [False, True])
def test_attention_rows_beside_a_rising_one(prefix, dtype, hd):
    """Two heads whose rows share the matrix cores' tiles: of head 0 every score is 840, of head 1 they rise by
    more than 8 powers of two per chunk, so that its rows are rescaled at each of 511 chunks. Head 0's sums must
    not change with them. Bounds as above; head 1 sees the last chunk's positions with equal weights."""
    B, new, L, page, scale = 86, 64, 16384, 64, 0.12
    if prefix:
        B, new = 64, 1
    k, v = torch.zeros(L, 1, hd, dtype=dtype), torch.zeros(L, 1, hd, dtype=dtype)
    k[:, 0, 0], v[:L // 2] = 112.0, 1.0
    rise = torch.arange(L) // 32 % 256  # (twice from 0 on: bf16 holds whole numbers to 256)
    k[:, 0, 1], k[:, 0, 2] = rise.to(dtype), (torch.arange(L) // 8192 * 256).to(dtype)
    k, v, table = _one_pool(k, v, page)
    q = torch.zeros(B * new, 2, hd, dtype=dtype, device="cuda")
    q[:, 0, 0] = 62.5
    q[:, 1, 1], q[:, 1, 2] = 60.0, 60.0  # 60 * 0.12 * log2 e = 10.4 per chunk
    tables = table.expand(B, -1).contiguous()
    if prefix:
        kv = i32([L] * B)
        got = paged.shared_prefix_attention(q, kv, tables, table, L, k, v, scale)
        at = torch.full((B,), L - 1, device="cuda")
    else:
        kv = i32([L] * B)
        got = paged.paged_attention(q, kv, tables, k, v, scale, cu_seqlens=i32([b * new for b in range(B + 1)]), max_q=new)
        at = torch.arange(B * new, device="cuda") % new + L - new
    want = (L / 2 / (at + 1).double())[:, None]
    assert ((got[:, 0].double() - want).abs() <= torch.finfo(dtype).eps / 2 * want + (2 * 512 + 64) * 2.0 ** -24).all(), \
        (got[:, 0].double() - want).abs().max()
    assert (got[:, 1] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("power", [10, 25, 40])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("hd,new,prefix", [(128, 1, 0), (64, 1, 128), (128, 1, 256), (64, 40, 0), (128, 100, 0), (128, 100, 64)])
def test_attention_of_scores_of_any_size(hd, new, prefix, sign, power, dtype):
    """Scores of 50 sizes, 2^power times 0.12 or half of that apart: what has the largest has all the weight, in
    equal parts, also where the scores' products with log2 e are rounded by whole powers of two."""
    L, page = 1600, 64
    g = torch.Generator().manual_seed(power + new)
    order = torch.randperm(L, generator=g) % 50
    steps = order + 1 if sign > 0 else order - 50
    k, v = torch.zeros(L, 1, hd, dtype=dtype), torch.randn(L, 1, hd, generator=g).to(dtype)
    k[:, 0, 0] = (steps * 2.0 ** (min(power, 25) - 15)).to(dtype)  # exact, below fp16's largest
    scale = 0.12 * 2.0 ** (power - min(power, 25))
    kk, vv, table = _one_pool(k, v, page)
    q = torch.zeros(new, 2, hd, dtype=dtype)
    q[:, 0, 0], q[:, 1, 0] = 2.0 ** 15, 2.0 ** 14
    kw = dict(cu_seqlens=None if new == 1 else i32([0, new]))
    if prefix:
        got = paged.shared_prefix_attention(q.cuda(), i32([L]), table[None], table[:prefix // page].clone(), prefix, kk, vv, scale, **kw)
    else:
        got = paged.paged_attention(q.cuda(), i32([L]), table[None], kk, vv, scale, **kw)
    half = torch.finfo(dtype).eps / 2
    for i in range(new):
        seen = steps[:L - new + i + 1]
        best = v[:len(seen), 0][seen == seen.max()].double()
        # equal weights (the others' are below e^-61): their fp32 sum, one rounding
        bound = half * best.mean(0).abs() + (len(best) + 64) * 2.0 ** -23 * best.abs().mean(0) + 2.0 ** -25
        assert_within(got[i], best.mean(0).expand(2, -1), bound.expand(2, -1), f"token {i}")


# ---------------------------------------------------------------------------------- shared prefix
@pytest.mark.parametrize("prefix", [0, 4096])
@pytest.mark.parametrize("new", [1, 48])
def test_attention_many_small_weights(new, prefix):
    """fp16: one position whose weight is 2^25 times that of each of 8191 others, which alone have values.
    Their numerators e^-17.41 = 2^-25.1 are below the type's least half step; the answer is their sum. Held
    times 2^7 they are 2^-18.1, off by half of fp16's step of 2^-24 there: by 2^-6.9 of themselves."""
    L, hd, page = 8192, 64, 64
    k = torch.zeros(1, 1, L, hd, dtype=F16)
    v = torch.ones(1, 1, L, hd, dtype=F16)
    k[0, 0, 5, 0], v[0, 0, 5] = 4.3515625, 0.0
    k, v = k.view(1, L // page, page, hd).transpose(0, 1), v.view(1, L // page, page, hd).transpose(0, 1)
    table = torch.arange(L // page, dtype=torch.int32).cuda()[None]
    q = torch.zeros(new, 4, hd, dtype=F16)
    q[:, :, 0] = 4.0
    args = (k_to_tiles(k.contiguous()).cuda(), vt_to_tiles(v.contiguous()).cuda(), 1.0)
    cu = None if new == 1 else i32([0, new])
    if prefix:
        got = paged.shared_prefix_attention(q.cuda(), i32([L]), table, table[0, :prefix // page].clone(), prefix, *args, cu_seqlens=cu)
    else:
        got = paged.paged_attention(q.cuda(), i32([L]), table, *args, cu_seqlens=cu)
    for i in range(new):
        w = (L - new + i) * math.exp(-4.0 * 4.3515625)
        ref = w / (1 + w)
        assert ((got[i].double().cpu() - ref).abs() <= ref * (2.0 ** -6.9 + 2.0 ** -10) + 2.0 ** -25).all(), (i, got[i, 0, 0].item(), ref)


@pytest.mark.parametrize("dtype,hd", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("prefix", [0, 32])
@pytest.mark.parametrize("news", [[1, 1, 1], [2, 5, 3], [60, 3, 200]])
def test_attention_of_nan(news, prefix, dtype, hd):
    """A NaN in a row of q makes that row's head NaN, one in a k that is seen every row that sees it, and
    no other row."""
    lens, nq, nkv, page = [700, 64, 300], 6, 2, 32
    pg = Pages(lens, nkv, hd, page, dtype)
    q, cu = q_of(sum(news), nq, hd, dtype), rows_of(news)
    at = lens[0] - (news[0] + 1) // 2  # seen by half of the first sequence's rows
    pg.k[0][at, 1, 3] = float("nan")
    k = k_from_tiles(pg.k_pages.cpu())
    k[pg.table[0, at // page].item(), 1, at % page, 3] = float("nan")
    q[cu[1] + news[1] // 2, 0, 5] = float("nan")
    args = (k_to_tiles(k).cuda(), pg.vt_pages, 0.125)
    cus = None if max(news) == 1 else i32(cu)
    if prefix:  # (each sequence alone: the pages differ)
        got = torch.cat([paged.shared_prefix_attention(q[cu[b]:cu[b + 1]].cuda(), i32([n]), pg.table[b:b + 1], pg.table[b, :1].clone(),
                                                       prefix, *args, cu_seqlens=cus if cus is None else i32([0, news[b]]))
                         for b, n in enumerate(lens)])
    else:
        got = paged.paged_attention(q.cuda(), i32(lens), pg.table, *args, cu_seqlens=cus, max_q=max(news))
    got = got.cpu()
    for b, n in enumerate(lens):
        ref, bound = attention64(q[cu[b]:cu[b + 1]], pg.k[b], pg.v[b], 0.125, [n - news[b] + i for i in range(news[b])])
        bad = torch.isnan(ref)
        mine = got[cu[b]:cu[b + 1]]
        assert (torch.isnan(mine) == bad).all(), b
        assert_within(torch.where(bad, 0, mine), torch.where(bad, 0, ref), torch.where(bad, 1, bound))


@pytest.mark.parametrize("dtype,hd", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("news", [[1, 1], [60, 200]])
def test_attention_of_infinite_scores(news, dtype, hd):
    """An infinity in a k makes the rows whose q gives it +inf NaN, as the formula's inf - inf is, and has no
    weight in the rows that it gives -inf, the other positions' results unchanged."""
    lens, nq, nkv, page = [700, 300], 6, 2, 32
    pg = Pages(lens, nkv, hd, page, dtype)
    q, cu = q_of(sum(news), nq, hd, dtype), rows_of(news)
    k = k_from_tiles(pg.k_pages.cpu())
    at = [333, 299]
    for b, j in enumerate(at):
        k[pg.table[b, j // page].item(), 1, j % page, 3] = float("inf")
    got = paged.paged_attention(q.cuda(), i32(lens), pg.table, k_to_tiles(k).cuda(), pg.vt_pages, 0.125,
                                cu_seqlens=None if max(news) == 1 else i32(cu), max_q=max(news)).cpu()
    for b, n in enumerate(lens):
        mine, rows = got[cu[b]:cu[b + 1]], q[cu[b]:cu[b + 1]]
        where = [n - news[b] + i for i in range(news[b])]
        hit = torch.zeros(rows.shape[:2], dtype=torch.bool)
        hit[:, 3:] = torch.tensor([p >= at[b] for p in where])[:, None]
        nan = hit & (rows[:, :, 3] > 0)
        assert (mine.isnan() == nan[:, :, None]).all(), b
        without = torch.ones(n, dtype=torch.bool)
        without[at[b]] = False
        for present, choose in ((None, ~hit), (without, hit & ~nan)):
            ref, bound = attention64(rows, pg.k[b], pg.v[b], 0.125, where, present=present)
            assert_within(mine[choose], ref[choose], bound[choose], f"sequence {b}")


@pytest.mark.parametrize("dtype,hd,nq,nkv,page", LAYOUTS)
@pytest.mark.parametrize("prefix_pages", [1, 7])
@pytest.mark.parametrize("lens", [[1], [33, 1, 64, 5, 100], [700, 32, 31, 65, 7, 90] * 4])
def test_prefix_one_token(dtype, hd, nq, nkv, page, prefix_pages, lens):
    check_attention(lens, [1] * len(lens), nq, nkv, hd, page, dtype, cu=False, prefix=prefix_pages * page)


@pytest.mark.parametrize("dtype,hd,nq,nkv,page", LAYOUTS[:3])
@pytest.mark.parametrize("lens,news", [([70], [70]), ([100, 40, 31, 200], [31, 40, 1, 64]), ([5, 9, 33], [5, 0, 2])])
def test_prefix_ragged(dtype, hd, nq, nkv, page, lens, news):
    check_attention(lens, news, nq, nkv, hd, page, dtype, prefix=4 * page)


def test_prefix_longer_than_a_sequence():
    """Sequences that end inside the prefix see their part of it; padding (kv_lens 0) sees nothing."""
    prefix, page = 256, 64
    pg = Pages([20, 0, 0, 0], 2, 64, page, F16, prefix=prefix)
    kv = [276, 100, 256, 0]
    q = q_of(4, 4, 64, F16)
    table = torch.cat([torch.full((4, prefix // page), -1, dtype=torch.int32, device="cuda"), pg.table], 1)
    got = paged.shared_prefix_attention(q.cuda(), i32(kv), table, i32(pg.prefix_ids), prefix, pg.k_pages, pg.vt_pages, 0.125)
    for b, n in enumerate(kv):
        ref, bound = attention64(q[b:b + 1], torch.cat([pg.pk, pg.k[b]]), torch.cat([pg.pv, pg.v[b]]), 0.125, [n - 1])
        assert_within(got[b:b + 1], ref, bound, f"sequence {b}")
    assert (got[3] == 0).all()


def test_prefix_long_batch():
    """A prefix of many ranges for more rows than a block holds."""
    check_attention([(7 * i) % 90 + 1 for i in range(70)], [1] * 70, 8, 2, 128, 64, BF16, cu=False, prefix=2048)


# ------------------------------------------------------------------------- streams, graphs, together
def _setup(seed, lens, news, nq=8, nkv=2, hd=128, page=32, dtype=F16):
    pg = Pages(lens, nkv, hd, page, dtype, seed=seed)
    cu = rows_of(news)
    return pg, q_of(cu[-1], nq, hd, dtype, seed).cuda(), i32(lens), i32(cu)


def test_attention_on_another_stream():
    pg, q, kv, cu = _setup(3, [900, 40], [1, 1])
    want = paged.paged_attention(q, kv, pg.table, pg.k_pages, pg.vt_pages, 0.09)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [paged.paged_attention(q, kv, pg.table, pg.k_pages, pg.vt_pages, 0.09) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want, g) for g in got)


def test_two_graphs_at_new_lengths():
    """Two captured calls (workspaces of their own) replayed in turn and on two streams, with eager calls
    between, their lengths changed on the device between replays."""
    cases = []
    for seed, (lens, news, window) in enumerate([([900, 700, 1300], [1, 1, 1], 0), ([500, 800], [40, 7], 200)]):
        pg, q, kv, cu = _setup(seed, lens, news)
        kw = dict(cu_seqlens=None if max(news) == 1 else cu, max_q=max(news), window=window, sinks=4 if window else 0)

        def call(q=q, kv=kv, pg=pg, kw=kw):
            return paged.paged_attention(q, kv, pg.table, pg.k_pages, pg.vt_pages, 0.09, **kw)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        cases.append((graph, out, kv, lens, call))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        want = []
        for graph, out, kv, lens, call in cases:
            kv.copy_(i32([max(50, n - 37 * step) for n in lens]))
            want.append(call())
        torch.cuda.synchronize()
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                c[0].replay()
        torch.cuda.synchronize()
        for w, c in zip(want, cases):
            assert torch.equal(w, c[1]), f"replay {step}"


def test_serving_steps():
    """Prompts of a ragged batch appended behind a shared prefix, then decode steps of the batch (append,
    windowed and full attention, attention behind the prefix, log probabilities) against 64 bits; the
    steps' kernels captured once and replayed with new lengths."""
    nq, nkv, hd, page, dtype, prefix = 8, 2, 64, 32, F16, 64
    width = (nq + 2 * nkv) * hd
    news, steps, scale = [40, 3, 70], 4, hd ** -0.5
    B = len(news)
    g = torch.Generator().manual_seed(9)
    pool = 30
    k_pages = torch.full(paged.k_pages_shape(pool, nkv, page, hd), float("nan"), dtype=dtype, device="cuda")
    vt_pages = torch.full(paged.vt_pages_shape(pool, nkv, page, hd), float("nan"), dtype=dtype, device="cuda")
    ids = torch.randperm(pool, generator=g).to(torch.int32)
    head = ids[:2].tolist()
    table = torch.full((B, 6), -1, dtype=torch.int32)
    at = 2
    for b, n in enumerate(news):
        need = -(-(n + steps) // page)
        table[b, :2] = torch.tensor(head, dtype=torch.int32)
        table[b, 2:2 + need] = ids[at:at + need]
        at += need
    table = table.cuda()
    inv = freqs(hd).cuda()
    # the prefix, once, as a sequence of its own
    first = torch.randn(prefix, width, generator=g).to(dtype).cuda()
    paged.paged_append(first, i32([prefix]), i32([head]), k_pages, vt_pages, inv, nq, cu_seqlens=i32([0, prefix]))
    # the prompts behind it
    rows = torch.randn(sum(news), width, generator=g).to(dtype).cuda()
    lens = [prefix + n for n in news]
    kv, cu = i32(lens), i32(rows_of(news))
    q = paged.paged_append(rows, kv, table, k_pages, vt_pages, inv, nq, cu_seqlens=cu)

    def read(b, n):
        k = torch.cat([k_from_tiles(k_pages[int(p)]).transpose(0, 1) for p in table[b, :-(-n // page)]])[:n].cpu()
        v = torch.cat([v_from_tiles(vt_pages[int(p)]).transpose(0, 1) for p in table[b, :-(-n // page)]])[:n].cpu()
        return k, v

    full = paged.paged_attention(q, kv, table, k_pages, vt_pages, scale, cu_seqlens=cu, max_q=max(news))
    shared = paged.shared_prefix_attention(q, kv, table, i32(head), prefix, k_pages, vt_pages, scale, cu_seqlens=cu, max_q=max(news))
    for b, n in enumerate(news):
        r = slice(rows_of(news)[b], rows_of(news)[b + 1])
        k, v = read(b, lens[b])
        ref, bound = attention64(q[r].cpu(), k, v, scale, list(range(prefix, lens[b])))
        assert_within(full[r], ref, bound)
        assert_within(shared[r], ref, bound)
    # decode: one graph of a step, replayed
    x = torch.zeros(B, width, dtype=dtype, device="cuda")
    tokens = torch.zeros(B, dtype=torch.int64, device="cuda")
    head_w = torch.randn(nq * hd, 501, generator=g).to(dtype).cuda()

    def step():
        kv.add_(1)
        q = paged.paged_append(x, kv, table, k_pages, vt_pages, inv, nq)
        a = paged.paged_attention(q, kv, table, k_pages, vt_pages, scale)
        w = paged.paged_attention(q, kv, table, k_pages, vt_pages, scale, window=24, sinks=2)
        s = paged.shared_prefix_attention(q, kv, table, i32_head, prefix, k_pages, vt_pages, scale)
        logits = (a + w + s).reshape(B, -1) @ head_w
        return q, a, w, s, logits, token_logprobs(logits, tokens, top=3)

    i32_head = i32(head)
    x.copy_(torch.randn(B, width, generator=g).to(dtype))
    step()  # eager
    lens = [n + 1 for n in lens]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, a, w, s, logits, answer = step()
    for i in range(steps - 1):
        x.copy_(torch.randn(B, width, generator=g).to(dtype))
        tokens.copy_(torch.randint(0, 501, (B,), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        lens = [n + 1 for n in lens]
        assert kv.tolist() == lens
        for b in range(B):
            k, v = read(b, lens[b])
            ref, bound = attention64(q[b:b + 1].cpu(), k, v, scale, [lens[b] - 1])
            assert_within(a[b:b + 1], ref, bound)
            assert_within(s[b:b + 1], ref, bound)
            ref, bound = attention64(q[b:b + 1].cpu(), k, v, scale, [lens[b] - 1], 24, 2)
            assert_within(w[b:b + 1], ref, bound)
        lp = torch.log_softmax(logits.double(), -1)
        assert (answer.logprob.double() - lp.gather(1, tokens[:, None])[:, 0]).abs().max() <= 2.0 ** -16 * (1 + lp.abs().max())
        assert torch.equal(answer.top_ids, torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :3])
