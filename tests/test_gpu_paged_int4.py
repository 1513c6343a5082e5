"""kernels.paged_int4 on the GPU: appended bytes and values read back against the format's definition, to the bit, and
attention over the pages against 64 bits, at the lengths, masks, values and layouts where they can go wrong, and a serving step
of all of them together."""

import pytest
import torch

from _paged import assert_within, rows_of
from _paged_int4 import Pages4, attention64, get, put, quantise, values
from kernels.paged_int4 import kv_int4_shape, paged_append_int4, paged_attention_int4, paged_read_int4

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
LAYOUTS = [(F16, 128, 128, 12, 2, 64), (BF16, 128, 64, 32, 8, 32), (F16, 128, 32, 20, 1, 32), (F16, 64, 32, 14, 2, 96),
           (BF16, 64, 64, 16, 16, 128)]  # dtype, hd, group, nq, nkv, page


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def q_of(T, nq, hd, dtype, seed=0):
    g = torch.Generator().manual_seed(100 + seed)
    return (1.3 * torch.randn(T, nq, hd, generator=g)).to(dtype)


def freqs(hd, theta=1e6):
    return 1.0 / (theta ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd))


def same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


# ------------------------------------------------------------------------------------------ append
def rope64(x, pos, inv_freq):
    a = pos.double()[:, None] * inv_freq.double()
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi = x.double().chunk(2, -1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1), torch.cat([lo.abs() + hi.abs()] * 2, -1)


def check_append(lens, news, nq, nkv, hd, group, page, dtype, rope_pos=None, rotate=True, cu=True, rows=None, in_place=False,
                 max_pages=None, room=None, seed=0, x=None):
    """Appends `news` tokens to sequences of `lens` positions (with them) and checks q, the pool's every byte and what is
    read back."""
    pg = Pages4([max(0, n - m) for n, m in zip(lens, news)], nkv, hd, group, page, dtype, seed=seed,
                room=room or [max(n, 0) for n in lens], max_pages=max_pages)
    starts = rows_of(news)
    T = rows or starts[-1]
    if x is None:
        x = torch.randn(T, nq + 2 * nkv, hd, generator=torch.Generator().manual_seed(seed + 50)).to(dtype)
    inv = freqs(hd) if rotate else None
    want = pg.pool.cpu().clone()
    qkv = x.reshape(T, -1).cuda()
    out = qkv.view(T, nq + 2 * nkv, hd)[:, :nq] if in_place else None
    q = paged_append_int4(qkv, i32(lens), pg.table, pg.pool, None if inv is None else inv.cuda(), nq,
                          cu_seqlens=i32(starts) if cu else None, rope_pos=None if rope_pos is None else rope_pos.cuda(), out=out).cpu()
    half = torch.finfo(dtype).eps / 2
    table = pg.table.cpu()
    held = torch.zeros(T, dtype=torch.bool)
    back = [torch.zeros(T, nkv, hd, dtype=dtype) for _ in "kv"]
    for b, (n, m) in enumerate(zip(lens, news)):
        r = torch.arange(starts[b], starts[b + 1])
        p = torch.arange(n - m, n)
        if rotate:
            y, size = rope64(x[r, :nq + nkv], p if rope_pos is None else rope_pos[r], inv)
        else:
            y, size = x[r, :nq + nkv].double(), torch.zeros(())
        # q: one rounding of the result; cos and sin to 2^-22, two products and a sum in fp32
        tol = half * y.abs() + 2.0 ** -21 * size + (2.0 ** -25 if dtype == F16 and rotate else 0)
        off, fine = (q[r].double() - y[:, :nq]).abs(), torch.isfinite(y[:, :nq])
        assert ((off <= tol[:, :nq]) | ~fine).all(), f"q of sequence {b}"
        k = y[:, nq:].float().to(dtype)
        for i in range(m):
            t = int(p[i])
            if t < 0 or t >= table.shape[1] * page or not 0 <= int(table[b, t // page]) < want.shape[0]:
                continue
            held[r[i]] = True
            kq, vq = quantise(k[i], group), quantise(x[r[i], nq + nkv:], group)
            put(want[int(table[b, t // page]), :, t % page // 32], t % 32, hd, kq, vq)
            for o, z in zip(back, (kq, vq)):
                o[r[i]] = values(*z).float().to(dtype)
    got = pg.pool.cpu()
    nan = torch.isnan(got) & torch.isnan(want)  # NaN offsets: any NaN
    assert torch.equal(got.view(torch.int16)[~nan], want.view(torch.int16)[~nan]) and torch.equal(torch.isnan(got), torch.isnan(want))
    if in_place:  # the k and v columns and the rows behind the batch keep their values
        assert torch.equal(qkv.view(T, nq + 2 * nkv, hd)[:, nq:].cpu(), x[:, nq:])
    outs = [torch.full((T, nkv, hd), 7.0, dtype=dtype, device="cuda") for _ in "kv"]
    paged_read_int4(i32(lens), pg.table, pg.pool, cu_seqlens=i32(starts) if cu else None, out=tuple(outs))
    for o, w in zip(outs, back):
        o = o.cpu()
        assert (o[starts[-1]:] == 7.0).all()
        o, w = o[:starts[-1]], w[:starts[-1]]
        assert torch.equal(torch.isnan(o), torch.isnan(w)) and torch.equal(torch.nan_to_num(o), torch.nan_to_num(w))
    return pg


@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", LAYOUTS + [(F16, 128, 64, 3, 1, 32), (BF16, 64, 32, 5, 5, 64)])
@pytest.mark.parametrize("lens", [[1], [33, 1, 64, 100], [500, 32, 31, 65, 7, 1, 90, 96, 97]])
def test_append_one_token(dtype, hd, group, nq, nkv, page, lens):
    check_append(lens, [1] * len(lens), nq, nkv, hd, group, page, dtype, cu=False)


@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", LAYOUTS)
@pytest.mark.parametrize("lens,news", [([1], [1]), ([70], [70]), ([100, 40, 31, 200], [31, 40, 1, 64]),
                                       ([64, 0, 5, 97, 33], [32, 0, 5, 97, 2]), ([300, 129], [255, 128]),
                                       ([32] * 40, [1] * 40), ([63, 63], [31, 33])])
def test_append_ragged(dtype, hd, group, nq, nkv, page, lens, news):
    """Chunks that begin and end inside the new tokens, sequences without new tokens, whole chunks."""
    check_append(lens, news, nq, nkv, hd, group, page, dtype)


@pytest.mark.parametrize("hd,group,nq,nkv,B", [(64, 32, 4, 2, 1100), (128, 64, 3, 3, 700), (128, 128, 2, 1, 300), (64, 64, 7, 1, 500)])
def test_append_many_sequences(hd, group, nq, nkv, B):
    """So many chunks that a workgroup takes several or all of a token's heads."""
    check_append([33 + b % 3 for b in range(B)], [b % 3 for b in range(B)], nq, nkv, hd, group, 32, F16)


@pytest.mark.parametrize("cu", [False, True])
def test_append_positions_apart_from_the_cache(cu):
    """rope_pos far away, and beyond 32 bits."""
    pos = torch.tensor([1_000_000, 0, 131_071, 2 ** 33 + 5])
    check_append([5, 40, 64, 65], [1, 1, 1, 1], 4, 2, 128, 64, 32, F16, rope_pos=pos, cu=cu)


@pytest.mark.parametrize("cu", [False, True])
@pytest.mark.parametrize("dtype,hd,group", [(BF16, 64, 64), (F16, 64, 32), (F16, 128, 32)])
def test_append_without_rotation(cu, dtype, hd, group):
    check_append([5, 40, 64], [1, 1, 1], 4, 4, hd, group, 32, dtype, rotate=False, cu=cu)


@pytest.mark.parametrize("cu", [False, True])
def test_append_in_place(cu):
    check_append([5, 40, 64], [1, 1, 1], 8, 2, 128, 128, 32, F16, cu=cu, in_place=True, rows=5)


@pytest.mark.parametrize("cu", [False, True])
def test_append_where_there_is_no_page(cu):
    """Positions below 0 (kv_lens below the new tokens), past the table, and on absent pages: q is turned, nothing is
    written, and what is read back is zeros."""
    check_append([0, 70, 40], [1, 1, 1], 4, 2, 128, 64, 32, F16, cu=cu, room=[0, 64, 32], max_pages=2)
    if cu:
        check_append([10, 70, 40], [30, 50, 33], 4, 2, 128, 32, 32, F16, room=[10, 64, 32], max_pages=2)


def test_append_page_ids_outside_the_pool():
    pg = Pages4([40, 40], 2, 128, 128, 32, F16)
    pg.table[0, 1], pg.table[1, 1] = 10 ** 6, -7
    before = pg.pool.clone()
    qkv = torch.randn(2, 8 * 128, device="cuda").half()
    paged_append_int4(qkv, i32([40, 40]), pg.table, pg.pool, freqs(128).cuda(), 4)
    assert same_bits(before, pg.pool)
    for y in paged_read_int4(i32([40, 40]), pg.table, pg.pool):
        assert (y == 0).all()


SPECIAL = {
    "one value": lambda x, f: torch.full_like(x, 0.7),
    "zeros": lambda x, f: torch.zeros_like(x) * torch.where(torch.arange(x.shape[-1]) % 2 == 0, 1.0, -1.0).to(x.dtype),
    "two values a step of the type apart": lambda x, f: torch.where(x > 0, 1.0 + f.eps, 1.0).to(x.dtype),
    "the type's largest": lambda x, f: torch.where(x > 0, f.max, f.min).to(x.dtype),
    "the largest alone": lambda x, f: torch.full_like(x, f.max),
    "the type's smallest": lambda x, f: (torch.randint(-20, 21, x.shape) * f.smallest_normal * f.eps).to(x.dtype),
    "around the smallest normal": lambda x, f: (x.double() * f.smallest_normal * 4).to(x.dtype),
    "far from zero": lambda x, f: (x.float() * 0.05 + 900).to(x.dtype),
    "one dim of many times the others": lambda x, f: torch.where(torch.arange(x.shape[-1]) == 37, 200 * x, x),
    "half way between codes": lambda x, f: torch.randint(0, 31, x.shape).to(x.dtype) / 2,
    "a NaN": lambda x, f: torch.where(torch.arange(x.shape[-1]) == 3, float("nan"), x),
    "infinities": lambda x, f: torch.where(torch.arange(x.shape[-1]) == 40, -float("inf"), torch.where(torch.arange(x.shape[-1]) == 63, float("inf"), x)),
}


@pytest.mark.parametrize("what", SPECIAL)
@pytest.mark.parametrize("dtype,hd,group", [(F16, 128, 32), (BF16, 128, 128), (F16, 64, 64), (BF16, 64, 32)])
@pytest.mark.parametrize("cu", [False, True])
def test_append_of_special_values(what, dtype, hd, group, cu):
    """The quantiser's edges, by its definition to the bit (no rotation, so that k holds them too)."""
    torch.manual_seed(5)
    x = SPECIAL[what](torch.randn(3, 4 + 2 * 2, hd).to(dtype), torch.finfo(dtype)).to(dtype)
    check_append([5, 40, 64], [1, 1, 1], 4, 2, hd, group, 32, dtype, rotate=False, cu=cu, x=x)


def test_append_of_what_is_quantised_keeps_it():
    """Values that the format holds are read back as they went in, and appended again give the same values (within the
    steps' own rounding: half a step of fp16 of 7.5 steps and of the offset)."""
    pg = Pages4([70, 70], 2, 128, 32, 32, F16)
    k, v = paged_read_int4(i32([70, 70]), pg.table, pg.pool, 140, cu_seqlens=i32([0, 70, 140]))
    qkv = torch.cat([torch.zeros(140, 2, 128, dtype=F16, device="cuda"), k, v], 1).reshape(140, -1)
    again = Pages4([0, 0], 2, 128, 32, 32, F16, room=[70, 70])
    paged_append_int4(qkv, i32([70, 70]), again.table, again.pool, None, 2, cu_seqlens=i32([0, 70, 140]))
    k2, v2 = paged_read_int4(i32([70, 70]), again.table, again.pool, 140, cu_seqlens=i32([0, 70, 140]))
    for a, b in ((k, k2), (v, v2)):
        size = a.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
        assert ((a.double() - b.double()).abs() <= 4 * torch.finfo(F16).eps * size).all()


def test_append_rows_behind_the_batch_and_strides():
    """A padded batch: rows behind the last sequence keep their values; qkv and outputs strided; pages of a pool that
    holds two layers."""
    nq, nkv, hd, page, group = 4, 2, 128, 32, 64
    shape = kv_int4_shape(5, nkv, page, hd, group)
    pool = torch.full((5, 2) + shape[1:], 3.0, dtype=F16, device="cuda")
    wide = torch.randn(6, 2 * (nq + 2 * nkv) * hd, device="cuda").half()
    qkv = wide[:, :(nq + 2 * nkv) * hd]
    big = torch.full((6, nq + 3, hd), 9.0, dtype=F16, device="cuda")
    table = i32([[0], [3], [4]])
    for cu in (None, i32([0, 1, 2, 3])):
        big.fill_(9.0)
        q = paged_append_int4(qkv, i32([7, 8, 9]), table, pool[:, 1], freqs(hd).cuda(), nq, cu_seqlens=cu, out=big[:, :nq])
        assert q.data_ptr() == big.data_ptr()
        assert (big[3:] == 9.0).all() and (big[:, nq:] == 9.0).all() and not (big[:3, :nq] == 9.0).any(-1).any()
        assert (pool[:, 0] == 3.0).all()
        both = torch.full((6, 2, nkv + 1, hd), 7.0, dtype=F16, device="cuda")
        paged_read_int4(i32([7, 8, 9]), table, pool[:, 1], cu_seqlens=cu, out=(both[:, 0, :nkv], both[:, 1, :nkv]))
        assert (both[3:] == 7.0).all() and (both[:, :, nkv:] == 7.0).all()
        v = values(*quantise(qkv.view(6, -1, hd)[:3, nq + nkv:].cpu(), group)).float().half()
        assert torch.equal(both[:3, 1, :nkv].cpu(), v)


def test_past_four_gibibytes():
    """Pages whose offsets pass 32 bits, in bytes and in elements."""
    nq, nkv, hd, page, group = 2, 2, 128, 512, 32
    pages = 60000  # 4.9e9 elements, 9.8 GB
    pool = torch.empty(kv_int4_shape(pages, nkv, page, hd, group), dtype=F16, device="cuda")
    ids = [pages - 1, 29000, 3]
    table = i32([[p] for p in ids])
    pool[table[:, 0].long()] = 0
    qkv = torch.randn(3, (nq + 2 * nkv) * hd, device="cuda").half()
    lens = i32([300, 2, 1])
    paged_append_int4(qkv, lens, table, pool, None, nq)
    x = qkv.view(3, -1, hd).cpu()
    want = [values(*quantise(t, group)).float().half() for t in (x[:, nq:nq + nkv], x[:, nq + nkv:])]
    for y, w in zip(paged_read_int4(lens, table, pool), want):
        assert torch.equal(y.cpu(), w)
    for b, n in enumerate([300, 2, 1]):
        kq, _ = get(pool[ids[b], :, (n - 1) // 32].cpu(), (n - 1) % 32, hd)
        assert torch.equal(kq[0], quantise(x[b, nq:nq + nkv], group)[0])
    pool[table[:, 0].long()] = 0
    paged_append_int4(qkv, i32([1, 1, 1]), table, pool, None, nq)
    one = paged_attention_int4(q_of(3, nq, hd, F16).cuda(), i32([1, 1, 1]), table, pool, 0.1)
    v = values(*quantise(x[:, nq + nkv:], group))
    # one position: its v, its weight (times step and code) rounded to fp16, the result too
    assert ((one.cpu().double() - v).abs() <= 2.0 ** -11 * (v.abs() + 8 * 0.5)).all()


# ------------------------------------------------------------------------------------------ reading
@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", LAYOUTS)
def test_read_whole_sequences(dtype, hd, group, nq, nkv, page):
    lens, news = [200, 33, 1, 0, 96, 500], [200, 20, 1, 0, 96, 41]
    pg = Pages4(lens, nkv, hd, group, page, dtype)
    cu = rows_of(news)
    k, v = paged_read_int4(i32(lens), pg.table, pg.pool, cu[-1], cu_seqlens=i32(cu))
    for y, quant in ((k, pg.kq), (v, pg.vq)):
        for b, (n, m) in enumerate(zip(lens, news)):
            want = values(*(t[n - m:] for t in quant[b])).float().to(dtype)
            assert torch.equal(y[cu[b]:cu[b + 1]].cpu(), want), b
    k, v = paged_read_int4(i32(lens), pg.table, pg.pool)
    for y, quant in ((k, pg.kq), (v, pg.vq)):
        for b, n in enumerate(lens):
            assert torch.equal(y[b].cpu(), values(*(t[-1] for t in quant[b])).float().to(dtype) if n else torch.zeros(nkv, hd, dtype=dtype))


# --------------------------------------------------------------------------------------- attention
def check_attention(lens, news, nq, nkv, hd, group, page, dtype, window=0, sinks=0, cu=True, rows=None, max_q="given", seed=0, v_scale=1.0):
    pg = Pages4([max(n, 0) for n in lens], nkv, hd, group, page, dtype, seed=seed, v_scale=v_scale)
    starts = rows_of(news)
    T = rows or max(1, starts[-1])
    q = q_of(T, nq, hd, dtype, seed)
    scale = hd ** -0.5
    out = torch.full((T, nq, hd), 7.0, dtype=dtype, device="cuda")
    got = paged_attention_int4(q.cuda(), i32(lens), pg.table, pg.pool, scale, window=window, sinks=sinks,
                               cu_seqlens=i32(starts) if cu else None, max_q=max(1, max(news)) if max_q == "given" else max_q, out=out)
    assert got is out
    for b, (n, m) in enumerate(zip(lens, news)):
        r = slice(starts[b], starts[b + 1])
        ref, bound = attention64(q[r], pg.kq[b], pg.vq[b], scale, [n - m + i for i in range(m)], window, sinks)
        assert_within(got[r], ref, bound, f"sequence {b}")
    assert (out[starts[-1]:] == 7.0).all()


@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", LAYOUTS)
@pytest.mark.parametrize("lens", [[1], [33, 1, 64, 0, 100], [700, 32, 31, 65, 7, 2000, 90], [5000]])
def test_attention_one_token(dtype, hd, group, nq, nkv, page, lens):
    check_attention(lens, [1] * len(lens), nq, nkv, hd, group, page, dtype, cu=False)


@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", LAYOUTS)
@pytest.mark.parametrize("lens,news", [([70], [70]), ([100, 40, 31, 200], [31, 40, 1, 64]),
                                       ([64, 0, 5, 97, 33, 12], [32, 0, 5, 97, 2, 0]), ([400], [3]), ([260, 900], [130, 140])])
def test_attention_ragged(dtype, hd, group, nq, nkv, page, lens, news):
    check_attention(lens, news, nq, nkv, hd, group, page, dtype)


@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", [
    (F16, 64, 32, 4, 2, 32), (BF16, 64, 64, 3, 1, 64), (F16, 64, 64, 2, 2, 96), (BF16, 64, 32, 16, 2, 32), (F16, 64, 64, 5, 1, 32),
    (BF16, 128, 32, 12, 2, 64), (F16, 128, 64, 1, 1, 32), (F16, 128, 128, 8, 1, 32), (BF16, 128, 128, 24, 2, 32)])
def test_attention_few_query_heads(dtype, hd, group, nq, nkv, page):
    """Heads and tokens whose rows fill a quarter of a tile, a half, or more, with the numbers of sequences that find their
    ranges in either way; ranges of one chunk, of a group's and of others between."""
    for lens in ([700, 32, 31, 65, 7, 2000, 90], [5000], [3, 641, 0, 673], [833 + 32 * i for i in range(4)], [1281 + 32 * i for i in range(9)]):
        check_attention(lens, [1] * len(lens), nq, nkv, hd, group, page, dtype, cu=False)
    check_attention([700, 2000, 90, 4, 1700], [2, 1, 2, 0, 2], nq, nkv, hd, group, page, dtype)
    check_attention([700, 2000, 90, 33], [2, 1, 2, 2], nq, nkv, hd, group, page, dtype, window=900, sinks=3)
    check_attention([1 + (97 * i) % 700 for i in range(70)], [1] * 70, nq, nkv, hd, group, page, dtype, cu=False)


@pytest.mark.parametrize("dtype,hd,group", [(F16, 128, 128), (BF16, 128, 64), (F16, 128, 32), (BF16, 64, 64), (F16, 64, 32)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 2)])
def test_attention_blocks_of_whole_sequences(dtype, hd, group, window, sinks):
    """So many blocks that none is cut along its positions, of 128 rows and of 64."""
    check_attention([900, 33], [880, 20], 32, 16, hd, group, 32, dtype, window, sinks)
    check_attention([40 + 31 * i for i in range(21)] + [400], [1] * 20 + [30, 340], 16, 16, hd, group, 32, dtype, window, sinks)


@pytest.mark.parametrize("dtype,hd,group", [(F16, 128, 128), (BF16, 128, 64), (F16, 128, 32), (BF16, 64, 64), (F16, 64, 32)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 2)])
def test_attention_long_prompts_beside_tokens(dtype, hd, group, window, sinks):
    """Blocks of 64 rows that are cut along their positions; and tiles of 16 rows, up to 20 a sequence."""
    check_attention([900] + [40 + 131 * i for i in range(12)], [180] + [1] * 12, 2, 1, hd, group, 32, dtype, window, sinks)
    check_attention([1900] + [40 + 131 * i for i in range(12)], [80] + [1, 3] * 6, 4, 1, hd, group, 32, dtype, window, sinks)
    check_attention([60, 59, 3], [60, 40, 3], 10, 2, hd, group, 32, dtype, window, sinks)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 33), (100, 70), (5000, 9), (64, 1000), (0, 5)])
@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", LAYOUTS[:4])
def test_attention_window(dtype, hd, group, nq, nkv, page, window, sinks):
    check_attention([1, 300, 97, 640], [1] * 4, nq, nkv, hd, group, page, dtype, window, sinks, cu=False)
    check_attention([10, 300, 97, 640], [10, 70, 97, 5], nq, nkv, hd, group, page, dtype, window, sinks)


@pytest.mark.parametrize("window,sinks", [(1024, 0), (1500, 40)])
@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", LAYOUTS[:4])
def test_attention_window_over_ranges(dtype, hd, group, nq, nkv, page, window, sinks):
    """Windows whose chunks, with those of the sinks a gap before them, are cut into several ranges that a merge joins."""
    lens = [6000, 300, 3100, 1, 4500]
    check_attention(lens, [1] * 5, nq, nkv, hd, group, page, dtype, window, sinks, cu=False)
    check_attention(lens, [3, 2, 1, 1, 2], nq, nkv, hd, group, page, dtype, window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1300, 5)])
def test_attention_ranges_of_many_sequences(window, sinks):
    """More sequences than a wave has lanes: the ranges are found in a launch of their own; empty ones among them."""
    lens = [(37 * i) % 90 for i in range(150)]
    lens[3], lens[50], lens[99] = 5000, 3300, 2500
    check_attention([max(n, 1) for n in lens], [1] * 150, 4, 2, 128, 128, 32, F16, window, sinks, cu=False)
    check_attention(lens, [min(n, i % 3) for i, n in enumerate(lens)], 8, 2, 64, 32, 32, BF16, window, sinks)
    check_attention(lens, [min(n, 55 if i % 40 == 10 else 1) for i, n in enumerate(lens)], 4, 1, 64, 64, 32, F16, window, sinks)


@pytest.mark.parametrize("new", [200, 600])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 3), (40, 100)])
@pytest.mark.parametrize("dtype,hd,group,nq,nkv,page", [(F16, 128, 128, 4, 2, 64), (BF16, 64, 32, 3, 1, 32), (BF16, 128, 32, 2, 2, 32),
                                                        (F16, 64, 64, 7, 1, 64), (F16, 128, 64, 8, 1, 32)])
def test_attention_prompts(dtype, hd, group, nq, nkv, page, window, sinks, new):
    """Blocks of many rows whose masks begin and end inside them, behind cached positions and from 0."""
    check_attention([new, new + 333, 50], [new, new - 31, 50], nq, nkv, hd, group, page, dtype, window, sinks)


def test_attention_long_contexts_beside_prompts():
    """A batch that decodes and prefills at once: one token after many positions beside whole prompts."""
    check_attention([9000, 300, 17000, 40], [1, 300, 2, 1], 4, 1, 64, 32, 32, F16)
    check_attention([9000, 300, 17000, 40], [1, 300, 2, 1], 4, 1, 128, 128, 32, BF16)


def test_attention_past_four_gibibytes():
    """Pages whose offsets pass 32 bits give what the same pages in a small pool give, in every form."""
    nq, nkv, hd, page, group = 4, 2, 128, 512, 32
    pages = 60000
    pg = Pages4([1000, 1500], nkv, hd, group, page, F16)
    big = torch.empty(kv_int4_shape(pages, nkv, page, hd, group), dtype=F16, device="cuda")
    ids = torch.linspace(pages - 1, 2, pg.pool.shape[0]).to(torch.int32).cuda()  # of the small pool's pages
    big[ids.long()] = pg.pool
    table = torch.where(pg.table >= 0, ids[pg.table.clamp(min=0).long()], -1).to(torch.int32)
    for news in ([1, 1], [60, 3], [300, 200]):
        q, cu = q_of(sum(news), nq, hd, F16).cuda(), None if max(news) == 1 else i32(rows_of(news))
        want, got = (paged_attention_int4(q, i32([1000, 1500]), t, pool, 0.09, cu_seqlens=cu, max_q=max(news))
                     for t, pool in ((pg.table, pg.pool), (table, big)))
        assert same_bits(want, got), news


def test_attention_of_thousands_of_sequences_beside_a_prompt():
    """So many that tiles of 16 rows for the longest would be a million and more: in blocks, and without the prompt in tiles.
    All sequences read the same pages."""
    B, nkv, hd, page = 9000, 8, 64, 32
    pg = Pages4([400], nkv, hd, 64, page, F16)
    lens = torch.arange(B, dtype=torch.int32) % 400 + 1
    table = pg.table.expand(B, -1).contiguous()
    for first in (320, 1):
        lens[0] = 400
        cu = torch.cat([torch.zeros(1), torch.arange(B) + first]).to(torch.int32)
        q = q_of(B - 1 + first, nkv, hd, F16)
        got = paged_attention_int4(q.cuda(), lens.cuda(), table, pg.pool, 0.125, cu_seqlens=cu.cuda(), max_q=first).cpu()
        for b in (0, 1, 31, 32, 399, 4567, B - 1):
            n, r = int(lens[b]), slice(int(cu[b]), int(cu[b + 1]))
            ref, bound = attention64(q[r], *(tuple(t[:n] for t in x[0]) for x in (pg.kq, pg.vq)), 0.125, list(range(n - (r.stop - r.start), n)))
            assert_within(got[r], ref, bound, f"sequence {b}")


@pytest.mark.parametrize("v_scale", [2.0 ** -12, 3000.0])
@pytest.mark.parametrize("dtype,hd,group", [(F16, 128, 128), (BF16, 64, 32)])
def test_attention_of_small_and_large_values(v_scale, dtype, hd, group):
    """v far from 1: the weights are held against the largest step."""
    check_attention([400, 1500], [1, 1], 4, 2, hd, group, 32, dtype, cu=False, v_scale=v_scale)
    check_attention([400, 700], [150, 100], 4, 2, hd, group, 32, dtype, v_scale=v_scale)


def test_attention_positions_below_zero():
    """kv_lens below the new tokens' count: the tokens at positions below 0 give zeros."""
    pg = Pages4([10, 3], 2, 128, 64, 32, F16)
    q = q_of(20, 4, 128, F16)
    for max_q in (12, None):
        got = paged_attention_int4(q.cuda(), i32([10, 3]), pg.table, pg.pool, 0.1, cu_seqlens=i32([0, 12, 20]), max_q=max_q)
        for b, (lo, hi, n) in enumerate([(0, 12, 10), (12, 20, 3)]):
            ref, bound = attention64(q[lo:hi], pg.kq[b], pg.vq[b], 0.1, [n - (hi - lo) + i for i in range(hi - lo)])
            assert_within(got[lo:hi], ref, bound)
        assert (got[:2] == 0).all() and (got[12:17] == 0).all()


@pytest.mark.parametrize("news", [[1, 1, 1], [200, 3, 90]])
def test_attention_absent_pages(news):
    """Ids outside the pool hide their positions, as does a table shorter than the sequence."""
    pg = Pages4([300, 100, 96], 2, 64, 32, 32, BF16, max_pages=10)
    table = pg.table.clone()
    table[0, 2], table[0, 5], table[1, 3], table[2, :3] = -1, 10 ** 6, 2 ** 30, -5
    q = q_of(sum(news), 6, 64, BF16)
    cu = rows_of(news)
    for max_pages, lens in ((10, [300, 100, 96]), (4, [300, 100, 96])):
        got = paged_attention_int4(q.cuda(), i32(lens), table[:, :max_pages], pg.pool, 0.125,
                                   cu_seqlens=None if max(news) == 1 else i32(cu), max_q=max(news))
        for b, n in enumerate(lens):
            ok = torch.tensor([i < max_pages * 32 and 0 <= int(table[b, i // 32]) < pg.pool.shape[0] for i in range(n)])
            ref, bound = attention64(q[cu[b]:cu[b + 1]], pg.kq[b], pg.vq[b], 0.125, torch.arange(n)[-news[b]:].tolist(), present=ok)
            assert_within(got[cu[b]:cu[b + 1]], ref, bound, f"sequence {b}")
        assert (got[cu[2]:cu[3]] == 0).all()


def test_attention_max_q_bounds_what_is_computed():
    """Rows past max_q of a sequence are not computed, the others are."""
    pg = Pages4([50, 60], 2, 64, 64, 32, F16)
    q = q_of(24, 4, 64, F16)
    out = torch.full((24, 4, 64), 7.0, dtype=F16, device="cuda")
    paged_attention_int4(q.cuda(), i32([50, 60]), pg.table, pg.pool, 0.125, cu_seqlens=i32([0, 20, 24]), max_q=5, out=out)
    for b, lo, n, first in ((0, 0, 5, 30), (1, 20, 4, 56)):
        ref, bound = attention64(q[lo:lo + n], pg.kq[b], pg.vq[b], 0.125, [first + i for i in range(n)])
        assert_within(out[lo:lo + n], ref, bound)
    assert (out[5:20] == 7.0).all()


@pytest.mark.parametrize("news", [[1, 1], [150, 33]])
def test_attention_strides(news):
    """q a view of the projection's rows, out a view of wider rows, pages of a two-layer pool, a table that is a slice of a
    wider one."""
    nq, nkv, hd, page = 4, 2, 128, 32
    pg = Pages4([200, 150], nkv, hd, 32, page, F16)
    pool = torch.full((pg.pool.shape[0], 2) + tuple(pg.pool.shape[1:]), float("nan"), dtype=F16, device="cuda")
    pool[:, 1] = pg.pool
    T = sum(news)
    wide = q_of(T, nq + 4, hd, F16).cuda()
    out = torch.full((T, nq + 3, hd), 7.0, dtype=F16, device="cuda")
    table = torch.cat([pg.table, pg.table], 1)
    cu = rows_of(news)
    paged_attention_int4(wide[:, :nq], i32([200, 150]), table[:, :pg.table.shape[1]], pool[:, 1], 0.09,
                         cu_seqlens=None if max(news) == 1 else i32(cu), max_q=max(news), out=out[:, :nq])
    for b, L in enumerate([200, 150]):
        ref, bound = attention64(wide[cu[b]:cu[b + 1], :nq].cpu(), pg.kq[b], pg.vq[b], 0.09, list(range(L - news[b], L)))
        assert_within(out[cu[b]:cu[b + 1], :nq], ref, bound)
    assert (out[:, nq:] == 7.0).all()


@pytest.mark.parametrize("dtype,hd,group", [(F16, 64, 32), (BF16, 128, 128)])
@pytest.mark.parametrize("news", [[1], [40], [150]])
def test_attention_large_scores(news, dtype, hd, group):
    """Scores of both signs up to some hundreds: the maximum is subtracted before the exponential."""
    pg = Pages4([400], 1, hd, group, 32, dtype)
    q = 40 * q_of(news[0], 4, hd, dtype)
    got = paged_attention_int4(q.cuda(), i32([400]), pg.table, pg.pool, 0.125, cu_seqlens=None if news == [1] else i32([0, news[0]]))
    ref, bound = attention64(q, pg.kq[0], pg.vq[0], 0.125, list(range(400 - news[0], 400)))
    assert_within(got, ref, bound)


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -20, 2.0 ** 12, 2.0 ** 90])
@pytest.mark.parametrize("new", [1, 150])
def test_attention_of_q_of_any_size(size, new):
    """bf16 rows of q far outside fp16's range, their scores brought back by the softmax's scale (1e-20 .. 1e20), and rows of
    very unlike sizes side by side."""
    pg = Pages4([500], 2, 128, 64, 32, BF16)
    q = q_of(new, 4, 128, BF16).double()
    scale = min(max(0.09 / size, 2e-20), 5e19)
    q = (q * (0.09 / scale)).to(BF16)
    q[:, 1] = (q[:, 1].double() * 2.0 ** -30).to(BF16)
    q[:, 2] = 0
    got = paged_attention_int4(q.cuda(), i32([500]), pg.table, pg.pool, scale, cu_seqlens=None if new == 1 else i32([0, new]))
    ref, bound = attention64(q, pg.kq[0], pg.vq[0], scale, list(range(500 - new, 500)))
    assert_within(got, ref, bound)


def one_pool(kq, vq, hd, page, dtype):
    """Pages of one sequence's (code, step, z) [L, 1, ..] in order, and their table."""
    L, groups = kq[0].shape[0], kq[1].shape[-1]
    pool = torch.zeros(kv_int4_shape(L // page, 1, page, hd, hd // groups), dtype=dtype)
    flat = pool.view(L // 32, -1)
    for r in range(32):
        put(flat, r, hd, tuple(t[r::32, 0] for t in kq), tuple(t[r::32, 0] for t in vq))
    return pool.cuda(), torch.arange(L // page, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("new", [1, 64])
def test_attention_of_equal_scores_far_from_zero(new, dtype, hd):
    """131072 positions of one score, 840, the first half of value 1 and the others of 0: every weight is the same, whatever
    the maximum's product with scale log2 e loses in rounding. A weight times its step is rounded alike for all, half a
    step of fp16 of a value of 8 steps less 7: (8 + 7) 2^-12 of a 1/8 step."""
    B, L, page = (170 if new == 1 else 3), 131072, 64
    k = torch.zeros(L, 1, hd, dtype=dtype)
    k[:, 0, 0] = 112.0
    kq = quantise(k, hd)
    code = torch.where(torch.arange(L) < L // 2, 15, 8)[:, None, None].expand(L, 1, hd).to(torch.uint8)
    vq = (code, torch.full((L, 1, 1), 1 / 7.0).to(dtype), torch.zeros(L, 1, 1, dtype=dtype))
    pool, table = one_pool(kq, vq, hd, page, dtype)
    one = float(values(*(t[:1] for t in vq))[0, 0, 0])
    q = torch.zeros(B * new, 1, hd, dtype=dtype, device="cuda")
    q[:, 0, 0] = 62.5
    got = paged_attention_int4(q, i32([L] * B), table.expand(B, -1).contiguous(), pool, 0.12,
                               cu_seqlens=None if new == 1 else i32([new * b for b in range(B + 1)]), max_q=new)
    n = torch.arange(L - new + 1, L + 1, device="cuda").double().repeat(B)[:, None, None]
    want = one * (L / 2) / n
    bound = want * (torch.finfo(dtype).eps / 2 + 2.0 ** -12) + (2 * 4096 + 64) * 2.0 ** -24
    assert ((got.double() - want).abs() <= bound).all(), (got.double() - want).abs().max()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("power", [10, 25, 40])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("hd,new", [(128, 1), (64, 1), (64, 40), (128, 100)])
def test_attention_of_scores_of_any_size(hd, new, sign, power, dtype):
    """Scores of 50 sizes, 2^power times 0.12 or half of that apart: what has the largest has all the weight, in equal parts,
    also where the scores' products with log2 e are rounded by whole powers of two."""
    L, page = 1600, 64
    g = torch.Generator().manual_seed(power + new)
    order = torch.randperm(L, generator=g) % 50
    steps = order + 1 if sign > 0 else order - 50
    # k = offset in the group's first half, 0 in the others: exact, below fp16's largest
    kz = (steps * 2.0 ** (min(power, 25) - 15)).to(dtype)[:, None, None].expand(L, 1, hd // 32).clone()
    kz[..., 1:] = 0
    kq = (torch.full((L, 1, hd), 8, dtype=torch.uint8), torch.zeros(L, 1, hd // 32, dtype=dtype), kz)
    vq = quantise(torch.randn(L, 1, hd, generator=g).to(dtype), 32)
    v = values(*vq)
    scale = 0.12 * 2.0 ** (power - min(power, 25))
    pool, table = one_pool(kq, vq, hd, page, dtype)
    q = torch.zeros(new, 2, hd, dtype=dtype)
    q[:, 0, 0], q[:, 1, 0] = 2.0 ** 15, 2.0 ** 14
    got = paged_attention_int4(q.cuda(), i32([L]), table[None], pool, scale, cu_seqlens=None if new == 1 else i32([0, new]))
    half = torch.finfo(dtype).eps / 2
    for i in range(new):
        seen = steps[:L - new + i + 1]
        at = (seen == seen.max()).nonzero()[:, 0]
        best = v[at, 0]
        size = (vq[1][at, 0].double().repeat_interleave(32, -1) * 8).mean(0)
        bound = half * best.mean(0).abs() + 2.0 ** -12 * size + (len(best) + 64) * 2.0 ** -23 * (best.abs().mean(0) + 3 * size) + 2.0 ** -25
        assert_within(got[i], best.mean(0).expand(2, -1), bound.expand(2, -1), f"token {i}")


@pytest.mark.parametrize("new", [1, 48])
def test_attention_many_small_weights(new):
    """One position whose weight is 2^25 times that of each of 8191 others, which alone have values: the answer is their sum.
    Held times 2^8 they are 2^-17.1, off by half of fp16's step of 2^-24 there, 2^-7.9 of themselves."""
    L, hd, page = 8192, 64, 64
    k = torch.zeros(L, 1, hd, dtype=F16)
    k[5, 0, 0] = 4.3515625
    z = k[..., :32].amax(-1, keepdim=True).repeat(1, 1, 2)
    kq = (torch.full((L, 1, hd), 8, dtype=torch.uint8), torch.zeros(L, 1, 2, dtype=F16), z)
    kq[2][..., 1] = 0
    vq = (torch.full((L, 1, hd), 15, dtype=torch.uint8), torch.ones(L, 1, 2, dtype=F16), torch.zeros(L, 1, 2, dtype=F16))
    vq[0][5] = 8
    pool, table = one_pool(kq, vq, hd, page, F16)
    q = torch.zeros(new, 4, hd, dtype=F16)
    q[:, :, 0] = 4.0
    got = paged_attention_int4(q.cuda(), i32([L]), table[None], pool, 1.0, cu_seqlens=None if new == 1 else i32([0, new]))
    for i in range(new):
        w = (L - new + i) * torch.exp(torch.tensor(-4.0 * 4.3515625, dtype=torch.float64))
        ref = 7 * w / (1 + w)
        assert ((got[i].double().cpu() - ref).abs() <= ref * (2.0 ** -7.9 + 2.0 ** -10) + 2.0 ** -25).all(), (i, got[i, 0, 0].item(), ref)


@pytest.mark.parametrize("dtype,hd,group", [(F16, 64, 32), (BF16, 128, 128), (F16, 128, 64)])
@pytest.mark.parametrize("news", [[1, 1, 1], [2, 5, 3], [60, 3, 200]])
def test_attention_of_nan(news, dtype, hd, group):
    """A NaN or an infinity in a row of q makes that row's head NaN; a k that is NaN the rows that see it; a v that is NaN the
    dims of its group in the rows that see it; and nothing else."""
    lens, nq, nkv, page = [700, 64, 300], 6, 2, 32
    pg = Pages4(lens, nkv, hd, group, page, dtype)
    q, cu = q_of(sum(news), nq, hd, dtype), rows_of(news)
    at = lens[0] - (news[0] + 1) // 2  # seen by half of the first sequence's rows
    pg.kq[0][2][at, 1, 0] = float("nan")
    at_v = lens[2] - (news[2] + 1) // 2
    pg.vq[2][2][at_v, 0, -1], pg.vq[2][1][at_v, 0, -1] = float("nan"), 0.0
    for b, p in ((0, at), (2, at_v)):
        page_id = int(pg.table[b, p // page])
        block = pg.pool[page_id, :, p % page // 32].cpu()
        put(block, p % 32, hd, tuple(t[p] for t in pg.kq[b]), tuple(t[p] for t in pg.vq[b]))
        pg.pool[page_id, :, p % page // 32] = block.cuda()
    q[cu[1] + news[1] // 2, 0, 5] = float("nan")
    q[cu[1], 3, 7] = float("inf")
    got = paged_attention_int4(q.cuda(), i32(lens), pg.table, pg.pool, 0.125, cu_seqlens=None if max(news) == 1 else i32(cu), max_q=max(news)).cpu()
    for b, n in enumerate(lens):
        rows = torch.nan_to_num(q[cu[b]:cu[b + 1]], nan=0.0, posinf=0.0)
        where = [n - news[b] + i for i in range(news[b])]
        clean_k, clean_v = (tuple(torch.nan_to_num(t) if t.is_floating_point() else t for t in x[b]) for x in (pg.kq, pg.vq))
        ref, bound = attention64(rows, clean_k, clean_v, 0.125, where)
        bad = (~torch.isfinite(q[cu[b]:cu[b + 1]])).any(-1)[..., None].expand(-1, -1, hd).clone()
        sees = torch.tensor(where)[:, None] >= torch.tensor([at, at_v])
        if b == 0:
            bad[:, 3:] |= sees[:, :1, None]
        if b == 2:
            bad[:, :3, hd - group:] |= sees[:, 1:, None]
        mine = got[cu[b]:cu[b + 1]]
        assert (torch.isnan(mine) == bad).all(), b
        assert_within(torch.where(bad, 0, mine), torch.where(bad, 0, ref), torch.where(bad, 1, bound))


# ------------------------------------------------------- attention of values at the format's edges
# forms of the call by (new tokens of the first sequence, of the others, sequences): its heads are one kv head's
FORMS = {"one token": (1, 1, 2), "tiles": (40, 7, 3), "cut blocks": (400, 400, 2), "whole blocks": (340, 340, 80), "blocks of 64": (340, 1, 13)}
EDGES = [(F16, 128, 128), (F16, 64, 32), (BF16, 128, 32), (BF16, 128, 64), (BF16, 64, 64)]


def flat(values, hd, group, first=False):
    """(code, step, z) of one kv head whose groups (first: the first alone, the others 0) are constant, values[p] at position p."""
    z = values[:, None, None].expand(-1, 1, hd // group).clone()
    if first:
        z[..., 1:] = 0
    return torch.full((len(values), 1, hd), 8, dtype=torch.uint8), torch.zeros_like(z), z


def attend_one_pool(form, kq, vq, hd, dtype, q1, scale, nq=1):
    """Attention in one of the FORMS, every sequence over the same pages of one kv head, every head's row q1 [hd]: [(rows, first
    position)] of each sequence's results, as float64."""
    first, others, B = FORMS[form]
    L, page = kq[0].shape[0], 64
    pool, table = one_pool(kq, vq, hd, page, dtype)
    news = [first] + [others] * (B - 1)
    T = sum(news)
    q = q1.to(dtype).expand(T, nq, hd).contiguous().cuda()
    got = paged_attention_int4(q, i32([L] * B), table.expand(B, -1).contiguous(), pool, scale,
                               cu_seqlens=None if T == B else i32(rows_of(news)), max_q=first).cpu().double()
    return [(got[lo:hi], L - (hi - lo)) for lo, hi in zip(rows_of(news), rows_of(news)[1:])]


@pytest.mark.parametrize("scores", ["equal", "just below the lag"])
@pytest.mark.parametrize("dtype,hd,group", EDGES)
@pytest.mark.parametrize("form", FORMS)
def test_attention_of_constant_groups(form, dtype, hd, group, scores):
    """V whose groups have no step at any position, and scores that are equal or rise by 5.95 powers of two after the first
    positions, which is less than a maximum may lag. The answer is a weighted mean of the offsets: fp32 sums of n
    weights and products (n + 64) 2^-23, and 2^-16 for exponents up to 2^7 in size."""
    first, _, B = FORMS[form]
    half = torch.finfo(dtype).eps / 2
    for L in (832, 8192) if first == 1 else (8192,):
        p = torch.arange(L).double()
        s = torch.where(p < 512, 0.0, 4.125) if scores != "equal" else torch.full((L,), 1.0)
        kq = flat(s.to(dtype), hd, group, first=True)
        w = torch.exp(s.double() - s.max())
        q1 = torch.zeros(hd)
        q1[0] = 1.0
        kinds = {"zero": 0 * p, "one": 0 * p + 1, "a thousand": 0 * p + 1000, "the largest": 0 * p + (65504.0 if dtype == F16 else 2.0 ** 80),
                 "by position": p % 256, "of both signs": 30000 * (1 - 2 * (p % 2)), "once": torch.where(p == 700, 2.0 ** 15, 0.0)}
        for name, v in kinds.items():
            vq = flat(v.to(dtype), hd, group)
            v = vq[2][:, 0, 0].double()
            n = torch.cumsum(w, 0)
            ref, around = torch.cumsum(w * v, 0) / n, torch.cumsum(w * v.abs(), 0) / n
            bound = around * ((L + 64) * 2.0 ** -23 + 2.0 ** -16) + half * ref.abs() * 1.01 + 2.0 ** -25
            for rows, at in attend_one_pool(form, kq, vq, hd, dtype, q1, 1.0):
                r = slice(at, at + rows.shape[0])
                assert_within(rows[:, 0], ref[r, None].expand(-1, hd), bound[r, None].expand(-1, hd), f"{name}, {L} positions")


EDGE_VALUES = {
    "zeros": lambda x, f: torch.zeros_like(x),
    "zeros, then values": lambda x, f: torch.where(torch.arange(len(x))[:, None, None] < 130, 0, x),
    "values, then one value": lambda x, f: torch.where(torch.arange(len(x))[:, None, None] < 130, x, 3.0),
    "one value, then small ones": lambda x, f: torch.where(torch.arange(len(x))[:, None, None] < 130, 3.0, x * 2.0 ** -10),
    "two values a step of the type apart": lambda x, f: torch.where(x > 0, 1.0 + f.eps, 1.0),
    "far from zero": lambda x, f: x.float() * 0.05 + 900,
    "one dim of many times the others": lambda x, f: torch.where(torch.arange(x.shape[-1]) == 37, 200 * x, x),
    "the smallest": lambda x, f: torch.randint(-20, 21, x.shape) * (2.0 ** -24 if f.bits == 16 and f.eps < 2 ** -8 else 2.0 ** -70),
    "zeros, then large ones": lambda x, f: torch.where(torch.arange(len(x))[:, None, None] < 130, 0, x.double() * (10000.0 if f.eps < 2 ** -8 else 2.0 ** 30)),
}


@pytest.mark.parametrize("what", EDGE_VALUES)
@pytest.mark.parametrize("dtype,hd,group", EDGES)
@pytest.mark.parametrize("lens,news", [([300, 1200], [1, 1]), ([300, 1200], [40, 9]), ([450, 1200], [400, 330])])
def test_attention_of_edge_values(lens, news, dtype, hd, group, what):
    """v of the quantiser's edges, and steps that appear only after positions without one."""
    check_edge(lens, news, dtype, hd, group, EDGE_VALUES[what])


@pytest.mark.parametrize("lens,news", [([300, 1200], [1, 1]), ([300, 1200], [40, 9]), ([450, 1200], [400, 330])])
@pytest.mark.parametrize("hd,group", [(128, 32), (128, 128), (64, 64)])
@pytest.mark.parametrize("power", [45, 60, 80])
def test_attention_of_zeros_before_large_values(lens, news, hd, group, power):
    """bf16 v: zeros, then values of 2^power, more than fp32's range of exponents above the least step that the weights' unit
    tells apart."""
    check_edge(lens, news, BF16, hd, group, lambda x, f: torch.where(torch.arange(len(x))[:, None, None] < 130, 0, x.double() * 2.0 ** power))


@pytest.mark.parametrize("lens,news", [([300, 1200], [1, 1]), ([300, 1200], [40, 9]), ([450, 1200], [400, 330])])
@pytest.mark.parametrize("hd,group", [(128, 32), (128, 128), (64, 64)])
def test_attention_near_the_limit_of_bf16(lens, news, hd, group):
    """k and v of up to 2^90 in size, q as much smaller."""
    check_edge(lens, news, BF16, hd, group, lambda x, f: x.double() * 2.0 ** 87, k_size=2.0 ** 85)


def check_edge(lens, news, dtype, hd, group, make, k_size=None):
    nq, nkv, page = 2, 1, 64
    pg = Pages4(lens, nkv, hd, group, page, dtype, seed=11)
    pool, table = pg.pool.cpu(), pg.table.cpu()
    for b, n in enumerate(lens):
        x = torch.randn(n, nkv, hd, generator=torch.Generator().manual_seed(b)).to(dtype)
        if k_size:
            pg.kq[b] = quantise((x.flip(0).double() * k_size).to(dtype), group)
        pg.vq[b] = quantise(make(x, torch.finfo(dtype)).to(dtype), group)
        for p in range(n):
            put(pool[int(table[b, p // page]), :, p % page // 32], p % 32, hd, tuple(t[p] for t in pg.kq[b]), tuple(t[p] for t in pg.vq[b]))
    pg.pool.copy_(pool)
    cu = rows_of(news)
    q = (q_of(cu[-1], nq, hd, dtype).double() / (k_size or 1)).to(dtype)
    got = paged_attention_int4(q.cuda(), i32(lens), pg.table, pg.pool, hd ** -0.5, cu_seqlens=None if max(news) == 1 else i32(cu), max_q=max(news))
    for b, n in enumerate(lens):
        ref, bound = attention64(q[cu[b]:cu[b + 1]], pg.kq[b], pg.vq[b], hd ** -0.5, list(range(n - news[b], n)))
        assert_within(got[cu[b]:cu[b + 1]], ref, bound, f"sequence {b}")


@pytest.mark.parametrize("dtype,hd,group", EDGES)
@pytest.mark.parametrize("form", ["tiles", "cut blocks", "whole blocks", "blocks of 64"])
def test_attention_of_a_later_large_value(form, dtype, hd, group):
    """The step of a position that a row does not see has no part in how its weights are held: a v of far more than the others'
    size at a late position, small ones before, each row against a bound of what it sees alone."""
    L = 512
    g = torch.Generator().manual_seed(3)
    kq = quantise((1.3 * torch.randn(L, 1, hd, generator=g)).to(dtype), group)
    v = torch.randn(L, 1, hd, generator=g) * (2.0 ** -11 if dtype == F16 else 1.0)
    v[-12] = (60000.0 if dtype == F16 else 2.0 ** 40) * (1 - 2 * (torch.arange(hd) % 2))
    vq = quantise(v.to(dtype), group)
    q1 = torch.randn(hd, generator=g)
    for rows, at in attend_one_pool(form, kq, vq, hd, dtype, q1, hd ** -0.5)[:2]:
        for i in range(0, rows.shape[0], 1 if rows.shape[0] < 50 else 13):
            n = at + i + 1
            ref, bound = attention64(q1.to(dtype).expand(1, 1, hd), *(tuple(t[:n] for t in x) for x in (kq, vq)), hd ** -0.5, [n - 1])
            assert_within(rows[i:i + 1], ref, bound, f"row at {n - 1}")


@pytest.mark.parametrize("dtype,hd,group", EDGES)
@pytest.mark.parametrize("cu", [False, True])
def test_values_near_the_largest_are_finite(cu, dtype, hd, group):
    """Groups from the type's lowest to its largest value: their outermost codes are by up to the step's rounding beyond, and
    are read as the largest."""
    big = torch.finfo(dtype).max
    x = torch.randn(3, 2 + 2 * 2, hd)
    x = torch.stack([torch.where(x[0] > 0, big, -big), torch.where(x[1] > 0, big, big / 2), torch.where(x[2] > 0, -big, big / 4)]).to(dtype)
    pg = check_append([5, 40, 64], [1, 1, 1], 2, 2, hd, group, 32, dtype, rotate=False, cu=cu, x=x)
    for i, y in enumerate(paged_read_int4(i32([5, 40, 64]), pg.table, pg.pool, 3, cu_seqlens=i32([0, 1, 2, 3]) if cu else None)):
        want = values(*quantise(x[:, 2 + 2 * i:4 + 2 * i], group)).clamp(-big, big).to(dtype)
        assert torch.isfinite(y).all() and torch.equal(y.cpu(), want)


@pytest.mark.parametrize("hd,group", [(128, 128), (128, 32), (64, 64)])
@pytest.mark.parametrize("L", [64, 4096])
@pytest.mark.parametrize("form", FORMS)
def test_attention_near_the_largest_value_is_finite(form, L, hd, group):
    """fp16 v of -65504 and 65504 in every group, the same at every position: the answer is what is read, half a step of fp16
    more for the weights times their steps, of values of 8 steps and an offset of half a step."""
    if FORMS[form][0] > L:
        L = 512
    v = torch.where(torch.arange(hd) % 3 == 0, -65504.0, 65504.0).half()
    vq = quantise(v.expand(L, 1, hd), group)
    want = values(*(t[:1] for t in vq))[0, 0].clamp(-65504, 65504)
    kq = flat(torch.ones(L).half(), hd, group, first=True)
    q1 = torch.zeros(hd)
    q1[0] = 1.0
    for rows, _ in attend_one_pool(form, kq, vq, hd, F16, q1, 1.0, nq=2):
        off = (rows - want).abs()
        assert torch.isfinite(rows).all() and (off <= 65504 * (2.0 ** -11 + 2.0 ** -12 + (L + 64) * 2.0 ** -23)).all(), off.max()


def test_what_is_read_back_attended_to_in_16_bits():
    """Sequences moved to 16-bit pages through what is read back, whose attention is within its own bound of 64 bits over those
    values."""
    import _paged
    from kernels import paged

    lens, nq, nkv, hd, page = [300, 41, 700], 8, 2, 128, 32
    pg = Pages4(lens, nkv, hd, 64, page, F16)
    cu = i32(rows_of(lens))
    k, v = paged_read_int4(i32(lens), pg.table, pg.pool, sum(lens), cu_seqlens=cu)
    pages = pg.pool.shape[0]
    k16 = torch.zeros(paged.k_pages_shape(pages, nkv, page, hd), dtype=F16, device="cuda")
    v16 = torch.zeros(paged.vt_pages_shape(pages, nkv, page, hd), dtype=F16, device="cuda")
    qkv = torch.cat([torch.zeros(sum(lens), nq, hd, dtype=F16, device="cuda"), k, v], 1).reshape(sum(lens), -1)
    paged.paged_append(qkv, i32(lens), pg.table, k16, v16, None, nq, cu_seqlens=cu)
    q = q_of(3, nq, hd, F16)
    got = paged.paged_attention(q.cuda(), i32(lens), pg.table, k16, v16, 0.09)
    for b, n in enumerate(lens):
        r = slice(rows_of(lens)[b], rows_of(lens)[b + 1])
        ref, bound = _paged.attention64(q[b:b + 1], k[r].cpu(), v[r].cpu(), 0.09, [n - 1])
        assert_within(got[b:b + 1], ref, bound, f"sequence {b}")


# ------------------------------------------------------------------------- streams, graphs, together
def test_on_another_stream():
    pg = Pages4([900, 40], 2, 128, 32, 32, F16, seed=3)
    q, kv = q_of(2, 8, 128, F16, 3).cuda(), i32([900, 40])
    want = paged_attention_int4(q, kv, pg.table, pg.pool, 0.09)
    back = paged_read_int4(kv, pg.table, pg.pool)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [paged_attention_int4(q, kv, pg.table, pg.pool, 0.09) for _ in range(3)]
        again = paged_read_int4(kv, pg.table, pg.pool)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want, g) for g in got) and all(torch.equal(a, b) for a, b in zip(back, again))


def test_append_and_read_on_another_stream_and_in_a_graph():
    """Both forms, captured and replayed on a side stream at new lengths, with eager calls between."""
    nq, nkv, hd, group, page = 6, 2, 128, 32, 32
    for news in ([1, 1, 1], [40, 1, 70]):
        T, lens = sum(news), [200, 40, 130]
        cu = None if max(news) == 1 else i32(rows_of(news))
        pg = Pages4([250] * 3, nkv, hd, group, page, F16)
        other = pg.pool.clone()
        qkv, kv, inv = torch.randn(T, (nq + 2 * nkv) * hd, device="cuda").half(), i32(lens), freqs(hd).cuda()

        def call(pool):
            q = paged_append_int4(qkv, kv, pg.table, pool, inv, nq, cu_seqlens=cu)
            return (q,) + tuple(paged_read_int4(kv, pg.table, pool, T, cu_seqlens=cu))

        call(other)
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            outs = call(pg.pool)
        call(pg.pool)
        for step in range(4):
            kv.copy_(i32([n + 13 * step for n in lens]))
            qkv.copy_(torch.randn(qkv.shape, device="cuda"))
            want = call(other)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)
            assert all(same_bits(a, b) for a, b in zip(outs, want)) and same_bits(pg.pool, other), step


def test_two_graphs_at_new_lengths():
    """Two captured calls (workspaces of their own) replayed in turn and on two streams, with eager calls between, their lengths
    changed on the device between replays."""
    cases = []
    for seed, (lens, news, window, group) in enumerate([([900, 700, 1300], [1, 1, 1], 0, 128), ([500, 800], [40, 7], 200, 32),
                                                        ([900, 800], [200, 150], 0, 64)]):
        pg = Pages4(lens, 2, 128, group, 32, F16, seed=seed)
        cu = rows_of(news)
        q, kv, cu = q_of(cu[-1], 8, 128, F16, seed).cuda(), i32(lens), i32(cu)
        kw = dict(cu_seqlens=None if max(news) == 1 else cu, max_q=max(news), window=window, sinks=4 if window else 0)

        def call(q=q, kv=kv, pg=pg, kw=kw):
            return paged_attention_int4(q, kv, pg.table, pg.pool, 0.09, **kw)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        cases.append((graph, out, kv, lens, call))
    streams = [torch.cuda.Stream() for _ in cases]
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
    """Prompts of a ragged batch appended and attended to, then decode steps of the batch (append, full and windowed
    attention) captured once and replayed at new lengths, against 64 bits over what the pages hold; the sequences then move
    to 16-bit pages through what is read back, where the 16-bit attention gives the same."""
    from kernels import paged

    nq, nkv, hd, page, dtype, group = 8, 2, 64, 32, F16, 32
    width = (nq + 2 * nkv) * hd
    news, steps, scale = [40, 3, 150], 4, hd ** -0.5
    B = len(news)
    g = torch.Generator().manual_seed(9)
    need = [-(-(n + steps) // page) for n in news]
    ids = torch.randperm(sum(need) + 3, generator=g).to(torch.int32)
    pool = torch.full(kv_int4_shape(len(ids), nkv, page, hd, group), float("nan"), dtype=dtype, device="cuda")
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    for b in range(B):
        table[b, :need[b]] = ids[sum(need[:b]):sum(need[:b + 1])]
    table, inv = table.cuda(), freqs(hd).cuda()
    rows = torch.randn(sum(news), width, generator=g).to(dtype).cuda()
    lens, kv, cu = list(news), i32(news), i32(rows_of(news))
    q = paged_append_int4(rows, kv, table, pool, inv, nq, cu_seqlens=cu)

    def held(b, n):
        blocks = pool.cpu()
        parts = [get(blocks[int(table[b, p // page]), :, p % page // 32], p % 32, hd) for p in range(n)]
        return tuple(tuple(torch.stack([p[i][j] for p in parts]) for j in range(3)) for i in range(2))

    o = paged_attention_int4(q, kv, table, pool, scale, cu_seqlens=cu, max_q=max(news))
    for b, n in enumerate(news):
        r = slice(rows_of(news)[b], rows_of(news)[b + 1])
        kq, vq = held(b, n)
        assert all(torch.equal(x, y) for x, y in zip(vq, quantise(rows[r].view(n, -1, hd)[:, nq + nkv:].cpu(), group)))
        ref, bound = attention64(q[r].cpu(), kq, vq, scale, list(range(n)))
        assert_within(o[r], ref, bound)
    x = torch.zeros(B, width, dtype=dtype, device="cuda")

    def step():
        kv.add_(1)
        q = paged_append_int4(x, kv, table, pool, inv, nq)
        return q, paged_attention_int4(q, kv, table, pool, scale), paged_attention_int4(q, kv, table, pool, scale, window=24, sinks=2)

    x.copy_(torch.randn(B, width, generator=g).to(dtype))
    step()  # eager
    lens = [n + 1 for n in lens]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, a, w = step()
    for _ in range(steps - 1):
        x.copy_(torch.randn(B, width, generator=g).to(dtype))
        graph.replay()
        torch.cuda.synchronize()
        lens = [n + 1 for n in lens]
        assert kv.tolist() == lens
        for b in range(B):
            kq, vq = held(b, lens[b])
            for got, win, sinks in ((a, 0, 0), (w, 24, 2)):
                ref, bound = attention64(q[b:b + 1].cpu(), kq, vq, scale, [lens[b] - 1], win, sinks)
                assert_within(got[b:b + 1], ref, bound)
    # to 16-bit pages
    all_rows = i32(rows_of(lens))
    k, v = paged_read_int4(kv, table, pool, sum(lens), cu_seqlens=all_rows)
    k16 = torch.zeros(paged.k_pages_shape(len(ids), nkv, page, hd), dtype=dtype, device="cuda")
    v16 = torch.zeros(paged.vt_pages_shape(len(ids), nkv, page, hd), dtype=dtype, device="cuda")
    qkv = torch.cat([torch.zeros(sum(lens), nq, hd, dtype=dtype, device="cuda"), k, v], 1).reshape(sum(lens), -1)
    paged.paged_append(qkv, kv, table, k16, v16, None, nq, cu_seqlens=all_rows)
    b16 = paged.paged_attention(q, kv, table, k16, v16, scale)
    # k and v rounded to fp16 in between: scores by some 2^-12 |q||k|, here below 2^-8 in all
    assert ((a.double() - b16.double()).abs() <= 2.0 ** -7 * (1 + a.double().abs())).all()
