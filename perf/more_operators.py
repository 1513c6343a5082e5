"""The operators of a paged cache held in 4 bits, as a serving program calls them.

A case is a dict of plain values: its `kind` names one of the operators below, the rest are sizes and
options. `listed()` has the standing ones, `draw(rng)` gives others of the same ranges.

  append  the qkv projection's rows of a step's new tokens: RoPE on q and k, k and v quantised into the
          cache's pages (`paged_append_int4`), and what the pages now hold for the new tokens read back
          (`paged_read_int4`), as a prompt's own attention takes it.
  read    the values of whole sequences back from the pages (`paged_read_int4`), as where a sequence moves
          to a 16-bit cache or to another machine.
  attend  grouped-query attention of the new tokens over the pages, causal, in full or over a sliding window
          with a few first positions that stay visible (`paged_attention_int4`).

`own` false: the plain form, elementary torch operations in 32 bits (k's rotation in 64, as the codes hang
on it), rounded once at the end. `own` true: the framework's calls.

A pool's element [page][kv head][chunk of 32 positions] is a block of 16-bit words of the cache's type: the
bytes below. A position has, per kv head and group of `group` dims, a step and an offset z of the type; its
value is z + (code - 8) step.
  codes of k, 16 hd bytes: position r, dim d = 32 s + 8 kb + e. Row i = 4 (r / 8) + r % 4 of half
    h = r / 4 % 2; the 16-byte unit is 16 kb + i (with head_dim 128 of half h's 64 units, with 64 the
    unit's 8 bytes h); in it 8 bytes per pair of steps s / 2, 4 per e / 4, the byte 0, 2, 1, 3 of e % 4 and
    its low (s even) or high four bits.
  codes of v, 16 hd bytes: position r, dim d = 16 b + c. Unit 16 (r / 8) + c of 64 per 4 blocks b / 4;
    in it 8 bytes per pair of blocks, 4 per r / 4 % 2, the byte 0, 2, 1, 3 of r % 4, low (b even) or high.
  steps and offsets of k, then of v, 128 bytes per group: [position / 8][step, z][8 positions].
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path
from types import SimpleNamespace as Bag

import torch

own = False

THETA = 1_000_000.0
INF = float("inf")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# The most a drawn case may cost, as (bytes or flops / 50), the larger: under the largest listed case's.
COST_CAP = 2.0e9


# ------------------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one decoded token of one conversation, the small model's heads: the calls' latency
        dict(name="append_1token", kind="append", seqs=1, new_lo=1, new_hi=1, ctx_lo=900, ctx_hi=900, heads=12,
             kv_heads=2, head_dim=128, group=128, dtype="fp16", page=64, shifted=False),
        # a decode step of a full batch far into long contexts, whose old pages a window has released
        dict(name="append_batch", kind="append", seqs=96, new_lo=1, new_hi=1, ctx_lo=500, ctx_hi=150000, heads=32,
             kv_heads=8, head_dim=128, group=64, dtype="bf16", page=64, shifted=False),
        # prompts of mixed lengths admitted together, some behind a cached beginning; angles at
        # positions of their own (an edited context)
        dict(name="append_prompts", kind="append", seqs=7, new_lo=40, new_hi=2500, ctx_lo=0, ctx_hi=1000, heads=28,
             kv_heads=4, head_dim=128, group=32, dtype="fp16", page=32, shifted=True),
        # one short conversation leaves the 4-bit cache: latency
        dict(name="read_short", kind="read", seqs=1, ctx_lo=700, ctx_hi=700, kv_heads=2, head_dim=128, group=128,
             dtype="fp16", page=64),
        # a batch of long contexts moves elsewhere: the values' bytes
        dict(name="read_batch", kind="read", seqs=9, ctx_lo=100, ctx_hi=16000, kv_heads=8, head_dim=128, group=32,
             dtype="bf16", page=128),
        # one decoded token on a windowed layer, deep in a conversation: latency
        dict(name="attend_1token", kind="attend", seqs=1, new_lo=1, new_hi=1, ctx_lo=6000, ctx_hi=6000, heads=12,
             kv_heads=2, head_dim=128, group=128, dtype="fp16", page=64, window=1024, sinks=4),
        # a decode step of a ragged batch on a full layer: the caches' bytes
        dict(name="attend_batch", kind="attend", seqs=64, new_lo=1, new_hi=1, ctx_lo=30, ctx_hi=16000, heads=28,
             kv_heads=4, head_dim=128, group=128, dtype="bf16", page=64, window=0, sinks=0),
        # the same with small heads, each its own kv head, and the finest groups: most words beside the codes
        dict(name="attend_heads", kind="attend", seqs=40, new_lo=1, new_hi=1, ctx_lo=100, ctx_hi=9000, heads=20,
             kv_heads=20, head_dim=64, group=32, dtype="fp16", page=32, window=0, sinks=0),
        # two very long contexts, one kv head: the work of a sequence split over the card
        dict(name="attend_long", kind="attend", seqs=2, new_lo=1, new_hi=1, ctx_lo=90001, ctx_hi=120000, heads=8,
             kv_heads=1, head_dim=128, group=64, dtype="bf16", page=256, window=0, sinks=0),
        # ragged prompts on a windowed layer: the matrix cores and the mask's two edges
        dict(name="attend_prompts", kind="attend", seqs=5, new_lo=100, new_hi=4000, ctx_lo=0, ctx_hi=700, heads=32,
             kv_heads=8, head_dim=128, group=128, dtype="bf16", page=128, window=1000, sinks=5),
        # a chunk of a long prompt after what is cached of it, small heads
        dict(name="attend_chunk", kind="attend", seqs=1, new_lo=509, new_hi=509, ctx_lo=20000, ctx_hi=20000,
             heads=14, kv_heads=2, head_dim=64, group=64, dtype="fp16", page=32, window=0, sinks=0),
    ]


HEADS = [(12, 2, 128), (28, 4, 128), (32, 8, 128), (20, 20, 64), (14, 2, 64), (8, 1, 128), (24, 8, 64)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng) -> dict:
    kind = rng.choice(["append", "read", "attend", "attend"])
    nq, nkv, hd = rng.choice(HEADS)
    c = dict(kind=kind, kv_heads=nkv, head_dim=hd, group=rng.choice([32, 64, 128] if hd == 128 else [32, 64]),
             dtype=rng.choice(["fp16", "bf16"]), page=rng.choice([32, 64, 64, 128, 256]))
    if kind == "read":
        return c | dict(seqs=rng.randint(1, 12), ctx_lo=rng.choice([1, 50]), ctx_hi=_log(rng, 100, 20000))
    c |= dict(heads=nq)
    if rng.random() < 0.5:  # one token per sequence
        c |= dict(seqs=_log(rng, 1, 128), new_lo=1, new_hi=1, ctx_lo=rng.choice([0, 1, 100]), ctx_hi=_log(rng, 200, 20000))
    else:
        new = _log(rng, 8, 4000)
        c |= dict(seqs=rng.randint(1, 8), new_lo=max(1, new // rng.choice([1, 3, 20])), new_hi=new, ctx_lo=0,
                  ctx_hi=rng.choice([0, _log(rng, 20, 10000)]))
    if kind == "append":
        return c | dict(shifted=rng.random() < 0.3)
    window = rng.choice([0, 0, _log(rng, 60, 5000)])
    return c | dict(window=window, sinks=rng.choice([0, 1, 4, 40]) if window else 0)


def draw(rng) -> dict:
    while True:
        c = _draw(rng)
        if _cost(c) <= COST_CAP and _score_bytes(c) <= 6e9:
            return c


# --------------------------------------------------------------------------- lengths of a case
def lengths(c: dict) -> tuple[list[int], list[int]]:
    """New tokens (read back: rows) and cached positions before them of every sequence: the longest first,
    the shortest second, the rest spread over the logarithm."""
    new_lo, new_hi = c.get("new_lo", 0), c.get("new_hi", 0)
    r = random.Random(c["seqs"] * 1009 + new_hi * 31 + c["ctx_hi"])

    def some(lo, hi):
        v = [max(lo, min(hi, int(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1)))))) for _ in range(c["seqs"])]
        v[0] = hi
        if len(v) > 1:
            v[1] = lo
        return v

    if c["kind"] == "read":  # whole sequences
        return some(c["ctx_lo"], c["ctx_hi"]), [0] * c["seqs"]
    return some(new_lo, new_hi), some(c["ctx_lo"], c["ctx_hi"])


def _pairs(new, ctx, window, sinks):
    """Visible (token, position) pairs of one sequence, and the positions that any token sees."""
    total = 0
    for p in range(ctx, ctx + new):
        n = p + 1
        if window and n > window:
            n = window + min(sinks, n - window)
        total += n
    first = max(0, ctx + 1 - window) if window else 0
    return total, ctx + new - first + min(sinks, first)


def work(case: dict) -> dict:
    c = case
    new, ctx = lengths(c)
    nkv, hd, T = c["kv_heads"], c["head_dim"], sum(new)
    held = nkv * (hd + 8 * (hd // c["group"]))  # bytes of a position: codes, steps and offsets of k and v
    if c["kind"] == "read":
        return {"bytes": T * (held + 4 * nkv * hd), "flops": 4.0 * T * nkv * hd}
    nq = c["heads"]
    if c["kind"] == "append":
        return {"bytes": T * (2 * (nq + 2 * nkv) * hd + 2 * nq * hd + held + 4 * nkv * hd) + 8 * c["seqs"],
                "flops": T * hd * (3.0 * (nq + nkv) + 12.0 * nkv)}
    pairs = keys = 0
    for n, x in zip(new, ctx):
        p, k = _pairs(n, x, c["window"], c["sinks"])
        pairs, keys = pairs + p, keys + k
    return {"bytes": 2 * T * nq * hd * 2 + keys * held, "flops": 4.0 * hd * nq * pairs}


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def _score_bytes(c):
    """The padded 32-bit scores of the plain form, and its padded K and V."""
    new, ctx = lengths(c)
    most = len(new) * max(n + x for n, x in zip(new, ctx))
    if c["kind"] != "attend":
        return 0
    return 4 * most * (c["heads"] * max(new) + 2 * c["kv_heads"] * c["head_dim"])


# -------------------------------------------------------------------------------- the 4-bit format
@functools.lru_cache(maxsize=None)
def _places(hd: int, device: str):
    """Of a position r and each of its hd / 2 bytes, for k and for v: the byte's place in the block, [32,
    hd / 2], and the dims of its low and high four bits, [hd / 2]."""
    perm = [0, 2, 1, 3]
    out = []
    for what in "kv":
        other = 32 if what == "k" else 16
        low = [d for d in range(hd) if d // other % 2 == 0]
        at = []
        for r in range(32):
            row = []
            for d in low:
                if what == "k":
                    s, kb, e = d // 32, d // 8 % 4, d % 8
                    half, unit = r // 4 % 2, 16 * kb + 4 * (r // 8) + r % 4
                    a = half * 1024 + unit * 16 + s // 2 * 8 if hd == 128 else unit * 16 + half * 8
                    row.append(a + e // 4 * 4 + perm[e % 4])
                else:
                    b, t = d // 16, d // 32
                    row.append(16 * hd + t // 2 * 1024 + (16 * (r // 8) + d % 16) * 16 + t % 2 * 8 + r // 4 % 2 * 4 + perm[r % 4])
            at.append(row)
        low = torch.tensor(low, device=device)
        out.append((torch.tensor(at, device=device), low, low + other))
    return out


@functools.lru_cache(maxsize=None)
def _codes_at(hd: int, device: str):
    """Byte and shift of the code of (position r, dim d), [32, hd] each, for k and for v."""
    out = []
    for at, low, high in _places(hd, device):
        byte = torch.empty(32, hd, dtype=torch.long, device=device)
        shift = torch.empty(32, hd, dtype=torch.uint8, device=device)
        byte[:, low], byte[:, high] = at, at
        shift[:, low], shift[:, high] = 0, 4
        out.append((byte, shift))
    return out


def _quantise(x, group, dt):
    """Codes [.., hd] (int64), steps and offsets [.., hd / group] (32 bits, values of dt) of x [.., hd]."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = ((hi * 0.5 - lo * 0.5) / 7.5).to(dt).float()
    z = ((lo * 0.5 + hi * 0.5) + step * 0.5).to(dt).float()
    code = torch.where(step > 0, (torch.round((g - z) / step) + 8).clamp(0, 15), 8.0)
    return code.long().flatten(-2), step.squeeze(-1), z.squeeze(-1)


def _blocks(pool):
    """The pool's bytes and its params: uint8 [.., bytes] and [.., (k, v), group, position / 8, (step, z), 8]."""
    n = pool.shape[-1]
    hd = 64 if n < 2000 else 128
    groups = (n - 16 * hd) // 128
    return pool.view(torch.uint8), pool[..., 16 * hd:].unflatten(-1, (2, groups, 4, 2, 8)), hd, hd // groups


def _values(pool, which):
    """The values of k (0) or v (1) of blocks [.., words], as 32 bits [.., 32, hd]."""
    b8, params, hd, group = _blocks(pool)
    byte, shift = _codes_at(hd, str(pool.device))[which]
    code = ((b8[..., byte] >> shift) & 15).float() - 8.0
    p = params[..., which, :, :, :, :].float()  # [.., group, 4, 2, 8]
    step, z = p[..., 0, :].flatten(-2).transpose(-1, -2), p[..., 1, :].flatten(-2).transpose(-1, -2)  # [.., 32, groups]
    return (z[..., None] + code.unflatten(-1, (-1, group)) * step[..., None]).flatten(-2)


def _store(pool, where, r, which, x):
    """Quantises x [n, nkv, hd] into positions r [n] of the blocks where = (page [n], chunk [n])."""
    b8, params, hd, group = _blocks(pool)
    at, low, high = _places(hd, str(pool.device))[which]
    code, step, z = _quantise(x, group, pool.dtype)
    page, chunk = where
    h = torch.arange(pool.shape[1], device=pool.device)
    b8[page[:, None, None], h[:, None], chunk[:, None, None], at[r][:, None]] = (code[..., low] + 16 * code[..., high]).to(torch.uint8)
    g = torch.arange(hd // group, device=pool.device)
    for i, t in enumerate((step, z)):
        params[page[:, None, None], h[:, None], chunk[:, None, None], which, g, (r // 8)[:, None, None], i,
               (r % 8)[:, None, None]] = t.to(pool.dtype)


# ------------------------------------------------------------------------------------ the inputs
def prepare(case: dict, seed: int) -> Bag:
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32)

    new, ctx = lengths(c)
    nq, nkv, hd, page, B, T = c.get("heads", 0), c["kv_heads"], c["head_dim"], c["page"], c["seqs"], sum(new)
    kv = [n + x for n, x in zip(new, ctx)]
    need = [-(-n // page) for n in kv]
    width = max(need) + 1
    # the pages a call touches: an append only the last ones of each sequence (the others' ids are -1
    # here, as where a sliding window has released them), the others all of them
    first = [x // page if c["kind"] == "append" else 0 for x in ctx]
    rows = [[-1] * width for _ in range(B)]
    count = sum(n - f for n, f in zip(need, first)) + 3
    ids = torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist()
    for b in range(B):
        for i in range(first[b], need[b]):
            rows[b][i] = ids.pop()
    groups = hd // c["group"]
    pool = torch.empty(count, nkv, page // 32, 16 * hd + 128 * groups, device="cuda", dtype=dt)
    # what earlier appends left: values of a broad bulk, a dim of k in 16 some times as large as the others
    wide = 1.0 + 3.0 * (torch.rand(hd, device="cuda", generator=g) < 1 / 16)
    at, low, high = zip(*_places(hd, "cuda"))
    per = max(1, (1 << 22) // (nkv * page * hd))
    for i in range(0, count, per):
        part = pool[i:i + per]
        b8, params, _, _ = _blocks(part)
        for which in (0, 1):
            x = randn(part.shape[0], nkv, page // 32, 32, hd)
            code, step, z = _quantise((x * wide if which == 0 else x).to(dt), c["group"], dt)
            b8[..., at[which].flatten()] = (code[..., low[which]] + 16 * code[..., high[which]]).to(torch.uint8).flatten(-2)
            for j, t in enumerate((step, z)):
                params[..., which, :, :, j, :] = t.transpose(-1, -2).unflatten(-1, (4, 8)).to(dt)
    s = Bag(kind=c["kind"], pool=pool, heads=nq, rows=T, max_q=max(new), most=max(kv), scale=hd ** -0.5,
            table=torch.tensor(rows, dtype=torch.int32, device="cuda"),
            kv_lens=torch.tensor(kv, dtype=torch.int32, device="cuda"),
            cu=torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32))
    if c["kind"] == "append":
        s.qkv = randn(T, (nq + 2 * nkv) * hd).to(dt)
        s.inv_freq = 1.0 / (THETA ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float32) / hd))
        s.rope_pos = torch.randint(0, 100000, (T,), device="cuda", generator=g) if c["shifted"] else None
    elif c["kind"] == "attend":
        s.q = (1.5 * randn(T, nq, hd)).to(dt)
        s.window, s.sinks = c["window"], c["sinks"]
    return s


# ------------------------------------------------------------------------------- one pass through
def run(s: Bag):
    if own:
        return _framework(s)
    return {"append": _append, "read": _read, "attend": _attend}[s.kind](s)


@functools.lru_cache(maxsize=None)
def _module():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "llm-decode-kernels_amd"))
    from kernels import paged_int4

    return paged_int4


def _framework(s: Bag):
    p = _module()
    cu = s.cu if s.max_q > 1 else None  # None: one token per sequence
    if s.kind == "append":
        q = p.paged_append_int4(s.qkv, s.kv_lens, s.table, s.pool, s.inv_freq, s.heads, cu_seqlens=cu, rope_pos=s.rope_pos)
        return q, *p.paged_read_int4(s.kv_lens, s.table, s.pool, s.rows, cu_seqlens=cu)
    if s.kind == "read":
        return p.paged_read_int4(s.kv_lens, s.table, s.pool, s.rows, cu_seqlens=s.cu)
    return p.paged_attention_int4(s.q, s.kv_lens, s.table, s.pool, s.scale, cu_seqlens=cu, max_q=s.max_q,
                                  window=s.window, sinks=s.sinks)


# ------------------------------------------------------------------------------- the plain forms
def _rows(s, T):
    """Of every token: its sequence and its position in the cache."""
    t = torch.arange(T, device=s.cu.device)
    seq = torch.searchsorted(s.cu[1:], t.to(torch.int32), right=True)
    return seq, s.kv_lens[seq].long() - s.cu[seq + 1].long() + t


def _read(s):
    seq, p = _rows(s, s.rows)
    page = s.pool.shape[2] * 32
    at = s.table[seq, p // page].long()
    # by whole blocks: the chunks that hold the rows, then each row of its chunk
    key, inverse = torch.unique(at * (page // 32) + p % page // 32, return_inverse=True)
    blocks = s.pool[key // (page // 32), :, key % (page // 32)]  # [n, nkv, words]
    r = p % 32
    return tuple(_values(blocks, i)[inverse, :, r].to(s.pool.dtype) for i in (0, 1))


def _append(s):
    T, nq, nkv = s.qkv.shape[0], s.heads, s.pool.shape[1]
    hd = s.qkv.shape[1] // (nq + 2 * nkv)
    page, dt = s.pool.shape[2] * 32, s.pool.dtype
    x = s.qkv.view(T, nq + 2 * nkv, hd)
    seq, p = _rows(s, T)
    ang = (p if s.rope_pos is None else s.rope_pos).double()[:, None] * s.inv_freq.double()
    c, n = ang.cos()[:, None], ang.sin()[:, None]

    def turned(y, c, n):
        lo, hi = y.chunk(2, -1)
        return torch.cat([lo * c - hi * n, hi * c + lo * n], -1)

    q = turned(x[:, :nq].float(), c.float(), n.float()).to(dt)
    k = turned(x[:, nq:nq + nkv].double(), c, n).float().to(dt)
    at = s.table[seq, p // page].long()
    for which, y in enumerate((k, x[:, nq + nkv:])):
        _store(s.pool, (at, p % page // 32), p % 32, which, y)
    return q, *_read(s)


def _attend(s):
    T, nq, hd = s.q.shape
    B, nkv, page, M = s.kv_lens.shape[0], s.pool.shape[1], s.pool.shape[2] * 32, s.max_q
    seq, p = _rows(s, T)
    i = torch.arange(T, device=s.q.device) - s.cu[seq].long()
    q = torch.zeros(B, M, nq, hd, device=s.q.device)
    q[seq, i] = s.q.float()
    q = q.view(B, M, nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, -1, hd)
    at = s.table[:, :-(-s.most // page)].clamp(min=0).long()
    blocks = s.pool[at].transpose(1, 2).flatten(2, 3)  # [B, nkv, chunks, words]
    k = _values(blocks, 0).flatten(2, 3)
    scores = torch.matmul(q * s.scale, k.transpose(-1, -2).contiguous()).view(B, nkv, nq // nkv, M, -1)
    del k
    pos = (s.kv_lens - s.cu[1:] + s.cu[:-1]).long()[:, None, None] + torch.arange(M, device=q.device)[:, None]
    j = torch.arange(scores.shape[-1], device=q.device)
    seen = j <= pos
    if s.window:
        seen &= (j > pos - s.window) | (j < s.sinks)
    scores.masked_fill_(~seen[:, None, None], -INF)
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(m == -INF, 0.0, m)).view(B, nkv, -1, scores.shape[-1])
    del scores
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, _values(blocks, 1).flatten(2, 3)) / torch.where(total == 0, 1.0, total)
    o = o.view(B, nkv, nq // nkv, M, hd).permute(0, 3, 1, 2, 4).reshape(B, M, nq, hd)
    return o[seq, i].to(s.q.dtype)


# --------------------------------------------------------------------- the definitions in 64 bits
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attention}[case["kind"]](s, case)


def _exact_value(s, c, b, j, h, which):
    """Values of k or v of positions j of sequence b and kv head h, in 64 bits, [n, hd]: each element's code,
    step and offset looked up by address."""
    hd, groups, page = c["head_dim"], c["head_dim"] // c["group"], c["page"]
    words = 16 * hd + 128 * groups
    bytes_, halves = s.pool.view(torch.uint8).flatten(), s.pool.flatten()
    j = j[:, None]
    d = torch.arange(hd, device=j.device)
    block = (s.table[b].long()[j // page] * c["kv_heads"] + h) * (page // 32) + j % page // 32
    r = j % 32
    if which == 0:
        step32, inner = d // 32, d % 8
        unit = (d % 32 // 8) * 16 + (r // 8) * 4 + r % 4
        half = r % 8 // 4
        byte = unit * 16 + (half * 1024 + (step32 // 2) * 8 if hd == 128 else half * 8)
        high = step32 % 2
    else:
        inner = r % 8
        byte = 16 * hd + (d // 64) * 1024 + ((r // 8) * 16 + d % 16) * 16 + (d % 64 // 32) * 8
        high = d % 32 // 16
    byte = byte + (inner // 4) * 4 + (inner % 4 % 2) * 2 + inner % 4 // 2
    code = (bytes_[block * (2 * words) + byte].long() >> (4 * high)) % 16
    param = block * words + 16 * hd + (which * groups + d // c["group"]) * 64 + (r // 8) * 16 + r % 8
    return halves[param + 8].double() + (code - 8).double() * halves[param].double()


def _exact_read(s, c):
    cu, lens = s.cu.tolist(), s.kv_lens.tolist()
    out = []
    for which in (0, 1):
        y = torch.empty(cu[-1], c["kv_heads"], c["head_dim"], dtype=torch.float64, device=s.pool.device)
        for b, n in enumerate(lens):
            j = torch.arange(n - cu[b + 1] + cu[b], n, device=s.pool.device)
            for h in range(c["kv_heads"]):
                y[cu[b]:cu[b + 1], h] = _exact_value(s, c, b, j, h, which)
        out.append(y)
    return out


def _exact_append(s, c):
    nq, nkv, hd, group, dt = s.heads, c["kv_heads"], c["head_dim"], c["group"], s.pool.dtype
    T, dev = s.qkv.shape[0], s.pool.device
    cu, lens = s.cu.tolist(), s.kv_lens.tolist()
    pos = torch.cat([torch.arange(n - cu[b + 1] + cu[b], n, device=dev) for b, n in enumerate(lens)])
    angle = (pos if s.rope_pos is None else s.rope_pos).double()[:, None] * s.inv_freq.double()[None]
    # the pair (x_j, x_{j + hd/2}) as one complex number, turned
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=dev), angle)
    rows = s.qkv.double().view(T, nq + 2 * nkv, hd)
    w = torch.complex(rows[:, :nq + nkv, :hd // 2].contiguous(), rows[:, :nq + nkv, hd // 2:].contiguous()) * turn[:, None]
    w = torch.cat([w.real, w.imag], -1)
    out = [w[:, :nq]]
    for x in (w[:, nq:].float().to(dt).double(), rows[:, nq + nkv:]):
        y = torch.empty_like(x)
        for d in range(0, hd, group):
            a = x[..., d:d + group]
            low, high = a.min(-1, keepdim=True).values, a.max(-1, keepdim=True).values
            step = ((high - low) / 15).float().to(dt).double()
            z = (low + 7.5 * (high - low) / 15 + step / 2).float().to(dt).double()
            code = torch.clamp(torch.round((a - z) / torch.where(step == 0, 1.0, step)), -8, 7)
            y[..., d:d + group] = z + code * step
        out.append(y)
    return out


def _exact_attention(s, c):
    T, nq, hd = s.q.shape
    nkv = c["kv_heads"]
    cu, lens = s.cu.tolist(), s.kv_lens.tolist()
    out = torch.zeros(T, nq, hd, dtype=torch.float64, device=s.q.device)
    for b in range(len(lens)):
        j = torch.arange(lens[b], device=s.q.device)
        for h in range(nkv):
            k, v = (_exact_value(s, c, b, j, h, i) for i in (0, 1))
            kt = k.T.contiguous()
            for lo in range(cu[b], cu[b + 1], 256):
                hi = min(lo + 256, cu[b + 1])
                p = lens[b] - cu[b + 1] + torch.arange(lo, hi, device=s.q.device)[:, None]
                hidden = j > p
                if s.window:
                    hidden |= (j <= p - s.window) & (j >= s.sinks)
                for n in range(h * nq // nkv, (h + 1) * nq // nkv):
                    x = s.q[lo:hi, n].double() @ kt * s.scale
                    out[lo:hi, n] = torch.softmax(x.masked_fill(hidden, -INF), -1) @ v
    return out
