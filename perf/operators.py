"""The operators of a batch that decodes over a paged cache, as a serving program calls them.

A case is a dict of plain values: its `kind` names one of the operators below, the rest are sizes and
options. `listed()` has the standing ones, `draw(rng)` gives others of the same ranges.

  append    the qkv projection's rows of a step's new tokens: RoPE on q and k, k and v written into
            the cache's pages (`paged_append`). One token per sequence, or the ragged rows of prompts.
  attend    grouped-query attention of the new tokens over the pages, causal, in full or over a sliding
            window with a few first positions that stay visible (`paged_attention`).
  prefix    the same for a batch whose sequences all begin with one long prompt, whose pages they share
            (`shared_prefix_attention`).
  logprobs  log probability of a given token of each row of logits, the entropy, and the most likely
            tokens (`token_logprobs`), as a program answers with them or scores a text.

`own` false: the plain form, elementary torch operations in 32 bits (positions' angles in 64), rounded
once at the end. `own` true: the framework's calls.

The pages hold the matrix cores' operand order: K in tiles [page/32][2 row halves][head_dim/32][16 rows]
[32 dims], row i of half h at position 8 (i / 4) + 4 h + i % 4 of its 32; V^T in tiles [page/32]
[head_dim/16][16 dims][32 positions].
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path
from types import SimpleNamespace as Bag

import torch

own = False

THETA = 1_000_000.0
INF = float("inf")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}

# The most a drawn case may cost, as (bytes or flops / 50), the larger: under the largest listed case's.
COST_CAP = 2.0e9


# ------------------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one decoded token of one conversation, the small model's heads: the call's latency
        dict(name="append_1token", kind="append", seqs=1, new_lo=1, new_hi=1, ctx_lo=900, ctx_hi=900, heads=12,
             kv_heads=2, head_dim=128, dtype="fp16", page=64, shifted=False),
        # a decode step of a full batch far into long contexts, whose old pages a window has released
        dict(name="append_batch", kind="append", seqs=96, new_lo=1, new_hi=1, ctx_lo=500, ctx_hi=150000, heads=32,
             kv_heads=8, head_dim=128, dtype="bf16", page=64, shifted=False),
        # prompts of mixed lengths admitted together, some behind a cached beginning; angles at
        # positions of their own (an edited context)
        dict(name="append_prompts", kind="append", seqs=7, new_lo=40, new_hi=2500, ctx_lo=0, ctx_hi=1000, heads=28,
             kv_heads=4, head_dim=128, dtype="fp16", page=32, shifted=True),
        # one decoded token on a windowed layer, deep in a conversation: latency
        dict(name="attend_1token", kind="attend", seqs=1, new_lo=1, new_hi=1, ctx_lo=6000, ctx_hi=6000, heads=12,
             kv_heads=2, head_dim=128, dtype="fp16", page=64, window=1024, sinks=4),
        # a decode step of a ragged batch on a full layer: the caches' bytes
        dict(name="attend_batch", kind="attend", seqs=64, new_lo=1, new_hi=1, ctx_lo=30, ctx_hi=16000, heads=28,
             kv_heads=4, head_dim=128, dtype="bf16", page=64, window=0, sinks=0),
        # ragged prompts on a windowed layer: the matrix cores and the mask's two edges
        dict(name="attend_prompts", kind="attend", seqs=5, new_lo=100, new_hi=4000, ctx_lo=0, ctx_hi=700, heads=32,
             kv_heads=8, head_dim=128, dtype="bf16", page=128, window=1000, sinks=5),
        # a chunk of a long prompt after what is cached of it, small heads
        dict(name="attend_chunk", kind="attend", seqs=1, new_lo=509, new_hi=509, ctx_lo=20000, ctx_hi=20000,
             heads=16, kv_heads=16, head_dim=64, dtype="fp16", page=32, window=0, sinks=0),
        # a few answers sampled from one prompt
        dict(name="prefix_8", kind="prefix", seqs=8, new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=100, prefix=2048, heads=12,
             kv_heads=2, head_dim=128, dtype="fp16", page=64),
        # a large batch behind one long set of instructions, each with a question and answer of its own
        dict(name="prefix_128", kind="prefix", seqs=128, new_lo=1, new_hi=1, ctx_lo=20, ctx_hi=900, prefix=16384,
             heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=128),
        # one sampled row of a decode step with the five best alternatives
        dict(name="logprobs_1row", kind="logprobs", rows=1, vocab=151936, width=151936, top=5, dtype="fp16"),
        # a decode batch's rows in fp32, an odd vocabulary in wider rows
        dict(name="logprobs_batch", kind="logprobs", rows=77, vocab=50257, width=50304, top=20, dtype="fp32"),
        # a scored text: every position's token
        dict(name="logprobs_text", kind="logprobs", rows=1900, vocab=151936, width=151936, top=20, dtype="bf16"),
    ]


HEADS = [(12, 2, 128), (28, 4, 128), (32, 8, 128), (16, 16, 64), (14, 2, 64), (8, 1, 128), (24, 8, 64)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng) -> dict:
    kind = rng.choice(["append", "attend", "prefix", "logprobs"])
    if kind == "logprobs":
        vocab = _log(rng, 4000, 200000)
        return dict(kind=kind, rows=_log(rng, 1, 2000), vocab=vocab, width=vocab + rng.choice([0, 0, 1, 47]),
                    top=rng.choice([0, 1, 5, 8, 20, 20, 50]), dtype=rng.choice(["fp16", "bf16", "fp32"]))
    nq, nkv, hd = rng.choice(HEADS)
    c = dict(kind=kind, heads=nq, kv_heads=nkv, head_dim=hd, dtype=rng.choice(["fp16", "bf16"]),
             page=rng.choice([32, 64, 64, 128, 256]))
    if kind == "prefix":
        new = rng.choice([1, 1, 1, 3])
        return c | dict(seqs=_log(rng, 2, 128), new_lo=1, new_hi=new, ctx_lo=rng.choice([0, 1, 20]), ctx_hi=_log(rng, 30, 2000),
                        prefix=c["page"] * max(1, _log(rng, 256, 16384) // c["page"]))
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
    """New tokens and cached positions before them of every sequence (with a shared prefix, the ones
    past it): the longest first, the shortest second, the rest spread over the logarithm."""
    r = random.Random(c["seqs"] * 1009 + c["new_hi"] * 31 + c["ctx_hi"])

    def some(lo, hi):
        v = [max(lo, min(hi, int(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1)))))) for _ in range(c["seqs"])]
        v[0] = hi
        if len(v) > 1:
            v[1] = lo
        return v

    return some(c["new_lo"], c["new_hi"]), some(c["ctx_lo"], c["ctx_hi"])


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
    if c["kind"] == "logprobs":
        n = c["rows"] * c["vocab"]
        # exp, two sums and their products; the answers in 32 bits, the ids in 64
        return {"bytes": n * (4 if c["dtype"] == "fp32" else 2) + c["rows"] * (16 + 12 * c["top"]), "flops": 6.0 * n}
    new, ctx = lengths(c)
    nq, nkv, hd, T = c["heads"], c["kv_heads"], c["head_dim"], sum(new)
    if c["kind"] == "append":
        return {"bytes": 2 * T * (nq + 2 * nkv) * hd * 2 + 8 * c["seqs"] + 4 * T, "flops": 3.0 * T * (nq + nkv) * hd}
    pairs = keys = 0
    if c["kind"] == "attend":
        for n, x in zip(new, ctx):
            p, k = _pairs(n, x, c["window"], c["sinks"])
            pairs, keys = pairs + p, keys + k
    else:
        keys = c["prefix"]
        for n, x in zip(new, ctx):
            p, k = _pairs(n, x, 0, 0)
            pairs, keys = pairs + p + n * c["prefix"], keys + k
    return {"bytes": 2 * T * nq * hd * 2 + keys * nkv * hd * 4, "flops": 4.0 * hd * nq * pairs}


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def _score_bytes(c):
    """The padded 32-bit scores of the plain form."""
    if c["kind"] not in ("attend", "prefix"):
        return 0
    new, ctx = lengths(c)
    return 4 * c["heads"] * len(new) * max(new) * (max(n + x for n, x in zip(new, ctx)) + c.get("prefix", 0))


# ------------------------------------------------------------------------------------ the inputs
def prepare(case: dict, seed: int) -> Bag:
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32)

    if c["kind"] == "logprobs":
        # a row of logits: a broad bulk and, as a model gives them, a few tokens far above it
        x = torch.empty(c["rows"], c["width"], device="cuda", dtype=dt)
        for r in range(0, c["rows"], 256):
            y = 2.5 * randn(min(256, c["rows"] - r), c["width"])
            high = torch.randint(0, c["vocab"], (y.shape[0], 40), device="cuda", generator=g)
            y.scatter_add_(1, high, 4.0 + 3.0 * randn(y.shape[0], 40).abs())
            x[r:r + 256] = y.to(dt)
        logits = x[:, :c["vocab"]]
        # the given tokens: half of them the row's likely ones, as in a generated text
        tokens = torch.randint(0, c["vocab"], (c["rows"],), device="cuda", generator=g)
        tokens = torch.where(torch.arange(c["rows"], device="cuda") % 2 == 0, logits.argmax(-1), tokens)
        return Bag(kind=c["kind"], logits=logits, tokens=tokens, top=c["top"])

    new, ctx = lengths(c)
    nq, nkv, hd, page, B, T = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["seqs"], sum(new)
    prefix = c.get("prefix", 0)
    kv = [n + x for n, x in zip(new, ctx)]  # past the prefix
    need = [-(-n // page) for n in kv]
    width = max(need) + 1
    # the pages a call touches: an append only the last ones of each sequence (the others' ids are -1
    # here, as where a sliding window has released them), the attention all of them
    first = [x // page if c["kind"] == "append" else 0 for x in ctx]
    rows = [[-1] * width for _ in range(B)]
    count = sum(n - f for n, f in zip(need, first)) + prefix // page + 3
    ids = torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist()
    head = [ids.pop() for _ in range(prefix // page)]
    for b in range(B):
        for i in range(first[b], need[b]):
            rows[b][i] = ids.pop()
    k = torch.empty(count, nkv, page // 32, 2, hd // 32, 16, 32, device="cuda", dtype=dt)
    vt = torch.empty(count, nkv, page // 32, hd // 16, 16, 32, device="cuda", dtype=dt)
    for t in (k, vt):
        for i in range(0, count, 1024):
            t[i:i + 1024] = randn(*t[i:i + 1024].shape).to(dt)
    s = Bag(kind=c["kind"], k=k, vt=vt, heads=nq, max_q=max(new), most=max(kv), scale=hd ** -0.5, prefix=prefix,
            table=torch.tensor([head + r for r in rows], dtype=torch.int32, device="cuda"),
            kv_lens=torch.tensor([prefix + n for n in kv], dtype=torch.int32, device="cuda"),
            cu=torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32))
    if c["kind"] == "append":
        s.qkv = randn(T, (nq + 2 * nkv) * hd).to(dt)
        s.inv_freq = 1.0 / (THETA ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float32) / hd))
        s.rope_pos = torch.randint(0, 100000, (T,), device="cuda", generator=g) if c["shifted"] else None
        return s
    s.q = (1.5 * randn(T, nq, hd)).to(dt)
    s.window, s.sinks = c.get("window", 0), c.get("sinks", 0)
    if prefix:
        s.prefix_table = torch.tensor(head, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------------------- one pass through
def run(s: Bag):
    if own:
        return _framework(s)
    return {"append": _append, "attend": _attend, "prefix": _prefix, "logprobs": _logprobs}[s.kind](s)


def _framework(s: Bag):
    pkg = str(Path(__file__).resolve().parent.parent / "llm-decode-kernels_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    if s.kind == "logprobs":
        from kernels.sample import token_logprobs

        r = token_logprobs(s.logits, s.tokens, top=s.top)
        return r.logprob, r.entropy, r.top_logprobs, r.top_ids
    from kernels import paged

    cu = s.cu if s.max_q > 1 else None  # None: one token per sequence
    if s.kind == "append":
        q = paged.paged_append(s.qkv, s.kv_lens, s.table, s.k, s.vt, s.inv_freq, s.heads, cu_seqlens=cu,
                               rope_pos=s.rope_pos)
        return q, s.k, s.vt
    if s.kind == "prefix":
        return paged.shared_prefix_attention(s.q, s.kv_lens, s.table, s.prefix_table, s.prefix, s.k, s.vt, s.scale,
                                             cu_seqlens=cu, max_q=s.max_q)
    return paged.paged_attention(s.q, s.kv_lens, s.table, s.k, s.vt, s.scale, cu_seqlens=cu, max_q=s.max_q,
                                 window=s.window, sinks=s.sinks)


# ------------------------------------------------------------------------------- the plain forms
def _rows(s, T):
    """Of every token: its sequence and its position in the cache."""
    t = torch.arange(T, device=s.cu.device)
    seq = torch.searchsorted(s.cu[1:], t.to(torch.int32), right=True)
    return seq, s.kv_lens[seq].long() - s.cu[seq + 1].long() + t


def _linear(k_tiles, vt_tiles):
    """Pages' tiles as 32-bit K and V, [.., page, hd]."""
    *lead, c, _, ns, _, _ = k_tiles.shape
    n = len(lead)
    k = k_tiles.float().reshape(*lead, c, 2, ns, 4, 4, 32).permute(*range(n), n, n + 3, n + 1, n + 4, n + 2, n + 5)
    v = vt_tiles.float().permute(*range(n), n, n + 3, n + 1, n + 2)
    return k.reshape(*lead, c * 32, ns * 32), v.reshape(*lead, c * 32, ns * 32)


def _append(s):
    T, nq, nkv = s.qkv.shape[0], s.heads, s.k.shape[1]
    page, hd = s.k.shape[2] * 32, s.k.shape[4] * 32
    x = s.qkv.float().view(T, nq + 2 * nkv, hd)
    seq, p = _rows(s, T)
    ang = (p if s.rope_pos is None else s.rope_pos).double()[:, None] * s.inv_freq.double()
    c, n = ang.cos().float()[:, None], ang.sin().float()[:, None]
    lo, hi = x[:, :nq + nkv].chunk(2, -1)
    roped = torch.cat([lo * c - hi * n, hi * c + lo * n], -1).to(s.qkv.dtype)
    at, o = s.table[seq, p // page].long(), p % page
    i = 4 * (o % 32 // 8) + o % 4  # the row of its half tile
    s.k[at, :, o // 32, o % 8 // 4, :, i] = roped[:, nq:].reshape(T, nkv, hd // 32, 32)
    s.vt[at, :, o // 32, :, :, o % 32] = x[:, nq + nkv:].to(s.vt.dtype).reshape(T, nkv, hd // 16, 16)
    return roped[:, :nq].contiguous(), s.k, s.vt


def _softmax_v(scores, v):
    """Of masked scores (-inf): the weighted sums of v, zeros where nothing is visible."""
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(m == -INF, 0.0, m))
    z = e.sum(-1, keepdim=True)
    return torch.matmul(e, v) / torch.where(z == 0, 1.0, z)


def _padded_q(s):
    """q by sequence, [B, nkv, group, max_q, hd], and where each token stands in it."""
    T, nq, hd = s.q.shape
    B, nkv = s.kv_lens.shape[0], s.k.shape[1]
    seq, p = _rows(s, T)
    i = torch.arange(T, device=s.q.device) - s.cu[seq].long()
    q = torch.zeros(B, s.max_q, nq, hd, device=s.q.device)
    q[seq, i] = s.q.float()
    return q.view(B, s.max_q, nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4), seq, i


def _positions(s):
    """[B, max_q]: the position of each padded token."""
    return (s.kv_lens - s.cu[1:] + s.cu[:-1]).long()[:, None] + torch.arange(s.max_q, device=s.q.device)


def _own_kv(s):
    """Each sequence's K and V past the prefix, padded to the longest, [B, nkv, L, hd]."""
    page = s.k.shape[2] * 32
    at = s.table[:, s.prefix // page:][:, :-(-s.most // page)].clamp(min=0).long()
    k, v = _linear(s.k[at], s.vt[at])
    return k.transpose(1, 2).flatten(2, 3), v.transpose(1, 2).flatten(2, 3)


def _attend(s):
    q, seq, i = _padded_q(s)
    k, v = _own_kv(s)
    B, nkv, g, M, hd = q.shape
    scores = torch.matmul(q.reshape(B, nkv, g * M, hd) * s.scale, k.transpose(-1, -2).contiguous()).view(B, nkv, g, M, -1)
    p, j = _positions(s)[:, :, None], torch.arange(k.shape[2], device=k.device)
    seen = j <= p
    if s.window:
        seen &= (j > p - s.window) | (j < s.sinks)
    scores.masked_fill_(~seen[:, None, None], -INF)
    o = _softmax_v(scores.view(B, nkv, g * M, -1), v).view(q.shape)
    return o.permute(0, 3, 1, 2, 4).reshape(B, M, nkv * g, hd)[seq, i].to(s.q.dtype)


def _prefix(s):
    q, seq, i = _padded_q(s)
    B, nkv, g, M, hd = q.shape
    q = q.reshape(B, nkv, g * M, hd) * s.scale
    kp, vp = (t.transpose(0, 1).reshape(nkv, -1, hd) for t in _linear(s.k[s.prefix_table.long()], s.vt[s.prefix_table.long()]))
    k, v = _own_kv(s)
    L = k.shape[2]
    first = torch.matmul(q.transpose(0, 1).reshape(nkv, -1, hd), kp.transpose(-1, -2).contiguous())
    first = first.view(nkv, B, g * M, -1).transpose(0, 1)
    scores = torch.cat([first, torch.matmul(q, k.transpose(-1, -2).contiguous())], -1).view(B, nkv, g, M, -1)
    j = torch.arange(s.prefix + L, device=k.device)
    scores.masked_fill_(~(j <= _positions(s)[:, :, None])[:, None, None], -INF)
    scores = scores.view(B, nkv, g * M, -1)
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(m == -INF, 0.0, m))
    z = e.sum(-1, keepdim=True)
    e0 = e[..., :s.prefix].transpose(0, 1).reshape(nkv, -1, s.prefix)
    o = torch.matmul(e0, vp).view(nkv, B, g * M, hd).transpose(0, 1) + torch.matmul(e[..., s.prefix:], v)
    o = (o / torch.where(z == 0, 1.0, z)).view(B, nkv, g, M, hd)
    return o.permute(0, 3, 1, 2, 4).reshape(B, M, nkv * g, hd)[seq, i].to(s.q.dtype)


def _logprobs(s):
    x = s.logits.float()
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = y.exp()
    z = e.sum(-1, keepdim=True)
    log_z = z.log()
    entropy = log_z - torch.where(e > 0, e * y, 0.0).sum(-1, keepdim=True) / z
    logprob = y.gather(1, s.tokens[:, None]) - log_z
    # the order of (value, lowest index first) as one integer
    u = (x + 0.0).view(torch.int32).long()
    key = torch.where(u < 0, u ^ 0x7FFFFFFF, u) * 2 ** 32 - torch.arange(x.shape[1], device=x.device)
    ids = key.topk(s.top, -1).indices
    return logprob[:, 0], entropy[:, 0], y.gather(1, ids) - log_z, ids


# --------------------------------------------------------------------- the definitions in 64 bits
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if s.kind == "logprobs":
        return _exact_logprobs(s)
    return _exact_append(s) if s.kind == "append" else _exact_attention(s)


def _exact_logprobs(s):
    out = [[], [], [], []]
    for r in range(0, s.logits.shape[0], 128):
        x = s.logits[r:r + 128].double()
        logp = torch.log_softmax(x, -1)
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s.top]
        out[0].append(logp[torch.arange(x.shape[0], device=x.device), s.tokens[r:r + 128]])
        out[1].append(-torch.special.xlogy(logp.exp(), logp.exp()).sum(-1))
        out[2].append(torch.gather(logp, 1, ids))
        out[3].append(ids)
    return tuple(torch.cat(o) for o in out)


def _slots(s, b, positions, hd):
    """Flat places in the K and V^T pools of a sequence's positions, per kv head: [n, nkv, hd] each."""
    page, nkv, dev = s.k.shape[2] * 32, s.k.shape[1], s.k.device
    p = positions[:, None, None]
    block = (s.table[b].long()[positions // page][:, None, None] * nkv + torch.arange(nkv, device=dev)[:, None]) * page * hd
    d = torch.arange(hd, device=dev)
    chunk = block + p % page // 32 * 32 * hd
    r = p % 32
    at_k = chunk + ((r % 8 // 4) * (hd // 32) + d // 32) * 512 + (r // 8 * 4 + r % 4) * 32 + d % 32
    at_v = chunk + d // 16 * 512 + d % 16 * 32 + r
    return at_k, at_v


def _exact_append(s):
    nq, nkv = s.heads, s.k.shape[1]
    hd = s.k.shape[4] * 32
    k, vt = s.k.double(), s.vt.double()
    q = torch.empty(s.qkv.shape[0], nq, hd, dtype=torch.float64, device=k.device)
    cu, lens = s.cu.tolist(), s.kv_lens.tolist()
    for b in range(len(lens)):
        lo, hi = cu[b], cu[b + 1]
        p = torch.arange(lens[b] - (hi - lo), lens[b], device=k.device)
        r = p if s.rope_pos is None else s.rope_pos[lo:hi]
        # the pair (x_j, x_{j + hd/2}) as one complex number, turned
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=k.device), r.double()[:, None] * s.inv_freq.double()[None])
        rows = s.qkv[lo:hi].double().view(hi - lo, -1, hd)
        z = torch.complex(rows[:, :nq + nkv, :hd // 2].contiguous(), rows[:, :nq + nkv, hd // 2:].contiguous()) * turn[:, None]
        z = torch.cat([z.real, z.imag], -1)
        q[lo:hi] = z[:, :nq]
        at_k, at_v = _slots(s, b, p, hd)
        k.view(-1)[at_k] = z[:, nq:]
        vt.view(-1)[at_v] = rows[:, nq + nkv:]
    return q, k, vt


def _exact_attention(s):
    T, nq, hd = s.q.shape
    nkv = s.k.shape[1]
    cu, lens = s.cu.tolist(), s.kv_lens.tolist()
    out = torch.zeros(T, nq, hd, dtype=torch.float64, device=s.q.device)
    for b in range(len(lens)):
        j = torch.arange(lens[b], device=s.q.device)
        at_k, at_v = _slots(s, b, j, hd)
        k, v = s.k.view(-1)[at_k].double(), s.vt.view(-1)[at_v].double()
        for lo in range(cu[b], cu[b + 1], 256):
            hi = min(lo + 256, cu[b + 1])
            p = lens[b] - cu[b + 1] + torch.arange(lo, hi, device=s.q.device)[:, None]
            hidden = j > p
            if s.window:
                hidden |= (j <= p - s.window) & (j >= s.sinks)
            for h in range(nq):
                x = s.q[lo:hi, h].double() @ k[:, h * nkv // nq].T.contiguous() * s.scale
                w = torch.softmax(x.masked_fill(hidden, -INF), -1)
                out[lo:hi, h] = w @ v[:, h * nkv // nq]
    return out
