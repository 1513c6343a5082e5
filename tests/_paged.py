"""A paged cache for the tests: pools filled from plain K and V, and the operators in 64 bits."""

from __future__ import annotations

import torch

from kernels.attention import k_to_tiles, vt_to_tiles

INF = float("inf")


class Pages:
    """Sequences with `lens[b]` cached positions in pages that are scattered over a pool; every other
    position of the pool holds `fill`. k, v [b]: [len, n_kv, hd] of the sequence."""

    def __init__(self, lens, nkv, hd, page, dtype, seed=0, fill=float("nan"), extra=2, max_pages=None, room=None,
                 prefix=0, v_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.hd, self.nkv, self.dtype = list(lens), page, hd, nkv, dtype
        room = list(room or lens)  # positions that have a page
        width = max_pages or max(1, max(-(-n // page) for n in room))
        need = [min(-(-n // page), width) for n in room]
        total = sum(need) + extra + prefix // page
        ids = torch.randperm(total, generator=g).tolist()
        self.prefix_ids = [ids.pop() for _ in range(prefix // page)]
        table = torch.full((len(self.lens), width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = ids.pop()
        k = torch.full((total, nkv, page, hd), fill, dtype=dtype)
        v = torch.full((total, nkv, page, hd), fill, dtype=dtype)
        self.k, self.v = [], []

        def put(row, n):
            kk = (1.3 * torch.randn(n, nkv, hd, generator=g)).to(dtype)
            vv = (v_scale * torch.randn(n, nkv, hd, generator=g)).to(dtype)
            for i in range(0, n, page):
                m = min(page, n - i)
                if i // page >= len(row) or row[i // page] < 0:
                    continue  # positions without a page
                k[row[i // page], :, :m] = kk[i:i + m].transpose(0, 1)
                v[row[i // page], :, :m] = vv[i:i + m].transpose(0, 1)
            return kk, vv

        if prefix:
            self.pk, self.pv = put(self.prefix_ids, prefix)
        for b, n in enumerate(self.lens):
            kk, vv = put(table[b].tolist(), n)
            self.k.append(kk)
            self.v.append(vv)
        self.table = table.cuda()
        self.k_pages, self.vt_pages = k_to_tiles(k).cuda(), vt_to_tiles(v).cuda()
        self.generator = g


def rows_of(news):
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return cu


def attention64(q, k, v, scale, positions, window=0, sinks=0, present=None):
    """q [n, nq, hd] at `positions` over k, v [len, nkv, hd] in 64 bits, on the CPU. Returns (out, bound):
    the largest error of a computation that rounds the softmax's numerators and the result to q's type,
    with fp32 scores and sums. present: positions that exist (bool [len])."""
    n, nq, hd = q.shape
    L, nkv = k.shape[:2]
    half = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(n, nq, hd, dtype=torch.float64)
    bound = torch.zeros_like(out)
    j = torch.arange(L)
    for i in range(n):
        p = positions[i]
        seen = j <= p
        if window:
            seen &= (j > p - window) | (j < sinks)
        if present is not None:
            seen &= present
        at = seen.nonzero()[:, 0]
        if not len(at):
            continue
        for h in range(nq):
            kk, vv = k[at, h * nkv // nq].double(), v[at, h * nkv // nq].double()
            qq = q[i, h].double()
            s = kk @ qq * scale
            w = torch.exp(s - s.max())
            z = w.sum()
            out[i, h] = w @ vv / z
            around = w @ vv.abs() / z
            # numerators: half a step each (fp16's below 2^-14: 2^-25); scores: hd fp32 products and sums of
            # |q||k| each, and the exponent's own rounding, doubled for numerator and sum; result: half a step
            ds = (kk.abs() @ qq.abs() * scale).max() * (hd + 8) * 2.0 ** -24
            small = 2.0 ** -25 * vv.abs().sum(0) / z if q.dtype == torch.float16 else 0.0
            bound[i, h] = half * (around + out[i, h].abs()) * (1 + 2 ** -6) + around * (2 * ds + (len(at) + 64) * 2.0 ** -23) + small + 2.0 ** -25
    return out, bound


def assert_within(got, ref, bound, what=""):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    d = (got - ref).abs()
    assert (d <= bound).all(), f"{what}: error {d.max():.3e}, {(d / bound).max():.2f} of its bound"
