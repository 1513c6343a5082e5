"""A paged cache in 4 bits for the tests: the format from its definition, pools of scattered pages, and attention
over the values they hold in 64 bits."""

from __future__ import annotations

import functools

import torch

from kernels.paged_int4 import kv_int4_shape


def quantise(x, group):
    """(codes uint8 [.., hd], step, z [.., hd / group] of x's dtype) of x [.., hd], by the definition's steps in fp32."""
    dt = x.dtype
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    fine = torch.isfinite(g).all(-1)
    step = ((hi * 0.5 - lo * 0.5) / 7.5).to(dt)
    z = ((lo * 0.5 + hi * 0.5) + step.float() * 0.5).to(dt)
    step = torch.where(fine, step, torch.zeros((), dtype=dt))
    z = torch.where(fine, z, torch.full((), float("nan"), dtype=dt))
    s = step.float()[..., None]
    code = torch.where(s > 0, (torch.round((g - z.float()[..., None]) / torch.where(s > 0, s, 1.0)) + 8).clamp(0, 15), torch.tensor(8.0))
    return code.flatten(-2).to(torch.uint8), step, z


def values(code, step, z):
    """In 64 bits."""
    group = code.shape[-1] // step.shape[-1]
    return (z.double()[..., None] + (code.double() - 8).unflatten(-1, (-1, group)) * step.double()[..., None]).flatten(-2)


@functools.lru_cache(maxsize=None)
def places(hd, groups):
    """For every position r and dim d: (byte, shift) of k's and of v's code; for every r and group: the word of k's step and
    of v's (the offset is 8 words on)."""
    perm = (0, 2, 1, 3)
    k = torch.zeros(32, hd, 2, dtype=torch.long)
    v = torch.zeros(32, hd, 2, dtype=torch.long)
    for r in range(32):
        for d in range(hd):
            unit = 16 * (d // 8 % 4) + 4 * (r // 8) + r % 4
            half = r // 4 % 2
            at = 1024 * half + 16 * unit + 8 * (d // 64) if hd == 128 else 16 * unit + 8 * half
            k[r, d] = torch.tensor([at + 4 * (d // 4 % 2) + perm[d % 4], 4 * (d // 32 % 2)])
            at = 16 * hd + 1024 * (d // 64) + 16 * (16 * (r // 8) + d % 16) + 8 * (d // 32 % 2) + 4 * (r // 4 % 2) + perm[r % 4]
            v[r, d] = torch.tensor([at, 4 * (d // 16 % 2)])
    r, g = torch.arange(32)[:, None], torch.arange(groups)
    step_k = 16 * hd + 64 * g + 16 * (r // 8) + r % 8
    return k, v, step_k, step_k + 64 * groups


def put(block, r, hd, kq, vq):
    """Writes position r of a block [words] (any leading dims): kq, vq = (code, step, z) with the same leading dims."""
    groups = kq[1].shape[-1]
    b8 = block.view(torch.uint8)
    for place, step_at, (code, step, z) in zip(places(hd, groups)[:2], places(hd, groups)[2:], (kq, vq)):
        for high in (0, 1):
            d = (place[r, :, 1] == 4 * high).nonzero()[:, 0]
            at = place[r, d, 0]
            keep = b8[..., at] & (0x0F if high else 0xF0)
            b8[..., at] = keep | (code[..., d] << (4 * high))
        block[..., step_at[r]], block[..., step_at[r] + 8] = step, z


def get(block, r, hd):
    """((code, step, z) of k, of v) at position r."""
    groups = (block.shape[-1] - 16 * hd) // 128
    k, v, sk, sv = places(hd, groups)
    b8 = block.view(torch.uint8)
    return tuple(((b8[..., p[r, :, 0]] >> p[r, :, 1].to(torch.uint8)) & 15, block[..., s[r]], block[..., s[r] + 8])
                 for p, s in ((k, sk), (v, sv)))


class Pages4:
    """Sequences with `lens[b]` cached positions in pages scattered over a pool; of every other position of the pool the
    codes are random, the steps infinite and the offsets NaN. kq, vq [b]: (code, step, z) of the sequence, [len, n_kv, ..]."""

    def __init__(self, lens, nkv, hd, group, page, dtype, seed=0, extra=2, max_pages=None, room=None, v_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.hd, self.nkv, self.dtype, self.group = [max(0, n) for n in lens], page, hd, nkv, dtype, group
        room = list(room or self.lens)
        width = max_pages or max(1, max(-(-n // page) for n in room))
        need = [min(-(-n // page), width) for n in room]
        total = sum(need) + extra
        ids = torch.randperm(total, generator=g).tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = ids.pop()
        shape = kv_int4_shape(total, nkv, page, hd, group)
        pool = torch.randint(0, 256, (*shape[:-1], 2 * shape[-1]), generator=g, dtype=torch.uint8).view(dtype)
        par = pool[..., 16 * hd:].unflatten(-1, (-1, 2, 8))
        par[..., 0, :], par[..., 1, :] = float("inf"), float("nan")
        self.kq, self.vq = [], []
        wide = 1.0 + 3.0 * (torch.rand(hd, generator=g) < 1 / 16)  # a few large dims, as k's
        for b, n in enumerate(self.lens):
            kq = quantise((1.3 * wide * torch.randn(n, nkv, hd, generator=g)).to(dtype), group)
            vq = quantise((v_scale * torch.randn(n, nkv, hd, generator=g)).to(dtype), group)
            self.kq.append(kq)
            self.vq.append(vq)
            for r in range(32):
                p = torch.arange(r, max(n, r), 32)
                p = p[(p // page < width)]
                if len(p):
                    at = table[b].long()[p // page]
                    p, at = p[at >= 0], at[at >= 0]
                    blocks = pool[at, :, p % page // 32]
                    put(blocks, r, hd, tuple(t[p] for t in kq), tuple(t[p] for t in vq))
                    pool[at, :, p % page // 32] = blocks
        self.table, self.pool, self.generator = table.cuda(), pool.cuda(), g


def attention64(q, kq, vq, scale, positions, window=0, sinks=0, present=None):
    """q [n, nq, hd] at `positions` over one sequence's quantised k and v in 64 bits, on the CPU. Returns (out, bound): the
    largest error of a computation that takes the codes exactly, scores, weights and sums in fp32, rounds each weight
    times its step to fp16, and the result to q's type."""
    n, nq, hd = q.shape
    L, nkv = kq[0].shape[:2]
    gq, group = nq // nkv, hd // kq[1].shape[-1]
    half = torch.finfo(q.dtype).eps / 2
    out, bound = torch.zeros(n, nq, hd, dtype=torch.float64), torch.zeros(n, nq, hd, dtype=torch.float64)
    if not n or not L:
        return out, bound
    pos, j = torch.tensor(positions)[:, None], torch.arange(L)
    seen = j <= pos
    if window:
        seen &= (j > pos - window) | (j < sinks)
    if present is not None:
        seen &= present
    some = seen.any(1)
    wide = lambda t: t.double().repeat_interleave(group, -1)  # noqa: E731
    for h in range(nkv):
        k, v = (values(*(t[:, h] for t in x)) for x in (kq, vq))
        ks, kz, vs, vz = (wide(t[:, h]).abs() for t in (*kq[1:], *vq[1:]))
        off = (vq[0][:, h].double() - 8).abs()
        for i in range(h * gq, (h + 1) * gq):
            x = q[:, i].double()
            s = torch.where(seen, x @ k.T * scale, -float("inf"))
            m = torch.where(some, s.max(1).values, 0.0)[:, None]
            w = torch.where(seen, torch.exp(s - m), 0.0)
            tot = torch.where(some, w.sum(1), 1.0)[:, None]
            w = w / tot
            o = w @ torch.where(seen.any(0)[:, None], v, 0.0)
            # A score: fp32 sums over hd products of q with codes to 15 and with -8, of step and offset, and q itself, which is
            # kept to 2^-34 of its row's largest; its exponent: the difference to the maximum times a rounded factor.
            ds = scale * (x.abs() @ (2 * kz + 31 * ks).T * (hd + 16) * 2.0 ** -24 + x.abs().max(1).values[:, None] * (kz + 8 * ks).sum(1) * 2.0 ** -34)
            ds = torch.where(seen, ds, 0.0)
            dw = ds + ds.max(1).values[:, None] + torch.where(seen, m - s + 4, 0.0) * 2.0 ** -22
            # a weight times its step: half a step of fp16, or 2^-33 of the largest step; fp32 products and sums of the uncentred codes
            vsz, vzz, ofz = (torch.where(seen.any(0)[:, None], t, 0.0) for t in (vs, vz, off))
            e = (w * dw) @ torch.where(seen.any(0)[:, None], v.abs(), 0.0) + (w * dw).sum(1)[:, None] * o.abs()
            e = e + w @ (vsz * ofz) * 2.0 ** -12 * 1.01 + 8 * 2.0 ** -33 * vsz.max() * seen.sum(1)[:, None] / tot
            e = e + w @ (23 * vsz + vzz) * (seen.sum(1)[:, None] + 64) * 2.0 ** -24
            e = e + half * o.abs() * 1.01 + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
            out[:, i], bound[:, i] = torch.where(some[:, None], o, 0.0), e
    return out, bound
