"""Several sequences over one cache of pages on gfx950 (libldk_amd.so): `paged_append` rotates the new
tokens' q and k and writes k and v into the pages (`ldk_paged_append`), `paged_attention` attends over
them, in full or over a sliding window with a few first positions that stay visible
(`ldk_paged_attention`), and `shared_prefix_attention` does so for a batch whose sequences begin with
the same pages, reading those once (`ldk_shared_prefix_attention`).

They are the batch's counterparts of kernels.attention, whose `decode_attention` and
`prefill_attention` serve one sequence over one static cache (the attention block of the reference's
runner, kernels/e2e/model.py:212-243).

A step of ragged sequences, each of its tensors on the device and re-read by a captured graph:

    q = paged_append(qkv, kv_lens, block_table, k_pages, vt_pages, inv_freq, n_heads, cu_seqlens)
    o = paged_attention(q, kv_lens, block_table, k_pages, vt_pages, scale, cu_seqlens, max_q)

- k_pages [pages, n_kv, page/32, 2, hd/32, 16, 32] and vt_pages [pages, n_kv, page/32, hd/16, 16, 32],
  fp16 or bf16, hold the static cache's tiles (`kernels.attention.k_to_tiles` / `vt_to_tiles` of
  [pages, n_kv, page, hd] and their inverses convert); page a multiple of 32, hd 64 or 128. The first
  dimension may have any stride (a pool of several layers' pages), the others are contiguous.
- block_table int32 [B, max_pages]: position p of sequence b is in page block_table[b, p // page]; an
  id outside the pool is no page (nothing is written there, its positions are not attended to).
- cu_seqlens int32 [B + 1]: the new tokens of sequence b are the rows cu_seqlens[b]:cu_seqlens[b + 1];
  None: one new token per sequence, row b. kv_lens int32 [B]: positions in the cache with the new
  tokens, which are the last of them. Rows behind the last sequence's are left as they were (of an
  output that is not given: undefined).
"""

from __future__ import annotations

import torch

from kernels import _lib
from kernels.attention import CHUNK

HEAD_DIMS = (64, 128)


def k_pages_shape(pages: int, n_kv: int, page: int, head_dim: int = 128) -> tuple:
    return (pages, n_kv, page // CHUNK, 2, head_dim // 32, 16, 32)


def vt_pages_shape(pages: int, n_kv: int, page: int, head_dim: int = 128) -> tuple:
    return (pages, n_kv, page // CHUNK, head_dim // 16, 16, 32)


def _pool(k_pages: torch.Tensor, vt_pages: torch.Tensor, what: str):
    """(pages, n_kv, page, head_dim, k page stride, vt page stride) of a pool, checked."""
    ks, vs = k_pages.shape, vt_pages.shape
    if len(ks) != 7 or len(vs) != 6:
        raise ValueError(f"{what}: k_pages and vt_pages must be k_pages_shape and vt_pages_shape, got "
                         f"{tuple(ks)} and {tuple(vs)}")
    pages, nkv, cpp, hd = ks[0], ks[1], ks[2], ks[4] * 32
    page = cpp * CHUNK
    if (ks[3] != 2 or ks[5] != 16 or ks[6] != 32 or vs[0] != pages or vs[1] != nkv or vs[2] != cpp
            or vs[3] * 16 != hd or vs[4] != 16 or vs[5] != 32):
        raise ValueError(f"{what}: k_pages and vt_pages must be k_pages_shape and vt_pages_shape of one pool, "
                         f"got {tuple(ks)} and {tuple(vs)}")
    if k_pages.dtype != vt_pages.dtype:
        raise ValueError(f"{what}: k_pages {k_pages.dtype} and vt_pages {vt_pages.dtype} differ")
    per = nkv * page * hd
    kst, vst = (per, per) if pages == 1 else (k_pages.stride(0), vt_pages.stride(0))
    for t in (k_pages, vt_pages):
        if not (t.is_contiguous() or (pages and t[0].is_contiguous())):
            raise ValueError(f"{what}: a page's tiles must be contiguous")
    return pages, nkv, page, hd, kst, vst


def _batch(kv_lens: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor | None, rows: int, what: str):
    """(B, table row stride), of checked lengths, table and row bounds."""
    B = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    if kv_lens.dtype != torch.int32 or B < 0 or (B > 1 and kv_lens.stride(0) != 1):
        raise ValueError(f"{what}: kv_lens must be a contiguous int32 [B]")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B or (
            block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"{what}: block_table must be int32 [{B}, max_pages] with contiguous rows")
    if cu_seqlens is None:
        if rows < B:
            raise ValueError(f"{what}: {rows} rows for {B} sequences of one token (cu_seqlens=None)")
    elif cu_seqlens.dtype != torch.int32 or cu_seqlens.shape != (B + 1,) or cu_seqlens.stride(0) != 1:
        raise ValueError(f"{what}: cu_seqlens must be a contiguous int32 [{B + 1}]")
    return B, block_table.stride(0) if B > 1 else block_table.shape[1]


def _heads(t: torch.Tensor, dtype: torch.dtype, hd: int, what: str, name: str) -> None:
    if t.dim() != 3 or t.shape[2] != hd or t.dtype != dtype:
        raise ValueError(f"{what}: {name} must be {dtype} [tokens, heads, {hd}], got {t.dtype} {tuple(t.shape)}")


def _check_out(out: torch.Tensor, rows: int, heads: int, hd: int, dtype: torch.dtype, what: str) -> None:
    _heads(out, dtype, hd, what, "out")
    if out.shape[0] != rows or out.shape[1] != heads or out.stride(2) != 1 or (heads > 1 and out.stride(1) != hd):
        raise ValueError(f"{what}: out must be [{rows}, {heads}, {hd}] with contiguous heads, got "
                         f"{tuple(out.shape)} strides {out.stride()}")


def _row_stride(t: torch.Tensor, width: int) -> int:
    return t.stride(0) if t.shape[0] > 1 else width


def paged_append(qkv: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, k_pages: torch.Tensor,
                 vt_pages: torch.Tensor, inv_freq: torch.Tensor | None, n_heads: int,
                 cu_seqlens: torch.Tensor | None = None, rope_pos: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """qkv [tokens, (n_heads + 2 n_kv) * hd], the projection's rows, in the cache's dtype; inv_freq fp32
    [hd/2], or None for no rotation; rope_pos int64 [tokens]: positions to turn q and k by instead of
    their cache positions. Writes the rotated k and v at their positions' pages and returns the
    rotated q [tokens, n_heads, hd], into `out` where given (which may be qkv's own q columns).
    Angles are reduced in 64 bits, the rotation is fp32, rounded once. Two tokens of one call may not
    share a position of a page."""
    what = "paged_append"
    pages, nkv, page, hd, kst, vst = _pool(k_pages, vt_pages, what)
    width = (n_heads + 2 * nkv) * hd
    if qkv.dim() != 2 or qkv.shape[1] != width or qkv.dtype != k_pages.dtype:
        raise ValueError(f"{what}: qkv must be {k_pages.dtype} [tokens, {width}], got {qkv.dtype} {tuple(qkv.shape)}")
    T = qkv.shape[0]
    B, ldt = _batch(kv_lens, block_table, cu_seqlens, T, what)
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.shape != (hd // 2,) or inv_freq.stride(0) != 1):
        raise ValueError(f"{what}: inv_freq must be a contiguous float32 [{hd // 2}]")
    if rope_pos is not None and (rope_pos.dtype != torch.int64 or rope_pos.shape != (T,) or (T > 1 and rope_pos.stride(0) != 1)):
        raise ValueError(f"{what}: rope_pos must be a contiguous int64 [{T}]")
    if out is not None:
        _check_out(out, T, n_heads, hd, qkv.dtype, what)
    dev = _lib.require_gpu(qkv, kv_lens, block_table, k_pages, vt_pages, inv_freq, cu_seqlens, rope_pos, out, what=what)
    q = torch.empty((T, n_heads, hd), dtype=qkv.dtype, device=dev) if out is None else out
    if not T or not B:
        return q
    x = qkv
    if x.stride(1) != 1 or x.data_ptr() % 16 or _row_stride(x, width) % 8:
        x = x.contiguous()
    with _lib.device_guard(dev):
        st = _lib.load().ldk_paged_append(
            _lib.ptr(x), _row_stride(x, width), _lib.dtype_code(x.dtype), _lib.ptr(cu_seqlens), _lib.ptr(kv_lens),
            _lib.ptr(block_table), ldt, block_table.shape[1], _lib.ptr(rope_pos), _lib.ptr(inv_freq),
            _lib.ptr(k_pages), kst, _lib.ptr(vt_pages), vst, pages, page, _lib.ptr(q), _row_stride(q, n_heads * hd),
            T, B, n_heads, nkv, hd, _lib.stream(dev))
    _lib.check(st, what)
    return q


def _attend(what, q, kv_lens, block_table, prefix_table, prefix_len, k_pages, vt_pages, scale, cu_seqlens, max_q, window,
            sinks, out):
    pages, nkv, page, hd, kst, vst = _pool(k_pages, vt_pages, what)
    _heads(q, k_pages.dtype, hd, what, "q")
    T, nq = q.shape[0], q.shape[1]
    B, ldt = _batch(kv_lens, block_table, cu_seqlens, T, what)
    if prefix_table is not None and (prefix_table.dtype != torch.int32 or prefix_table.dim() != 1
                                     or prefix_table.shape[0] * page < prefix_len
                                     or (prefix_table.shape[0] > 1 and prefix_table.stride(0) != 1)):
        raise ValueError(f"{what}: prefix_table must be a contiguous int32 of at least {prefix_len // page} pages")
    if out is not None:
        _check_out(out, T, nq, hd, q.dtype, what)
    dev = _lib.require_gpu(q, kv_lens, block_table, prefix_table, k_pages, vt_pages, cu_seqlens, out, what=what)
    o = torch.empty((T, nq, hd), dtype=q.dtype, device=dev) if out is None else out
    if not T or not B:
        return o
    x = q
    if x.stride(2) != 1 or (nq > 1 and x.stride(1) != hd) or x.data_ptr() % 16 or _row_stride(x, 0) % 8:
        x = x.contiguous()
    if cu_seqlens is None:
        max_q = 1
    elif max_q is None:
        max_q = T
    lib = _lib.load()
    with _lib.device_guard(dev):
        need = lib.ldk_paged_attention_workspace_bytes(T, B, max_q, prefix_len, nq, nkv, hd)
        if need < 0:
            _lib.check(-need, what)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        if prefix_table is None:
            st = lib.ldk_paged_attention(
                _lib.ptr(x), _row_stride(x, nq * hd), _lib.dtype_code(x.dtype), _lib.ptr(cu_seqlens), _lib.ptr(kv_lens),
                _lib.ptr(block_table), ldt, block_table.shape[1], _lib.ptr(k_pages), kst, _lib.ptr(vt_pages), vst, pages,
                page, _lib.ptr(o), _row_stride(o, nq * hd), T, B, max_q, nq, nkv, hd, window, sinks, float(scale),
                _lib.ptr(ws), need, _lib.stream(dev))
        else:
            st = lib.ldk_shared_prefix_attention(
                _lib.ptr(x), _row_stride(x, nq * hd), _lib.dtype_code(x.dtype), _lib.ptr(cu_seqlens), _lib.ptr(kv_lens),
                _lib.ptr(block_table), ldt, block_table.shape[1], _lib.ptr(prefix_table), prefix_len, _lib.ptr(k_pages),
                kst, _lib.ptr(vt_pages), vst, pages, page, _lib.ptr(o), _row_stride(o, nq * hd), T, B, max_q, nq, nkv, hd,
                float(scale), _lib.ptr(ws), need, _lib.stream(dev))
    _lib.check(st, what)
    return o


def paged_attention(q: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, k_pages: torch.Tensor,
                    vt_pages: torch.Tensor, scale: float, cu_seqlens: torch.Tensor | None = None,
                    max_q: int | None = None, window: int = 0, sinks: int = 0,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal grouped-query attention of q [tokens, n_heads, hd] (paged_append's) over the pages, which
    hold the tokens' own k and v: the token at position p sees the positions j <= p of its sequence
    with window == 0, j > p - window or j < sinks. max_q: the most new tokens that a sequence has (a
    host number that chooses the launch; rows past it are not computed; None: as many as there are
    rows). Returns [tokens, n_heads, hd]; a token that sees nothing gives zeros. scale > 0."""
    return _attend("paged_attention", q, kv_lens, block_table, None, 0, k_pages, vt_pages, scale, cu_seqlens, max_q,
                   window, sinks, out)


def shared_prefix_attention(q: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor,
                            prefix_table: torch.Tensor, prefix_len: int, k_pages: torch.Tensor,
                            vt_pages: torch.Tensor, scale: float, cu_seqlens: torch.Tensor | None = None,
                            max_q: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """paged_attention (no window) for a batch whose sequences share their first prefix_len positions,
    whole pages: those are read through prefix_table (int32 [>= prefix_len / page]) once for all
    sequences instead of once for each, the rest through block_table, whose entries before them are not
    read. kv_lens counts the prefix; a sequence shorter than it sees its part of it."""
    if prefix_len <= 0:
        raise ValueError(f"shared_prefix_attention: prefix_len={prefix_len} must be positive (paged_attention "
                         "serves a batch without a prefix)")
    return _attend("shared_prefix_attention", q, kv_lens, block_table, prefix_table, prefix_len, k_pages, vt_pages,
                   scale, cu_seqlens, max_q, 0, 0, out)
