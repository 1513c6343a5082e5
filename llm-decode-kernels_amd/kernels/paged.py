"""Several sequences over one cache of pages on gfx950 (libldk_amd.so): `paged_append` rotates the new
tokens' q and k and writes k and v into the pages (`ldk_paged_append`), `paged_attention` attends over
them, in full or over a sliding window with a few first positions that stay visible
(`ldk_paged_attention`), and `shared_prefix_attention` does so for a batch whose sequences begin with
the same pages, which it reads once for tokens that are few (`ldk_shared_prefix_attention`).

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


_CODES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


# The checks below run on every call of every layer of a step, so they read each property once and test
# the good case in one expression; what is wrong is found out when something is.
def _pool(k_pages: torch.Tensor, vt_pages: torch.Tensor, what: str):
    """(pages, n_kv, page, head_dim, k page stride, vt page stride) of a pool, checked."""
    ks, vs = k_pages.shape, vt_pages.shape
    if len(ks) != 7 or len(vs) != 6:
        raise ValueError(f"{what}: k_pages and vt_pages must be k_pages_shape and vt_pages_shape, got "
                         f"{tuple(ks)} and {tuple(vs)}")
    pages, nkv, cpp, halves, steps, rows, dims = ks
    if halves != 2 or rows != 16 or dims != 32 or vs != (pages, nkv, cpp, 2 * steps, 16, 32):
        raise ValueError(f"{what}: k_pages and vt_pages must be k_pages_shape and vt_pages_shape of one pool, "
                         f"got {tuple(ks)} and {tuple(vs)}")
    if k_pages.dtype is not vt_pages.dtype:
        raise ValueError(f"{what}: k_pages {k_pages.dtype} and vt_pages {vt_pages.dtype} differ")
    per = nkv * cpp * steps * (CHUNK * 32)
    if k_pages.is_contiguous() and vt_pages.is_contiguous():
        return pages, nkv, cpp * CHUNK, steps * 32, per, per
    for t in (k_pages, vt_pages):
        if not (t.is_contiguous() or (pages and t[0].is_contiguous())):
            raise ValueError(f"{what}: a page's tiles must be contiguous")
    return (pages, nkv, cpp * CHUNK, steps * 32, k_pages.stride(0) if pages > 1 else per,
            vt_pages.stride(0) if pages > 1 else per)


def _batch(kv_lens: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor | None, rows: int, what: str):
    """(B, max_pages, table row stride), of checked lengths, table and row bounds."""
    if kv_lens.dtype is not torch.int32 or kv_lens.dim() != 1 or not kv_lens.is_contiguous():
        raise ValueError(f"{what}: kv_lens must be a contiguous int32 [B]")
    B = kv_lens.shape[0]
    ts = block_table.shape
    if block_table.dtype is not torch.int32 or len(ts) != 2 or ts[0] != B or not (
            block_table.is_contiguous() or ts[1] <= 1 or block_table.stride(1) == 1):
        raise ValueError(f"{what}: block_table must be int32 [{B}, max_pages] with contiguous rows")
    if cu_seqlens is None:
        if rows < B:
            raise ValueError(f"{what}: {rows} rows for {B} sequences of one token (cu_seqlens=None)")
    elif cu_seqlens.dtype is not torch.int32 or cu_seqlens.shape != (B + 1,) or not cu_seqlens.is_contiguous():
        raise ValueError(f"{what}: cu_seqlens must be a contiguous int32 [{B + 1}]")
    return B, ts[1], block_table.stride(0) if B > 1 else ts[1]


def _rows3(t: torch.Tensor, rows: int, heads: int, hd: int, dtype: torch.dtype, what: str, name: str) -> int:
    """The row stride of t [rows, heads, hd] with contiguous heads; 0: its heads are not."""
    if t.shape != (rows, heads, hd) or t.dtype is not dtype:
        raise ValueError(f"{what}: {name} must be {dtype} [{rows}, {heads}, {hd}], got {t.dtype} {tuple(t.shape)}")
    if t.is_contiguous():
        return heads * hd
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != hd):
        return 0
    return t.stride(0) if rows > 1 else heads * hd


def _out_stride(out: torch.Tensor, rows: int, heads: int, hd: int, dtype: torch.dtype, what: str) -> int:
    ldo = _rows3(out, rows, heads, hd, dtype, what, "out")
    if not ldo:
        raise ValueError(f"{what}: out must have contiguous heads, got strides {out.stride()}")
    return ldo


def _device(what: str, first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """The index of the GPU that all tensors are on."""
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            dev = -1
    if dev < 0:
        _lib.require_gpu(first, *others, what=what)
    return dev


def _call(entry, dev: int, args: tuple, what: str) -> None:
    """entry(*args, the device's current stream), with that device current. The callers hold the tensors
    whose addresses the arguments are."""
    cur = torch._C._cuda_getDevice()
    if cur == dev:
        st = entry(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with _lib.device_guard(torch.device("cuda", dev)):
            st = entry(*args, torch._C._cuda_getCurrentRawStream(dev))
    if st:
        _lib.check(st, what)


def _addr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def paged_append(qkv: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, k_pages: torch.Tensor,
                 vt_pages: torch.Tensor, inv_freq: torch.Tensor | None, n_heads: int,
                 cu_seqlens: torch.Tensor | None = None, rope_pos: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """qkv [tokens, (n_heads + 2 n_kv) * hd], the projection's rows, in the cache's dtype; inv_freq fp32
    [hd/2], or None for no rotation; rope_pos int64 [tokens]: positions to turn q and k by instead of
    their cache positions. Writes the rotated k and v at their positions' pages and returns the
    rotated q [tokens, n_heads, hd], into `out` where given (which may be qkv's own q columns).
    Angles are reduced in 64 bits, the rotation is fp32, rounded once. A token at a position without a page
    (below 0, where kv_lens is below the new tokens' number, too) has its q turned and writes no k and v.
    Two tokens of one call may not share a position of a page."""
    what = "paged_append"
    pages, nkv, page, hd, kst, vst = _pool(k_pages, vt_pages, what)
    width = (n_heads + 2 * nkv) * hd
    dtype = qkv.dtype
    if qkv.dim() != 2 or qkv.shape[1] != width or dtype is not k_pages.dtype:
        raise ValueError(f"{what}: qkv must be {k_pages.dtype} [tokens, {width}], got {qkv.dtype} {tuple(qkv.shape)}")
    T = qkv.shape[0]
    B, max_pages, ldt = _batch(kv_lens, block_table, cu_seqlens, T, what)
    if inv_freq is not None and (inv_freq.dtype is not torch.float32 or inv_freq.shape != (hd // 2,)
                                 or not inv_freq.is_contiguous()):
        raise ValueError(f"{what}: inv_freq must be a contiguous float32 [{hd // 2}]")
    if rope_pos is not None and (rope_pos.dtype is not torch.int64 or rope_pos.shape != (T,)
                                 or not rope_pos.is_contiguous()):
        raise ValueError(f"{what}: rope_pos must be a contiguous int64 [{T}]")
    ldq = n_heads * hd if out is None else _out_stride(out, T, n_heads, hd, dtype, what)
    dev = _device(what, qkv, kv_lens, block_table, k_pages, vt_pages, inv_freq, cu_seqlens, rope_pos, out)
    q = torch.empty((T, n_heads, hd), dtype=dtype, device=qkv.device) if out is None else out
    if not T or not B:
        return q
    x = qkv
    if not x.is_contiguous() and (x.stride(1) != 1 or (T > 1 and x.stride(0) % 8)):
        x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    _call(_lib.load().ldk_paged_append, dev,
          (x.data_ptr(), x.stride(0) if T > 1 else width, _CODES.get(dtype, -1), _addr(cu_seqlens), kv_lens.data_ptr(),
           block_table.data_ptr(), ldt, max_pages, _addr(rope_pos), _addr(inv_freq), k_pages.data_ptr(), kst,
           vt_pages.data_ptr(), vst, pages, page, q.data_ptr(), ldq, T, B, n_heads, nkv, hd), what)
    return q


def _attend(what, q, kv_lens, block_table, prefix_table, prefix_len, k_pages, vt_pages, scale, cu_seqlens, max_q, window,
            sinks, out):
    pages, nkv, page, hd, kst, vst = _pool(k_pages, vt_pages, what)
    dtype = k_pages.dtype
    if q.dim() != 3:
        raise ValueError(f"{what}: q must be {dtype} [tokens, heads, {hd}], got {q.dtype} {tuple(q.shape)}")
    T, nq, _ = q.shape
    ldq = _rows3(q, T, nq, hd, dtype, what, "q")
    B, max_pages, ldt = _batch(kv_lens, block_table, cu_seqlens, T, what)
    if prefix_table is not None and (prefix_table.dtype is not torch.int32 or prefix_table.dim() != 1
                                     or prefix_table.shape[0] * page < prefix_len or not prefix_table.is_contiguous()):
        raise ValueError(f"{what}: prefix_table must be a contiguous int32 of at least {prefix_len // page} pages")
    ldo = nq * hd if out is None else _out_stride(out, T, nq, hd, dtype, what)
    dev = _device(what, q, kv_lens, block_table, prefix_table, k_pages, vt_pages, cu_seqlens, out)
    if out is not None:
        o = out
    else:  # (a copy of a contiguous q's form takes the least time)
        o = torch.empty_like(q) if q.is_contiguous() else torch.empty((T, nq, hd), dtype=dtype, device=q.device)
    if not T or not B:
        return o
    x = q
    if not ldq or ldq % 8:
        x, ldq = x.contiguous(), nq * hd
    if x.data_ptr() % 16:
        x, ldq = x.clone(memory_format=torch.contiguous_format), nq * hd
    if cu_seqlens is None:
        max_q = 1
    elif max_q is None:
        max_q = T
    lib = _lib.load()
    need = lib.ldk_paged_attention_workspace_bytes(T if cu_seqlens is not None else B, B, max_q, max_pages * page, window, sinks,
                                                   prefix_len, nq, nkv, hd)
    if need < 0:
        _lib.check(-need, what)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    head = (x.data_ptr(), ldq, _CODES.get(dtype, -1), _addr(cu_seqlens), kv_lens.data_ptr(), block_table.data_ptr(), ldt,
            max_pages)
    pool = (k_pages.data_ptr(), kst, vt_pages.data_ptr(), vst, pages, page, o.data_ptr(), ldo, T, B, max_q, nq, nkv, hd)
    if prefix_table is None:
        _call(lib.ldk_paged_attention, dev, head + pool + (window, sinks, scale, _addr(ws), need), what)
    else:
        _call(lib.ldk_shared_prefix_attention, dev,
              head + (prefix_table.data_ptr(), prefix_len) + pool + (scale, _addr(ws), need), what)
    return o


def paged_attention(q: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, k_pages: torch.Tensor,
                    vt_pages: torch.Tensor, scale: float, cu_seqlens: torch.Tensor | None = None,
                    max_q: int | None = None, window: int = 0, sinks: int = 0,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal grouped-query attention of q [tokens, n_heads, hd] (paged_append's) over the pages, which
    hold the tokens' own k and v: the token at position p sees the positions j <= p of its sequence
    with window == 0, j > p - window or j < sinks. max_q: the most new tokens that a sequence has (a
    host number that chooses the launch; rows past it are not computed; None: as many as there are
    rows). Returns [tokens, n_heads, hd]; a token that sees nothing gives zeros. scale > 0.

    k may hold anything at positions that a token does not see, v at those that no token of the call
    sees (its weights are 0, and 0 x NaN is NaN). max_q chooses one kernel for the call: a batch that
    decodes over long contexts beside prompts runs faster as two calls."""
    return _attend("paged_attention", q, kv_lens, block_table, None, 0, k_pages, vt_pages, scale, cu_seqlens, max_q,
                   window, sinks, out)


def shared_prefix_attention(q: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor,
                            prefix_table: torch.Tensor, prefix_len: int, k_pages: torch.Tensor,
                            vt_pages: torch.Tensor, scale: float, cu_seqlens: torch.Tensor | None = None,
                            max_q: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """paged_attention (no window) for a batch whose sequences share their first prefix_len positions,
    whole pages: those are read through prefix_table (int32 [>= prefix_len / page]), the rest through
    block_table, whose entries before them are not read. The prefix is read once for all sequences where
    max_q * n_heads / n_kv <= 128, else by each sequence's rows for themselves, as paged_attention does: a
    batch of single tokens beside a prompt runs faster as two calls. kv_lens counts the prefix; a sequence
    shorter than it sees its part of it."""
    if prefix_len <= 0:
        raise ValueError(f"shared_prefix_attention: prefix_len={prefix_len} must be positive (paged_attention "
                         "serves a batch without a prefix)")
    return _attend("shared_prefix_attention", q, kv_lens, block_table, prefix_table, prefix_len, k_pages, vt_pages,
                   scale, cu_seqlens, max_q, 0, 0, out)
