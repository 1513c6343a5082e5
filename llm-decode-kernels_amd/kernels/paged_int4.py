"""The paged cache of kernels.paged held in 4 bits, on gfx950 (libldk_amd.so): `paged_append_int4` rotates the new
tokens' q and k and quantises k and v into the pages (`ldk_paged_append_int4`), `paged_attention_int4` attends over them
(`ldk_paged_attention_int4`), and `paged_read_int4` gives the values back as rows (`ldk_paged_read_int4`).

A step of ragged sequences, as with kernels.paged:

    q = paged_append_int4(qkv, kv_lens, block_table, kv_pages, inv_freq, n_heads, cu_seqlens)
    o = paged_attention_int4(q, kv_lens, block_table, kv_pages, scale, cu_seqlens, max_q)

- kv_pages [pages, n_kv, page/32, words], fp16 or bf16 (the type of qkv and q, and of the steps and offsets that it
  holds beside the codes): `kv_int4_shape`. page a multiple of 32, hd 64 or 128. The first dimension may have any stride,
  the others are contiguous. It holds both k and v: per kv head and position hd bytes of codes and 8 bytes per
  group, 3.8 (group 128) to 3.2 (32) times less than 16-bit pages.
- Each position's k and v are quantised for themselves, per kv head and group of 32, 64 or 128 dims, to value = z + (code - 8)
  step with codes 0..15 over the group's range. Smaller groups follow dims of unlike sizes, as k's often are, at 0.25
  bits per value for each halving from 128 to 64, 0.5 to 32. step and z are rounded to the dtype, so that a group far from 0
  is held to its offset's rounding. A group with a NaN or an infinity reads as NaN.
- block_table, kv_lens and cu_seqlens are kernels.paged's, absent pages and padded batches too. Two sequences of a call may
  append to one page, as each byte is one position's alone, but not at one position.

The reference keeps one static fp16 cache (kernels/e2e/model.py:192-243) and has no counterpart.
"""

from __future__ import annotations

import torch

from kernels import _lib
from kernels.attention import CHUNK
from kernels.paged import _CODES, _addr, _batch, _call, _device, _out_stride, _rows3

# words of a chunk's block: its head_dim and groups
_BLOCKS = {16 * hd + 128 * n: (hd, n) for hd in (64, 128) for n in (1, 2, 4) if hd // n >= 32}


def kv_int4_shape(pages: int, n_kv: int, page: int, head_dim: int = 128, group: int | None = None) -> tuple:
    """The shape of kv_pages; group None: one per head."""
    words = 16 * head_dim + 128 * (head_dim // (group or head_dim))
    if _BLOCKS.get(words) != (head_dim, head_dim // (group or head_dim)) or head_dim % (group or head_dim):
        raise ValueError(f"kv_int4_shape: head_dim={head_dim} (64 or 128) in groups of {group} (32, 64 or 128, at most head_dim)")
    if page % CHUNK:
        raise ValueError(f"kv_int4_shape: page={page} must be a multiple of {CHUNK}")
    return (pages, n_kv, page // CHUNK, words)


def _pool(kv_pages: torch.Tensor, what: str):
    """(pages, n_kv, page, head_dim, group, page stride) of a pool, checked."""
    shape = kv_pages.shape
    if len(shape) != 4 or shape[3] not in _BLOCKS:
        raise ValueError(f"{what}: kv_pages must be kv_int4_shape, got {tuple(shape)}")
    pages, nkv, cpp, words = shape
    hd, groups = _BLOCKS[words]
    per = nkv * cpp * words
    if kv_pages.is_contiguous():
        return pages, nkv, cpp * CHUNK, hd, hd // groups, per
    if not (pages and kv_pages[0].is_contiguous()):
        raise ValueError(f"{what}: a page's blocks must be contiguous")
    return pages, nkv, cpp * CHUNK, hd, hd // groups, kv_pages.stride(0) if pages > 1 else per


def paged_append_int4(qkv: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, kv_pages: torch.Tensor,
                      inv_freq: torch.Tensor | None, n_heads: int, cu_seqlens: torch.Tensor | None = None,
                      rope_pos: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """kernels.paged.paged_append into 4-bit pages: qkv [tokens, (n_heads + 2 n_kv) * hd] in the pages' dtype; inv_freq fp32
    [hd/2], or None for no rotation; rope_pos int64 [tokens]: positions to turn q and k by instead of their cache
    positions. Quantises the rotated k and v into their positions' pages and returns the rotated q [tokens,
    n_heads, hd], into `out` where given (which may be qkv's own q columns). k is rotated in 64 bits and rounded
    to fp32, then to the dtype, before it is quantised. A token at a position without a page has its q turned
    and writes nothing. Two tokens of one call may not share a position of a page."""
    what = "paged_append_int4"
    pages, nkv, page, hd, group, stride = _pool(kv_pages, what)
    width = (n_heads + 2 * nkv) * hd
    dtype = qkv.dtype
    if qkv.dim() != 2 or qkv.shape[1] != width or dtype is not kv_pages.dtype:
        raise ValueError(f"{what}: qkv must be {kv_pages.dtype} [tokens, {width}], got {qkv.dtype} {tuple(qkv.shape)}")
    T = qkv.shape[0]
    B, max_pages, ldt = _batch(kv_lens, block_table, cu_seqlens, T, what)
    if inv_freq is not None and (inv_freq.dtype is not torch.float32 or inv_freq.shape != (hd // 2,)
                                 or not inv_freq.is_contiguous()):
        raise ValueError(f"{what}: inv_freq must be a contiguous float32 [{hd // 2}]")
    if rope_pos is not None and (rope_pos.dtype is not torch.int64 or rope_pos.shape != (T,)
                                 or not rope_pos.is_contiguous()):
        raise ValueError(f"{what}: rope_pos must be a contiguous int64 [{T}]")
    ldq = n_heads * hd if out is None else _out_stride(out, T, n_heads, hd, dtype, what)
    dev = _device(what, qkv, kv_lens, block_table, kv_pages, inv_freq, cu_seqlens, rope_pos, out)
    q = torch.empty((T, n_heads, hd), dtype=dtype, device=qkv.device) if out is None else out
    if not T or not B:
        return q
    x = qkv
    if not x.is_contiguous() and (x.stride(1) != 1 or (T > 1 and x.stride(0) % 8)):
        x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    _call(_lib.load().ldk_paged_append_int4, dev,
          (x.data_ptr(), x.stride(0) if T > 1 else width, _CODES.get(dtype, -1), _addr(cu_seqlens), kv_lens.data_ptr(),
           block_table.data_ptr(), ldt, max_pages, _addr(rope_pos), _addr(inv_freq), kv_pages.data_ptr(), stride, pages, page,
           q.data_ptr(), ldq, T, B, n_heads, nkv, hd, group), what)
    return q


def paged_read_int4(kv_lens: torch.Tensor, block_table: torch.Tensor, kv_pages: torch.Tensor, rows: int | None = None,
                    cu_seqlens: torch.Tensor | None = None,
                    out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The values that the pages hold, (k, v), each [rows, n_kv, hd] of the pages' dtype: the rows cu_seqlens[b]:
    cu_seqlens[b + 1] are the last of sequence b's kv_lens[b] positions (None: its last position, row b), z + (code - 8)
    step rounded once, at most the dtype's largest number. rows: as many as cu_seqlens ends with, or more (a host number;
    without cu_seqlens or with `out` it need not be given). Rows at positions without a page, or below 0, are zeros; rows
    behind the last sequence's are left as they were (of outputs that are not given: undefined)."""
    what = "paged_read_int4"
    pages, nkv, page, hd, group, stride = _pool(kv_pages, what)
    dtype = kv_pages.dtype
    if rows is None:
        if out is None and cu_seqlens is not None:
            raise ValueError(f"{what}: rows must be given with cu_seqlens")
        rows = kv_lens.shape[0] if out is None else out[0].shape[0]
    B, max_pages, ldt = _batch(kv_lens, block_table, cu_seqlens, rows, what)
    ld = [nkv * hd] * 2 if out is None else [_out_stride(t, rows, nkv, hd, dtype, what) for t in out]
    dev = _device(what, kv_pages, kv_lens, block_table, cu_seqlens, *(out or ()))
    if out is None:
        out = tuple(torch.empty((2, rows, nkv, hd), dtype=dtype, device=kv_pages.device))
    k, v = out
    if not rows or not B:
        return k, v
    _call(_lib.load().ldk_paged_read_int4, dev,
          (_CODES.get(dtype, -1), _addr(cu_seqlens), kv_lens.data_ptr(), block_table.data_ptr(), ldt, max_pages,
           kv_pages.data_ptr(), stride, pages, page, k.data_ptr(), ld[0], v.data_ptr(), ld[1], rows, B, nkv, hd, group), what)
    return k, v


def paged_attention_int4(q: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, kv_pages: torch.Tensor,
                         scale: float, cu_seqlens: torch.Tensor | None = None, max_q: int | None = None, window: int = 0,
                         sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """kernels.paged.paged_attention over 4-bit pages: causal grouped-query attention of q [tokens, n_heads, hd]
    (paged_append_int4's) over the values that the pages hold, the tokens' own k and v included. The token at position p
    sees the positions j <= p of its sequence with window == 0, j > p - window or j < sinks. max_q: the most new
    tokens that a sequence has (a host number that chooses the launch; rows past it are not computed; None: as many as
    there are rows). Returns [tokens, n_heads, hd]; a token that sees nothing gives zeros. scale > 0.

    A NaN in a position's k or v reaches the tokens that see it and no other. bf16 k and v are taken up to 2^90 in size.
    max_q chooses one kernel for the call: a batch that decodes over long contexts beside prompts runs faster as two calls."""
    what = "paged_attention_int4"
    pages, nkv, page, hd, group, stride = _pool(kv_pages, what)
    dtype = kv_pages.dtype
    if q.dim() != 3:
        raise ValueError(f"{what}: q must be {dtype} [tokens, heads, {hd}], got {q.dtype} {tuple(q.shape)}")
    T, nq, _ = q.shape
    ldq = _rows3(q, T, nq, hd, dtype, what, "q")
    B, max_pages, ldt = _batch(kv_lens, block_table, cu_seqlens, T, what)
    ldo = nq * hd if out is None else _out_stride(out, T, nq, hd, dtype, what)
    dev = _device(what, q, kv_lens, block_table, kv_pages, cu_seqlens, out)
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
    need = lib.ldk_paged_attention_int4_workspace_bytes(T if cu_seqlens is not None else B, B, max_q, max_pages * page,
                                                        window, sinks, nq, nkv, hd)
    if need < 0:
        _lib.check(-need, what)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _call(lib.ldk_paged_attention_int4, dev,
          (x.data_ptr(), ldq, _CODES.get(dtype, -1), _addr(cu_seqlens), kv_lens.data_ptr(), block_table.data_ptr(), ldt,
           max_pages, kv_pages.data_ptr(), stride, pages, page, o.data_ptr(), ldo, T, B, max_q, nq, nkv, hd, group, window,
           sinks, scale, _addr(ws), need), what)
    return o
