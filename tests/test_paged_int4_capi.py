"""kernels.paged_int4's argument checks on the CPU: the C entries refuse bad arguments with a status and a message before
any launch, the Python wrappers before the library is called."""

import ctypes

import pytest
import torch

from kernels import _lib, paged_int4

P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4104)  # 8-byte aligned only
PAGE = 2 * 2 * (16 * 128 + 128)  # words of a page: 2 kv heads, 2 chunks, group 128


def status(st):
    return st, _lib.load().ldk_last_error().decode()


BASE = dict(dtype=_lib.F16, cu=None, kv=P, table=P, ldt=8, max_pages=8, pool=P, stride=PAGE, pages=10, page=64, T=4, B=4, nq=12,
            nkv=2, hd=128, group=128)


def append(**kw):
    a = {**BASE, **dict(qkv=P, ldqkv=16 * 128, rope_pos=None, inv=P, q=P, ldq=12 * 128), **kw}
    return status(_lib.load().ldk_paged_append_int4(
        a["qkv"], a["ldqkv"], a["dtype"], a["cu"], a["kv"], a["table"], a["ldt"], a["max_pages"], a["rope_pos"], a["inv"],
        a["pool"], a["stride"], a["pages"], a["page"], a["q"], a["ldq"], a["T"], a["B"], a["nq"], a["nkv"], a["hd"], a["group"], None))


def read(**kw):
    a = {**BASE, **dict(k=P, v=P, ldk=256, ldv=256), **kw}
    return status(_lib.load().ldk_paged_read_int4(
        a["dtype"], a["cu"], a["kv"], a["table"], a["ldt"], a["max_pages"], a["pool"], a["stride"], a["pages"], a["page"], a["k"],
        a["ldk"], a["v"], a["ldv"], a["T"], a["B"], a["nkv"], a["hd"], a["group"], None))


def attend(**kw):
    a = {**BASE, **dict(q=P, ldq=12 * 128, out=P, ldo=12 * 128, max_q=1, window=0, sinks=0, scale=0.1, ws=P, ws_bytes=1 << 40), **kw}
    return status(_lib.load().ldk_paged_attention_int4(
        a["q"], a["ldq"], a["dtype"], a["cu"], a["kv"], a["table"], a["ldt"], a["max_pages"], a["pool"], a["stride"], a["pages"],
        a["page"], a["out"], a["ldo"], a["T"], a["B"], a["max_q"], a["nq"], a["nkv"], a["hd"], a["group"], a["window"], a["sinks"],
        a["scale"], a["ws"], a["ws_bytes"], None))


COMMON = [(dict(kv=None), _lib.ERR_INVALID), (dict(table=None), _lib.ERR_INVALID), (dict(pool=None), _lib.ERR_INVALID),
          (dict(dtype=_lib.F32), _lib.ERR_INVALID), (dict(hd=96), _lib.ERR_UNSUPPORTED), (dict(group=16), _lib.ERR_UNSUPPORTED),
          (dict(group=256), _lib.ERR_UNSUPPORTED), (dict(hd=64, group=128), _lib.ERR_UNSUPPORTED), (dict(group=0), _lib.ERR_UNSUPPORTED),
          (dict(nkv=0), _lib.ERR_INVALID), (dict(T=0), _lib.ERR_INVALID), (dict(T=(1 << 24) + 1), _lib.ERR_INVALID),
          (dict(B=0), _lib.ERR_INVALID), (dict(B=5), _lib.ERR_INVALID), (dict(page=48), _lib.ERR_UNSUPPORTED),
          (dict(page=0), _lib.ERR_UNSUPPORTED), (dict(pages=0), _lib.ERR_INVALID), (dict(max_pages=0), _lib.ERR_INVALID),
          (dict(ldt=7), _lib.ERR_INVALID), (dict(max_pages=1 << 26, ldt=1 << 26), _lib.ERR_INVALID),
          (dict(stride=PAGE - 8), _lib.ERR_INVALID), (dict(group=32), _lib.ERR_INVALID), (dict(stride=1 << 31), _lib.ERR_UNSUPPORTED),
          (dict(stride=PAGE + 4), _lib.ERR_ALIGN), (dict(pool=ODD), _lib.ERR_ALIGN), (dict(kv=ctypes.c_void_p(4098)), _lib.ERR_ALIGN)]
HEADS = [(dict(nq=13), _lib.ERR_INVALID), (dict(nq=0), _lib.ERR_INVALID), (dict(nq=8192), _lib.ERR_INVALID)]


@pytest.mark.parametrize("kw,code", COMMON + HEADS + [
    (dict(qkv=None), _lib.ERR_INVALID), (dict(q=None), _lib.ERR_INVALID), (dict(ldqkv=16 * 128 - 8), _lib.ERR_INVALID),
    (dict(ldq=12 * 128 - 8), _lib.ERR_INVALID), (dict(qkv=ODD), _lib.ERR_ALIGN), (dict(q=ODD), _lib.ERR_ALIGN),
    (dict(ldqkv=16 * 128 + 4), _lib.ERR_ALIGN), (dict(rope_pos=ctypes.c_void_p(4100)), _lib.ERR_ALIGN)])
def test_append_refuses(kw, code):
    st, msg = append(**kw)
    assert st == code and "paged_append_int4" in msg


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(k=None), _lib.ERR_INVALID), (dict(v=None), _lib.ERR_INVALID), (dict(ldk=248), _lib.ERR_INVALID),
    (dict(ldv=248), _lib.ERR_INVALID), (dict(k=ODD), _lib.ERR_ALIGN), (dict(v=ODD), _lib.ERR_ALIGN), (dict(ldv=260), _lib.ERR_ALIGN)])
def test_read_refuses(kw, code):
    st, msg = read(**kw)
    assert st == code and "paged_read_int4" in msg


LONG = dict(max_pages=128, ldt=128)  # tables long enough for a workspace


@pytest.mark.parametrize("kw,code", COMMON + HEADS + [
    (dict(q=None), _lib.ERR_INVALID), (dict(out=None), _lib.ERR_INVALID), (dict(max_q=0), _lib.ERR_INVALID),
    (dict(max_q=5), _lib.ERR_INVALID), (dict(window=-1), _lib.ERR_INVALID), (dict(sinks=-1), _lib.ERR_INVALID),
    (dict(scale=0.0), _lib.ERR_INVALID), (dict(scale=-1.0), _lib.ERR_INVALID), (dict(scale=float("nan")), _lib.ERR_INVALID),
    (dict(ws=None, **LONG), _lib.ERR_INVALID), (dict(ws_bytes=16, **LONG), _lib.ERR_INVALID), (dict(ldo=12 * 128 - 8), _lib.ERR_INVALID),
    (dict(T=65536, B=65536), _lib.ERR_INVALID), (dict(ldo=12 * 128 + 4), _lib.ERR_ALIGN), (dict(out=ODD), _lib.ERR_ALIGN),
    (dict(ws=ODD), _lib.ERR_ALIGN)])
def test_attention_refuses(kw, code):
    st, msg = attend(**kw)
    assert st == code and "paged_attention_int4" in msg


def test_workspace_queries():
    query = _lib.load().ldk_paged_attention_int4_workspace_bytes
    ok = (4, 4, 1, 8192, 0, 0, 12, 2, 128)
    assert query(*ok) > 0
    assert query(4, 4, 1, 256, 0, 0, 12, 2, 128) == 0
    for at, bad in ((0, 0), (1, 0), (1, 65536), (2, 0), (3, 0), (3, 1 << 26), (4, -1), (5, -1), (6, 13), (7, 0), (8, 96)):
        assert query(*ok[:at], bad, *ok[at + 1:]) == -_lib.ERR_INVALID


@pytest.mark.parametrize("B,new,gq,nkv,hd", [(201, 80, 4, 8, 128), (1001, 80, 4, 8, 128), (64, 45, 7, 4, 128), (9, 300, 1, 2, 64), (3000, 20, 8, 2, 128),
                                             (12, 2, 100, 1, 64)])
def test_workspace_follows_the_rows(B, new, gq, nkv, hd):
    """One prompt beside many tokens: partials of 16 rows of fp32 for the rows that there are (a sequence's last 16 not full) and for
    ranges past each sequence's first, not for as many as the longest has of every sequence."""
    lib = _lib.load()
    T, tile = B - 1 + new, 16 * (2 + hd) * 4
    need = lib.ldk_paged_attention_int4_workspace_bytes(T, B, new, 65536, 0, 0, gq * nkv, nkv, hd)
    tiles, longest = T * gq // 16 + B, -(-new * gq // 16)
    plan = 4 * (2 * B + 1 + B + 512 + B // 4)
    assert 0 < need <= (1.25 * tiles + 512 // nkv + longest) * nkv * tile + plan


# ------------------------------------------------------------------------------- the Python wrappers
@pytest.mark.parametrize("hd,group", [(128, None), (128, 128), (128, 64), (128, 32), (64, None), (64, 32)])
def test_shape(hd, group):
    shape = paged_int4.kv_int4_shape(5, 3, 96, hd, group)
    assert shape == (5, 3, 3, 16 * hd + 128 * hd // (group or hd))
    # bytes of a position: codes of k and v, and 4 bytes of step and offset per group of each
    assert 2 * shape[3] == 32 * (hd + 8 * hd // (group or hd))


@pytest.mark.parametrize("page,hd,group", [(32, 96, None), (32, 128, 16), (32, 128, 48), (32, 64, 128), (48, 128, 128), (32, 256, 256), (32, 128, 256)])
def test_shape_refuses(page, hd, group):
    with pytest.raises(ValueError, match="kv_int4_shape"):
        paged_int4.kv_int4_shape(4, 2, page, hd, group)


def _args(**kw):
    a = dict(qkv=torch.zeros(3, 8 * 128, dtype=torch.float16), q=torch.zeros(3, 4, 128, dtype=torch.float16),
             kv=torch.ones(3, dtype=torch.int32), table=torch.zeros(3, 2, dtype=torch.int32),
             pool=torch.zeros(paged_int4.kv_int4_shape(4, 2, 64), dtype=torch.float16), inv=torch.zeros(64))
    return {**a, **kw}


def _append(cu=None, rope_pos=None, out=None, **kw):
    a = _args(**kw)
    return paged_int4.paged_append_int4(a["qkv"], a["kv"], a["table"], a["pool"], a["inv"], 4, cu_seqlens=cu, rope_pos=rope_pos, out=out)


def _attend(cu=None, out=None, **kw):
    a = _args(**kw)
    return paged_int4.paged_attention_int4(a["q"], a["kv"], a["table"], a["pool"], 0.1, cu_seqlens=cu, out=out)


def _read(cu=None, out=None, rows=3, **kw):
    a = _args(**kw)
    return paged_int4.paged_read_int4(a["kv"], a["table"], a["pool"], rows, cu_seqlens=cu, out=out)


@pytest.mark.parametrize("call", [_append, _attend, _read])
@pytest.mark.parametrize("kw,match", [
    (dict(kv=torch.ones(3, dtype=torch.int64)), "kv_lens"), (dict(kv=torch.ones(6, dtype=torch.int32)[::2]), "kv_lens"),
    (dict(table=torch.zeros(2, 2, dtype=torch.int32)), "block_table"), (dict(table=torch.zeros(3, 2)), "block_table"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int32).t()), "block_table"),
    (dict(cu=torch.zeros(3, dtype=torch.int32)), "cu_seqlens"), (dict(cu=torch.zeros(4, dtype=torch.int64)), "cu_seqlens"),
    (dict(pool=torch.zeros(4, 2, 64, 128, dtype=torch.float16)), "kv_pages"), (dict(pool=torch.zeros(4, 2, 2176, dtype=torch.float16)), "kv_pages"),
    (dict(pool=torch.zeros(4, 4, 2, 2176, dtype=torch.float16)[:, ::2]), "contiguous"),
    (dict(kv=torch.ones(4, dtype=torch.int32), table=torch.zeros(4, 2, dtype=torch.int32)), "rows")])
def test_wrappers_refuse(call, kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


@pytest.mark.parametrize("call", [_append, _attend])
@pytest.mark.parametrize("kw,match", [
    (dict(pool=torch.zeros(paged_int4.kv_int4_shape(4, 2, 64), dtype=torch.bfloat16)), "bfloat16"),
    (dict(out=torch.zeros(3, 5, 128, dtype=torch.float16)), "out"), (dict(out=torch.zeros(3, 4, 128)), "out"),
    (dict(out=torch.zeros(3, 128, 4, dtype=torch.float16).transpose(1, 2)), "out")])
def test_wrappers_refuse_outputs(call, kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


@pytest.mark.parametrize("kw,match", [(dict(qkv=torch.zeros(3, 7 * 128, dtype=torch.float16)), "qkv"),
                                      (dict(qkv=torch.zeros(3, 8 * 128)), "qkv"), (dict(inv=torch.zeros(32)), "inv_freq"),
                                      (dict(inv=torch.zeros(64).half()), "inv_freq"),
                                      (dict(rope_pos=torch.zeros(2, dtype=torch.int64)), "rope_pos"),
                                      (dict(rope_pos=torch.zeros(3, dtype=torch.int32)), "rope_pos")])
def test_append_wrapper_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _append(**kw)


def test_read_wrapper_refuses():
    row = torch.zeros(3, 2, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="rows must be given"):
        _read(cu=torch.zeros(4, dtype=torch.int32), rows=None)
    for bad in (row[:2], row.float(), row[:, :1], row.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError, match="out"):
            _read(out=(row, bad))


def test_wrappers_refuse_cpu_tensors():
    for call in (_append, _attend, _read):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
