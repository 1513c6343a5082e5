"""The paged operators' and token_logprobs' argument checks on the CPU: the C entries refuse bad arguments
with a status and a message before any launch, the Python wrappers before the library is called."""

import ctypes

import pytest
import torch

from kernels import _lib, paged
from kernels.sample import token_logprobs

P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4104)  # 8-byte aligned only


def status(st):
    return st, _lib.load().ldk_last_error().decode()


APPEND = dict(qkv=P, ldqkv=16 * 128, dtype=_lib.F16, cu=None, kv=P, table=P, ldt=8, max_pages=8, rope_pos=None, inv=P, k=P,
              kps=2 * 64 * 128, vt=P, vps=2 * 64 * 128, pages=10, page=64, q=P, ldq=12 * 128, T=4, B=4, nq=12, nkv=2, hd=128)


def append(**kw):
    a = {**APPEND, **kw}
    return status(_lib.load().ldk_paged_append(
        a["qkv"], a["ldqkv"], a["dtype"], a["cu"], a["kv"], a["table"], a["ldt"], a["max_pages"], a["rope_pos"], a["inv"],
        a["k"], a["kps"], a["vt"], a["vps"], a["pages"], a["page"], a["q"], a["ldq"], a["T"], a["B"], a["nq"], a["nkv"],
        a["hd"], None))


ATTEND = dict(q=P, ldq=12 * 128, dtype=_lib.F16, cu=None, kv=P, table=P, ldt=8, max_pages=8, k=P, kps=2 * 64 * 128, vt=P,
              vps=2 * 64 * 128, pages=10, page=64, out=P, ldo=12 * 128, T=4, B=4, max_q=1, nq=12, nkv=2, hd=128, window=0,
              sinks=0, scale=0.1, ws=P, ws_bytes=1 << 40)


def attend(**kw):
    a = {**ATTEND, **kw}
    return status(_lib.load().ldk_paged_attention(
        a["q"], a["ldq"], a["dtype"], a["cu"], a["kv"], a["table"], a["ldt"], a["max_pages"], a["k"], a["kps"], a["vt"],
        a["vps"], a["pages"], a["page"], a["out"], a["ldo"], a["T"], a["B"], a["max_q"], a["nq"], a["nkv"], a["hd"],
        a["window"], a["sinks"], a["scale"], a["ws"], a["ws_bytes"], None))


def prefix(ptable=P, prefix_len=128, **kw):
    a = {**ATTEND, **kw}
    return status(_lib.load().ldk_shared_prefix_attention(
        a["q"], a["ldq"], a["dtype"], a["cu"], a["kv"], a["table"], a["ldt"], a["max_pages"], ptable, prefix_len, a["k"],
        a["kps"], a["vt"], a["vps"], a["pages"], a["page"], a["out"], a["ldo"], a["T"], a["B"], a["max_q"], a["nq"],
        a["nkv"], a["hd"], a["scale"], a["ws"], a["ws_bytes"], None))


LONG = dict(max_pages=128, ldt=128)  # tables long enough for a workspace
COMMON = [(dict(kv=None), _lib.ERR_INVALID), (dict(table=None), _lib.ERR_INVALID), (dict(k=None), _lib.ERR_INVALID),
          (dict(vt=None), _lib.ERR_INVALID), (dict(dtype=_lib.F32), _lib.ERR_INVALID), (dict(hd=96), _lib.ERR_UNSUPPORTED),
          (dict(nq=13), _lib.ERR_INVALID), (dict(nq=0), _lib.ERR_INVALID), (dict(nkv=0), _lib.ERR_INVALID),
          (dict(T=0), _lib.ERR_INVALID), (dict(T=(1 << 24) + 1), _lib.ERR_INVALID), (dict(B=0), _lib.ERR_INVALID),
          (dict(B=5), _lib.ERR_INVALID), (dict(page=48), _lib.ERR_UNSUPPORTED), (dict(page=0), _lib.ERR_UNSUPPORTED),
          (dict(pages=0), _lib.ERR_INVALID), (dict(max_pages=0), _lib.ERR_INVALID), (dict(ldt=7), _lib.ERR_INVALID),
          (dict(max_pages=1 << 26, ldt=1 << 26), _lib.ERR_INVALID), (dict(kps=2 * 64 * 128 - 8), _lib.ERR_INVALID),
          (dict(vps=0), _lib.ERR_INVALID), (dict(kps=1 << 31), _lib.ERR_UNSUPPORTED), (dict(kps=2 * 64 * 128 + 4), _lib.ERR_ALIGN), (dict(k=ODD), _lib.ERR_ALIGN),
          (dict(vt=ODD), _lib.ERR_ALIGN), (dict(kv=ctypes.c_void_p(4098)), _lib.ERR_ALIGN)]


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(qkv=None), _lib.ERR_INVALID), (dict(q=None), _lib.ERR_INVALID), (dict(ldqkv=16 * 128 - 8), _lib.ERR_INVALID),
    (dict(ldq=12 * 128 - 8), _lib.ERR_INVALID), (dict(qkv=ODD), _lib.ERR_ALIGN), (dict(q=ODD), _lib.ERR_ALIGN),
    (dict(ldqkv=16 * 128 + 4), _lib.ERR_ALIGN), (dict(rope_pos=ctypes.c_void_p(4100)), _lib.ERR_ALIGN)])
def test_append_refuses(kw, code):
    st, msg = append(**kw)
    assert st == code and "paged_append" in msg


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(q=None), _lib.ERR_INVALID), (dict(out=None), _lib.ERR_INVALID), (dict(max_q=0), _lib.ERR_INVALID),
    (dict(max_q=5), _lib.ERR_INVALID), (dict(window=-1), _lib.ERR_INVALID), (dict(sinks=-1), _lib.ERR_INVALID),
    (dict(scale=0.0), _lib.ERR_INVALID), (dict(scale=-1.0), _lib.ERR_INVALID), (dict(scale=float("nan")), _lib.ERR_INVALID),
    (dict(ws=None, **LONG), _lib.ERR_INVALID), (dict(ws_bytes=16, **LONG), _lib.ERR_INVALID), (dict(ldo=12 * 128 - 8), _lib.ERR_INVALID),
    (dict(ldo=12 * 128 + 4), _lib.ERR_ALIGN), (dict(out=ODD), _lib.ERR_ALIGN), (dict(ws=ODD), _lib.ERR_ALIGN)])
def test_attention_refuses(kw, code):
    st, msg = attend(**kw)
    assert st == code and "paged_attention" in msg


@pytest.mark.parametrize("kw,code", [(dict(ptable=None), _lib.ERR_INVALID), (dict(prefix_len=100), _lib.ERR_INVALID),
                                     (dict(prefix_len=64 * 9), _lib.ERR_INVALID), (dict(prefix_len=-64), _lib.ERR_INVALID),
                                     (dict(scale=0.0), _lib.ERR_INVALID), (dict(ws_bytes=16), _lib.ERR_INVALID)])
def test_prefix_refuses(kw, code):
    st, msg = prefix(**kw)
    assert st == code and "shared_prefix_attention" in msg


def test_workspace_queries():
    lib = _lib.load()
    ok = (4, 4, 1, 8192, 0, 0, 0, 12, 2, 128)
    assert lib.ldk_paged_attention_workspace_bytes(*ok) > 0
    assert lib.ldk_paged_attention_workspace_bytes(4, 4, 1, 512, 0, 0, 0, 12, 2, 128) == 0
    for at, bad in ((0, 0), (1, 0), (1, 65536), (2, 0), (3, 0), (3, 1 << 26), (4, -1), (5, -1), (6, -1), (7, 13), (8, 0), (9, 96)):
        assert lib.ldk_paged_attention_workspace_bytes(*ok[:at], bad, *ok[at + 1:]) == -_lib.ERR_INVALID
    assert lib.ldk_token_logprobs_workspace_bytes(2000, 1000, 5) == 0
    for bad in ((0, 10, 1), (1, 0, 0), (1, 10, 11), (1, 100, 65), (1, 10, -1)):
        assert lib.ldk_token_logprobs_workspace_bytes(*bad) == -_lib.ERR_INVALID


def logprobs(x=P, ld=100, dtype=_lib.F32, tok=P, rows=2, V=100, top=3, lp=P, ent=P, tl=P, ti=P, ws=P, ws_bytes=1 << 30):
    return status(_lib.load().ldk_token_logprobs(x, ld, dtype, tok, rows, V, top, lp, ent, tl, ti, ws, ws_bytes, None))


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), _lib.ERR_INVALID), (dict(tok=None), _lib.ERR_INVALID), (dict(lp=None), _lib.ERR_INVALID),
    (dict(ent=None), _lib.ERR_INVALID), (dict(tl=None), _lib.ERR_INVALID), (dict(ti=None), _lib.ERR_INVALID),
    (dict(rows=0), _lib.ERR_INVALID), (dict(V=0), _lib.ERR_INVALID), (dict(top=101), _lib.ERR_INVALID),
    (dict(top=65), _lib.ERR_INVALID), (dict(ld=99), _lib.ERR_INVALID), (dict(dtype=7), _lib.ERR_INVALID),
    (dict(x=ctypes.c_void_p(4098)), _lib.ERR_ALIGN), (dict(tok=ctypes.c_void_p(4100)), _lib.ERR_ALIGN),
    (dict(rows=1, V=100000, ld=100000, ws=None, ws_bytes=0), _lib.ERR_INVALID)])
def test_logprobs_refuses(kw, code):
    st, msg = logprobs(**kw)
    assert st == code and "token_logprobs" in msg


# ------------------------------------------------------------------------------- the Python wrappers
def _args(**kw):
    a = dict(qkv=torch.zeros(3, 8 * 128, dtype=torch.float16), q=torch.zeros(3, 4, 128, dtype=torch.float16),
             kv=torch.ones(3, dtype=torch.int32), table=torch.zeros(3, 2, dtype=torch.int32),
             k=torch.zeros(paged.k_pages_shape(4, 2, 64), dtype=torch.float16),
             vt=torch.zeros(paged.vt_pages_shape(4, 2, 64), dtype=torch.float16), inv=torch.zeros(64))
    return {**a, **kw}


def _append(cu=None, rope_pos=None, out=None, **kw):
    a = _args(**kw)
    return paged.paged_append(a["qkv"], a["kv"], a["table"], a["k"], a["vt"], a["inv"], 4, cu_seqlens=cu, rope_pos=rope_pos, out=out)


def _attend(cu=None, out=None, **kw):
    a = _args(**kw)
    return paged.paged_attention(a["q"], a["kv"], a["table"], a["k"], a["vt"], 0.1, cu_seqlens=cu, out=out)


@pytest.mark.parametrize("call", [_append, _attend])
@pytest.mark.parametrize("kw,match", [
    (dict(kv=torch.ones(3, dtype=torch.int64)), "kv_lens"), (dict(kv=torch.ones(6, dtype=torch.int32)[::2]), "kv_lens"),
    (dict(table=torch.zeros(2, 2, dtype=torch.int32)), "block_table"), (dict(table=torch.zeros(3, 2)), "block_table"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int32).t()), "block_table"),
    (dict(cu=torch.zeros(3, dtype=torch.int32)), "cu_seqlens"), (dict(cu=torch.zeros(4, dtype=torch.int64)), "cu_seqlens"),
    (dict(k=torch.zeros(4, 2, 64, 128, dtype=torch.float16)), "k_pages"),
    (dict(vt=torch.zeros(paged.vt_pages_shape(5, 2, 64), dtype=torch.float16)), "one pool"),
    (dict(vt=torch.zeros(paged.vt_pages_shape(4, 2, 64))), "differ"),
    (dict(k=torch.zeros(paged.k_pages_shape(4, 4, 64), dtype=torch.float16)[:, ::2]), "contiguous"),
    (dict(kv=torch.ones(4, dtype=torch.int32), table=torch.zeros(4, 2, dtype=torch.int32)), "rows"),
    (dict(out=torch.zeros(3, 5, 128, dtype=torch.float16)), "out"), (dict(out=torch.zeros(3, 4, 128)), "out"),
    (dict(out=torch.zeros(3, 128, 4, dtype=torch.float16).transpose(1, 2)), "out")])
def test_wrappers_refuse(call, kw, match):
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


def test_wrappers_refuse_cpu_tensors():
    for call in (_append, _attend):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(RuntimeError, match="GPU"):
        token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))


def test_prefix_wrapper_refuses():
    a = _args()
    call = lambda table, n: paged.shared_prefix_attention(a["q"], a["kv"], a["table"], table, n, a["k"], a["vt"], 0.1)  # noqa: E731
    with pytest.raises(ValueError, match="prefix_table"):
        call(torch.zeros(1, dtype=torch.int32), 128)
    with pytest.raises(ValueError, match="prefix_table"):
        call(torch.zeros(2, dtype=torch.int64), 128)
    with pytest.raises(ValueError, match="positive"):
        call(torch.zeros(2, dtype=torch.int32), 0)
