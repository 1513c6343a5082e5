"""Sampling's bookkeeping on the GPU.

`greedy_step`: argmax of the last logits row, then out[pos] = idx,
tok = idx, pos += 1, as one HIP launch (libldk_amd.so `ldk_greedy_step`).

This is the greedy step of the reference's GraphDecoder (kernels/e2e/run.py:69-74). It replaces
`logits.argmax(-1)` inside captured decode graphs: torch's vocabulary-sized argmax reduces across
workgroups through a semaphore buffer cleared with a memset node, which is not reliable under
repeated hipGraph replay on this platform.

`token_logprobs` (`ldk_token_logprobs`): what an answer is returned or a text is scored with, the
log probability of a given token of every row of logits, the row's entropy and its most likely
tokens, with every logit read once.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from kernels import _lib

MAX_TOP = 64  # most alternatives per row (csrc/logprobs.hip, kTopMax)


def greedy_step(logits: torch.Tensor, tok: torch.Tensor, pos: torch.Tensor,
                out: torch.Tensor | None = None) -> None:
    """logits: [..., V] (the last row is used); tok: int64 tensor of one element; pos: int64
    tensor of one element; out: optional int64 [L] token log. Updates tok, out and pos in place."""
    V = logits.shape[-1]
    row = logits.reshape(-1, V)[-1]
    if row.stride(0) != 1:
        row = row.contiguous()
    for t, name in ((tok, "tok"), (pos, "pos")):
        if t.dtype != torch.int64 or t.numel() != 1:
            raise ValueError(f"greedy_step: {name} must be one int64 element")
    if out is not None and (out.dtype != torch.int64 or not out.is_contiguous()):
        raise ValueError("greedy_step: out must be a contiguous int64 tensor")
    dev = _lib.require_gpu(row, tok, pos, out, what="greedy_step")
    with _lib.device_guard(dev):
        st = _lib.load().ldk_greedy_step(
            _lib.ptr(row), _lib.dtype_code(row.dtype), V, _lib.ptr(tok), _lib.ptr(out),
            0 if out is None else out.numel(), _lib.ptr(pos), _lib.stream(dev))
    _lib.check(st, "greedy_step")


class TokenLogprobs(NamedTuple):
    """token_logprobs' answer, of the logits' leading shape (natural logarithms)."""

    logprob: torch.Tensor       # fp32 [...]: of the given token; NaN for one outside [0, V)
    entropy: torch.Tensor       # fp32 [...]
    top_logprobs: torch.Tensor  # fp32 [..., top], descending
    top_ids: torch.Tensor       # int64 [..., top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """logits [..., V] (fp16, bf16 or fp32); tokens int64 of the leading shape; top: 0..64
    alternatives per row, at most V (ties go to the lowest index, NaN counts as the largest, as
    torch.argmax). log_softmax(logits)[tokens], the softmax's entropy and the `top` largest log
    probabilities with their indexes, in fp32. -inf logits (masked words) have probability 0; a row
    that holds +inf or NaN, or nothing but -inf, gives NaN."""
    lead, V = logits.shape[:-1], logits.shape[-1]
    if tokens.dtype is not torch.int64 or tokens.shape != lead:
        raise ValueError(f"token_logprobs: tokens must be int64 of shape {tuple(lead)}, got "
                         f"{tokens.dtype} {tuple(tokens.shape)}")
    code = _lib.dtype_code(logits.dtype)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"token_logprobs: top={top} outside 0..{min(MAX_TOP, V)}")
    dev = logits.get_device()
    if dev < 0 or tokens.get_device() != dev:
        _lib.require_gpu(logits, tokens, what="token_logprobs")
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    rows = x.shape[0]
    if not x.is_contiguous() and (x.stride(1) != 1 or (rows > 1 and x.stride(0) < V)):
        x = x.contiguous()
    tok = tokens if tokens.is_contiguous() else tokens.contiguous()
    lib = _lib.load()
    need = lib.ldk_token_logprobs_workspace_bytes(rows, V, top) if rows else 0
    if need < 0:
        _lib.check(-need, "token_logprobs")
    device = logits.device
    ids = torch.empty(lead + (top,), dtype=torch.int64, device=device)
    # the fp32 answers as parts of one allocation
    top_lp, logprob, entropy = torch.empty(rows * (top + 2), dtype=torch.float32, device=device).split(
        (rows * top, rows, rows))
    top_lp = top_lp.view(lead + (top,))
    if logits.dim() != 2:
        logprob, entropy = logprob.view(lead), entropy.view(lead)
    if rows:
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        p, n = logprob.data_ptr(), 4 * rows  # (an empty top_lp has no address)
        with _lib.device_guard(device):
            st = lib.ldk_token_logprobs(
                x.data_ptr(), x.stride(0), code, tok.data_ptr(), rows, V, top, p, p + n, p - n * top,
                ids.data_ptr(), None if ws is None else ws.data_ptr(), need, _lib.stream(device))
        if st:
            _lib.check(st, "token_logprobs")
    return TokenLogprobs(logprob, entropy, top_lp, ids)
