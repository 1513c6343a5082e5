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
    V = logits.shape[-1]
    lead = logits.shape[:-1]
    if tokens.dtype != torch.int64 or tokens.shape != lead:
        raise ValueError(f"token_logprobs: tokens must be int64 of shape {tuple(lead)}, got "
                         f"{tokens.dtype} {tuple(tokens.shape)}")
    code = _lib.dtype_code(logits.dtype)
    dev = _lib.require_gpu(logits, tokens, what="token_logprobs")
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    rows = x.shape[0]
    if x.stride(1) != 1 or (rows > 1 and x.stride(0) < V):
        x = x.contiguous()
    tok = tokens.reshape(-1).contiguous()
    logprob = torch.empty(lead, dtype=torch.float32, device=dev)
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"token_logprobs: top={top} outside 0..{min(MAX_TOP, V)}")
    top_lp = torch.empty(lead + (top,), dtype=torch.float32, device=dev)
    top_ids = torch.empty(lead + (top,), dtype=torch.int64, device=dev)
    if rows:
        with _lib.device_guard(dev):
            lib = _lib.load()
            need = lib.ldk_token_logprobs_workspace_bytes(rows, V, top)
            if need < 0:
                _lib.check(-need, "token_logprobs")
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            st = lib.ldk_token_logprobs(_lib.ptr(x), x.stride(0), code, _lib.ptr(tok), rows, V, top,
                                        _lib.ptr(logprob), _lib.ptr(entropy), _lib.ptr(top_lp), _lib.ptr(top_ids),
                                        _lib.ptr(ws), need, _lib.stream(dev))
        _lib.check(st, "token_logprobs")
    return TokenLogprobs(logprob, entropy, top_lp, top_ids)
