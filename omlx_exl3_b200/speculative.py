"""Speculative sampling: which drafted tokens stand, and what comes after them (exl3_verify_drafts).

The reference leaves MTP drafting and its verification to oMLX's scheduler (one sequence, T = 0 in its published
numbers); here a whole batch is decided on the GPU, without the host looking at a probability. The random numbers are
inputs, so a step can be replayed.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import check, dtype_code, lib, stream_ptr
from .paged import _need, _workspace


def verify_drafts(target_logits: torch.Tensor, draft_tokens: torch.Tensor, cu_rows: torch.Tensor, u: torch.Tensor,
                  noise: torch.Tensor, max_drafts: int, draft_logits: torch.Tensor | None = None,
                  temperature: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Verify drafted tokens against the target's probabilities. Returns (tokens (seqs, max_drafts + 1) int64,
    count (seqs) int32, accept_prob (drafts) f32).

    Sequence s has target rows cu_rows[s] .. cu_rows[s + 1] - 1 (at least one): all but the last judge one draft each.
    target_logits (rows, n) and draft_logits (rows - seqs, n), fp16, bf16 or fp32 alike; draft_tokens (rows - seqs) int64;
    temperature (seqs) f32, 0 for greedy, None for 1; u (rows - seqs) f32 in [0, 1); noise (seqs, n) f32, positive
    and exponentially distributed. Without draft_logits the drafts were given outright (a lookup): q is one-hot.

    A draft x stands while u < min(1, p(x) / q(x)); the next token is drawn from max(0, p - q) after a rejection, else
    from the last row's p, as the first largest w(v) / noise[s, v]. tokens holds the accepted drafts, the next token,
    then -1; count is the accepted drafts + 1. A row without any finite probability accepts nothing and gives -1.
    """
    dt = target_logits.dtype
    code = dtype_code(dt)
    dev = target_logits.device
    if dev.type != "cuda":
        raise ValueError("EXL3 kernels take CUDA tensors")
    _need(target_logits.dim() == 2 and cu_rows.dim() == 1 and cu_rows.shape[0] >= 2, "target_logits (rows, n), cu_rows (seqs + 1)")
    rows, n = target_logits.shape
    seqs = cu_rows.shape[0] - 1
    drafts = rows - seqs
    _need(n >= 1 and drafts >= 0 and max_drafts >= 0, "each sequence needs at least one target row")
    if cu_rows.dtype != torch.int32 or draft_tokens.dtype != torch.int64:
        raise TypeError("cu_rows must be int32 and draft_tokens int64")
    if u.dtype != torch.float32 or noise.dtype != torch.float32 or (temperature is not None and temperature.dtype != torch.float32):
        raise TypeError("u, noise and temperature must be fp32")
    _need(draft_tokens.shape == (drafts,) and u.shape == (drafts,), "draft_tokens and u must be (rows - seqs)")
    _need(noise.shape == (seqs, n) and (temperature is None or temperature.shape == (seqs,)),
          "noise must be (seqs, n) and temperature (seqs)")
    _need(cu_rows.is_contiguous() and draft_tokens.is_contiguous() and u.is_contiguous()
          and (temperature is None or temperature.is_contiguous()), "cu_rows, draft_tokens, u and temperature must be contiguous")
    matrices = [target_logits, noise]
    if draft_logits is not None:
        if draft_logits.dtype != dt:
            raise TypeError("draft_logits must have target_logits' dtype")
        _need(draft_logits.shape == (drafts, n), "draft_logits must be (rows - seqs, n)")
        matrices.append(draft_logits)
    for m in matrices:
        _need(m.stride(1) == 1 and (m.shape[0] < 2 or m.stride(0) >= n), "logits and noise need contiguous, non-overlapping rows")
    for t in (draft_tokens, cu_rows, u, noise, draft_logits, temperature):
        _need(t is None or t.device == dev, "all tensors must be on one device")
    tokens = torch.empty((seqs, max_drafts + 1), dtype=torch.int64, device=dev)
    count = torch.empty(seqs, dtype=torch.int32, device=dev)
    prob = torch.empty(drafts, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        stream = stream_ptr(dev)
        need = ctypes.c_size_t()
        check(lib().exl3_verify_workspace(rows, seqs, n, ctypes.byref(need)), "exl3_verify_workspace")
        ws = _workspace(dev, stream, need.value)
        check(lib().exl3_verify_drafts(target_logits.data_ptr(), max(target_logits.stride(0), n),
                                       None if draft_logits is None or drafts == 0 else draft_logits.data_ptr(),
                                       n if draft_logits is None else max(draft_logits.stride(0), n), code, rows, seqs, n,
                                       draft_tokens.data_ptr() if drafts else None, cu_rows.data_ptr(),
                                       None if temperature is None else temperature.data_ptr(),
                                       u.data_ptr() if drafts else None, noise.data_ptr(), max(noise.stride(0), n),
                                       max_drafts, tokens.data_ptr(), count.data_ptr(), prob.data_ptr() if drafts else None,
                                       ws.data_ptr(), ws.numel(), stream), "exl3_verify_drafts")
    return tokens, count, prob
