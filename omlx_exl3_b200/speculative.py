"""Speculative sampling: which drafted tokens stand, and what comes after them (exl3_verify_drafts).

The reference leaves MTP drafting and its verification to oMLX's scheduler (one sequence, T = 0 in its published
numbers); here a whole batch is decided on the GPU, without the host looking at a probability. The random numbers are
inputs, so a step can be replayed.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import check, dtype_code, lib, stream_ptr
from .paged import _F32, _I32, _get_device, _row_stride, _workspace


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
    dev = target_logits.get_device()
    if dev < 0:
        raise ValueError("EXL3 kernels take CUDA tensors")
    if _get_device() != dev:                      # the kernels launch on the current device
        with torch.cuda.device(dev):
            return verify_drafts(target_logits, draft_tokens, cu_rows, u, noise, max_drafts, draft_logits, temperature)
    if target_logits.dim() != 2 or cu_rows.dim() != 1 or cu_rows.numel() < 2:
        raise ValueError("need target_logits (rows, n) and cu_rows (seqs + 1)")
    rows, n = target_logits.shape
    seqs = cu_rows.numel() - 1
    drafts = rows - seqs
    if n < 1 or drafts < 0 or max_drafts < 0:
        raise ValueError("each sequence needs at least one target row")
    if cu_rows.dtype is not _I32 or draft_tokens.dtype is not torch.int64:
        raise TypeError("cu_rows must be int32 and draft_tokens int64")
    if u.dtype is not _F32 or noise.dtype is not _F32 or (temperature is not None and temperature.dtype is not _F32):
        raise TypeError("u, noise and temperature must be fp32")
    if draft_tokens.shape != (drafts,) or u.shape != (drafts,):
        raise ValueError("draft_tokens and u must be (rows - seqs)")
    if temperature is not None and temperature.shape != (seqs,):
        raise ValueError("temperature must be (seqs)")
    if not (cu_rows.is_contiguous() and draft_tokens.is_contiguous() and u.is_contiguous()
            and (temperature is None or temperature.is_contiguous())):
        raise ValueError("cu_rows, draft_tokens, u and temperature must be contiguous")
    if not (draft_tokens.get_device() == cu_rows.get_device() == u.get_device() == noise.get_device() == dev):
        raise ValueError("all tensors must be on one device")
    ld, noise_ld = _row_stride(target_logits, rows, n, "target_logits"), _row_stride(noise, seqs, n, "noise")
    draft_ptr, draft_ld, temp_ptr = None, n, None
    if draft_logits is not None:
        if draft_logits.dtype is not dt:
            raise TypeError("draft_logits must have target_logits' dtype")
        if draft_logits.get_device() != dev:
            raise ValueError("all tensors must be on one device")
        draft_ld = _row_stride(draft_logits, drafts, n, "draft_logits")
        if drafts:
            draft_ptr = draft_logits.data_ptr()
    if temperature is not None:
        if temperature.get_device() != dev:
            raise ValueError("all tensors must be on one device")
        temp_ptr = temperature.data_ptr()
    tokens = draft_tokens.new_empty((seqs, max_drafts + 1))
    count = cu_rows.new_empty(seqs)
    prob = u.new_empty(drafts)
    stream = stream_ptr(dev)
    size = ctypes.c_size_t()
    check(lib().exl3_verify_workspace(rows, seqs, n, size), "exl3_verify_workspace")
    ws = _workspace(dev, stream, size.value)
    status = lib().exl3_verify_drafts(target_logits.data_ptr(), ld, draft_ptr, draft_ld, code, rows, seqs, n,
                                      draft_tokens.data_ptr() if drafts else None, cu_rows.data_ptr(), temp_ptr,
                                      u.data_ptr() if drafts else None, noise.data_ptr(), noise_ld, max_drafts,
                                      tokens.data_ptr(), count.data_ptr(), prob.data_ptr() if drafts else None, ws.data_ptr(),
                                      ws.numel(), stream)
    if status:
        check(status, "exl3_verify_drafts")
    return tokens, count, prob
