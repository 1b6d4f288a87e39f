"""Speculative sampling: which drafted tokens stand, and what comes after them (exl3_verify_drafts).

The reference leaves MTP drafting and its verification to oMLX's scheduler (one sequence, T = 0 in its published
numbers); here a whole batch is decided on the GPU, without the host looking at a probability. The random numbers are
inputs, so a step can be replayed.
"""
from __future__ import annotations

import torch

from ._lib import torch_calls


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
    then -1; count is the accepted drafts + 1. A row without any finite probability (all logits -inf, one of them NaN or, but
    for T = 0, +inf) accepts nothing and gives -1.
    """
    return torch_calls().verify_drafts(target_logits, draft_tokens, cu_rows, u, noise, max_drafts, draft_logits, temperature)
