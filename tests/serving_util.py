"""A stand-in for the decoder on the CPU, for tests of the engine: logits that depend on every token of a sequence, read back from
its pages."""
import random
from types import SimpleNamespace

import torch

VOCAB = 97


def history_logits(tokens):
    """What the stand-in gives after these tokens."""
    rng = random.Random(str(tokens))
    return torch.tensor([rng.random() * 4 for _ in range(VOCAB)])


def greedy_text(prompt, max_new):
    """The text the stand-in writes after the prompt at T = 0."""
    tokens = list(prompt)
    for _ in range(max_new):
        tokens.append(int(history_logits(tokens).argmax()))
    return tokens[len(prompt):]


class HistoryModel:
    """Writes each fed token to its page slot and reads the whole sequence from there. `fail`: called with the number of the
    step before it is done; `spoil`: whether a history's logits are NaN."""

    def __init__(self, fail=lambda step: None, spoil=lambda tokens: False):
        self.cfg = SimpleNamespace(vocab_size=VOCAB, max_position_embeddings=1000)
        self.rope_cos = torch.zeros(1)
        self.fail, self.spoil = fail, spoil
        self.steps, self.fed, self.asked = 0, [], []

    def make_paged_cache(self, num_pages, page_size):
        from omlx_exl3_b200 import PagedKVCache
        return PagedKVCache(1, 1, 1, num_pages, page_size, device="cpu", dtype=torch.float32)

    def forward_paged(self, tokens, cache, batch, rows=None):
        assert ((tokens >= 0) & (tokens < VOCAB)).all(), "a token that the embedding does not have"
        self.steps += 1
        self.fed.append(batch.total_rows)
        self.asked.append(batch.total_rows if rows is None else rows.numel())
        k, logits, at = cache.k[0], [], 0
        for s, n in enumerate(batch.rows):
            total, table = int(batch.lens[s]), batch.page_table[s].tolist()
            for i in range(n):
                pos = total - n + i
                k[table[pos // cache.page_size], 0, pos % cache.page_size, 0] = float(tokens[at + i])
                text = [int(k[table[p // cache.page_size], 0, p % cache.page_size, 0]) for p in range(pos + 1)]
                logits.append(torch.full((VOCAB,), float("nan")) if self.spoil(text) else history_logits(text))
            at += n
        self.fail(self.steps)                                          # after the pages were written, as a late failure is
        out = torch.stack(logits)
        return out if rows is None else out[rows]

    def gather_logits(self, local):
        return local


def on_cpu(monkeypatch):
    """The engine's GPU parts replaced: the verification by its definition, uploads by plain tensors."""
    from omlx_exl3_b200 import serving
    from test_verify_gpu import _plain

    def verify(target, tokens, cu, u, noise, most, draft_logits=None, temperature=None):
        return _plain(target, tokens, cu.tolist(), u, noise, most, draft_logits, temperature)
    monkeypatch.setattr(serving, "verify_drafts", verify)
    monkeypatch.setattr(serving, "check_paged_status", lambda device: None)
    monkeypatch.setattr(serving.PagedEngine, "_upload", lambda self, values, dtype: torch.tensor(values, dtype=dtype))
