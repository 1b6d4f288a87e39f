"""A small engine over the paged cache: many sequences, prompts in chunks, drafts verified on the GPU.

The reference's scheduler (continuous batching, MTP drafting and verification) is oMLX's; PagedEngine is the least
that runs the paged operators as a server does. One step is one batch: a chunk of the prompts that are not read yet, and for
every other sequence its last token with the drafts that a proposer offers. Its logits go to verify_drafts, what was not
accepted leaves the cache again, and the host reads one small tensor of tokens a step.

    engine = PagedEngine(model, num_pages=4096)
    engine.add("a", prompt_ids, max_new=200, temperature=0.7)
    while engine.running:
        for key, tokens in engine.step().items(): ...

cancel() drops a sequence; engine.failed names those that left because the model gave no probabilities for them.
"""
from __future__ import annotations

import itertools
from dataclasses import dataclass, field

import torch

from .model import Qwen3EXL3
from .paged import check_paged_status
from .speculative import verify_drafts


def lookup_drafts(tokens: list[int], most: int, longest: int = 3) -> list[int]:
    """Drafts from the sequence's own text: what followed the last earlier occurrence of its final tokens (the longest
    of up to `longest` that occurs), at most `most` of it."""
    for n in range(min(longest, len(tokens) - 1), 0, -1):
        tail = tokens[-n:]
        for at in range(len(tokens) - n - 1, -1, -1):
            if tokens[at:at + n] == tail:
                return tokens[at + n:at + n + most]
    return []


@dataclass
class _Sequence:
    tokens: list[int]                   # prompt and what was generated
    prompt: int                         # tokens of the prompt
    max_new: int
    temperature: float
    stop: frozenset
    new: list[int] = field(default_factory=list)


class PagedEngine:
    def __init__(self, model: Qwen3EXL3, num_pages: int, page_size: int = 64, chunk: int = 512, max_drafts: int = 4,
                 propose=lookup_drafts, seed: int = 0, check_every: int = 64):
        """chunk: prompt rows of a step; max_drafts: drafts of a sequence and step (0: none); propose(tokens, most) -> drafts, of
        which no more than that are fed, and none from the first that is no token of the model on."""
        if chunk < 1 or max_drafts < 0:
            raise ValueError("chunk must be one or more and max_drafts zero or more")
        self.model, self.chunk, self.max_drafts, self.propose = model, chunk, max_drafts, propose
        self.device = model.rope_cos.device
        self.cache = model.make_paged_cache(num_pages, page_size)
        self.check_every, self._unchecked = check_every, 0
        self._gen = torch.Generator(device=self.device)
        self._gen.manual_seed(seed)
        self._seqs: dict = {}
        self._set_back: set = set()                                 # sequences that gave their pages up and wait
        self.failed: dict = {}                                      # sequences that left without an end, and why
        self.drafted = self.accepted = 0

    @property
    def running(self) -> int:
        return len(self._seqs)

    def add(self, key, prompt: list[int], max_new: int, temperature: float = 0.0, stop=()) -> None:
        """Queue a sequence; temperature 0 is greedy, `stop` are token ids that end it."""
        if not prompt or max_new < 1 or not temperature >= 0:
            raise ValueError("need a prompt, max_new of one or more and a temperature of zero or more")
        if len(prompt) + max_new > self.model.cfg.max_position_embeddings:
            raise ValueError(f"{len(prompt)} + {max_new} tokens exceed max_position_embeddings")
        if not all(self._known(t) for t in prompt):                 # the embedding would fault on the GPU
            raise ValueError("the prompt has tokens outside the model's vocabulary")
        self.cache.add(key)
        self.failed.pop(key, None)
        self._seqs[key] = _Sequence(list(prompt), len(prompt), max_new, float(temperature), frozenset(stop))

    def _drop(self, key) -> None:
        self.cache.release(key)
        del self._seqs[key]
        self._set_back.clear()                                      # pages came back: all may try again

    def cancel(self, key) -> None:
        """A sequence leaves the engine, whatever it was doing; its pages come back. KeyError if there is none under `key`."""
        if key not in self._seqs:
            raise KeyError(key)
        self._drop(key)

    def _known(self, token: int) -> bool:
        return 0 <= token < self.model.cfg.vocab_size

    def _drafts(self, s: _Sequence) -> list[int]:
        most = min(self.max_drafts, s.max_new - len(s.new) - 1)
        drafts = list(self.propose(s.tokens, most))[:most] if most > 0 else []
        return list(itertools.takewhile(self._known, drafts))

    def _upload(self, values: list, dtype) -> torch.Tensor:
        return torch.tensor(values, dtype=dtype).pin_memory().to(self.device, non_blocking=True)

    def step(self) -> dict:
        """One batch; returns the new tokens of the sequences that have some (finished ones leave the engine). A step that raises
        changes nothing: the next one feeds the same rows. A sequence for which the model gives no probabilities leaves too, and
        `failed` names it.

        Where the pool is short of pages, drafts are left out first, then prompts wait; if nothing can be fed, the youngest sequence
        gives its pages up and is read again once another has left. MemoryError, naming them, if all that is left are sequences
        that the whole pool could not hold (cancel() them)."""
        if not self._seqs:
            return {}
        feeds = self._feeds()
        while not feeds:
            holders = [key for key in self._seqs if self.cache.length(key)]
            if len(holders) > 1:
                self._give_up(holders[-1])
                self._set_back.add(holders[-1])
            elif self._set_back:
                self._set_back.clear()
            else:
                keys = ", ".join(repr(key) for key in self._seqs)
                raise MemoryError(f"the pool of {self.cache.num_pages} pages cannot hold the next token of {keys}")
            feeds = self._feeds()
        judged = [(key, s, drafts) for key, s, _, drafts, wanted in feeds if wanted]
        lengths = {key: self.cache.length(key) for key, *_ in feeds}
        try:
            picked = self._run(feeds, judged)
        except BaseException:                                       # as before the step: its rows leave the cache again
            for key, length in lengths.items():
                self.cache.truncate(key, length)
            raise
        return self._keep(judged, picked, lengths)

    def _give_up(self, key) -> None:
        """A sequence's pages come back; all it has is its prompt from now on."""
        self.cache.truncate(key, 0)
        self._seqs[key].prompt = len(self._seqs[key].tokens)

    def _feeds(self) -> list:
        """What the next step feeds, as (key, sequence, rows, drafts, whether logits are wanted), within the free pages: a row of
        every decoding sequence, prompts in order of arrival, then drafts."""
        size = self.cache.page_size
        reading, decoding, drafts = [], [], {}
        for key, s in self._seqs.items():
            if len(s.tokens) > self.cache.num_pages * size:         # the whole pool could not hold what its next token needs
                if self.cache.length(key):
                    self._give_up(key)
            elif self.cache.length(key) < s.prompt:
                reading.append(key)
            else:
                decoding.append(key)
        spare, grant = self.cache.free_pages, {}

        def take(key, want):                                        # rows granted, of the `want` more that the sequence would have
            nonlocal spare
            at = self.cache.length(key) + grant.get(key, 0)
            held = -(-at // size)
            n = max(0, min(want, (held + spare) * size - at))
            spare -= -(-(at + n) // size) - held
            if n:
                grant[key] = grant.get(key, 0) + n
            return n

        decoding = [key for key in decoding if take(key, 1)]
        room = self.chunk
        for key in reading:
            if room and key not in self._set_back:
                room -= take(key, min(self._seqs[key].prompt - self.cache.length(key), room))
        for key in decoding:
            offered = self._drafts(self._seqs[key])
            drafts[key] = offered[:take(key, len(offered))]
        feeds = []
        for key, s in self._seqs.items():
            if key in drafts:
                feeds.append((key, s, [s.tokens[-1]] + drafts[key], drafts[key], True))
            elif key in grant:                                      # its prompt, as far as this step's chunk goes
                have = self.cache.length(key)
                feeds.append((key, s, s.tokens[have:have + grant[key]], [], have + grant[key] == s.prompt))
        return feeds

    def _run(self, feeds: list, judged: list) -> list:
        """The batch through the model and the verification; for each judged sequence its tokens and their count."""
        batch = self.cache.extend([(key, len(rows)) for key, _, rows, _, _ in feeds])
        tokens = self._upload([t for _, _, rows, _, _ in feeds for t in rows], torch.int64)
        # rows whose logits are wanted: a decoding sequence's all, a finished prompt's last
        at, rows, cu = 0, [], [0]
        for _, _, fed, drafts, wanted in feeds:
            at += len(fed)
            if wanted:
                rows += range(at - len(drafts) - 1, at)
                cu.append(len(rows))
        logits = self.model.forward_paged(tokens, self.cache, batch, self._upload(rows, torch.int64))
        picked = self._verify(self.model.gather_logits(logits), judged, cu) if judged else []
        self._unchecked += 1
        if self.check_every and self._unchecked >= self.check_every:
            self._unchecked = 0
            check_paged_status(self.device)
        return picked

    def _verify(self, logits: torch.Tensor, judged: list, cu: list[int]) -> list:
        drafts = [t for _, _, d in judged for t in d]
        most = max(len(d) for _, _, d in judged)
        n, vocab = len(judged), logits.shape[1]
        noise = torch.empty((n, vocab), device=self.device).exponential_(generator=self._gen).clamp_(min=1e-20)
        u = torch.rand(len(drafts), device=self.device, generator=self._gen)
        picked, count, _ = verify_drafts(logits, self._upload(drafts, torch.int64), self._upload(cu, torch.int32), u, noise, most,
                                         temperature=self._upload([s.temperature for _, s, _ in judged], torch.float32))
        return torch.cat([picked, count[:, None]], 1).tolist()      # the step's one wait for the GPU

    def _keep(self, judged: list, picked: list, lengths: dict) -> dict:
        """Take a finished step's tokens over, and what was not accepted out of the cache."""
        out = {}
        for (key, s, d), row in zip(judged, picked):
            got = row[:row[-1]]
            dead = got[-1] < 0                                      # no token after the drafts that stand
            if dead:
                got.pop()
            self.drafted += len(d)
            self.accepted += len(got) - (not dead)
            end = next((i + 1 for i, t in enumerate(got) if t in s.stop), len(got))
            got = got[:min(end, s.max_new - len(s.new))]
            s.tokens += got
            s.new += got
            if got:
                out[key] = got
            ended = len(s.new) >= s.max_new or (got and got[-1] in s.stop)
            if dead and not ended:
                self.failed[key] = "the model gave no probabilities"
            if dead or ended:
                self._drop(key)
            elif lengths[key] >= s.prompt:                          # its last token and the drafts that stand stay cached
                self.cache.truncate(key, lengths[key] + len(got))
        return out

    def generate(self, prompts: list[list[int]], max_new: int, temperature: float = 0.0, stop=()) -> list[list[int]]:
        """All of the prompts' continuations, by an engine that runs nothing else. If it raises, none of them stays behind."""
        if self._seqs:
            raise ValueError("generate needs an engine without running sequences")
        done = {i: [] for i in range(len(prompts))}
        try:
            for i, p in enumerate(prompts):
                self.add(i, p, max_new, temperature, stop)
            while self.running:
                for i, got in self.step().items():
                    done[i] += got
                for i in done:
                    if i in self.failed:
                        raise RuntimeError(f"prompt {i}: {self.failed[i]}")
            check_paged_status(self.device)
        finally:
            for key in list(self._seqs):
                self._drop(key)
        return [done[i] for i in range(len(prompts))]
