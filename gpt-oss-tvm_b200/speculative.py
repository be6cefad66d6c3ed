"""Speculative decoding on the engine: drafts looked up in the text so far, one
forward over every sequence's drafts, and the test that keeps the target's
distribution.

A step of ``SpeculativeDecoder`` takes the last token of each sequence and up
to ``draft_len`` drafts after it, runs them as one chunk a sequence over the
paged cache (``Engine.extend_batch``), keeps the drafts that ``verify_drafts``
accepts and the token drawn after them, and pops the rest from the cache.
Greedy (temperature 0) it gives the tokens of plain greedy decoding of the same
forward, only several a step.

    eng = Engine.random(config, seed=0, max_batch_size=2, max_chunk=5, kv_dtype="float8_e4m3")
    tokens = SpeculativeDecoder(eng, draft_len=4).generate([[1, 2, 3], [4, 5]], 32)
"""
from __future__ import annotations

import torch

from .engine import Engine


def prompt_lookup(tokens: list[int], n: int, ngram: int = 3) -> list[int]:
    """Up to n tokens that followed the last earlier occurrence of the text's
    last ``ngram`` tokens (or fewer, down to one); none if there is no such."""
    if n <= 0:
        return []
    for k in range(min(ngram, len(tokens) - 1), 0, -1):
        tail = tokens[-k:]
        for i in range(len(tokens) - k - 1, -1, -1):
            if tokens[i:i + k] == tail:
                return tokens[i + k:i + k + n]
    return []


class SpeculativeDecoder:
    """Decodes a batch of sequences of ``engine`` (created with max_chunk of at
    least draft_len + 1).  draft: (tokens so far, n) -> up to n drafts, without
    a distribution of their own.  Tokens are drawn from softmax(logits /
    temperature), without the top-p cut of ``Engine.sample``.  The random numbers
    come from one seeded generator, so a run can be repeated."""

    def __init__(self, engine: Engine, draft_len: int = 4, draft=prompt_lookup, temperature: float = 0.0,
                 seed: int = 0):
        if draft_len < 0 or draft_len + 1 > engine.max_chunk:
            raise ValueError(f"draft_len {draft_len} needs an engine with max_chunk {draft_len + 1} or more "
                             f"(it has {engine.max_chunk})")
        self.engine, self.draft_len, self.draft, self.temperature = engine, draft_len, draft, float(temperature)
        self.generator = torch.Generator(device=engine.device)
        self.generator.manual_seed(seed)
        self.drafted = self.accepted = self.steps = 0

    def _draws(self, n: int) -> torch.Tensor:
        return torch.rand(n, generator=self.generator, device=self.engine.device)

    def step(self, texts: dict[int, list[int]], room: dict[int, int]) -> None:
        """One forward for the sequences of ``texts`` (sequence id -> tokens,
        whose last is not in the cache yet); appends what it yields, at most
        room[id] tokens.  Raises RuntimeError when the device reports a wait that
        ran out, with texts and cache as they were before the step."""
        eng, seqs = self.engine, list(texts)
        chunks = []
        for s in seqs:
            most = min(self.draft_len, room[s] - 1)
            drafts = list(self.draft(texts[s], most))
            if len(drafts) > max(most, 0):
                raise ValueError(f"{len(drafts)} drafts where at most {most} were asked for")
            chunks.append([texts[s][-1]] + drafts)
        logits, ids, row_start = eng.extend_batch(chunks, seqs)
        greedy = self.temperature < 1e-6
        accepted, nxt = eng.verify(logits, ids, row_start, None if greedy else self._draws(ids.numel()),
                                   None if greedy else self._draws(len(seqs)), temperature=self.temperature)
        n, workspace = len(seqs), eng.chunk_workspace()
        got = torch.cat([accepted, nxt, workspace.error_word()]).tolist()
        if got[-1] or min(got[n:2 * n]) < 0:
            workspace.reset()
            for s, c in zip(seqs, chunks):
                eng.popn(s, len(c))
            raise RuntimeError(f"a speculative step failed on the device (attention error bits {got[-1]:#x}, next "
                               f"tokens {got[n:2 * n]})")
        for s, c, a, t in zip(seqs, chunks, got[:n], got[n:2 * n]):
            texts[s] += c[1:1 + a] + [t]
            if len(c) - 1 > a:
                eng.popn(s, len(c) - 1 - a)
            self.drafted += len(c) - 1
            self.accepted += a
        self.steps += 1

    def generate(self, prompts: list[list[int]], max_new_tokens: int) -> list[list[int]]:
        """max_new_tokens tokens after each prompt (sequences 0, 1, .. of the
        engine's cache, which is cleared first)."""
        eng = self.engine
        if not prompts or len(prompts) > eng.max_batch_size:
            raise ValueError(f"1 to {eng.max_batch_size} prompts (max_batch_size), got {len(prompts)}")
        if any(len(p) == 0 for p in prompts):
            raise ValueError("a prompt needs a token")
        eng.clear_kv_cache()
        texts = {s: [int(t) for t in p] for s, p in enumerate(prompts)}
        for s, text in texts.items():
            eng.paged_kv_cache.add_sequence(s)
            if len(text) > 1:
                eng.prefill(text[:-1], s)
        want = {s: len(t) + max_new_tokens for s, t in texts.items()}
        while True:
            live = {s: t for s, t in texts.items() if len(t) < want[s]}
            if not live:
                return [texts[s][len(p):] for s, p in enumerate(prompts)]
            self.step(live, {s: want[s] - len(t) for s, t in live.items()})
