"""Beam search: for every prompt the ``beams`` most probable continuations are carried on side by side.

The beams of a prompt are requests of the cache like any other.  Behind the prompt the first one is
forked: all share the prompt's pages.  Every step feeds each beam's last token, ranks all continuations of
a prompt's beams (``sampling.beams``) and puts the beams' contents in the order of the choice
(``CacheManager.reorder``): filled pages change hands in the block tables, unfilled pages and recurrent
states move on the device.  Attention reads the pages that a prompt's beams share once for all of them
(``kernels.shared_prefix``).

A hypothesis is finished by the end-of-sequence token or by the length limit; its score is its log
probability divided by (number of generated tokens) ** length_penalty.  A prompt is done when it has
``beams`` finished hypotheses none of which is worse than the best running beam's score would be now.

The reference has no beam search; its nearest relative is ``generate_greedy_cached``
(src/utils/generation.py:7-46), which is the case of one beam.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field

from ..kernels import ops
from ..sampling.beams import BeamSelector
from .step import StepEntry

NO_SCORE = float("-inf")


@dataclass
class Hypothesis:
    """A continuation: its generated tokens and its score (log probability over length)."""
    token_ids: list[int]
    score: float


@dataclass
class _Search:
    """One prompt's beams: their request ids, tokens and log probabilities, by label."""
    prompt: list[int]
    ids: list[str]
    tokens: "list[list[int]]" = field(default_factory=list)
    scores: "list[float]" = field(default_factory=list)
    finished: "list[Hypothesis]" = field(default_factory=list)


def choose(search: _Search, candidates: "list[tuple[float, int, int]]", beams: int, eos: int,
           penalty: float) -> "tuple[list[int], list[int]]":
    """The next beams from the ranked continuations: (parent, token) of each label.  A continuation that
    ends is a finished hypothesis if it is among the first ``beams``; the others become beams, each where
    its parent is as long as that place is free, so that few contents move."""
    chosen: "list[tuple[float, int, int]]" = []
    for rank, (score, parent, token) in enumerate(candidates):
        if token == eos:
            if rank < beams:
                tokens = search.tokens[parent] + [token]
                search.finished.append(Hypothesis(tokens, score / len(tokens) ** penalty))
        elif len(chosen) < beams:
            chosen.append((score, parent, token))
    labels: "list[tuple[float, int, int] | None]" = [None] * beams
    rest = []
    for entry in chosen:
        if labels[entry[1]] is None:
            labels[entry[1]] = entry
        else:
            rest.append(entry)
    for label in range(beams):
        if labels[label] is None:
            # (no continuation left: the beam stays in the batch and counts no more)
            labels[label] = rest.pop(0) if rest else (NO_SCORE, label, 0)
    tokens = [search.tokens[parent] + [token] for _, parent, token in labels]
    search.tokens, search.scores = tokens, [score for score, _, _ in labels]
    return [parent for _, parent, _ in labels], [token for _, _, token in labels]


def is_done(search: _Search, beams: int, penalty: float) -> bool:
    best = max(search.scores)
    if best == NO_SCORE:
        return True
    if len(search.finished) < beams:
        return False
    worst = sorted(h.score for h in search.finished)[-beams]
    return worst >= best / len(search.tokens[0]) ** penalty


class BeamSearch:
    def __init__(self, runner, cache, beams: int, max_batch_tokens: int,
                 length_penalty: float = 1.0) -> None:
        if type(beams) is not int or not 1 <= beams <= ops.MAX_BEAMS:
            raise ValueError(f"beam search takes 1 to {ops.MAX_BEAMS} beams, got {beams}")
        if beams > cache.max_seqs:
            raise ValueError(f"{beams} beams are more than the {cache.max_seqs} requests that are live "
                             f"at a time (decode_batch_size)")
        if beams > max_batch_tokens:
            raise ValueError(f"{beams} beams are more than the {max_batch_tokens} tokens of a step "
                             f"(max_batch_tokens)")
        if not isinstance(length_penalty, (int, float)) or not abs(length_penalty) <= 1e300:
            raise ValueError("length_penalty must be a finite number")
        self.runner, self.cache, self.beams = runner, cache, beams
        self.max_batch_tokens, self.penalty = max_batch_tokens, float(length_penalty)
        # twice as many as beams: even if half of them end, there are enough that go on
        self.take = min(2 * beams, ops.MAX_TAKE)
        self.groups = min(cache.max_seqs, max_batch_tokens) // beams
        self.selector = BeamSelector(runner.device, self.groups, self.take)

    def _pages(self, prompt: "list[int]", max_new_tokens: int) -> int:
        """Pages that a prompt's beams may need together: the prompt's once, and for every beam what is
        generated (the last token is never fed), with the page in which the prompt ends."""
        page = self.cache.page_size
        total = -(-(len(prompt) + max_new_tokens - 1) // page)
        return len(prompt) // page + self.beams * (total - len(prompt) // page)

    def run(self, prompts: "list[list[int]]", max_new_tokens: int, eos_token_id: int,
            name: str) -> "list[list[Hypothesis]]":
        """For every prompt its finished hypotheses, best first (up to ``beams``).  As many prompts at a
        time as there are slots and pages for, and tokens in a step."""
        # (scores of continuations of all lengths stay numbers: far within 1e308)
        if abs(self.penalty) * math.log10(max(max_new_tokens, 2)) > 200.0:
            raise ValueError(f"length_penalty {self.penalty} is too large for {max_new_tokens} tokens")
        have = self.cache.num_free_pages()
        for prompt in prompts:
            if self._pages(prompt, max_new_tokens) > have:
                raise ValueError(f"a prompt of {len(prompt)} tokens with {self.beams} beams of "
                                 f"{max_new_tokens} may need {self._pages(prompt, max_new_tokens)} "
                                 f"pages, the cache has {have}")
        results: "list[list[Hypothesis]]" = []
        at = 0
        while at < len(prompts):
            wave, need = [], 0
            while at < len(prompts) and len(wave) < self.groups:
                need += self._pages(prompts[at], max_new_tokens)
                if wave and need > have:
                    break
                wave.append(_Search(list(prompts[at]),
                                    [f"{name}-{at}-{b}" for b in range(self.beams)]))
                at += 1
            try:
                self._run_wave(wave, max_new_tokens, eos_token_id)
            finally:
                for search in wave:
                    for request_id in search.ids:
                        if self.cache.has(request_id):
                            self.cache.release(request_id)
            for search in wave:
                ranked = sorted(search.finished, key=lambda h: -h.score)
                results.append(ranked[: self.beams])
        return results

    def _run_wave(self, wave: "list[_Search]", max_new_tokens: int, eos: int) -> None:
        live = []
        for search in wave:
            # the prompt, in portions, by the first beam; its continuations are ranked from one row
            for start in range(0, len(search.prompt), self.max_batch_tokens):
                portion = search.prompt[start: start + self.max_batch_tokens]
                last = start + len(portion) == len(search.prompt)
                logits = self.runner.step([StepEntry(search.ids[0], portion,
                                                     [len(portion) - 1] if last else [])])
            search.tokens, search.scores = [[]] * self.beams, [0.0] + [NO_SCORE] * (self.beams - 1)
            candidates = self.selector.select(logits, [[0.0]], self.take)[0]
            self.runner.check_status()
            _, tokens = choose(search, candidates, self.beams, eos, self.penalty)
            if max_new_tokens > 1 and not is_done(search, self.beams, self.penalty):
                self.cache.fork(search.ids[0], search.ids[1:])
                live.append((search, tokens))
            else:
                self._finish(search)
        for generated in range(2, max_new_tokens + 1):
            if not live:
                break
            logits = self.runner.step([StepEntry(request_id, [token], [0])
                                       for search, tokens in live
                                       for request_id, token in zip(search.ids, tokens)])
            ranked = self.selector.select(logits, [search.scores for search, _ in live], self.take)
            self.runner.check_status()
            going, parents = [], []
            for (search, _), candidates in zip(live, ranked):
                source, tokens = choose(search, candidates, self.beams, eos, self.penalty)
                if generated == max_new_tokens or is_done(search, self.beams, self.penalty):
                    self._finish(search)
                    for request_id in search.ids:
                        self.cache.release(request_id)
                else:
                    going.append((search, tokens))
                    parents.append(source)
            if going:
                self.cache.reorder([search.ids for search, _ in going], parents)
            live = going

    def _finish(self, search: _Search) -> None:
        """The beams that still run are hypotheses too, ended by the length (of a prompt that is done,
        none of them is better than what it has)."""
        for tokens, score in zip(search.tokens, search.scores):
            if score > NO_SCORE and tokens:
                search.finished.append(Hypothesis(tokens, score / len(tokens) ** self.penalty))
