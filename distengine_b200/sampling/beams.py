"""Choosing the next beams of a beam search: the best continuations over the beams of a prompt and the
vocabulary, by their whole log probability.

One kernel call ranks scores + log_softmax(logits) over all beams of every prompt
(``kernels.ops.beam_select``); the chosen scores, beams and tokens come back to the host in one copy.
The reference decodes greedily only (src/layers/sampler.py:5-8).
"""

from __future__ import annotations

import torch

from ..kernels import ops


class BeamSelector:
    """Buffers for ``groups`` prompts of which ``take`` continuations each are chosen at most."""

    def __init__(self, device: torch.device, groups: int, take: int) -> None:
        self.device, self.groups, self.take = device, groups, take
        self._buffer = torch.zeros(3 * groups * take, dtype=torch.int32, device=device)
        self._host = torch.zeros(3 * groups * take, dtype=torch.int32).pin_memory()
        self._scratch: "torch.Tensor | None" = None

    def select(self, logits: torch.Tensor, scores: "list[list[float]]",
               take: int) -> "list[list[tuple[float, int, int]]]":
        """logits [groups * beams, vocabulary] float32, ``scores`` each beam's log probability so far
        (minus infinity: a beam that does not count).  Returns for every group up to ``take``
        (log probability, beam, token), best first; synchronises to bring them to the host."""
        groups, beams = len(scores), len(scores[0])
        if groups > self.groups or take > self.take:
            raise ValueError(f"the selector was made for {self.groups} groups and {self.take} "
                             f"continuations, got {groups} and {take}")
        n = groups * take
        best, beam, token = (self._buffer[i * n: (i + 1) * n].view(groups, take) for i in range(3))
        size = ops.beam_scratch(groups, beams, logits.shape[1], take)
        if self._scratch is None or self._scratch.numel() < size:
            self._scratch = torch.empty(size, dtype=torch.uint8, device=self.device)
        ops.beam_select(logits, torch.tensor(scores, dtype=torch.float32).to(self.device),
                        best.view(torch.float32), beam, token, self._scratch)
        self._host[: 3 * n].copy_(self._buffer[: 3 * n])
        host = self._host[: 3 * n].view(3, groups, take)
        columns = (host[0].view(torch.float32).tolist(), host[1].tolist(), host[2].tolist())
        return [[(s, b, t) for s, b, t in zip(*rows) if b >= 0] for rows in zip(*columns)]
