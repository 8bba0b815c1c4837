"""Beam search above the step function: the most probable continuations of a prompt, several at a time.

The beams of a prompt are requests of the engine.  A step runs all beams of all prompts as one decode batch, `ops.beam_select` chooses
the best continuations over beams and vocabulary on the device (one more per beam and end token than there are beams, so that enough are
left when some of them end), and `Engine.reorder` makes the requests go on with the beams chosen: pages are shared until a beam writes
them, states are copied.

A continuation that ends (an end token among the first `beams` choices of its step, or the most tokens) is a finished one; finished
ones are ordered by the sum of their tokens' log probabilities over length^length_penalty, the end token's probability included.  A
prompt is done when it has `beams` finished ones and no running one can be better than the worst of them any more.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..cache.pages import OutOfPages, TooManyRequests
from ..csrc import ops
from ..csrc.ops import BEAM_CHOICES
from .engine import Engine, EngineError, StepEntry, check_prompt


@dataclass
class Continuation:
    tokens: List[int]
    score: float          # the sum of log probabilities over length^length_penalty
    ended: bool           # on an end token (which is not among the tokens)


@dataclass
class _Prompt:
    index: int
    names: List[tuple]
    outputs: List[List[int]] = field(default_factory=list)     # of the running beams
    scores: List[float] = field(default_factory=list)
    finished: List[Continuation] = field(default_factory=list)


class BeamSearch:
    """`run(prompts)` gives every prompt its `beams` best continuations, best first."""

    def __init__(self, engine: Engine, beams: int, max_new_tokens: int, length_penalty: float = 1.0, eos_token_ids: Sequence[int] = (),
                 prefill_chunk: int = 2048):
        if beams < 1 or beams > 128:
            raise ValueError(f"{beams} beams: between 1 and 128 are taken")
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1")
        if beams > engine.cache.books.max_requests:
            raise ValueError(f"{beams} beams need as many request slots; the engine has {engine.cache.books.max_requests}")
        if beams > engine.max_batch_tokens:
            raise ValueError(f"{beams} beams are as many tokens a step; the engine takes {engine.max_batch_tokens}")
        self.engine, self.beams, self.most, self.penalty = engine, int(beams), int(max_new_tokens), float(length_penalty)
        self.eos = set(int(t) for t in eos_token_ids if 0 <= int(t) < engine.vocab)
        self.chunk = max(1, min(int(prefill_chunk), engine.max_batch_tokens))

    def run(self, prompts: Sequence[Sequence[int]]) -> List[List[Continuation]]:
        plist = [[int(t) for t in p] for p in prompts]
        for p in plist:
            check_prompt(self.engine, p)
            if len(p) + self.most - 1 > self.engine.max_context:
                raise EngineError(f"a prompt of {len(p)} tokens and {self.most} new ones pass the context of {self.engine.max_context}")
        at_once = max(1, min(self.engine.cache.books.max_requests, self.engine.max_batch_tokens) // self.beams)
        out: List[List[Continuation]] = []
        while len(out) < len(plist):
            group = plist[len(out):len(out) + at_once]
            try:
                out += self._group(group)
            except (OutOfPages, TooManyRequests):
                if len(group) == 1:
                    raise
                at_once = len(group) // 2        # pages, or slots that other requests leave, for fewer
        self.engine.check_kernel_status()
        return out

    # -- one batch of prompts ------------------------------------------------------------------
    def _group(self, plist) -> List[List[Continuation]]:
        group = [_Prompt(i, [("beam", i, 0)]) for i in range(len(plist))]
        opened = []
        try:
            for g, p in zip(group, plist):
                self.engine.open_request(g.names[0])
                opened.append(g.names[0])
                logits = None
                for a in range(0, len(p), self.chunk):
                    part = p[a:a + self.chunk]
                    logits = self.engine.step([StepEntry(g.names[0], part, [len(part) - 1] if a + len(part) == len(p) else [])])
                g.scores, g.outputs = [0.0], [[]]
                self._choose([g], logits, opened)
            running = [g for g in group if self._goes_on(g)]
            while running:
                logits = self.engine.step([StepEntry(n, [o[-1]], [0]) for g in running for n, o in zip(g.names, g.outputs)])
                self._choose(running, logits, opened)
                running = [g for g in running if self._goes_on(g)]
        finally:
            for name in opened:
                if self.engine.has_request(name):
                    self.engine.close_request(name)
        return [sorted(g.finished, key=lambda c: -c.score)[:self.beams] for g in group]

    def _final(self, total: float, length: int) -> float:
        return total / max(length, 1) ** self.penalty

    def _goes_on(self, g: _Prompt) -> bool:
        if not g.outputs:
            return False                       # every choice ended; its requests are closed
        length = len(g.outputs[0])
        if length >= self.most:
            g.finished += [Continuation(list(o), self._final(s, length), False) for o, s in zip(g.outputs, g.scores)]
        elif len(g.finished) < self.beams:
            return True
        else:
            # what the best running beam can come to: its sum only falls, and a positive penalty divides it by more as it grows
            best, last = max(g.scores), self.most if self.penalty > 0 else length
            if self._final(best, last) > sorted((c.score for c in g.finished), reverse=True)[self.beams - 1]:
                return True
        for n in g.names:
            self.engine.close_request(n)
        g.outputs = []
        return False

    def _choose(self, prompts: List[_Prompt], logits: torch.Tensor, opened: List[tuple]) -> None:
        """The next beams of prompts with equally many running beams each (a prompt with fewer has places that are not there)."""
        width = max(len(g.names) for g in prompts)
        scores = np.full((len(prompts), width), -np.inf, dtype=np.float32)
        for i, g in enumerate(prompts):
            scores[i, :len(g.scores)] = g.scores
        if any(len(g.names) < width for g in prompts):         # rows for the places that are not there
            rows, at = [], 0
            for g in prompts:
                rows += [at + min(k, len(g.names) - 1) for k in range(width)]
                at += len(g.names)
            logits = logits[torch.tensor(rows, device=logits.device)]
        scores = torch.from_numpy(scores.reshape(-1)).to(logits.device)
        # `beams` choices that go on are among the best beams + (end tokens) * width
        most = self.beams + len(self.eos) * width
        ahead = chosen = self._best(logits, scores, width, min(most, width * self.engine.vocab)) if most <= BEAM_CHOICES else None
        if chosen is None:                                     # all end tokens as one, with their probabilities together
            ahead = self._best(logits, scores, width, min(self.beams, width * self.engine.vocab))
            chosen = self._best(self._ends_as_one(logits), scores, width, min(self.beams + width, width * (self.engine.vocab + 1)))
        for i, g in enumerate(prompts):
            parents, outputs, totals = [], [], []
            for s, k, t in ahead[i][:self.beams]:
                if s != -np.inf and t in self.eos:
                    g.finished.append(Continuation(list(g.outputs[k]), self._final(s, len(g.outputs[k]) + 1), True))
            for s, k, t in chosen[i]:
                if s == -np.inf or len(parents) == self.beams:
                    break
                if t in self.eos or t == self.engine.vocab:
                    continue
                parents.append(k)
                outputs.append(g.outputs[k] + [t])
                totals.append(s)
            self._follow(g, parents, opened)
            g.outputs, g.scores = outputs, totals

    @staticmethod
    def _best(logits: torch.Tensor, scores: torch.Tensor, width: int, choices: int) -> List[List[tuple]]:
        """For each prompt (score, beam, token) of its best choices, best first."""
        prompts, dev = logits.shape[0] // width, logits.device
        best = torch.empty((prompts, choices), dtype=torch.float32, device=dev)
        beam, token = (torch.empty((prompts, choices), dtype=torch.int32, device=dev) for _ in range(2))
        ops.beam_select(logits, scores, width, best, beam, token)
        return [list(zip(*lists)) for lists in zip(best.tolist(), beam.tolist(), token.tolist())]

    def _ends_as_one(self, logits: torch.Tensor) -> torch.Tensor:
        """The logits with the end tokens masked and a token more, as probable as all of them together (its logit is rounded to float32,
        2^-24 of it: what the sum of a row's exponentials can be off by)."""
        ends = torch.tensor(sorted(self.eos), device=logits.device)
        x = logits[:, ends].double()
        x = torch.where(torch.isfinite(x), x, -torch.inf)
        out = torch.cat([logits, torch.logsumexp(x, dim=1, keepdim=True).float()], dim=1)
        out[:, ends] = -torch.inf
        return out

    def _follow(self, g: _Prompt, parents: List[int], opened: List[tuple]) -> None:
        """Makes the prompt's requests the chosen beams, as many as there are parents."""
        eng, had = self.engine, len(g.names)
        for k in parents[had:]:                                # more beams than before (the first step): forks
            name = ("beam", g.index, len(g.names))
            eng.fork_request(g.names[k], name)
            opened.append(name)
            g.names.append(name)
        now = parents[:had]
        if now and now != list(range(had)):
            eng.reorder(g.names[:had], now + [now[0]] * (had - len(now)))
        for n in g.names[len(parents):]:                       # fewer continuations than beams
            eng.close_request(n)
        del g.names[len(parents):]
