"""Decoding with drafted tokens: a step verifies a tree of guesses instead of making one token.

The guesses come from the request's own tokens (`LookupDrafts`): where its last few tokens stood before, what came behind them then is
a guess at what comes now; several such places make a tree.  A step runs the request's last token and the tree behind it
(`StepEntry.parents`), a token is drawn at every node from the logits there, and the path along which the tree guessed right is kept
(`Engine.accept`).  What is drawn at a node is what a step by step decoding would have drawn in its place (the same logits, the same
place of the request's random stream), so the output is the same: only the number of steps is smaller.  (In bfloat16 the logits of a
step with guesses can differ from a single step's in the last bits, as they do between batch sizes, and so can what is drawn where two
tokens are that close.  A step in which no request has a guess is a single step.)
"""
from __future__ import annotations

from collections import deque
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

from ..cache.pages import OutOfPages
from ..csrc.ops import TREE_TOKENS
from ..sampling import Sampler, SamplingParams, SamplingState
from .engine import Engine, EngineError, StepEntry, check_prompt
from .scheduler import fits_alone


class LookupDrafts:
    """Guesses from the tokens so far: the latest places where the last `most_match` .. 1 tokens stood before."""

    def __init__(self, tokens: Sequence[int], most_match: int = 3, branches: int = 4):
        self.tokens: List[int] = []
        self.most_match, self.branches = int(most_match), int(branches)
        self._places: Dict[tuple, List[int]] = {}       # n-gram -> where what follows it stands, the latest last
        self.extend(tokens)

    def extend(self, tokens: Sequence[int]) -> None:
        for t in tokens:
            at = len(self.tokens)
            for n in range(1, min(self.most_match, at) + 1):
                self._places.setdefault(tuple(self.tokens[at - n:at]), []).append(at)
            self.tokens.append(int(t))

    def tree(self, most: int) -> Tuple[List[int], List[int]]:
        """(tokens, parents) of up to `most` guesses behind the last token; parents are indices into the tokens, -1: the last token.
        Longer matches and later places come first."""
        tokens: List[int] = []
        parents: List[int] = []
        children: Dict[Tuple[int, int], int] = {}
        paths = 0
        seen = set()
        for n in range(min(self.most_match, len(self.tokens)), 0, -1):
            for place in reversed(self._places.get(tuple(self.tokens[len(self.tokens) - n:]), ())):
                if place in seen or place >= len(self.tokens):
                    continue
                seen.add(place)
                parent = -1
                for t in self.tokens[place:place + most]:
                    node = children.get((parent, t))
                    if node is None:
                        if len(tokens) == most:
                            break
                        node = children[(parent, t)] = len(tokens)
                        tokens.append(t)
                        parents.append(parent)
                    parent = node
                paths += 1
                if paths == self.branches or len(tokens) == most:
                    return tokens, parents
        return tokens, parents


@dataclass
class DraftStats:
    steps: int = 0            # steps of the engine behind the prompts
    tokens: int = 0           # tokens made by them
    drafted: int = 0          # guesses verified


@dataclass
class _Request:
    index: int
    drafts: LookupDrafts
    sampling: SamplingState
    pending: int = -1
    output: List[int] = field(default_factory=list)


class DraftDecoder:
    """`run(prompts, params)` generates up to `max_new_tokens` for every prompt, with up to `draft_tokens` guesses a step."""

    def __init__(self, engine: Engine, draft_tokens: int, max_new_tokens: int, eos_token_ids: Sequence[int] = (), prefill_chunk: int = 2048,
                 sampler: Optional[Sampler] = None):
        if not engine.takes_trees:
            raise EngineError("this model does not take trees of drafted tokens (a mixer keeps a state, or an attention that knows no trees)")
        if not 1 <= draft_tokens < TREE_TOKENS:
            raise ValueError(f"{draft_tokens} drafted tokens: between 1 and {TREE_TOKENS - 1} are taken")
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1")
        self.engine, self.most_drafts, self.most = engine, int(draft_tokens), int(max_new_tokens)
        self.eos = set(int(t) for t in eos_token_ids)
        self.chunk = max(1, min(int(prefill_chunk), engine.max_batch_tokens))
        self.sampler = sampler if sampler is not None else Sampler(engine.device)
        self.stats = DraftStats()

    def run(self, prompts: Sequence[Sequence[int]], params: Sequence[SamplingParams]) -> List[List[int]]:
        plist = [[int(t) for t in p] for p in prompts]
        if len(params) != len(plist):
            raise ValueError(f"{len(plist)} prompts and {len(params)} of sampling parameters")
        if any(p.adjusts_logits for p in params):
            raise ValueError("penalties and biases follow the tokens drawn so far: they cannot be had with drafted tokens")
        for p in plist:
            check_prompt(self.engine, p)
            if len(p) > self.engine.max_context:
                raise EngineError(f"the prompt has {len(p)} tokens; the context holds {self.engine.max_context}")
            if not fits_alone(self.engine.cache.books, min(len(p) + self.most - 1, self.engine.max_context), self.engine.max_batch_tokens):
                raise OutOfPages(f"a prompt of {len(p)} tokens and its continuation need more pages than there are")
        out: List[List[int]] = [[] for _ in plist]
        waiting = deque(_Request(i, LookupDrafts(p), SamplingState.start(s, p)) for i, (p, s) in enumerate(zip(plist, params)))
        running: List[_Request] = []
        names = set()
        try:
            while waiting or running:
                while waiting and len(running) < min(self.engine.cache.books.max_requests, self.engine.max_batch_tokens):
                    if not self._open(waiting[0], running, names, out):
                        break
                    waiting.popleft()
                if running:
                    self._step(running, waiting, names, out)
        finally:
            for n in list(names):
                self._close(n, names)
        self.engine.check_kernel_status()
        return out

    def _close(self, name, names) -> None:
        if self.engine.has_request(name):
            self.engine.close_request(name)
        names.discard(name)

    def _open(self, r: _Request, running, names, out) -> bool:
        """Reads a request's tokens and, where it has none yet, draws its first one; False where the pool has no room for it beside
        those that run."""
        eng, name = self.engine, ("drafts", r.index)
        books = eng.cache.books
        tokens = r.drafts.tokens[:-1] if r.output else r.drafts.tokens          # (put back: all but the token that waits)
        need = -(-(len(tokens) + 1) // books.page_tokens)
        if running and min(books.free_pages(), default=need) < need + len(running):
            return False
        eng.open_request(name)
        names.add(name)
        logits = None
        for a in range(0, len(tokens), self.chunk):
            part = tokens[a:a + self.chunk]
            last = a + len(part) == len(tokens) and not r.output
            logits = eng.step([StepEntry(name, part, [len(part) - 1] if last else [])])
        if r.output or self._take(r, [int(self.sampler.sample(logits, [r.sampling]).item())]):
            running.append(r)
        else:
            self._close(name, names)
            out[r.index] = r.output
        return True

    def _take(self, r: _Request, tokens: List[int]) -> bool:
        """Adds drawn tokens to the output, in order; False when the request ends with one of them."""
        for t in tokens:
            self.sampler.accept(r.sampling, t)
            if t in self.eos:
                return False
            r.output.append(t)
            r.drafts.extend([t])
            r.pending = t
            if len(r.output) >= self.most or len(r.drafts.tokens) > self.engine.max_context:
                return False
        return True

    def _entries(self, running: List[_Request], most: int):
        eng = self.engine
        share = eng.max_batch_tokens // len(running)
        trees, entries = [], []
        for r in running:
            name = ("drafts", r.index)
            # no guess that could not be kept: the output's end, the context's, the step's
            room = min(most, share - 1, self.most - len(r.output) - 1, eng.max_context - eng.request_length(name) - 1)
            tokens, parents = r.drafts.tree(room) if room > 0 else ([], [])
            trees.append(([r.pending] + tokens, [-1] + [p + 1 for p in parents]))
            entries.append(StepEntry(name, trees[-1][0], list(range(len(trees[-1][0]))), trees[-1][1]))
        if all(len(tokens) == 1 for tokens, _ in trees):       # nobody has a guess: a step by step decoding's step, captured as that one is
            entries = [StepEntry(e.request, e.tokens, [0]) for e in entries]
        return trees, entries

    def _step(self, running: List[_Request], waiting, names, out) -> None:
        eng, most = self.engine, self.most_drafts
        while True:
            trees, entries = self._entries(running, most)
            try:
                eng.check_step(entries)
                break
            except OutOfPages:
                if most > 0:
                    most //= 2                    # fewer guesses need fewer pages
                elif len(running) > 1:            # not even a token each: the newest gives up its pages and comes back later
                    waiting.appendleft(running.pop())
                    self._close(("drafts", waiting[0].index), names)
                else:
                    raise
        logits = eng.step(entries)
        self.stats.steps += 1
        # every node draws with the place of the stream that the token behind it has
        states = []
        for r, (tokens, parents) in zip(running, trees):
            depth: List[int] = []
            for p in parents:
                depth.append(0 if p < 0 else depth[p] + 1)
            states += [SamplingState(r.sampling.params, r.sampling.seed, r.sampling.drawn + d) for d in depth]
        drawn = self.sampler.sample(logits, states).tolist()
        accepted, at = {}, 0
        going: List[_Request] = []
        for r, (tokens, parents) in zip(running, trees):
            mine = drawn[at:at + len(tokens)]
            at += len(tokens)
            path = [0]
            while True:
                child = next((j for j in range(path[-1] + 1, len(tokens)) if parents[j] == path[-1] and tokens[j] == mine[path[-1]]), None)
                if child is None:
                    break
                path.append(child)
            new = [mine[j] for j in path]
            self.stats.drafted += len(tokens) - 1
            before = len(r.output)
            name = ("drafts", r.index)
            goes_on = self._take(r, new)
            self.stats.tokens += len(r.output) - before
            r.sampling.drawn += len(new)
            if goes_on:
                if entries[0].parents is not None:
                    accepted[name] = path
                going.append(r)
            else:
                self._close(name, names)
                out[r.index] = r.output
        if accepted:
            eng.accept(accepted)
        running[:] = going
