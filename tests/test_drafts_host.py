"""Drafted decoding above the step function, with a stand-in for the engine (no GPU)."""
import numpy as np
import pytest
import torch

from hk_b200.cache import CacheBooks
from hk_b200.engine import DraftDecoder
from hk_b200.sampling import SamplingParams
from test_beams_host import FakeEngine


class TreeEngine(FakeEngine):
    """A model of `logits_of(tokens)` that takes drafted trees."""

    takes_trees = True

    def __init__(self, logits_of, vocab, **options):
        super().__init__(logits_of, vocab, **options)
        self.cache.books = CacheBooks([None], page_tokens=4, num_pages=400, max_requests=4, max_context=self.max_context)
        self.trees, self.kinds = {}, []

    def check_step(self, entries):
        assert not any(e.request in self.trees for e in entries), "a tree waits for accept"

    def request_length(self, name):
        return len(self.texts[name])

    def step(self, entries):
        self.check_step(entries)
        trees = [e.parents is not None for e in entries]
        if not any(trees):
            if len(entries) > 1 or len(entries[0].tokens) == 1:
                self.kinds.append("plain")
            return super().step(entries)
        self.kinds.append("tree")
        rows = []
        for e in entries:
            texts = []
            for t, p in zip(e.tokens, e.parents):
                texts.append((texts[p] if p >= 0 else tuple(self.texts[e.request])) + (int(t),))
            rows += [self.logits_of(texts[i]) for i in e.want]
            self.trees[e.request] = texts
        return torch.from_numpy(np.stack(rows))

    def accept(self, accepted):
        for name, path in accepted.items():
            self.texts[name] = list(self.trees.pop(name)[path[-1]])

    def close_request(self, name):
        self.trees.pop(name, None)
        super().close_request(name)


class Argmax:
    def sample(self, logits, states):
        assert logits.shape[0] == len(states)
        for s in states:
            s.drawn += 1
        return logits.argmax(dim=1).int()

    def accept(self, state, token):
        state.history.append(token)


def model(seed, vocab, repeats):
    """Greedy text that never repeats a token (until all were), or that falls into cycles."""
    def logits_of(tokens):
        x = np.random.default_rng([seed, *[t + 1 for t in (tokens[-2:] if repeats else tokens)]]).standard_normal(vocab)
        if not repeats:
            x[list(set(tokens))] -= 100
        return x.astype(np.float32)
    return logits_of


def greedy(logits_of, prompt, most, eos=()):
    out = []
    while len(out) < most:
        t = int(logits_of(tuple(prompt) + tuple(out)).argmax())
        if t in eos:
            break
        out.append(t)
    return out


@pytest.mark.parametrize("repeats", [False, True])
@pytest.mark.parametrize("drafts", [1, 4, 9])
def test_drafted_decoding(drafts, repeats):
    logits_of = model(3, 300 if not repeats else 4, repeats)
    prompts = [[1], [2, 3], [0, 1, 2], [3, 2, 1]]
    eng = TreeEngine(logits_of, 300)
    decoder = DraftDecoder(eng, drafts, 40, sampler=Argmax())
    assert decoder.run(prompts, [SamplingParams(temperature=0.0)] * 4) == [greedy(logits_of, p, 40) for p in prompts]
    assert not eng.texts and (decoder.stats.drafted > 0) == repeats


def test_steps_without_a_guess_are_plain_steps():
    """What a step by step decoding would run, to the bit: no trees where no request has a guess."""
    logits_of = model(3, 300, False)
    eng = TreeEngine(logits_of, 300)
    DraftDecoder(eng, 8, 40, sampler=Argmax()).run([[1], [2, 3]], [SamplingParams(temperature=0.0)] * 2)
    assert set(eng.kinds) == {"plain"}
    # the last step of a request has no room for a guess that could be kept
    eng = TreeEngine(model(3, 4, True), 300)
    DraftDecoder(eng, 8, 12, sampler=Argmax()).run([[1, 2, 1, 2, 1]], [SamplingParams(temperature=0.0)])
    assert "tree" in eng.kinds


@pytest.mark.parametrize("repeats", [False, True])
def test_end_tokens(repeats):
    logits_of = model(5, 300 if not repeats else 4, repeats)
    full = greedy(logits_of, [1, 2], 40)
    eos = {full[17]}
    eng = TreeEngine(logits_of, 300)
    got = DraftDecoder(eng, 6, 40, eos_token_ids=eos, sampler=Argmax()).run([[1, 2]], [SamplingParams(temperature=0.0)])
    assert got == [greedy(logits_of, [1, 2], 40, eos)] and not eng.texts
