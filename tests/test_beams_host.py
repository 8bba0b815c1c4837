"""Beam search above the step function against a search that sorts all continuations, with stand-ins for the engine and the device's
choice (no GPU)."""
import itertools
import types

import numpy as np
import pytest
import torch

from hk_b200.engine.beams import BeamSearch
from ref_branches import beam_reference


class FakeEngine:
    """A model whose logits are a function of a request's tokens: `logits_of(tokens)`, float32 [vocab]."""

    def __init__(self, logits_of, vocab, max_requests=128, max_batch_tokens=2048, max_context=1000):
        self.logits_of, self.vocab = logits_of, vocab
        self.max_batch_tokens, self.max_context = max_batch_tokens, max_context
        self.cache = types.SimpleNamespace(books=types.SimpleNamespace(max_requests=max_requests))
        self.texts = {}
        self.steps = []

    def take_slot(self, name, tokens):
        from hk_b200.cache.pages import TooManyRequests
        assert name not in self.texts
        if len(self.texts) == self.cache.books.max_requests:
            raise TooManyRequests("no slot")
        self.texts[name] = tokens

    def open_request(self, name):
        self.take_slot(name, [])

    def close_request(self, name):
        del self.texts[name]

    def has_request(self, name):
        return name in self.texts

    def fork_request(self, name, new):
        self.take_slot(new, list(self.texts[name]))

    def reorder(self, names, parents):
        old = [list(self.texts[n]) for n in names]
        for n, p in zip(names, parents):
            self.texts[n] = list(old[p])

    def step(self, entries):
        self.steps.append(sum(len(e.tokens) for e in entries))
        rows = []
        for e in entries:
            for i, t in enumerate(e.tokens):
                self.texts[e.request].append(int(t))
                if i in e.want:
                    rows.append(self.logits_of(tuple(self.texts[e.request])))
        return torch.from_numpy(np.stack(rows)) if rows else None

    def check_kernel_status(self):
        pass


@pytest.fixture
def choice(monkeypatch):
    """`ops.beam_select` by its 64-bit form, within the sizes that it takes."""
    from hk_b200.csrc import ops

    def select(logits, scores, n_beams, out_scores, out_beams, out_tokens):
        choices = out_scores.shape[1]
        assert logits.dtype == scores.dtype == torch.float32 and logits.shape[0] == scores.shape[0] == out_scores.shape[0] * n_beams
        assert n_beams <= 256 and 1 <= choices <= min(256, n_beams * logits.shape[1])
        s, k, v = beam_reference(logits.numpy(), scores.numpy(), n_beams, choices)
        out_scores.copy_(torch.from_numpy(s.astype(np.float32)))
        out_beams.copy_(torch.from_numpy(k.astype(np.int32)))
        out_tokens.copy_(torch.from_numpy(v.astype(np.int32)))
    monkeypatch.setattr(ops, "beam_select", select)


def all_continuations(logits_of, vocab, prompt, beams, most, penalty, eos):
    """Beam search that sorts every continuation of every beam: (tokens, score, ended), best first."""
    live, finished = [((), 0.0)], []
    while live:
        options = []
        for k, (toks, s) in enumerate(live):
            x = logits_of(tuple(prompt) + toks).astype(np.float64)
            lp = x - (x.max() + np.log(np.exp(x - x.max()).sum()))
            options += [(-(s + lp[v]), k, v) for v in range(vocab) if np.isfinite(lp[v])]
        nxt = []
        for rank, (neg, k, v) in enumerate(sorted(options)):
            if v not in eos and len(nxt) < beams:
                nxt.append((live[k][0] + (v,), -neg))
            elif v in eos and rank < beams:
                finished.append((live[k][0], -neg / (len(live[k][0]) + 1) ** penalty, True))
        live = nxt
        if live and len(live[0][0]) >= most:
            finished += [(t, s / len(t) ** penalty, False) for t, s in live]
            live = []
        if live and len(finished) >= beams:
            best = max(s for _, s in live) / (most if penalty > 0 else len(live[0][0])) ** penalty
            if best <= sorted((f[1] for f in finished), reverse=True)[beams - 1]:
                live = []
    return sorted(finished, key=lambda f: -f[1])[:beams]


def random_model(seed, vocab, eos, lift):
    """Logits drawn from the text; those of the end tokens lie `lift` higher."""
    def logits_of(tokens):
        x = np.random.default_rng([seed, *[t + 1 for t in tokens]]).standard_normal(vocab) * 2
        x[sorted(eos)] += lift
        return x.astype(np.float32)
    return logits_of


def agree(mine, want, most):
    assert [c.tokens for c in mine] == [list(t) for t, _, _ in want]
    assert [c.ended for c in mine] == [e for _, _, e in want]
    # scores are float32 sums: each of up to `most` + 1 roundings is 2^-24 of a sum below 2^6 (a step's log probability is above -2^4)
    assert all(abs(c.score - s) <= (most + 1) * 2.0 ** -18 for c, (_, s, _) in zip(mine, want))


def test_two_likely_end_tokens_leave_the_better_continuation(choice):
    """Both end tokens are likelier than the one token that goes on with certainty: the beams that go on stay."""
    vocab, eos = 12, (0, 1)

    def logits_of(tokens):
        p = np.full(vocab, 1e-4)
        if len(tokens) == 1:                       # behind the prompt
            p[5:9] = 0.26, 0.25, 0.24, 0.23
        elif len(tokens) == 2:
            p[[0, 1, 4]] = 0.36, 0.34, 0.30
        else:
            p[4] = 1.0
        return np.log(p / p.sum()).astype(np.float32)
    got = BeamSearch(FakeEngine(logits_of, vocab), 4, 10, 1.0, eos).run([[3]])[0]
    agree(got, all_continuations(logits_of, vocab, [3], 4, 10, 1.0, set(eos)), 10)
    assert got[0].tokens == [5] + [4] * 9 and not got[0].ended and got[0].score > -0.27


@pytest.mark.parametrize("beams,ends", list(itertools.product((1, 2, 5), (0, 1, 2, 3, 7))) + [(100, 2), (128, 1), (128, 3)])
def test_beams_and_end_tokens(beams, ends, choice):
    """Up to (end tokens) ended choices a beam; with more than the operator's 256 choices too."""
    vocab = 11 if beams < 100 else 40
    for seed in range(3):
        eos = set(np.random.default_rng(seed).permutation(vocab)[:ends].tolist())
        logits_of = random_model(seed, vocab, eos, 6.0)
        prompts = [[1], [2, 3], [4]]
        most = 6 if beams < 100 else 4
        got = BeamSearch(FakeEngine(logits_of, vocab, max_requests=256), beams, most, 0.7, tuple(eos) + (vocab + 5, -1)).run(prompts)
        for p, mine in zip(prompts, got):
            agree(mine, all_continuations(logits_of, vocab, p, beams, most, 0.7, eos), most)


def test_every_token_ends(choice):
    vocab = 6
    logits_of = random_model(1, vocab, set(), 0.0)
    got = BeamSearch(FakeEngine(logits_of, vocab), 3, 5, 1.0, range(vocab)).run([[1]])[0]
    agree(got, all_continuations(logits_of, vocab, [1], 3, 5, 1.0, set(range(vocab))), 5)
    assert [c.tokens for c in got] == [[]] * 3 and all(c.ended for c in got)


class SmallPool(FakeEngine):
    """The same with room for `most` tokens in all requests together."""

    def __init__(self, logits_of, vocab, most, **options):
        super().__init__(logits_of, vocab, **options)
        self.most = most

    def step(self, entries):
        from hk_b200.cache.pages import OutOfPages
        if sum(map(len, self.texts.values())) + sum(len(e.tokens) for e in entries) > self.most:
            raise OutOfPages("no room")
        return super().step(entries)


@pytest.mark.parametrize("most", [30, 45, 60, 1000])
def test_prompts_that_do_not_fit_together(most, choice):
    """Fewer prompts at once where the pool has no room for as many as there are slots; an error only where one alone has none."""
    from hk_b200.cache.pages import OutOfPages
    logits_of = random_model(2, 11, {3}, 2.0)
    prompts = [[1, 2], [3], [4, 5, 6], [7], [8, 9]]
    eng = SmallPool(logits_of, 11, most)
    got = BeamSearch(eng, 3, 6, 1.0, (3,)).run(prompts)
    for p, mine in zip(prompts, got):
        agree(mine, all_continuations(logits_of, 11, p, 3, 6, 1.0, {3}), 6)
    assert not eng.texts
    with pytest.raises(OutOfPages):
        BeamSearch(SmallPool(logits_of, 11, 10), 3, 6, 1.0, (3,)).run(prompts)


def test_slots_that_other_requests_hold(choice):
    logits_of = random_model(2, 11, {3}, 2.0)
    eng = FakeEngine(logits_of, 11, max_requests=12)
    for i in range(5):
        eng.open_request(i)
    prompts = [[1, 2], [3], [4, 5, 6], [7], [8, 9]]
    got = BeamSearch(eng, 3, 6, 1.0, (3,)).run(prompts)
    for p, mine in zip(prompts, got):
        agree(mine, all_continuations(logits_of, 11, p, 3, 6, 1.0, {3}), 6)
    assert sorted(eng.texts) == list(range(5))


def test_more_beams_than_a_step_takes():
    """Known before any prompt is read."""
    eng = FakeEngine(random_model(1, 11, set(), 0.0), 11, max_batch_tokens=7)
    BeamSearch(eng, 7, 4)
    with pytest.raises(ValueError):
        BeamSearch(eng, 8, 4)


@pytest.mark.parametrize("bad", [[], [11], [-1], [3, 4, 99]])
def test_prompts_are_looked_at_before_any_is_read(bad, choice):
    from hk_b200.engine import EngineError
    eng = FakeEngine(random_model(1, 11, set(), 0.0), 11)
    with pytest.raises((EngineError, ValueError)):
        BeamSearch(eng, 2, 4).run([[1], [2], bad])
    assert not eng.steps


def test_drafted_requests_are_looked_at_before_any_is_read():
    """As the scheduler does: tokens outside the vocabulary, more than the pool holds, and sampling parameters for each prompt."""
    from hk_b200.cache import CacheBooks, OutOfPages
    from hk_b200.engine import DraftDecoder, EngineError
    from hk_b200.sampling import SamplingParams
    eng = FakeEngine(random_model(1, 11, set(), 0.0), 11, max_context=64)
    eng.takes_trees, eng.cache.books = True, CacheBooks([None], page_tokens=4, num_pages=5, max_requests=3, max_context=64)
    greedy = SamplingParams(temperature=0.0)
    for prompts, n, kind in (([[1], []], 2, ValueError), ([[1], [11]], 2, EngineError), ([[1], [2, -1]], 2, EngineError), ([[1], [2]], 1, ValueError),
                             ([[1], [2]], 3, ValueError), ([[1], [2] * 65], 2, EngineError), ([[1], [2] * 17], 2, OutOfPages)):
        with pytest.raises(kind):
            DraftDecoder(eng, 3, 5, sampler=object()).run(prompts, [greedy] * n)
    assert not eng.steps
