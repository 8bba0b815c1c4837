"""Several continuations of one request through the engine: drafted trees, forks, beams, drafted generation."""
import importlib
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import helpers
import plain_qwen3 as P

pytestmark = pytest.mark.gpu
ROOT = os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir)

# the engine's tolerances against the plain implementation: max |difference| relative to the largest |logit|
TOL = {torch.float32: 2e-5, torch.bfloat16: 2e-2}

_models = {}


def model(tmp_path_factory, which, dtype):
    if (which, dtype) not in _models:
        d = helpers.make_model_dir(tmp_path_factory.mktemp("branches"), which, dtype)
        _models[which, dtype] = (d,) + helpers.load_plain(d)
    return _models[which, dtype]


def random_tree(rng, count, vocab):
    parents = [-1] + [int(rng.integers(max(-1, i - 6), i)) for i in range(1, count)]
    return rng.integers(0, vocab, count).tolist(), parents


def path_to(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which,page", [("A", 4), ("B", 8), ("C", 16), ("D", 16), ("E", 32), ("F", 16), ("G", 8)])
def test_trees_against_the_plain_model(which, page, dtype, tmp_path_factory):
    """Every node of drafted trees sees its own path, before and after paths were accepted; beside a request whose tokens follow one
    another."""
    import hk_b200
    from hk_b200.engine import StepEntry
    d, cfg, w = model(tmp_path_factory, which, dtype)
    rng = np.random.default_rng(3)
    vocab = cfg["vocab_size"]
    eng = hk_b200.Engine(d, dtype=dtype, max_tokens=600, page_tokens=page, max_requests=4, max_context=200, max_batch_tokens=300)
    assert eng.takes_trees
    text = {r: rng.integers(0, vocab, n).tolist() for r, n in (("a", 37), ("b", 5), ("c", 64))}
    for r, ids in text.items():
        eng.open_request(r)
        eng.step([StepEntry(r, ids, [])])
    scale = max(np.abs(P.forward(cfg, w, ids)).max() for ids in text.values())
    for round_ in range(3):
        trees = {"a": random_tree(rng, int(rng.integers(1, 20)), vocab), "b": random_tree(rng, int(rng.integers(2, 40)), vocab)}
        chain = rng.integers(0, vocab, 7).tolist()
        entries = [StepEntry(r, toks, list(range(len(toks))), parents) for r, (toks, parents) in trees.items()] + [StepEntry("c", chain, [2, 6])]
        logits = eng.step(entries).float().cpu().numpy()
        at = 0
        for r, (toks, parents) in trees.items():
            leaves = [i for i in range(len(toks)) if i not in parents]
            for leaf in leaves:
                path = path_to(parents, leaf)
                want = P.forward(cfg, w, text[r] + [toks[i] for i in path])[-len(path):]
                off = np.abs(logits[[at + i for i in path]] - want).max()
                assert off <= TOL[dtype] * scale, (r, round_, off / scale)
            at += len(toks)
        want = P.forward(cfg, w, text["c"] + chain)
        assert np.abs(logits[at:] - want[[len(text["c"]) + 2, len(text["c"]) + 6]]).max() <= TOL[dtype] * scale
        text["c"] = text["c"] + chain
        accepted = {}
        for r, (toks, parents) in trees.items():
            path = path_to(parents, int(rng.integers(0, len(toks))))
            accepted[r] = path
            text[r] = text[r] + [toks[i] for i in path]
        eng.accept(accepted)
        assert all(eng.request_length(r) == len(ids) for r, ids in text.items())
        eng.cache.books.audit()
        # plain decoding goes on where the path ended
        nxt = {r: int(rng.integers(0, vocab)) for r in text}
        logits = eng.step([StepEntry(r, [t], [0]) for r, t in nxt.items()]).float().cpu().numpy()
        for row, (r, t) in zip(logits, nxt.items()):
            text[r] = text[r] + [t]
            assert np.abs(row - P.forward(cfg, w, text[r])[-1]).max() <= TOL[dtype] * scale
    eng.check_kernel_status()


def test_tree_refusals(tmp_path_factory):
    import hk_b200
    from hk_b200.engine import EngineError, StepEntry, UnknownRequest
    d, cfg, w = model(tmp_path_factory, "A", torch.float32)
    eng = hk_b200.Engine(d, dtype="float32", max_tokens=128, page_tokens=4, max_requests=3, max_context=100)
    eng.open_request("a")
    eng.step([StepEntry("a", [1, 2, 3], [])])
    for tokens, parents in (([4, 5], [-1]), ([4, 5], [-1, 1]), ([4, 5], [0, -1]), ([4, 5], [-2, -1]), ([], [])):
        with pytest.raises(EngineError):
            eng.step([StepEntry("a", tokens, [0] if tokens else [], parents)])
    with pytest.raises(EngineError):
        eng.accept({"a": [0]})                       # no tree
    assert eng.request_length("a") == 3
    eng.step([StepEntry("a", [4, 5, 6, 7], [0], [-1, 0, 0, 1])])
    for call in (lambda: eng.step([StepEntry("a", [8], [0])]), lambda: eng.fork_request("a", "b"), lambda: eng.reorder(["a"], [0])):
        with pytest.raises(EngineError):
            call()                                   # the tree waits for accept
    for kept in ([], [1], [0, 3], [0, 2, 3], [0, 1, 9], [0, 1, 1]):
        with pytest.raises(EngineError):
            eng.accept({"a": kept})
    with pytest.raises(UnknownRequest):
        eng.accept({"x": [0]})
    eng.accept({"a": [0, 1, 3]})
    assert eng.request_length("a") == 6
    eng.fork_request("a", "b")
    with pytest.raises(EngineError):
        eng.fork_request("a", "b")
    for parents in ([0], [0, 2], [-1, 0]):
        with pytest.raises(EngineError):
            eng.reorder(["a", "b"], parents)
    with pytest.raises(EngineError):
        eng.reorder(["a", "a"], [0, 0])
    eng.step([StepEntry("a", [4, 5], [0], [-1, -1])])
    eng.close_request("a")                           # with its tree
    eng.open_request("a")
    eng.step([StepEntry("a", [1], [0])])
    eng.cache.books.audit()


def test_models_that_take_no_trees(tmp_path):
    import hk_b200
    import kedanex_models
    from hk_b200.engine import DraftDecoder, EngineError, StepEntry
    d = kedanex_models.make_model_dir(tmp_path, "X", torch.float32)
    eng = hk_b200.Engine(d, dtype="float32", max_tokens=128, page_tokens=4, max_requests=2, max_context=64)
    assert not eng.takes_trees
    eng.open_request("a")
    with pytest.raises(EngineError):
        eng.step([StepEntry("a", [1, 2], [0], [-1, 0])])
    with pytest.raises(EngineError):
        DraftDecoder(eng, 4, 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("family,which", [("", "A"), ("", "C"), ("", "E"), ("kedanex", "X"), ("mifolorn", None), ("gezavik", None), ("nebanex", None),
                                          ("padodra", None), ("zazulix", None)])
def test_forks_go_on_like_requests_of_their_own(family, which, dtype, tmp_path):
    """A forked request, and beams that are reordered, give what requests with the same tokens of their own give, to the bit."""
    import hk_b200
    from hk_b200.engine import StepEntry
    if family:
        m = importlib.import_module(f"{family}_models")
        which = which or sorted(m.CONFIGS)[0]
        d = m.make_model_dir(tmp_path, which, dtype)
    else:
        d = helpers.make_model_dir(tmp_path, which, dtype)
    make = lambda: hk_b200.Engine(d, dtype=dtype, max_tokens=1024, page_tokens=4, max_requests=4, max_context=120)  # noqa: E731
    forked, apart = make(), make()
    rng = np.random.default_rng(1)
    vocab = forked.vocab
    prompt = rng.integers(0, vocab, 22).tolist()
    names = ["a", "b", "c", "d"]
    forked.open_request("a")
    forked.step([StepEntry("a", prompt, [])])
    for n in names[1:]:
        forked.fork_request("a", n)
    for n in names:
        apart.open_request(n)
        apart.step([StepEntry(n, prompt, [])])
    texts = {n: [] for n in names}
    orders = [None, [0, 0, 2, 2], None, [3, 2, 1, 0], [1, 1, 1, 1], None, [2, 0, 3, 3], [0, 1, 2, 3], None]
    for order in orders:
        toks = {n: int(rng.integers(0, vocab)) for n in names}
        got = forked.step([StepEntry(n, [toks[n]], [0]) for n in names])
        want = apart.step([StepEntry(n, [toks[n]], [0]) for n in names])
        assert torch.equal(got, want)
        for n in names:
            texts[n] = texts[n] + [toks[n]]
        if order is not None:
            forked.reorder(names, order)
            forked.cache.books.audit()
            texts = {n: texts[names[p]] for n, p in zip(names, order)}
            for n in names:                            # the same tokens again, in the same steps
                apart.close_request(n)
            for n in names:
                apart.open_request(n)
                apart.step([StepEntry(n, prompt, [])])
            for i in range(len(texts["a"])):
                apart.step([StepEntry(n, [texts[n][i]], [0]) for n in names])
    for n in names:
        forked.close_request(n)
    assert forked.free_pages() == [g.pool.num_pages for g in forked.cache.books.groups]
    forked.check_kernel_status()


def test_a_step_that_just_fits_the_shared_pages(tmp_path_factory):
    """All holders of a page write it in one step: the last of them needs no page of its own."""
    import hk_b200
    from hk_b200.cache import OutOfPages
    from hk_b200.engine import StepEntry
    d, cfg, w = model(tmp_path_factory, "A", torch.float32)
    eng = hk_b200.Engine(d, dtype="float32", max_tokens=16, page_tokens=4, max_requests=4, max_context=40)
    eng.open_request("a")
    eng.step([StepEntry("a", [1, 2, 3, 4, 5, 6], [])])
    eng.fork_request("a", "b")
    eng.fork_request("a", "c")                         # two pages held, two free: three writers need two copies
    got = eng.step([StepEntry(n, [t], [0]) for n, t in (("a", 7), ("b", 8), ("c", 9))]).cpu().numpy()
    for row, t in zip(got, (7, 8, 9)):
        want = P.forward(cfg, w, [1, 2, 3, 4, 5, 6, t])[-1]
        assert np.abs(row - want).max() <= TOL[torch.float32] * np.abs(want).max()
    assert eng.free_pages() == [0]
    eng.fork_request("a", "d")
    with pytest.raises(OutOfPages):
        eng.step([StepEntry("d", [1], [0])])
    eng.close_request("a")
    eng.step([StepEntry("d", [1], [0])])
    eng.cache.books.audit()


# ---- beams -----------------------------------------------------------------------------------------------------------------


def plain_beams(cfg, w, prompt, beams, most, penalty, eos):
    """Beam search in plain steps: (tokens, score, ended), best first."""
    live, finished = [([], 0.0)], []
    while live:
        options = []
        for k, (toks, s) in enumerate(live):
            x = P.forward(cfg, w, prompt + toks)[-1].astype(np.float64)
            lp = x - (x.max() + np.log(np.exp(x - x.max()).sum()))
            options += [(-(s + lp[v]), k, v) for v in np.argsort(-lp, kind="stable")[:2 * beams]]
        options = sorted(options)[:2 * beams]
        nxt = []
        for rank, (neg, k, v) in enumerate(options):
            if len(nxt) == beams:
                break
            toks = live[k][0]
            if v in eos:
                if rank < beams:
                    finished.append((toks, -neg / (len(toks) + 1) ** penalty, True))
                continue
            nxt.append((toks + [int(v)], -neg))
        live = nxt
        if live and len(live[0][0]) >= most:
            finished += [(t, s / len(t) ** penalty, False) for t, s in live]
            live = []
        if live and len(finished) >= beams:
            best = max(s for _, s in live) / (most if penalty > 0 else len(live[0][0])) ** penalty
            if best <= sorted((f[1] for f in finished), reverse=True)[beams - 1]:
                live = []
    return sorted(finished, key=lambda f: -f[1])[:beams]


@pytest.mark.parametrize("which,beams,most,penalty,eos", [("A", 1, 6, 1.0, ()), ("A", 4, 7, 1.0, ()), ("B", 3, 6, 0.0, ()), ("C", 5, 5, 2.0, ()),
                                                          ("A", 4, 9, 1.0, tuple(range(0, 256, 5))), ("B", 2, 8, 0.6, tuple(range(0, 512, 3)))])
def test_beam_search_against_plain_steps(which, beams, most, penalty, eos, tmp_path_factory):
    import hk_b200
    d, cfg, w = model(tmp_path_factory, which, torch.float32)
    prompts = helpers.prompts_for(which, np.random.default_rng(4), [3, 17, 9])
    eng = hk_b200.Engine(d, dtype="float32", max_tokens=1024, page_tokens=4, max_requests=2 * beams, max_context=100)
    got = hk_b200.beam_search_with_engine(eng, prompts, beams, most, penalty, eos_token_ids=eos)
    assert eng.free_pages() == [g.pool.num_pages for g in eng.cache.books.groups]
    for p, mine in zip(prompts, got):
        want = plain_beams(cfg, w, p, beams, most, penalty, set(eos))
        assert [c.tokens for c in mine] == [t for t, _, _ in want]
        assert [c.ended for c in mine] == [e for _, _, e in want]
        # float32 logits off by at most TOL of the largest (a few units), summed over the tokens
        assert all(abs(c.score - s) <= 1e-4 * most for c, (_, s, _) in zip(mine, want))


def test_beam_search_entry_points(tmp_path):
    import hk_b200
    from hk_b200.engine import EngineError
    d = helpers.make_model_dir(tmp_path, "A", torch.bfloat16)
    out = hk_b200.beam_search(d, [[1, 2, 3], [4, 5]], num_beams=3, max_new_tokens=5)
    assert len(out) == 2 and all(len(o) == 3 and all(len(c.tokens) == 5 for c in o) for o in out)
    assert all(o[0].score >= o[1].score >= o[2].score for o in out)
    eng = hk_b200.Engine(d, max_tokens=256, page_tokens=16, max_requests=4, max_context=64)
    for bad in (dict(num_beams=0), dict(num_beams=5), dict(max_new_tokens=0)):
        with pytest.raises(ValueError):
            hk_b200.beam_search_with_engine(eng, [[1]], **bad)
    with pytest.raises(EngineError):
        hk_b200.beam_search_with_engine(eng, [[1] * 60], num_beams=2, max_new_tokens=10)
    run = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "hk"), "run", d, "1,2,3", "-n", "5", "--beams", "3"], capture_output=True, text=True)
    assert run.returncode == 0 and [int(t) for t in run.stdout.split()] == out[0][0].tokens, run.stderr


def test_recurrent_beams(tmp_path):
    """Beams of a model with states: the best of one beam is the greedy continuation, and more beams find one at least as probable."""
    import hk_b200
    import kedanex_models
    d = kedanex_models.make_model_dir(tmp_path, "X", torch.float32)
    eng = hk_b200.Engine(d, dtype="float32", max_tokens=512, page_tokens=4, max_requests=4, max_context=80)
    prompts = kedanex_models.prompts("X", np.random.default_rng(2), [6, 11])
    greedy = hk_b200.generate_with_engine(eng, prompts, 6, temperature=0, eos_token_ids=())
    one = hk_b200.beam_search_with_engine(eng, prompts, 1, 6, 0.0, eos_token_ids=())
    assert [o[0].tokens for o in one] == greedy
    four = hk_b200.beam_search_with_engine(eng, prompts, 4, 6, 0.0, eos_token_ids=())
    for o, f in zip(one, four):
        assert len(f) == 4 and len({tuple(c.tokens) for c in f}) == 4 and f[0].score >= f[1].score


# ---- drafted generation --------------------------------------------------------------------------------------------------------


def repetitive(rng, vocab, n):
    piece = rng.integers(0, vocab, 9).tolist()
    return (piece * (n // 9 + 1))[:n]


@pytest.mark.parametrize("sampling", [dict(temperature=0), dict(temperature=0.7, top_k=20, seed=5), dict(temperature=1.0, top_p=0.8, min_p=0.05, seed=9)])
@pytest.mark.parametrize("which,page", [("A", 4), ("B", 16), ("C", 8)])
def test_drafted_generation_is_plain_generation(which, page, sampling, tmp_path_factory):
    import hk_b200
    from hk_b200.api import GenerationStats
    d, cfg, w = model(tmp_path_factory, which, torch.float32)
    rng = np.random.default_rng(6)
    vocab = cfg["vocab_size"]
    prompts = [repetitive(rng, vocab, n) for n in (20, 45, 7, 33, 61)] + [[3]]
    eng = hk_b200.Engine(d, dtype="float32", max_tokens=400, page_tokens=page, max_requests=3, max_context=110, max_batch_tokens=60)
    want = hk_b200.generate_with_engine(eng, prompts, 40, eos_token_ids=(), **sampling)
    for draft in (1, 7, 24):
        st = GenerationStats()
        got = hk_b200.generate_with_engine(eng, prompts, 40, eos_token_ids=(), draft_tokens=draft, stats=st, **sampling)
        assert got == want
        assert st.decode_tokens == sum(len(o) - 1 for o in got) and eng.free_pages() == [g.pool.num_pages for g in eng.cache.books.groups]
    eos = sorted({o[len(o) // 2] for o in want})
    want = hk_b200.generate_with_engine(eng, prompts, 40, eos_token_ids=eos, **sampling)
    assert hk_b200.generate_with_engine(eng, prompts, 40, eos_token_ids=eos, draft_tokens=9, **sampling) == want


def test_drafts_save_steps_where_the_text_repeats_itself(tmp_path_factory):
    import hk_b200
    from hk_b200.api import GenerationStats
    d, cfg, w = model(tmp_path_factory, "A", torch.float32)
    eng = hk_b200.Engine(d, dtype="float32", max_tokens=256, page_tokens=16, max_requests=1, max_context=128)
    # greedy text of a tiny random model falls into a cycle, which the guesses then follow
    st = GenerationStats()
    out = hk_b200.generate_with_engine(eng, [[1, 2, 3]], 100, temperature=0, eos_token_ids=(), draft_tokens=8, stats=st)
    assert len(out[0]) == 100 and st.decode_steps < 99


def test_drafted_generation_in_tight_pools_and_its_refusals(tmp_path_factory):
    import hk_b200
    from hk_b200.engine import EngineError
    d, cfg, w = model(tmp_path_factory, "A", torch.float32)
    rng = np.random.default_rng(7)
    prompts = [repetitive(rng, 256, n) for n in (18, 30)]
    wide = hk_b200.Engine(d, dtype="float32", max_tokens=512, page_tokens=4, max_requests=2, max_context=60)
    want = hk_b200.generate_with_engine(wide, prompts, 40, temperature=0, eos_token_ids=())          # ends at the context
    assert hk_b200.generate_with_engine(wide, prompts, 40, temperature=0, eos_token_ids=(), draft_tokens=16) == want
    tight = hk_b200.Engine(d, dtype="float32", max_tokens=64, page_tokens=4, max_requests=2, max_context=60)
    assert hk_b200.generate_with_engine(tight, prompts, 20, temperature=0, eos_token_ids=(), draft_tokens=30) == [o[:20] for o in want]
    for bad in (dict(draft_tokens=256), dict(draft_tokens=4, repeat_penalty=1.1)):
        with pytest.raises(ValueError):
            hk_b200.generate_with_engine(wide, prompts, 4, temperature=0, **bad)
    with pytest.raises(EngineError):
        hk_b200.generate_with_engine(wide, [[1] * 61], 4, temperature=0, draft_tokens=4)
    assert wide.free_pages() == [128]
    run = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "hk"), "run", d, ",".join(map(str, prompts[0])), "-n", "12", "--temp", "0", "--draft", "6",
                          "--dtype", "float32"], capture_output=True, text=True)
    assert run.returncode == 0 and [int(t) for t in run.stdout.split()] == want[0][:12], run.stderr
