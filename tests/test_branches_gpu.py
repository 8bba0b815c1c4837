"""Copied blocks, kept rows and the choice over beams and vocabulary against plain forms."""
import numpy as np
import pytest
import torch

from ref_branches import beam_reference

pytestmark = pytest.mark.gpu


# ---- blocks ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("pieces,rows,row_bytes,dtype", [(8, 64, 256, torch.bfloat16), (2, 16, 128, torch.float32), (1, 1, 1 << 20, torch.float32),
                                                         (3, 5, 20, torch.float32), (1, 1, 262148, torch.float32), (2, 7, 6, torch.bfloat16),
                                                         (1, 1, 36, torch.float32), (4, 16, 100, torch.bfloat16)])
def test_copied_blocks(pieces, rows, row_bytes, dtype):
    from hk_b200.csrc import ops
    rng = np.random.default_rng(1)
    arrays = [torch.randn(9 + a, pieces, rows, row_bytes // dtype.itemsize).to(dtype).cuda() for a in range(5)]
    before = [a.clone() for a in arrays]
    table = torch.tensor([[a.data_ptr(), a.shape[0], pieces, rows * row_bytes, row_bytes] for a in arrays], dtype=torch.int64).cuda()
    moves = [(0, 3, rows), (0, 5, max(1, rows // 2)), (2, 8, 1), (1, 4, 10 ** 6), (2, 6, 0), (7, 7, rows), (-1, 1, rows), (1, -1, rows), (40, 2, rows),
             (11, 7, rows)]       # the last lies inside two of the arrays only
    order = rng.permutation(len(moves))
    ops.copy_blocks(table, torch.tensor([moves[i] for i in order], dtype=torch.int32).cuda(), pieces * rows * row_bytes)
    for a, b in zip(arrays, before):
        want = b.clone()
        for s, d, r in moves:
            if 0 <= s < b.shape[0] and 0 <= d < b.shape[0] and s != d and r > 0:
                want[d, :, :r] = b[s, :, :r]
        assert torch.equal(a, want)


def test_no_moves_and_refusals():
    from hk_b200.csrc import ops
    a = torch.randn(4, 8, device="cuda")
    table = torch.tensor([[a.data_ptr(), 4, 1, 32, 32]], dtype=torch.int64).cuda()
    before = a.clone()
    ops.copy_blocks(table, torch.zeros((0, 3), dtype=torch.int32, device="cuda"), 32)
    assert torch.equal(a, before)
    moves = torch.zeros((1, 3), dtype=torch.int32, device="cuda")
    for bad in ((table[:, :4], moves, 32), (table, moves[:, :2], 32), (table, moves, 0), (table.int(), moves, 32), (table, moves.cpu(), 32)):
        with pytest.raises(ops.KernelError):
            ops.copy_blocks(*bad)


# ---- kept rows -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("G,hd,page,dtype", [(8, 128, 64, torch.bfloat16), (2, 64, 16, torch.float32), (3, 5, 4, torch.float32), (1, 3, 7, torch.bfloat16),
                                             (2, 16, 1, torch.bfloat16)])
def test_kept_rows(G, hd, page, dtype):
    from hk_b200.csrc import ops
    rng = np.random.default_rng(2)
    R, n, stride = 6, 300, -(-400 // page)
    pages = R * stride + 3
    caches = [torch.randn(pages, G, page, hd).to(dtype).cuda() for _ in range(4)]
    before = [c.clone() for c in caches]
    order = rng.permutation(pages)[:R * stride].reshape(R, stride).astype(np.int32)
    bt = torch.from_numpy(order).cuda()
    table = torch.tensor([[c.data_ptr(), G, hd * dtype.itemsize, bt.data_ptr()] for c in caches], dtype=torch.int64).cuda()
    kept = [[0], list(range(12)), [0, 1, 2, 5, 9, 30], sorted(rng.choice(n, 290, replace=False).tolist()), [], [1, 2, 3, 4, 299]]
    firsts = [0, 3, 61, 99, 5, 64]
    paths = np.full((R, 2 + 290), -1, dtype=np.int32)
    slots = [4, 0, 2, 1, 3, 5]
    for i in range(R):
        paths[i, :2] = slots[i], firsts[i]
        paths[i, 2:2 + len(kept[i])] = kept[i]
    ops.compact_rows(table, torch.from_numpy(paths).cuda(), R, stride, page, G, hd * dtype.itemsize, pages)
    for c, b in zip(caches, before):
        want = b.clone()
        for i in range(R):
            for to, row in enumerate(kept[i]):
                s, d = firsts[i] + row, firsts[i] + to
                want[order[slots[i], d // page], :, d % page] = b[order[slots[i], s // page], :, s % page]
        assert torch.equal(c, want)


def test_rows_outside_the_table_stay():
    from hk_b200.csrc import ops
    c = torch.randn(4, 1, 4, 8, device="cuda")
    before = c.clone()
    bt = torch.tensor([[0, 1], [2, -1], [9, 3]], dtype=torch.int32, device="cuda")
    table = torch.tensor([[c.data_ptr(), 1, 32, bt.data_ptr()]], dtype=torch.int64).cuda()
    paths = torch.tensor([[0, 3, 1, 7], [1, 2, 0, 3], [2, 0, 2, 5], [5, 0, 2, 3], [-1, 0, 2, 3], [0, -2, 2, 3]], dtype=torch.int32, device="cuda")
    ops.compact_rows(table, paths, 3, 2, 4, 1, 32, 4)
    want = before.clone()
    want[0, :, 3] = before[1, :, 0]            # row 4 of slot 0 to row 3; row 10 is none
    assert torch.equal(c, want)
    for bad in ((table[:, :3], paths), (table, paths[:, :1]), (table.int(), paths), (table, paths.long())):
        with pytest.raises(ops.KernelError):
            ops.compact_rows(*bad, 3, 2, 4, 1, 32, 4)
    with pytest.raises(ops.KernelError):
        ops.compact_rows(table, paths, 3, 0, 4, 1, 32, 4)


# ---- beams ----------------------------------------------------------------------------------------------------------------


def run_beams(ops, logits, scores, beams, choices):
    prompts = logits.shape[0] // beams
    out = torch.empty((prompts, choices), dtype=torch.float32, device="cuda")
    k, v = (torch.empty((prompts, choices), dtype=torch.int32, device="cuda") for _ in range(2))
    ops.beam_select(logits, scores, beams, out, k, v)
    return out.cpu().numpy(), k.cpu().numpy(), v.cpu().numpy()


def check_beams(ops, logits, scores, beams, choices):
    got = run_beams(ops, torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), beams, choices)
    want = beam_reference(logits, scores, beams, choices)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    finite = np.isfinite(want[0])
    assert np.array_equal(np.isneginf(got[0]), ~finite)
    # one rounding to float32 (2^-24 of the value) and the sum's exponentials (2 units in the last place of each, 2^-22 of the sum)
    assert (np.abs(got[0][finite] - want[0][finite]) <= 2.0 ** -24 * np.abs(want[0][finite]) + 2.0 ** -22).all()


@pytest.mark.parametrize("prompts,beams,choices,V", [(1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 6, 7), (1, 4, 8, 151936), (3, 5, 10, 32003), (16, 8, 16, 20000), (1, 16, 32, 1000),
                                                    (2, 2, 256, 4097), (1, 256, 256, 64), (5, 1, 2, 8193), (40, 8, 16, 151936), (1, 7, 100, 2048)])
def test_beams(prompts, beams, choices, V):
    from hk_b200.csrc import ops
    rng = np.random.default_rng(prompts * 1000 + beams)
    logits = (rng.standard_normal((prompts * beams, V)) * 3).astype(np.float32)
    check_beams(ops, logits, -(rng.random(prompts * beams) * 6).astype(np.float32), beams, choices)


@pytest.mark.parametrize("V", [1000, 9000, 70001])
def test_equal_logits_and_equal_beams(V):
    """Ties inside a beam, between beams, and all logits equal: the lowest beam and token first."""
    from hk_b200.csrc import ops
    rng = np.random.default_rng(4)
    coarse = np.round(rng.standard_normal((8, V)) * 2).astype(np.float32)
    check_beams(ops, coarse, np.zeros(8, dtype=np.float32), 4, 32)
    same = np.repeat(coarse[:1], 8, axis=0)
    check_beams(ops, same, np.full(8, -1.5, dtype=np.float32), 4, 16)
    check_beams(ops, np.zeros((8, V), dtype=np.float32), np.zeros(8, dtype=np.float32), 8, 64)


def test_climbing_logits():
    """Every tile's values above all before: the list of candidates is made anew again and again."""
    from hk_b200.csrc import ops
    rng = np.random.default_rng(8)
    up = np.sort(rng.standard_normal((12, 151936)).astype(np.float32), axis=1)
    for logits in (up, up[:, ::-1].copy()):
        check_beams(ops, logits, -(rng.random(12) * 0.1).astype(np.float32), 4, 8)
        check_beams(ops, np.repeat(logits, 60, axis=0)[:700], -(rng.random(700) * 0.1).astype(np.float32), 7, 100)


@pytest.mark.parametrize("leading", [1, 7, 40, 128])
def test_many_beams_and_choices(leading):
    """More parts' tokens than the threads of the choice hold: the best lie in a few beams, or in all."""
    from hk_b200.csrc import ops
    rng = np.random.default_rng(leading)
    logits = (rng.standard_normal((128, 40000)) * 3).astype(np.float32)
    scores = -(rng.random(128) * 2).astype(np.float32)
    scores[leading:] -= 40.0
    order = rng.permutation(128)
    check_beams(ops, logits[order], scores[order], 128, 256)


@pytest.mark.parametrize("V,allowed,choices", [(40000, 500, 16), (40000, 300, 256), (3000, 3000, 200), (5000, 4000, 256), (1500, 40, 100)])
def test_rows_that_allow_few_tokens(V, allowed, choices):
    """Most tokens masked, by -inf or NaN: groups of threads that hold nothing, and bars that are found late."""
    from hk_b200.csrc import ops
    rng = np.random.default_rng(V + choices)
    logits = (rng.standard_normal((6, V)) * 3).astype(np.float32)
    for row in logits:
        row[rng.permutation(V)[allowed:]] = -np.inf
        row[rng.random(V) < 0.02] = np.nan
    logits[1, rng.random(V) < 0.01] = np.inf
    check_beams(ops, logits, -(rng.random(6) * 3).astype(np.float32), 2, choices)
    check_beams(ops, np.repeat(logits, 120, axis=0)[:700], -(rng.random(700) * 3).astype(np.float32), 7, choices)


def test_beams_that_are_not_there_and_masked_logits():
    from hk_b200.csrc import ops
    rng = np.random.default_rng(5)
    logits = (rng.standard_normal((12, 5000)) * 3).astype(np.float32)
    scores = -(rng.random(12) * 3).astype(np.float32)
    first = scores.copy().reshape(3, 4)
    first[:, 1:] = -np.inf                                   # the first step: one beam a prompt
    check_beams(ops, logits, first.reshape(-1), 4, 8)
    masked = logits.copy()
    masked[:, :4990] = -np.inf                               # fewer tokens left than choices
    masked[3, 4995:] = np.nan
    masked[7, 4991] = np.inf
    masked[5] = -np.inf
    masked[8:] = -np.inf                                     # and none at all
    check_beams(ops, masked, scores, 4, 64)
    odd = scores.copy()
    odd[2], odd[6] = np.nan, np.inf
    check_beams(ops, logits, odd, 4, 8)
    lowest = np.where(rng.random((4, 3000)) < 0.999, np.float32(-3.4028234663852886e38), logits[:4, :3000]).astype(np.float32)
    check_beams(ops, lowest, scores[:4], 2, 8)


def test_large_and_small_logits():
    from hk_b200.csrc import ops
    rng = np.random.default_rng(6)
    logits = (rng.standard_normal((6, 3001)) * 3).astype(np.float32)
    check_beams(ops, logits * 1e4, np.zeros(6, dtype=np.float32), 3, 6)
    check_beams(ops, logits + 3e4, np.zeros(6, dtype=np.float32), 3, 6)
    check_beams(ops, logits * 1e-6, np.zeros(6, dtype=np.float32), 3, 6)
    check_beams(ops, logits, np.full(6, -1e6, dtype=np.float32) - np.arange(6, dtype=np.float32), 3, 6)


def test_beams_replayed_and_on_two_streams():
    """Two captured calls and one on another stream, side by side: none disturbs another's scratch."""
    from hk_b200.csrc import ops
    rng = np.random.default_rng(7)
    a, b = ((rng.standard_normal((16, 50000)) * 3).astype(np.float32) for _ in range(2))
    scores = -(rng.random(16) * 3).astype(np.float32)
    wants = [beam_reference(x, scores, 8, 16) for x in (a, b)]
    inputs = [torch.from_numpy(x).cuda() for x in (a, b)]
    s = torch.from_numpy(scores).cuda()
    outs, graphs = [], []
    run_beams(ops, inputs[0], s, 8, 16)
    for x in inputs:
        out = (torch.empty((2, 16), device="cuda"), torch.empty((2, 16), dtype=torch.int32, device="cuda"), torch.empty((2, 16), dtype=torch.int32, device="cuda"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.beam_select(x, s, 8, *out)
        outs.append(out)
        graphs.append(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        assert np.array_equal(out[1].cpu().numpy(), want[1]) and np.array_equal(out[2].cpu().numpy(), want[2])


def test_beams_of_many_calls_in_flight():
    """Calls that wait one behind the other for the GPU, on other inputs by turns: each starts beside the one before, on the same scratch."""
    from hk_b200.csrc import ops
    rng = np.random.default_rng(9)
    work = torch.randn(4096, 4096, device="cuda", dtype=torch.bfloat16)
    for beams, choices, V, rows in ((3, 6, 5936, 51), (8, 16, 30001, 64)):
        inputs = [((rng.standard_normal((rows, V)) * 3).astype(np.float32), -(rng.random(rows) * 3).astype(np.float32)) for _ in range(3)]
        wants = [beam_reference(x, s, beams, choices) for x, s in inputs]
        inputs = [(torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda()) for x, s in inputs]
        outs = [(torch.empty((rows // beams, choices), device="cuda"), *(torch.empty((rows // beams, choices), dtype=torch.int32, device="cuda") for _ in range(2)))
                for _ in range(60)]
        for _ in range(20):
            work @ work
        for i, out in enumerate(outs):
            ops.beam_select(*inputs[i % 3], beams, *out)
        torch.cuda.synchronize()
        for i, (score, beam, token) in enumerate(outs):
            want = wants[i % 3]
            assert np.array_equal(beam.cpu().numpy(), want[1]) and np.array_equal(token.cpu().numpy(), want[2])
            # (as in check_beams)
            assert (np.abs(score.cpu().numpy() - want[0]) <= 2.0 ** -24 * np.abs(want[0]) + 2.0 ** -22).all()


def test_beam_refusals():
    from hk_b200.csrc import ops
    logits, scores = torch.randn(6, 50, device="cuda"), torch.zeros(6, device="cuda")

    def call(logits=logits, scores=scores, beams=3, prompts=2, choices=6, kind=torch.int32, tokens=None):
        ops.beam_select(logits, scores, beams, torch.empty(prompts, choices, device="cuda"), torch.empty(prompts, choices, dtype=kind, device="cuda"),
                        torch.empty(prompts, tokens or choices, dtype=torch.int32, device="cuda"))

    call()
    for bad in (dict(logits=logits.cpu()), dict(logits=logits.half()), dict(logits=logits.t().contiguous().t()), dict(scores=scores[:5]), dict(beams=2), dict(beams=0),
                dict(choices=151), dict(choices=0), dict(kind=torch.int64), dict(tokens=5), dict(prompts=3), dict(choices=257, logits=torch.randn(6, 500, device="cuda"))):
        with pytest.raises(ops.KernelError):
            call(**bad)
