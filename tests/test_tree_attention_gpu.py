"""Attention of drafted token trees over the paged cache against a plain form in 64 bits."""
import numpy as np
import pytest
import torch

from ref_branches import TreeCase

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    if torch.cuda.is_available():
        from hk_b200.csrc import gemm_fast
        gemm_fast.check_status(torch.device("cuda", 0))


SHAPES = [
    # contexts, drafted tokens, heads, key heads, dim, page
    ([0], [1], 4, 2, 64, 16),
    ([1], [1], 32, 8, 128, 64),
    ([37], [5], 4, 4, 128, 16),
    ([0, 3, 200], [7, 0, 33], 8, 2, 64, 16),
    ([127, 128, 129], [1, 16, 31], 8, 8, 128, 64),
    ([1000, 20], [32, 32], 16, 2, 128, 16),
    ([255, 700], [64, 65], 8, 2, 128, 64),
    ([300], [256], 4, 1, 64, 128),
    ([513, 5, 90], [130, 1, 40], 10, 2, 128, 256),
    ([2100], [3], 5, 1, 128, 8),
    ([30000], [16], 8, 2, 128, 16),
    ([9000, 70, 12000], [64, 100, 17], 32, 8, 128, 16),
    ([15000], [64], 8, 2, 64, 64),
    ([40], [20], 6, 2, 80, 16),
    ([33, 65], [9, 18], 4, 2, 16, 5),
    ([61], [10], 2, 1, 256, 16),
    ([90], [12], 3, 1, 100, 7),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}+{s[1]}x{s[2]}/{s[3]}x{s[4]}p{s[5]}".replace(" ", ""))
def test_shapes(shape, dtype):
    from hk_b200.csrc import ops
    TreeCase(11, *shape, dtype=dtype).check(ops)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", ["tree", "chain", "full", "random", "none"])
def test_masks(mask, dtype):
    from hk_b200.csrc import ops
    TreeCase(5, [0, 150, 31], [40, 33, 1], 8, 2, 128, 16, dtype=dtype, mask=mask).check(ops)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128, 48])
@pytest.mark.parametrize("window,cap,sink", [(50, 0.0, 0), (3, 0.0, 2), (1, 30.0, 0), (0, 5.0, 1), (400, 20.0, 2), (128, 0.0, 0)])
def test_options(window, cap, sink, hd, dtype):
    from hk_b200.csrc import ops
    TreeCase(6, [300, 0, 129, 1000], [21, 40, 64, 9], 8, 2, hd, 16, window=window, cap=cap, sink=sink, dtype=dtype).check(ops)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sink", [0, 1])
def test_rows_that_see_nothing(sink, dtype):
    from hk_b200.csrc import ops
    case = TreeCase(7, [0, 0], [12, 70], 8, 2, 128, 16, dtype=dtype, mask="none", sink=sink)
    out = case.check(ops)
    for first, count in case.requests[:, 1:3].tolist():
        assert (out[first:first + count] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_that_are_not_seen_do_not_matter(bad, hd, dtype):
    """NaN and Inf in the keys and values of drafted tokens that no row sees, of rows outside the window and behind the last."""
    from hk_b200.csrc import ops
    case = TreeCase(8, [140, 0, 517], [30, 11, 70], 8, 2, hd, 16, window=100, dtype=dtype)
    hidden = {0: [3, 17, 29], 1: [4], 2: [0, 69]}
    for i, rows in hidden.items():
        for t in rows:
            case.see[i][:, t] = False
            case.ancestors[case.requests[i, 1]:case.requests[i, 1] + case.counts[i], t // 32] &= ~np.int32(np.uint32(1 << (t % 32)).view(np.int32))
    want, _, _ = case.reference()
    for i, rows in hidden.items():
        for row in [case.contexts[i] + t for t in rows] + list(range(max(0, case.contexts[i] - 99 - 20), max(0, case.contexts[i] - 99))):
            page, at = case.place(i, row)
            case.k[page, :, at] = bad
            case.v[page, :, at] = bad
        end = case.contexts[i] + case.counts[i]
        if end % case.page:
            page, at = case.place(i, end - 1)
            case.k[page, :, at + 1:] = bad
            case.v[page, :, at + 1:] = bad
    case.check(ops)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 128])
def test_seen_by_some_rows_only(hd, dtype):
    """A value of NaN reaches the rows that see it and no other."""
    from hk_b200.csrc import ops
    case = TreeCase(9, [100, 290], [24, 48], 8, 2, hd, 16, dtype=dtype)
    clean = case.run(ops).cpu()
    page, at = case.place(1, 290 + 7)
    case.v[page, :, at, 3] = float("nan")
    out = case.run(ops).cpu()
    first = case.requests[1, 1]
    sees = torch.zeros(case.n, dtype=torch.bool)
    sees[first:first + 48] = torch.from_numpy(case.see[1][:, 7])
    dims = torch.zeros(case.H * hd, dtype=torch.bool)
    dims[3::hd] = True
    assert out[sees][:, dims].isnan().all()
    assert torch.isfinite(out[sees][:, ~dims].float()).all()
    # a row that went through the exact path holds probabilities that were not rounded to bfloat16: within the rounding of both
    a, b = out[~sees].float(), clean[~sees].float()
    assert ((a - b).abs() <= 2.0 ** -6 * (b.abs() + 1.0)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_same_bits_twice_and_on_another_stream(dtype):
    from hk_b200.csrc import ops
    case = TreeCase(10, [900, 31, 4000], [33, 64, 17], 16, 4, 128, 16, dtype=dtype)
    first = case.run(ops)
    assert torch.equal(first, case.run(ops))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = case.run(ops)
    side.synchronize()
    assert torch.equal(first, again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_replayed_over_other_contexts(dtype):
    """A captured launch reads who has how many rows from the device: other lengths, the same graph."""
    from hk_b200.csrc import ops
    a = TreeCase(12, [500, 90], [16, 16], 8, 2, 128, 16, dtype=dtype)
    b = TreeCase(12, [333, 400], [16, 5], 8, 2, 128, 16, dtype=dtype, gap=1)
    pages, stride = max(a.num_pages, b.num_pages), 40
    k = torch.zeros(pages, 2, 16, 128, dtype=dtype, device="cuda")
    v, q = torch.zeros_like(k), torch.zeros(a.n, 8 * 128, dtype=dtype, device="cuda")
    table = torch.full((3, stride), -1, dtype=torch.int32, device="cuda")
    requests = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    ancestors, positions = torch.zeros(a.n, 1, dtype=torch.int32, device="cuda"), torch.zeros(a.n, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)

    def load(c):
        k[:c.num_pages].copy_(c.k)
        v[:c.num_pages].copy_(c.v)
        q[:c.n].copy_(c.q)
        table[:, :c.table.shape[1]].copy_(torch.from_numpy(c.table))
        requests.copy_(torch.from_numpy(c.requests))
        ancestors[:c.n].copy_(torch.from_numpy(c.ancestors))
        positions[:c.n].copy_(torch.from_numpy(c.positions))

    def call():
        ops.tree_attention(q, k, v, table, requests, ancestors, positions, out, 8, 2, 128, 16, 0, a.scale, 16, stride * 16)

    load(a)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for case in (a, b, a):
        load(case)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        want, weight, most = case.reference()
        tol = case.tolerance(weight, most)
        for first, count in case.requests[:, 1:3].tolist():
            rows = slice(first, first + count)
            assert (np.abs(out[rows].double().cpu().numpy() - want[rows]) <= tol[rows]).all()


def test_many_requests_and_bad_ones():
    """More requests than a warp has lanes, some without tokens; requests whose numbers lie outside the arrays are left out."""
    from hk_b200.csrc import ops
    rng = np.random.default_rng(3)
    case = TreeCase(13, [int(x) for x in rng.integers(0, 300, 70)], [int(x) for x in rng.integers(0, 9, 70)], 4, 2, 64, 16)
    clean = case.check(ops)
    bad = case.requests.copy()
    bad[3, 0], bad[5, 0], bad[9, 1], bad[11, 3], bad[12, 1] = -1, 71, case.n, 40 * 16, -2
    lost = [i for i in (3, 5, 9, 11, 12) if case.counts[i]]
    good, case.requests = case.requests, bad
    out = case.run(ops).cpu()
    skip = torch.zeros(case.n, dtype=torch.bool)
    for i in lost:
        skip[good[i, 1]:good[i, 1] + good[i, 2]] = True
    assert torch.equal(out[~skip], clean[~skip])
    assert (out[skip] == 7.0).all()


def test_offsets_past_32_bits():
    """Pages whose first element lies more than 2^32 bytes, and more than 2^31 elements, behind the pool's start."""
    from hk_b200.csrc import ops
    G, page, hd = 8, 64, 128
    num_pages = (1 << 31) // (G * page * hd) + 40
    case = TreeCase(14, [700], [20], 8, 8, hd, page)
    want, weight, most = case.reference()
    k = torch.empty((num_pages, G, page, hd), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    shift = num_pages - case.num_pages
    k[shift:].copy_(case.k)
    v[shift:].copy_(case.v)
    table = torch.from_numpy(np.where(case.table >= 0, case.table + shift, -1)).to("cuda").int()
    up = lambda a: torch.from_numpy(a).to("cuda")  # noqa: E731
    out = torch.empty((case.n, 8 * hd), dtype=torch.bfloat16, device="cuda")
    ops.tree_attention(case.q.cuda(), k, v, table, up(case.requests), up(case.ancestors), up(case.positions), out, 8, 8, hd, page, 0, case.scale, 20, 720)
    rows = slice(case.requests[0, 1], case.requests[0, 1] + 20)
    off = np.abs(out[rows].double().cpu().numpy() - want[rows])
    assert (off <= case.tolerance(weight, most)[rows]).all()


def test_refusals():
    from hk_b200.csrc import ops
    case = TreeCase(15, [20], [4], 4, 2, 64, 16)
    dev = "cuda"
    good = dict(q=case.q.to(dev), k=case.k.to(dev), v=case.v.to(dev), table=torch.from_numpy(case.table).to(dev),
                requests=torch.from_numpy(case.requests).to(dev), ancestors=torch.from_numpy(case.ancestors).to(dev),
                positions=torch.from_numpy(case.positions).to(dev), H=4, G=2, hd=64, page=16, window=0, scale=0.125, tokens=4, keys=24,
                cap=0.0, sink=False, sinks=None)

    def call(**change):
        a = dict(good, **change)
        out = a.get("out", torch.empty_like(a["q"]) if a["q"].is_cuda else torch.empty_like(good["q"]))
        ops.tree_attention(a["q"], a["k"], a["v"], a["table"], a["requests"], a["ancestors"], a["positions"], out, a["H"], a["G"], a["hd"], a["page"],
                           a["window"], a["scale"], a["tokens"], a["keys"], sink=a["sink"], sinks=a["sinks"], softcap=a["cap"])

    call()
    for change in (dict(q=case.q), dict(q=good["q"].float()), dict(H=3), dict(G=3), dict(hd=32), dict(page=8), dict(requests=good["requests"][:, :3]),
                   dict(requests=good["requests"].long()), dict(ancestors=good["ancestors"][:-1]), dict(positions=good["positions"][1:]),
                   dict(tokens=0), dict(tokens=33), dict(tokens=300), dict(keys=0), dict(keys=10 ** 6), dict(scale=0.0), dict(scale=float("nan")),
                   dict(cap=-1.0), dict(sinks=torch.zeros(4, device=dev)), dict(sink=True, sinks=torch.zeros(3, device=dev)),
                   dict(v=good["v"][:-1]), dict(table=good["table"].t()), dict(out=torch.empty(1, 256, dtype=torch.bfloat16, device=dev))):
        with pytest.raises(ops.KernelError):
            call(**change)
    torch.cuda.synchronize()


@pytest.mark.parametrize("lost", ["scores", "values"])
def test_all_rows_taken_again_behind_long_contexts(lost):
    """Every row of every request is lost to the tensor core: its scores jump by 2^100 in a late tile, or a value of NaN lies in a drafted
    row that none sees.  Taking them again lasts far longer than a wait may, and nothing gives up (the fixture looks)."""
    from hk_b200.csrc import ops
    m, count, context, G, hd, page = 20, 100, 4000, 8, 128, 16
    H, g = 2 * G, torch.Generator(device="cuda").manual_seed(3)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda") * 0.3
    pages = (context + count + page - 1) // page
    q, k, v = normal(m * count, H * hd), normal(m * pages, G, page, hd), normal(m * pages, G, page, hd)
    if lost == "scores":
        q.view(-1, H, hd)[:, :, 0] = 10.0
        k[:, :, :, 0] = 0.0
        k.view(m, pages, G, page, hd)[:, 150, :, :, 0] = 80.0
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    plain_v = v.clone()
    at = context + count - 1                                                     # the last drafted token, which no row sees, nor its own
    v.view(m, pages, G, page, hd)[:, at // page, :, at % page] = float("nan")
    if lost == "scores":
        v.copy_(plain_v)
    table = torch.arange(m * pages, dtype=torch.int32, device="cuda").view(m, pages)
    requests = torch.tensor([[i, i * count, count, context] for i in range(m)], dtype=torch.int32, device="cuda")
    bits = np.zeros((m * count, -(-count // 32)), dtype=np.uint32)
    for i in range(count - 1):
        bits[i::count, i // 32] = 1 << (i % 32)
    ancestors = torch.from_numpy(bits.view(np.int32)).cuda()
    positions = torch.arange(context, context + count, dtype=torch.int32, device="cuda").repeat(m)
    out = torch.empty_like(q)
    ops.tree_attention(q, k, v, table, requests, ancestors, positions, out, H, G, hd, page, 0, hd ** -0.5, count, context + count)
    torch.cuda.synchronize()
    for i in (0, 7, m - 1):
        rows = slice(i * count, (i + 1) * count)
        x = q[rows].double().view(count, G, 2, hd)
        kk, vv = (t.view(m, pages, G, page, hd)[i].transpose(0, 1).reshape(G, pages * page, hd)[:, :context + count].double() for t in (k, plain_v))
        scores = torch.einsum("tghd,gjd->tghj", x, kk) * hd ** -0.5
        see = torch.zeros(count, context + count, dtype=torch.bool, device="cuda")
        see[:, :context] = True
        own = torch.arange(count - 1, device="cuda")
        see[own, context + own] = True
        p = torch.softmax(scores.masked_fill(~see[:, None, None], float("-inf")), dim=-1)
        want = torch.einsum("tghj,gjd->tghd", p, vv).reshape(count, H * hd)
        weight = torch.einsum("tghj,gjd->tghd", p, vv.abs()).reshape(count, H * hd)
        # one rounding of the result (2^-8 of it); probabilities rounded where the tensor core did a part of the keys (2^-8 of each); scores
        # of up to 800 before the scale, summed 128 times in 32 bits (128 * 800 * 2^-24 / sqrt(128) = 5.4e-4, above and below: 2^-9)
        error = (out[rows].double() - want).abs()
        assert (error <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * weight).all()
