"""Tree attention over block tables with pages that are not there: such a key is not seen, whichever kernel runs."""
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


def holed(case, holes):
    """Takes pages of the block table away; the 64-bit form of what is left (see `TreeCase.reference`)."""
    G, hd, H, page = case.G, case.hd, case.H, case.page
    for i, logical, value in holes:
        case.table[case.requests[i, 0], logical] = value
    out, weight, most = np.full((case.n, H, hd), np.nan), np.zeros((case.n, H, hd)), 0.0
    for i, (slot, first, count, context) in enumerate(case.requests.tolist()):
        end = context + count
        pages = case.table[slot, np.arange(end) // page]
        there = (pages >= 0) & (pages < case.num_pages)
        at = np.where(there, pages, 0), np.arange(end) % page
        K, V = (t.double().numpy()[at[0], :, at[1]] for t in (case.k, case.v))          # [end, G, hd]
        see = np.concatenate([np.ones((count, context), dtype=bool), case.see[i]], axis=1) & there[None]
        if case.window:
            mine = case.positions[first:first + count].astype(np.int64)
            see &= np.concatenate([np.arange(context), mine])[None] > mine[:, None] - case.window
        for h in range(H):
            q = case.q[first:first + count, h * hd:(h + 1) * hd].double().numpy()
            for t in range(count):
                idx = np.nonzero(see[t])[0]
                kk, vv = K[idx, h // (H // G)], V[idx, h // (H // G)]
                s = kk @ q[t] * case.scale
                if len(idx):
                    most = max(most, float((np.abs(kk) @ np.abs(q[t])).max() * case.scale))
                if case.cap:
                    s = case.cap * np.tanh(s / case.cap)
                if case.sink:
                    s = np.append(s, float(case.sinks[h]) if case.sinks is not None else 0.0)
                if not len(s):
                    out[first + t, h] = 0.0
                    continue
                p = np.exp(s - s.max())
                p = (p / p.sum())[:len(idx)]
                out[first + t, h], weight[first + t, h] = p @ vv, p @ np.abs(vv)
    return out.reshape(case.n, -1), weight.reshape(case.n, -1), most


def check(case, holes):
    """The pool's first page is no request's and holds finite numbers, then NaN: nothing of it may come through."""
    from hk_b200.csrc import ops
    spare = next(p for p in range(case.num_pages) if not (case.table == p).any())
    case.table[case.table == 0] = spare
    for t in (case.k, case.v):
        t[spare] = t[0]
    want, weight, most = holed(case, holes)
    for first_page in (2.0, float("nan")):
        case.k[0], case.v[0] = first_page, first_page
        out = case.run(ops).cpu()
        for first, count in case.requests[:, 1:3].tolist():
            rows = slice(first, first + count)
            off = np.abs(out[rows].double().numpy() - want[rows])
            assert (off <= case.tolerance(weight, most)[rows]).all(), float(off.max())
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 64), (128, 128), (128, 256), (48, 16), (128, 6)])
@pytest.mark.parametrize("lost", [-1, "pages", 2 ** 31 - 1, -2 ** 31])
def test_pages_that_are_not_there(lost, hd, page, dtype):
    case = TreeCase(21, [700, 40, 1500, 3], [20, 70, 9, 5], 8, 2, hd, page, dtype=dtype)
    value = case.num_pages if lost == "pages" else lost
    need = [-(-(c + t) // page) for c, t in zip(case.contexts, case.counts)]
    holes = [(0, 0, value), (0, need[0] // 2, value), (0, need[0] - 1, value), (2, need[2] // 3, value), (2, need[2] // 2, value)]
    check(case, holes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [128, 48])
@pytest.mark.parametrize("window,cap,sink", [(100, 0.0, 2), (0, 20.0, 1), (30, 10.0, 0)])
def test_with_options(window, cap, sink, hd, dtype):
    case = TreeCase(22, [700, 40, 300], [20, 70, 9], 8, 2, hd, 16, window=window, cap=cap, sink=sink, dtype=dtype)
    check(case, [(0, 700 // 16 - 1, -1), (0, 700 // 16 - 3, case.num_pages), (1, 3, -1), (2, 300 // 16, -1)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [128, 64, 48])
def test_no_page_at_all(hd, dtype):
    """A request none of whose pages are there gives zeros; the others beside it what they give without it."""
    case = TreeCase(23, [260, 90], [12, 33], 8, 2, hd, 16, dtype=dtype)
    out = check(case, [(0, i, -1) for i in range(-(-272 // 16))])
    first, count = case.requests[0, 1:3].tolist()
    assert (out[first:first + count] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_behind_long_contexts(dtype):
    """A request cut among many shares, a page lost in some of them: all its parts belong together."""
    check(TreeCase(24, [9000, 70, 12000], [64, 100, 17], 16, 4, 128, 16, dtype=dtype), [(0, 200, -1), (0, 561, -1), (2, 3, 10 ** 6), (2, 751, -1)])
