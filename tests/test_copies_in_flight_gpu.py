"""Copies and kept rows one behind the other without a wait of the host: each reads what the one before wrote beside it, in blocks and rows
that share 32-byte sectors."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def busy():
    """Keeps the GPU at work until the calls behind it are all launched."""
    work = torch.randn(4096, 4096, device="cuda", dtype=torch.bfloat16)
    for _ in range(20):
        work @ work


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("size", [36, 52, 4100, 262148])
def test_chained_copies(size, captured):
    """Call i copies blocks (i, ..) to the blocks beside them, which call i + 1 copies on."""
    from hk_b200.csrc import ops
    n, arrays = 24, 6
    caches = [torch.randint(0, 2 ** 31 - 1, (n, size // 4), dtype=torch.int32, device="cuda") for _ in range(arrays)]
    table = torch.tensor([[c.data_ptr(), n, 1, size, size] for c in caches], dtype=torch.int64).cuda()
    # block b to the one behind it, for every third b, so that neighbours of a source are written in the same call
    chain = [[(b, b + 1, 1) for b in range(i % 3, n - 1, 3)] for i in range(30)]
    want = [c.cpu().clone() for c in caches]
    for moves in chain:
        for w in want:
            old = w.clone()
            for a, b, _ in moves:
                w[b] = old[a]
    moves = [torch.tensor(m, dtype=torch.int32, device="cuda") for m in chain]
    torch.cuda.synchronize()

    def call():
        for m in moves:
            ops.copy_blocks(table, m, size)
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graph.replay()
    else:
        busy()
        call()
    torch.cuda.synchronize()
    for c, w in zip(caches, want):
        assert torch.equal(c.cpu(), w)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("G,hd,page,dtype", [(3, 5, 4, torch.float32), (1, 3, 7, torch.bfloat16), (2, 10, 1, torch.bfloat16), (2, 64, 8, torch.bfloat16)])
def test_chained_kept_rows(G, hd, page, dtype, captured):
    """Every call moves rows up that the call before moved, behind one another and in pages that lie beside each other."""
    from hk_b200.csrc import ops
    rng = np.random.default_rng(3)
    R, stride = 5, -(-120 // page)
    pages = R * stride
    caches = [torch.randn(pages, G, page, hd).to(dtype).cuda() for _ in range(6)]
    order = rng.permutation(pages).reshape(R, stride).astype(np.int32)
    bt = torch.from_numpy(order).cuda()
    row = hd * dtype.itemsize
    table = torch.tensor([[c.data_ptr(), G, row, bt.data_ptr()] for c in caches], dtype=torch.int64).cuda()
    want = [c.cpu().clone() for c in caches]
    calls = []
    for _ in range(30):
        paths = np.full((R, 2 + 12), -1, dtype=np.int32)
        for r in range(R):
            paths[r, :2] = r, int(rng.integers(0, 60))
            paths[r, 2:] = np.sort(rng.choice(50, 12, replace=False))
        for w in want:
            old = w.clone()
            for r in range(R):
                for to, k in enumerate(paths[r, 2:].tolist()):
                    s, d = int(paths[r, 1]) + k, int(paths[r, 1]) + to
                    w[order[r, d // page], :, d % page] = old[order[r, s // page], :, s % page]
        calls.append(torch.from_numpy(paths).cuda())
    torch.cuda.synchronize()

    def call():
        for p in calls:
            ops.compact_rows(table, p, R, stride, page, G, row, pages)
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graph.replay()
    else:
        busy()
        call()
    torch.cuda.synchronize()
    for c, w in zip(caches, want):
        assert torch.equal(c.cpu(), w)
