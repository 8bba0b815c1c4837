"""What drafted trees and beams need on the host: packed trees, guesses from the text, command-line options (no GPU)."""
import numpy as np
import pytest

from hk_b200.engine.context import pack_trees
from hk_b200.engine.drafts import LookupDrafts


def test_packed_trees():
    rng = np.random.default_rng(0)
    lens = [5, 1, 70]
    parents = [[-1, 0, 0, 1, -1], None, [-1] + [int(rng.integers(-1, i)) for i in range(1, 70)]]
    packed, depth, words = pack_trees([4, 0, 2], [0, 5, 6], lens, [10, 0, 33], parents)
    assert words == 3 and packed.dtype == np.int32 and len(packed) == 12 + 76 * 3 + 76
    assert packed[:12].reshape(3, 4).tolist() == [[4, 0, 5, 10], [0, 5, 1, 0], [2, 6, 70, 33]]
    bits = packed[12:12 + 76 * 3].view(np.uint32).reshape(76, 3)
    assert packed[12 + 76 * 3:].tolist() == list(range(10, 15)) + [0] + list(range(33, 103))
    row = 0
    for n, tree in zip(lens, parents):
        for i in range(n):
            path, j = set(), i
            while j >= 0:
                path.add(j)
                j = (j - 1) if tree is None else tree[j]
            got = {32 * w + b for w in range(3) for b in range(32) if (int(bits[row + i, w]) >> b) & 1}
            assert got == path and depth[row + i] == len(path) - 1
        row += n


def test_tokens_that_follow_one_another():
    packed, depth, words = pack_trees([1], [0], [4], [7], [None])
    assert packed[4:8].tolist() == [1, 3, 7, 15] and depth.tolist() == [0, 1, 2, 3]


def test_guesses_follow_the_text():
    d = LookupDrafts([1, 2, 3, 4, 1, 2, 3, 5, 1, 2, 3])
    tokens, parents = d.tree(6)
    # the longest match, the latest place first: 5 1 2 3, then 4 1 ... from the earlier place, sharing nothing
    assert tokens[:4] == [5, 1, 2, 3] and parents[:4] == [-1, 0, 1, 2]
    assert tokens[4:] == [4, 1] and parents[4:] == [-1, 4]
    assert d.tree(0) == ([], []) and LookupDrafts([7]).tree(5) == ([], []) and LookupDrafts([]).tree(5) == ([], [])
    d.extend([4])
    assert d.tree(3) == ([1, 2, 3], [-1, 0, 1])


@pytest.mark.parametrize("seed", range(4))
def test_guesses_are_trees(seed):
    rng = np.random.default_rng(seed)
    d = LookupDrafts(rng.integers(0, 5, 50).tolist())
    for _ in range(40):
        most = int(rng.integers(1, 30))
        tokens, parents = d.tree(most)
        assert len(tokens) == len(parents) <= most and all(-1 <= p < i for i, p in enumerate(parents))
        assert len({(p, t) for p, t in zip(parents, tokens)}) == len(tokens), "two children of a node guess the same token"
        d.extend([int(rng.integers(0, 5))])


def test_command_line_options():
    from hk_b200.cli import BadUsage, parse_run_args
    g = parse_run_args(["m", "1,2", "--beams", "4", "--length-penalty", "0.5"])
    assert g["beams"] == 4 and g["length_penalty"] == 0.5 and g["draft"] == 0
    assert parse_run_args(["m", "1,2", "--draft", "8"])["draft"] == 8
    for bad in (["--beams", "0"], ["--beams", "129"], ["--draft", "-1"], ["--draft", "256"], ["--draft", "4", "--beams", "2"], ["--length-penalty", "x"],
                ["--draft", "4", "--repeat-penalty", "1.2"]):
        with pytest.raises(BadUsage):
            parse_run_args(["m", "1,2"] + bad)


def test_launches_go_to_the_device_of_their_tensors(monkeypatch):
    """With another device current, every entry point launches on its tensors' device and that one's stream (against stand-ins)."""
    import contextlib
    import types

    import torch

    from hk_b200.csrc import build, gemm_fast, ops
    current, launched = [1], []

    @contextlib.contextmanager
    def device(index):
        old, current[0] = current[0], index
        yield
        current[0] = old
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(ops, "_need", lambda *a, **k: None)
    monkeypatch.setattr(gemm_fast, "_sms", lambda d: 148)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: types.SimpleNamespace(data_ptr=lambda: 4096))

    def tell(*args):
        launched.append((current[0], args[-1]))
        return 0
    lib = types.SimpleNamespace(hk_copy_blocks=tell, hk_compact_rows=tell, hk_beam_select=tell, hk_beam_select_scratch=lambda *a: 64, hk_tree_attention=tell)
    monkeypatch.setattr(build, "load", lambda name: lib)

    class Fake:
        def __init__(self, index, shape, dtype=None):
            self.device, self.shape, self.dtype = types.SimpleNamespace(index=index), torch.Size(shape), dtype

        def get_device(self):
            return self.device.index

        def data_ptr(self):
            return 1024

        def is_contiguous(self):
            return True

    f, n = torch.float32, torch.int32
    for i in (0, 1):
        ops.copy_blocks(Fake(i, (2, 5)), Fake(i, (3, 3)), 64)
        ops.compact_rows(Fake(i, (2, 4)), Fake(i, (3, 6)), 4, 8, 16, 2, 256, 32)
        ops.beam_select(Fake(i, (6, 50), f), Fake(i, (6,), f), 3, Fake(i, (2, 6), f), Fake(i, (2, 6), n), Fake(i, (2, 6), n))
        ops.tree_attention(Fake(i, (4, 256), f), Fake(i, (9, 2, 16, 64), f), Fake(i, (9, 2, 16, 64), f), Fake(i, (2, 5), n), Fake(i, (1, 4), n),
                           Fake(i, (4, 1), n), Fake(i, (4,), n), Fake(i, (4, 256), f), 4, 2, 64, 16, 0, 0.125, 4, 60)
    assert launched == [(0, 100)] * 4 + [(1, 101)] * 4 and current == [1]


def test_beam_selection_refuses_rows_that_its_indexes_do_not_hold(monkeypatch):
    import types

    import torch

    from hk_b200.csrc import ops
    monkeypatch.setattr(ops, "_need", lambda *a, **k: None)

    def fake(*shape):
        return types.SimpleNamespace(shape=torch.Size(shape), dtype=None, get_device=lambda: 0)
    for vocab, beams in (((1 << 30) + 1, 1), (1 << 30, 2), (1 << 23, 256), (50, 257)):
        with pytest.raises(ops.KernelError, match="are taken"):
            ops.beam_select(fake(beams, vocab), fake(beams), beams, fake(1, 4), fake(1, 4), fake(1, 4))
