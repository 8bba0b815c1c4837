"""Plain 64-bit forms of the operators on drafted trees and beams, and the inputs of their tests."""
import math

import numpy as np
import torch


def tree_bits(see: np.ndarray, words: int) -> np.ndarray:
    """bool [count, count] -> int32 [count, words]: bit j of a row: it sees drafted token j."""
    out = np.zeros((see.shape[0], words), dtype=np.uint32)
    for i, j in zip(*np.nonzero(see)):
        out[i, j // 32] |= np.uint32(1 << (j % 32))
    return out.view(np.int32)


def tree_masks(kind: str, count: int, rng) -> np.ndarray:
    if kind == "chain":
        return np.tril(np.ones((count, count), dtype=bool))
    if kind == "full":
        return np.ones((count, count), dtype=bool)
    if kind == "random":
        return rng.random((count, count)) < 0.4
    if kind == "none":
        return np.zeros((count, count), dtype=bool)
    see = np.eye(count, dtype=bool)                       # a tree
    for i in range(1, count):
        see[i] |= see[rng.integers(max(0, i - 9), i)]
    return see


class TreeCase:
    """A batch of drafted trees over a paged cache, with rows of q that belong to no request between and behind the requests."""

    def __init__(self, seed, contexts, counts, H, G, hd, page, window=0, cap=0.0, sink=0, dtype=torch.bfloat16, mask="tree", device="cuda",
                 gap=1, q_std=1.5):
        rng = np.random.default_rng(seed)
        self.contexts, self.counts, self.H, self.G, self.hd, self.page = contexts, counts, H, G, hd, page
        self.window, self.cap, self.sink, self.dtype = window, cap, sink, dtype
        self.scale = 1.0 / math.sqrt(hd)
        R = len(contexts)
        self.words = -(-max(max(counts), 1) // 32)
        need = [-(-(c + t) // page) for c, t in zip(contexts, counts)]
        self.num_pages = sum(need) + 2
        order = rng.permutation(self.num_pages)
        self.table = np.full((R + 1, max(max(need), 1)), -1, dtype=np.int32)
        self.requests = np.zeros((R, 4), dtype=np.int32)
        self.n = sum(counts) + gap * (R + 1)
        self.ancestors = rng.integers(-2 ** 31, 2 ** 31, (self.n, self.words)).astype(np.int32)      # bits behind the last token mean nothing
        self.positions = np.zeros(self.n, dtype=np.int32)
        self.see = []
        slots = rng.permutation(R + 1)[:R]
        at, row = 0, gap
        for i in range(R):
            self.table[slots[i], :need[i]] = order[at:at + need[i]]
            at += need[i]
            self.requests[i] = (slots[i], row, counts[i], contexts[i])
            see = tree_masks(mask, counts[i], rng)
            self.see.append(see)
            if counts[i]:
                bits = tree_bits(see, self.words).view(np.uint32)
                for w in range(self.words):
                    inside = max(0, min(32, counts[i] - 32 * w))
                    keep = np.uint32((1 << inside) - 1) if inside < 32 else np.uint32(0xffffffff)
                    rows = self.ancestors[row:row + counts[i], w].view(np.uint32)
                    rows[:] = (rows & ~keep) | (bits[:, w] & keep)
                self.positions[row:row + counts[i]] = contexts[i] + (np.tril(see, -1).sum(1) if mask == "tree" else np.arange(counts[i]))
            row += counts[i] + gap
        g = torch.Generator().manual_seed(seed)
        self.q = (torch.randn(self.n, H * hd, generator=g) * q_std).to(dtype)
        self.k = torch.randn(self.num_pages, G, page, hd, generator=g).to(dtype)
        self.v = torch.randn(self.num_pages, G, page, hd, generator=g).to(dtype)
        self.sinks = torch.randn(H, generator=g) if sink == 2 else None
        self.device = device

    def place(self, i, row):
        """(page, row of the page) of a request's cache row."""
        return int(self.table[self.requests[i, 0], row // self.page]), row % self.page

    def reference(self):
        """(out in 64 bits, sum of p |v| in 64 bits, largest sum of |q_d k_d| * scale); rows of no request NaN."""
        H, G, hd = self.H, self.G, self.hd
        out = np.full((self.n, H, hd), np.nan)
        weight = np.zeros((self.n, H, hd))
        most = 0.0
        for i, (slot, first, count, context) in enumerate(self.requests.tolist()):
            if not count:
                continue
            end = context + count
            pages = self.table[slot, :-(-end // self.page)]
            K = self.k[pages].double().permute(1, 0, 2, 3).reshape(G, -1, hd)[:, :end].numpy()
            V = self.v[pages].double().permute(1, 0, 2, 3).reshape(G, -1, hd)[:, :end].numpy()
            see = np.concatenate([np.ones((count, context), dtype=bool), self.see[i]], axis=1)
            if self.window:
                mine = self.positions[first:first + count].astype(np.int64)
                at = np.concatenate([np.arange(context), mine])
                see &= at[None, :] > mine[:, None] - self.window
            for h in range(H):
                q = self.q[first:first + count, h * hd:(h + 1) * hd].double().numpy()
                for t in range(count):
                    idx = np.nonzero(see[t])[0]
                    kk, vv = K[h // (H // G)][idx], V[h // (H // G)][idx]
                    s = kk @ q[t] * self.scale
                    if len(idx):
                        most = max(most, float((np.abs(kk) @ np.abs(q[t])).max() * self.scale)) if np.isfinite(kk).all() else most
                    if self.cap:
                        s = self.cap * np.tanh(s / self.cap)
                    if self.sink:
                        s = np.append(s, float(self.sinks[h]) if self.sinks is not None else 0.0)
                    if not len(s):
                        out[first + t, h] = 0.0
                        continue
                    p = np.exp(s - s.max())
                    p = (p / p.sum())[:len(idx)]
                    out[first + t, h] = p @ vv
                    weight[first + t, h] = p @ np.abs(vv)
        return out.reshape(self.n, -1), weight.reshape(self.n, -1), most

    def run(self, ops, out=None):
        dev = self.device
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        q = self.q.to(dev)
        if out is None:
            out = torch.full_like(q, 7.0)
        ops.tree_attention(q, self.k.to(dev), self.v.to(dev), up(self.table), up(self.requests), up(self.ancestors), up(self.positions), out,
                           self.H, self.G, self.hd, self.page, self.window, self.scale, max(max(self.counts), 1),
                           max(1, max(c + t for c, t in zip(self.contexts, self.counts))), sum(self.contexts) + sum(self.counts),
                           sink=self.sink > 0, sinks=None if self.sinks is None else self.sinks.to(dev), softcap=self.cap)
        return out

    def tolerance(self, weight, most):
        """Element by element, relative to sum p |v|.  bfloat16: the probabilities and the result are each rounded to it (2^-8 each), the
        rest (32-bit scores of exponents below 2^6, exponentials, sums) stays below 2^-11.  float32: a score of hd products is off by at
        most hd 2^-24 of the sum of their sizes, and so is the exponent; sums of n terms by n 2^-24; each counted twice (numerator and
        denominator), the exponential, the division and the roundings by 16 2^-24 (a tanh form of the cap adds 2^-20 cap)."""
        if self.dtype == torch.bfloat16:
            return (2.0 ** -7 + 2.0 ** -11) * weight + 1e-30
        keys = max(c + t for c, t in zip(self.contexts, self.counts))
        return (2.0 ** -23 * (self.hd * most + keys + 16) + 2.0 ** -20 * self.cap) * weight + 1e-30

    def check(self, ops):
        out = self.run(ops).cpu()
        want, weight, most = self.reference()
        real = ~np.isnan(want).all(axis=1)
        for first, count in self.requests[:, 1:3].tolist():
            real[first:first + count] = True
        assert (out[torch.from_numpy(~real)] == 7.0).all(), "rows of no request were written"
        off = np.abs(out.double().numpy()[real] - want[real])
        tol = self.tolerance(weight, most)[real]
        assert np.isfinite(out[torch.from_numpy(real)].float().numpy()).all()
        worst = float((off / tol).max()) if off.size else 0.0
        assert worst <= 1.0, f"{worst:.3f} of the tolerance"
        return out


def beam_reference(logits: np.ndarray, scores: np.ndarray, beams: int, choices: int):
    """(scores float64, beams, tokens) [prompts, choices] of float32 logits [prompts * beams, V]."""
    rows, V = logits.shape
    x = logits.astype(np.float64)
    x[~np.isfinite(x)] = -np.inf
    with np.errstate(invalid="ignore", divide="ignore"):
        top = x.max(axis=1, keepdims=True)
        top = np.where(np.isfinite(top), top, 0.0)
        lse = top + np.log(np.exp(x - top).sum(axis=1, keepdims=True))
        s = x - lse + scores.astype(np.float64)[:, None]
    s[np.isnan(s)] = -np.inf
    s[~np.isfinite(scores)] = -np.inf
    s = s.reshape(rows // beams, beams * V)
    at = np.argsort(-s, axis=1, kind="stable")[:, :choices]
    return np.take_along_axis(s, at, axis=1), at // V, at % V
