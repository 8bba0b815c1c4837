"""The sums behind beam selection's scores on rows where most of the probability lies far from a thread's first logits."""
import numpy as np
import pytest
import torch

from ref_branches import beam_reference

pytestmark = pytest.mark.gpu

# A score is its logit and its beam's score less the logarithm of a sum, in 64 bits, rounded once (2^-24 of it).  The sum: each exponential
# is off by the approximation's 2 units in the last place (2^-22) and by the roundings of its exponent, a difference of two numbers of at
# most a half, each rounded twice (2^-26 and 2^-25), and rounded itself (2^-25): 2^-23 together; sixteen are added in four steps (2^-24
# each); all beyond that has 64 bits.  Relative, and so absolute in the logarithm.
SUM = 2.0 ** -22 + 2.0 ** -23 + 4 * 2.0 ** -24


def errors(logits, scores, beams, choices):
    from hk_b200.csrc import ops
    prompts = logits.shape[0] // beams
    out = torch.empty((prompts, choices), dtype=torch.float32, device="cuda")
    k, v = (torch.empty((prompts, choices), dtype=torch.int32, device="cuda") for _ in range(2))
    ops.beam_select(torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), beams, out, k, v)
    want = beam_reference(logits, scores, beams, choices)
    assert np.array_equal(v.cpu().numpy(), want[2]) and np.array_equal(k.cpu().numpy(), want[1])
    return np.abs(out.cpu().numpy() - want[0]) - 2.0 ** -24 * np.abs(want[0])


def rows_of(kind, rows, V, rng):
    x = (rng.standard_normal((rows, V)) * 2.5).astype(np.float32)
    if kind == "one ahead":                        # one token far ahead, anywhere in the row
        x[np.arange(rows), rng.integers(0, V, rows)] = 17 + 4 * rng.random(rows)
    elif kind == "late":                           # the same in the row's last quarter, where every thread has seen others before
        x[np.arange(rows), rng.integers(V - V // 4, V, rows)] = 17 + 4 * rng.random(rows)
    elif kind == "twelve":
        for r in x:
            r[rng.choice(V, 12, replace=False)] = 14 + rng.standard_normal(12)
    elif kind == "climbing":                       # every tile's values some 6 above those of the one before
        x += np.floor(np.arange(V) / 4096).astype(np.float32) * 6
    elif kind == "flat and one":                   # most of the sum in equal logits far below the largest
        x[:] = (-9 - 2 * rng.random((rows, 1))).astype(np.float32)
        x[np.arange(rows), rng.integers(0, V, rows)] = rng.random(rows).astype(np.float32)
        x[:, :7] += np.arange(7, dtype=np.float32) / 16
    elif kind == "flat":
        x[:] = (rng.standard_normal((rows, 1)) * 5).astype(np.float32)
    elif kind == "low":                            # the same far from zero, where logits lie 2^-4 apart
        x = (x * 16).round() / 16 + np.float32(1.5e6)
        x[np.arange(rows), rng.integers(0, V, rows)] += 9
    elif kind == "steps":                          # logits 64 and more apart, and up to the largest finite
        x = (np.float32(2.0) ** rng.integers(20, 100, (rows, V)).astype(np.float32) * rng.choice([-1, 1], (rows, V))).astype(np.float32)
    return np.ascontiguousarray(x)


@pytest.mark.parametrize("rows,V", [(4, 30001), (128, 40000), (600, 20000), (600, 4096)])
@pytest.mark.parametrize("kind", ["plain", "one ahead", "late", "twelve", "climbing", "flat and one", "flat", "low", "steps"])
def test_sums(kind, rows, V):
    rng = np.random.default_rng(rows + V)
    off = errors(rows_of(kind, rows, V, rng), np.zeros(rows, dtype=np.float32), 1, 4)
    assert off.max() <= SUM, f"{off.max():.2e}"


@pytest.mark.parametrize("rows", [4, 600])
def test_masked_rows(rows):
    """-inf, +inf and NaN among the logits of rows whose largest is the lowest finite number, a usual one or none."""
    rng = np.random.default_rng(rows)
    x = rows_of("late", rows, 20000, rng)
    for bad in (-np.inf, np.inf, np.nan):
        x[rng.random(x.shape) < 0.2] = bad
    x[1::4] = np.where(rng.random(x[1::4].shape) < 0.5, -np.inf, np.float32(-3.4028234663852886e38))
    x[2::4] = np.where(rng.random(x[2::4].shape) < 0.5, -np.inf, np.nan)
    x[3::4, :15000] = -np.inf
    from hk_b200.csrc import ops
    out = torch.empty((rows, 4), dtype=torch.float32, device="cuda")
    k, v = (torch.empty((rows, 4), dtype=torch.int32, device="cuda") for _ in range(2))
    ops.beam_select(torch.from_numpy(x).cuda(), torch.zeros(rows, device="cuda"), 1, out, k, v)
    want = beam_reference(x, np.zeros(rows, dtype=np.float32), 1, 4)
    got, finite = out.cpu().numpy(), np.isfinite(want[0])
    assert np.array_equal(np.isneginf(got), ~finite) and np.array_equal(v.cpu().numpy(), want[2])
    assert (np.abs(got[finite] - want[0][finite]) <= 2.0 ** -24 * np.abs(want[0][finite]) + SUM).all()
