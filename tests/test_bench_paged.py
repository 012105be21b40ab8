"""The CPU side of the paged workload's parity check where the reference's own code is not built: blocks
of the highest mean score, attention over their tokens in float64."""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_without_the_reference(monkeypatch):
    import bench
    from oracle import oracle as O
    monkeypatch.setattr(O, "ref_available", lambda: False)
    rng = np.random.RandomState(0)
    n, d = bench.P_BLOCK * (bench.P_TOP + 7), bench.P_DIM
    keys, vals = (rng.standard_normal((n, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal(d).astype(np.float32)
    blocks, out = bench.paged_decode_cpu(O, keys, vals, q)
    means = keys.astype(np.float64).reshape(-1, bench.P_BLOCK, d).mean(1)
    score = means @ q
    want = np.argsort(-score, kind="stable")[:bench.P_TOP]
    assert np.abs(np.diff(np.sort(score))).min() > 1e-5          # no two blocks next to a tie in fp32
    assert np.array_equal(np.sort(blocks), np.sort(want)) and np.array_equal(blocks, want)
    rows = np.concatenate([np.arange(b * bench.P_BLOCK, (b + 1) * bench.P_BLOCK) for b in want])
    x = keys[rows].astype(np.float64) @ q / np.sqrt(d)
    p = np.exp(x - x.max())
    p /= p.sum()
    v = vals[rows].astype(np.float64)
    # fp32: a score is off by d roundings of sum |q k| (and its scaling, the exponential), which moves a
    # weight's share by twice that; a sum of n weights by n roundings
    delta = (d + 4) * 2.0 ** -24 * (np.abs(keys[rows]) @ np.abs(q)).max() / np.sqrt(d) + 2.0 ** -22
    tol = (2 * delta + 2 * len(rows) * 2.0 ** -24) * (p @ np.abs(v))
    assert (np.abs(out - p @ v) <= tol).all()
