"""Filtered sampling where the border of top-p lies among very small weights: the
index that is drawn is one that the border's own uncertainty allows.

A weight is rounded to a whole multiple of 2^-s of the largest, s from n alone
and at least 40 up to 737280 logits, so each is off by at most 2^-41 and a
running sum of n of them by n 2^-41, without any statistics; the model's sums
in 64 bits add n 2^-53 of the mass."""
import numpy as np
import pytest

from test_gpu_sample_filtered import _run

pytestmark = pytest.mark.gpu


def _allowed(x, u, p):
    """Every index that the draw can give when each running sum is off by as much as rounding allows."""
    n, x = len(x), x.astype(np.float64)
    w = np.exp(x - x.max())
    order = np.argsort(-x, kind="stable")
    c = np.cumsum(w[order])
    near = n * 2.0 ** -41 + n * 2.0 ** -53 * c[-1]
    goal = np.float64(np.float32(p)) * c[-1]
    found = set()
    for cut in range(int(np.searchsorted(c, goal - 2 * near)) + 1, min(n, int(np.searchsorted(c, goal + 2 * near)) + 1) + 1):
        kept = np.sort(order[:cut])
        run = np.cumsum(w[kept])
        a, b = (np.searchsorted(run, np.float64(np.float32(u)) * run[-1] + d, side="right") for d in (-2 * near, 2 * near))
        found |= set(kept[int(a):int(b) + 1].tolist())
    return found


@pytest.mark.parametrize("rows,n", [(12, 151936), (6, 262147)])
def test_a_border_among_small_weights(ctx, rows, n):
    import torch
    rng = np.random.default_rng(n + rows)
    x = (rng.standard_normal((rows, n)) * 2.5).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    got = _run(ctx, torch, x, u, top_p=0.99999)
    sure = 0
    for r in range(rows):
        want = _allowed(x[r], u[r], 0.99999)
        assert got[r] in want, (r, got[r], want)
        sure += len(want) == 1
    assert sure >= rows - 1                                # (this seed's rows: the model decides nearly all of them alone)


def test_nothing_beyond_the_border_is_drawn(ctx):
    """u next to 1 draws the last kept index: with descending logits that is the border's own rank, to within its uncertainty."""
    import torch
    n = 151936
    rng = np.random.default_rng(9)
    x = -np.sort(-(rng.standard_normal((4, n)) * 2.5).astype(np.float32), axis=1)
    u = np.full(4, np.nextafter(np.float32(1), np.float32(0)), np.float32)
    for p in (0.5, 0.9, 0.99999):
        got = _run(ctx, torch, x, u, top_p=p)
        for r in range(4):
            assert got[r] in _allowed(x[r], u[r], p), (p, r, got[r])
