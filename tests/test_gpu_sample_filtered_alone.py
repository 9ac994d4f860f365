"""Filtered sampling: a draw follows from its row alone, whatever else is in
the batch."""
import numpy as np
import pytest

from test_gpu_sample_filtered import _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [5000, 20001, 40000, 100000, 151936, 262147])
def test_a_draw_does_not_depend_on_the_batch(ctx, n):
    """u = 0 draws the first index whose weight is not rounded away, and u next to 1 the last: rows whose ends have
    weights about the rounding's, alone and among other rows."""
    import torch
    rng = np.random.default_rng(n)
    rows = 24
    x = (rng.standard_normal((rows, n)) * 0.5).astype(np.float32)
    x[:, n // 2] = 8.0                                     # the largest; all other weights are at least 2^-17 or so
    x[:, 0] = 8.0 - np.linspace(36, 53, rows) * np.log(2)  # weights of 2^-36 to 2^-53
    x[:, -1] = x[::-1, 0]
    first, last = np.zeros(rows, np.float32), np.full(rows, np.nextafter(np.float32(1), np.float32(0)), np.float32)
    for kw in ({}, {"top_p": 0.97}):
        for u in (first, last, rng.random(rows).astype(np.float32)):
            alone = np.concatenate([_run(ctx, torch, x[r:r + 1], u[r:r + 1], **kw) for r in range(rows)])
            for batch in (2, 8, 18, 64, 200):
                at = np.resize(np.arange(rows), batch)
                got = _run(ctx, torch, torch.from_numpy(x).cuda()[torch.from_numpy(at).cuda()], u[at], **kw)
                assert np.array_equal(got, alone[at]), (batch, kw, got, alone[at])
