"""Filtered sampling against the 64-bit model: equal indices wherever no
decision lies so close to its border that the weights' rounding could cross it.

A weight is rounded to a multiple of 2^-s of the largest, s at least 40 (for
rows that a cluster holds), so it is off by at most 2^-41, and the sums are
exact; the n roundings are independent, each of standard deviation 2^-40 / sqrt(12), so a
running sum is off by 6 sqrt(n) 2^-40 / sqrt(12) at six standard deviations,
against a mass of at least 1; a weight itself is computed to 2^-48 of itself.  The model's own sums in 64 bits add n 2^-53 of the mass at most."""
import numpy as np
import pytest

import serving_ref as R

pytestmark = pytest.mark.gpu


def _run(ctx, torch, x, u, **kw):
    d = {}
    for name, a in kw.items():
        if a is not None:
            dt = np.int32 if name == "top_k" else np.float32
            d[name] = torch.from_numpy(np.broadcast_to(np.asarray(a, dt), (len(x),)).copy()).cuda()
    idx = torch.full((len(x),), -9, dtype=torch.int32, device="cuda")
    xd = x if isinstance(x, torch.Tensor) else torch.from_numpy(x).cuda()
    ctx.sample_filtered(xd, torch.from_numpy(np.asarray(u, np.float32)).cuda(), idx, **d)
    return idx.cpu().numpy()


def _check(ctx, torch, x, u, temperature=None, top_k=None, top_p=None, min_p=None, on_border=1):
    """on_border: how many rows may lie on a border (rows of equal logits have whole masses that meet p exactly)."""
    n = x.shape[1]
    near = 6 * np.sqrt(n / 12) * 2.0 ** -40 + 2.0 ** -48 + n * 2.0 ** -53
    got = _run(ctx, torch, x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    at = lambda a, r, v: v if a is None else np.broadcast_to(a, (len(x),))[r]  # noqa: E731
    sure = 0
    for r in range(len(x)):
        want, margin = R.sample(x[r], u[r], np.float64(np.float32(at(temperature, r, 1.0))), int(at(top_k, r, 0)),
                                at(top_p, r, 1.0), at(min_p, r, 0.0))
        if margin > near:
            assert got[r] == want, (r, got[r], want, margin)
            sure += 1
    assert sure >= len(x) - on_border
    return got


SETTINGS = [{}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 50}, {"top_p": 0.9}, {"min_p": 0.05},
            {"temperature": 1.7, "top_k": 40, "top_p": 0.8, "min_p": 0.02}, {"top_p": 0.001}, {"top_p": 0.99999},
            {"temperature": 0.3, "top_p": 0.95}, {"top_k": 3000, "top_p": 0.5}]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("rows,n", [(6, 1), (6, 2), (5, 33), (4, 1000), (3, 4097), (3, 32000), (2, 151936), (2, 262147)])
def test_matches_the_model(ctx, rows, n, kw):
    import torch
    rng = np.random.default_rng(n + rows)
    x = (rng.standard_normal((rows, n)) * 2.5).astype(np.float32)
    # (at top_p = 0.99999 the running mass moves by about 1e-10 of itself per index of a long row: rows may lie on a border)
    _check(ctx, torch, x, rng.random(rows).astype(np.float32), on_border=2 if kw.get("top_p") == 0.99999 and n > 100000 else 1, **kw)


@pytest.mark.parametrize("rows,n", [(8, 151936), (20, 100000), (16, 20001), (40, 9001), (70, 20000), (300, 5000)])
def test_rows_that_fill_the_machine_in_every_way(ctx, rows, n):
    """Each number of CTAs and threads per row that the number of rows asks for."""
    import torch
    rng = np.random.default_rng(n + rows)
    x = (rng.standard_normal((rows, n)) * 2.5).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    one = _check(ctx, torch, x, u, on_border=1, top_k=1000, top_p=0.9)
    assert np.array_equal(_check(ctx, torch, x[:1], u[:1], on_border=1, top_k=1000, top_p=0.9), one[:1])


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_ties_go_to_the_lowest_index(ctx, kw):
    """Few distinct values: every threshold falls among equal logits."""
    import torch
    rng = np.random.default_rng(17)
    x = rng.integers(-3, 3, (16, 3001)).astype(np.float32)
    x[3] = 1.5                                   # all equal
    x[4] = np.where(np.arange(3001) % 2, 0.0, -0.0)   # 0 and -0 are equal
    _check(ctx, torch, x, rng.random(16).astype(np.float32), on_border=3, **kw)


def test_rows_have_their_own_settings(ctx):
    import torch
    rng = np.random.default_rng(23)
    rows = 64
    x = (rng.standard_normal((rows, 5003)) * rng.uniform(0.5, 6, (rows, 1))).astype(np.float32)
    _check(ctx, torch, x, rng.random(rows).astype(np.float32), temperature=rng.choice([0.0, 0.5, 1.0, 2.0], rows).astype(np.float32),
           top_k=rng.choice([0, 1, 2, 64, 5002, 5003, 9999], rows).astype(np.int32),
           top_p=rng.choice([0.0, 0.3, 0.9, 1.0, 1.5], rows).astype(np.float32),
           min_p=rng.choice([0.0, 0.001, 0.3, 1.0], rows).astype(np.float32))


def test_special_logits(ctx):
    import torch
    inf, nan = np.inf, np.nan
    x = np.full((9, 777), -inf, np.float32)   # (and rows of one CTA: the others span several)
    x[1, 700] = -3e38
    x[2, :] = nan
    x[3, [5, 9]] = nan, 2.0
    x[4, [3, 600]] = inf                          # only infinities can be drawn
    x[5, :] = np.linspace(-3.4e38, 3.4e38, 777)
    x[6, :10] = 1e-42                             # subnormal and equal
    x[7, ::2] = 0.25
    x[8, [1, 2]] = 0.0, -200.0
    u = np.full(9, 0.6, np.float32)
    got = _check(ctx, torch, x, u, top_p=0.95)
    assert got[0] == -1 and got[2] == -1 and got[1] == 700 and got[3] == 9 and got[4] == 600 and got[8] == 1
    _check(ctx, torch, x, u, top_k=2)
    _check(ctx, torch, x, u, min_p=0.5, temperature=1e-3)
    _check(ctx, torch, x[[0, 1, 3, 6, 7, 8]], u[:6], temperature=inf)


def test_random_numbers_at_and_outside_the_ends(ctx):
    import torch
    x = np.tile(np.array([0.0, 1.0, -1.0, 0.5], np.float32), (6, 1))
    got = _run(ctx, torch, x, [0.0, -1.0, np.nan, np.nextafter(np.float32(1), np.float32(0)), 1.0, 7.0])
    assert got.tolist() == [0, 0, 0, 3, 3, 3]
    got = _run(ctx, torch, x, [0.0, -1.0, np.nan, 0.9999, 1.0, 7.0], top_k=2)   # keeps 1.0 and 0.5
    assert got.tolist() == [1, 1, 1, 3, 3, 3]
    got = _run(ctx, torch, x, [0.5] * 6, temperature=[0.0, -1.0, np.nan, 1e-30, 0.01, 1.0], top_k=0)
    assert got[:5].tolist() == [1] * 5


def test_strided_rows_and_no_rows(ctx):
    import torch
    rng = np.random.default_rng(3)
    big = torch.from_numpy((rng.standard_normal((5, 2048)) * 3).astype(np.float32)).cuda()
    x = big[:, 13:1014]
    u = rng.random(5).astype(np.float32)
    got = _run(ctx, torch, x, u, top_p=0.9)
    assert np.array_equal(got, _run(ctx, torch, x.contiguous(), u, top_p=0.9))
    assert _run(ctx, torch, big[:0], u[:0]).size == 0


def test_draws_follow_the_filtered_distribution(ctx):
    import torch
    logits = np.array([2.0, 1.0, 0.5, 0.0, -1.0, -np.inf, 1.5, -3.0], np.float32)
    R_ = 20000
    rng = np.random.default_rng(8)
    got = _run(ctx, torch, np.tile(logits, (R_, 1)), rng.random(R_).astype(np.float32), top_k=5, temperature=0.9)
    w = np.exp(logits.astype(np.float64) / 0.9)
    w[[4, 5, 7]] = 0
    w /= w.sum()
    counts = np.bincount(got, minlength=8)
    assert not counts[w == 0].any()
    assert np.all(np.abs(counts - R_ * w) <= 5 * np.sqrt(R_ * w * (1 - w)))


def test_captured_and_replayed(ctx):
    import torch
    rng = np.random.default_rng(4)
    x = torch.from_numpy((rng.standard_normal((3, 40000)) * 2).astype(np.float32)).cuda()
    u, idx = torch.tensor([0.1, 0.5, 0.9], device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    p = torch.full((3,), 0.9, device="cuda")
    before = torch.cuda.current_stream().cuda_stream
    s = torch.cuda.Stream()
    ctx.set_stream(s.cuda_stream)
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ctx.sample_filtered(x, u, idx, top_p=p)
        for step in range(4):
            x.copy_(torch.from_numpy((rng.standard_normal((3, 40000)) * 2).astype(np.float32)))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            want = [R.sample(r, v, p=0.9)[0] for r, v in zip(x.cpu().numpy(), u.cpu().numpy())]
            assert idx.tolist() == want, step
    finally:
        ctx.set_stream(before)


@pytest.mark.parametrize("n", [1_100_003, 5_000_000])
def test_rows_beyond_shared_memory(ctx, n):
    """A row that no cluster holds is read from memory at every step."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(2, n, generator=g, device="cuda") * 2
    u = np.array([0.3, 0.8], np.float32)
    for kw in ({"top_p": 0.9}, {"top_k": 500, "top_p": 0.7}, {"min_p": 0.001}):
        got = _run(ctx, torch, x, u, **kw)
        for r in range(2):
            want, margin = R.sample(x[r].cpu().numpy(), u[r], k=kw.get("top_k", 0), p=kw.get("top_p", 1.0), min_p=kw.get("min_p", 0.0))
            assert got[r] == want or margin < 1e-9


def test_many_equal_logits_in_long_rows(ctx):
    """The bin of the threshold holds more elements than are compared with one another, on several levels."""
    import torch
    rng = np.random.default_rng(31)
    n = 100_000
    x = np.empty((5, n), np.float32)
    x[0] = 0.5                                                    # one key
    x[1] = 1.0 + rng.integers(0, 3000, n).astype(np.float32) * np.float32(2.0 ** -23)   # 3000 neighbouring keys
    x[2] = rng.standard_normal(n).astype(np.float32) * np.float32(1e-3)    # all in a few bins, keys far apart
    x[3] = np.where(rng.random(n) < 0.5, 2.0, -1.0)
    x[4] = np.where(np.arange(n) < n - 700, -40.0, 1.0)
    u = rng.random(5).astype(np.float32)
    for kw in ({"top_k": 33333}, {"top_p": 0.37}, {"top_k": 60001, "top_p": 0.61}, {"top_k": 99_999, "top_p": 0.999}):
        _check(ctx, torch, x, u, on_border=3, **kw)
