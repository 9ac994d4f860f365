"""Attention over the 4-bit cache with scores of any size.

Every key of a request is one pattern times a power of two
c_j, so the score of position j is c_j (q . pattern), equal bit for bit for
equal c_j (each column of a product is summed in the same order), and the
largest is at least twice the next.  From 2^20 on (in base-2 units) every other
weight is 2^(-2^19) = 0 in any arithmetic, so the output is the mean of the
values at the largest: weights 1 / w each, summed in float32."""
import numpy as np
import pytest

import serving_ref as R
from test_gpu_kv4_attention import Case, _close, _decode

pytestmark = pytest.mark.gpu

LOG2E = 1.4426950408889634
HIGH, LOW = [3, 100, 101, 400, 550, 699], [0, 50, 333, 640]   # where c_j is largest and smallest


def _steep(hd, n_kv, exponent, heads, rows, scale, seed=1):
    """(case, q [rows, heads, hd]): the heads' largest scores are +-2^exponent in base-2 units, even heads positive."""
    c = Case(seed, [700], n_kv, hd, 16)
    rng = c.rng
    c.kq[:] = rng.integers(0, 16, hd, dtype=np.uint8)
    c.kq[..., 0] = 1                                   # a pattern that is not all zeros
    d = (2.0 ** rng.integers(-5, -2, 700)).astype(np.float16)
    d[HIGH], d[LOW] = 0.25, 2.0 ** -6
    for j in range(700):
        c.kd[c.tables[0, j // 16], :, j % 16] = d[j]
    pattern = c.kq[0, 0, 0].astype(np.float64) - 8
    q = np.abs(rng.standard_normal((rows, heads, hd))) * np.sign(pattern)
    top = np.where(np.arange(heads) % 2, -(2.0 ** -6), 0.25)      # the c_j that wins, with q's sign
    q *= (2.0 ** exponent / (scale * LOG2E * (q @ pattern) * np.abs(top)) * np.sign(top))[..., None]
    return c, q.astype(np.float32)


def _mean_of(c, at, heads):
    """The mean of the values at the even heads' and the odd heads' winners, and a bound on float32's error."""
    _, v = c.kv(0, 700)
    rep = heads // c.n_kv
    ref, tol = np.zeros((heads, c.hd)), np.zeros((heads, c.hd))
    for h in range(heads):
        w = v[at[h % 2], h // rep]
        ref[h] = w.mean(0)
        # the weights are equal; at most 64 additions before and in the joins and a division, in float32
        tol[h] = np.abs(w).mean(0) * 2 * 64 * 2.0 ** -24
    return ref, tol


EXPONENTS = [20, 23.4, 24, 24.3, 24.9, 25, 26.2, 27, 27.9, 28, 29.5, 31, 40, 64, 100]


@pytest.mark.parametrize("exponent", EXPONENTS)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_decode_scores_of_any_size(ctx, hd, exponent):
    import torch
    c, q = _steep(hd, 2, exponent, 14, 1, hd ** -0.5)
    _, out = _decode(ctx, torch, c.device(torch), 14, q=q)
    _close(out.cpu().numpy()[0], *_mean_of(c, (HIGH, LOW), 14))


@pytest.mark.parametrize("exponent", EXPONENTS)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_prefill_scores_of_any_size(ctx, hd, exponent):
    import torch
    new = 150
    c, q = _steep(hd, 2, exponent, 14, new, hd ** -0.5)
    c.device(torch)
    out = torch.full(q.shape, 7.0, device="cuda")
    ctx.kv4_attention_prefill(torch.from_numpy(q).cuda(), c.cache, c.t, c.l, torch.tensor([0, new], dtype=torch.int32, device="cuda"), out)
    got = out.cpu().numpy()
    for t in range(new):
        i = 700 - new + t
        _close(got[t], *_mean_of(c, ([j for j in HIGH if j <= i], [j for j in LOW if j <= i]), 14))


@pytest.mark.parametrize("prefill", [False, True])
def test_a_scale_whose_product_with_q_passes_float32(ctx, prefill):
    """scale 3e38 and q of about 2^20: the scores pass float32's largest number, their softmax does not."""
    import torch
    c, q = _steep(64, 2, 150, 8, 1, 3e38)
    c.device(torch)
    if prefill:
        out = torch.full(q.shape, 7.0, device="cuda")
        ctx.kv4_attention_prefill(torch.from_numpy(q).cuda(), c.cache, c.t, c.l, torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                                  out, scale=3e38)
    else:
        out = _decode(ctx, torch, c, 8, q=q, scale=3e38)[1]
    _close(out.cpu().numpy()[0], *_mean_of(c, (HIGH, LOW), 8))
