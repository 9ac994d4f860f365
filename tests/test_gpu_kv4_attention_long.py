"""Attention over the 4-bit cache over long requests: pieces of hundreds of CTAs
joined, windows and sinks of many tiles, steps of single tokens beside chunks,
and the prefill within the bound that its scaling of the weights allows."""
import numpy as np
import pytest

import serving_ref as R
from test_gpu_kv4_attention import Case, _check_prefill, _close, _decode

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ one request, every CTA
class Flat:
    """One request of n positions in consecutive pages, made at once."""

    def __init__(self, torch, seed, n, n_kv, hd, page):
        rng = np.random.default_rng(seed)
        pages = -(-n // page)
        shape = (pages, n_kv, page, hd)
        self.q4 = [rng.integers(0, 16, shape, dtype=np.uint8) for _ in range(2)]
        # values of the later positions are larger, so that a piece that is missing moves the output
        grow = np.linspace(0.05, 0.25, pages * page).reshape(pages, 1, page, 1)
        self.d = [R._bf16((rng.uniform(0.05, 0.2, (*shape[:3], hd // 32)) * f).astype(np.float32)).astype(np.float16) for f in (1.0, 4 * grow)]
        self.n, self.n_kv, self.hd = n, n_kv, hd
        self.cache = torch.from_numpy(R.pack(self.q4[0], self.d[0], self.q4[1], self.d[1])).cuda()
        self.t = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
        self.l = torch.tensor([n], dtype=torch.int32, device="cuda")
        self.lens, self.rng = [n], rng

    def kv(self):
        return [R.values(q, d).transpose(0, 2, 1, 3).reshape(-1, self.n_kv, self.hd)[:self.n] for q, d in zip(self.q4, self.d)]


@pytest.mark.parametrize("hd,n_kv,heads,n", [(32, 1, 7, 80011), (64, 1, 8, 40003), (64, 2, 14, 120000), (128, 1, 3, 66000)])
def test_decode_joins_of_more_than_sixteen_groups(ctx, hd, n_kv, heads, n):
    """A long document on few kv heads: pieces of hundreds of CTAs join in more groups than half a warp has lanes.

    The bound is the model's with the roundings of this split in the place of n / 4: a CTA has at most n_kv n / 16 / 592
    + 1 <= 27 tiles on four warps, so a warp adds at most 8 products of 32 positions (two MMA steps of 16 each), and the
    joins add 4, 16 and at most 64 pieces: fewer than 192 roundings, and four exponentials instead of one."""
    import torch
    c = Flat(torch, n, n, n_kv, hd, 64)
    ws = torch.zeros(ctx.kv4_workspace_bytes(heads, n_kv, hd), dtype=torch.uint8, device="cuda")
    q, out = _decode(ctx, torch, c, heads, ws=ws)
    for _ in range(3):                                # the tickets are zero again after every call
        assert torch.equal(_decode(ctx, torch, c, heads, q=q, ws=ws)[1], out)
    k, v = c.kv()
    got, rep = out.cpu().numpy()[0], heads // n_kv
    for h in range(heads):
        kk, vv, x = k[:, h // rep], v[:, h // rep], q[0, h].astype(np.float64)
        s = kk @ x * hd ** -0.5
        ds = (hd + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(x)).max() * hd ** -0.5 + 2.0 ** -22 * np.abs(s).max()
        p = np.exp(s - s.max())
        p /= p.sum()
        tol = (p @ np.abs(vv)) * (2 * ds + 4 * 2.0 ** -21 + 2 * 192 * 2.0 ** -24) + 2.0 ** -40 * p.max() * np.abs(vv).sum(0)
        _close(got[h], p @ vv, tol)


# ------------------------------------------------------------------ the prefill's windows and the tight bound
def _check_rows(ctx, torch, c, heads, new, window=0, sinks=0, step=1):
    """Every step-th row against the model; the largest weight is scaled to 2^15 in both kernels, so the f16 floor is 2^-40."""
    row0 = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = c.rng.standard_normal((row0[-1], heads, c.hd)).astype(np.float32)
    out = torch.full(q.shape, 7.0, device="cuda")
    ctx.kv4_attention_prefill(torch.from_numpy(q).cuda(), c.cache, c.t, c.l, torch.from_numpy(row0).cuda(), out, window=window, sinks=sinks)
    got = out.cpu().numpy()
    for r, n in enumerate(c.lens):
        for t in sorted({*range(0, new[r], step), new[r] - 1}) if new[r] else []:
            _close(got[row0[r] + t], *c.expect(r, q[row0[r] + t], n - new[r] + t, window, sinks, floor=2.0 ** -40))


@pytest.mark.parametrize("hd,heads,n_kv", [(32, 12, 2), (64, 14, 2), (128, 4, 2)])
@pytest.mark.parametrize("window,sinks", [(128, 0), (200, 5), (300, 140), (513, 1), (129, 300)])
def test_prefill_windows_and_sinks_over_many_tiles(ctx, hd, heads, n_kv, window, sinks):
    """Windows and sinks of more than a tile of 128 positions; NaN wherever no query of a chunk looks."""
    import torch
    c = Case(window + hd, [900, 1210, 130], n_kv, hd, 32)
    new = [300, 90, 130]
    for r, n in enumerate(c.lens):
        for j in range(sinks, max(0, n - new[r] - window + 1)):
            c.hide(r, j)
    _check_rows(ctx, torch, c.device(torch), heads, new, window, sinks, step=13)


@pytest.mark.parametrize("hd,heads,n_kv", [(32, 16, 1), (64, 6, 2), (128, 7, 1)])
def test_prefill_within_the_tight_bound(ctx, hd, heads, n_kv):
    import torch
    _check_rows(ctx, torch, Case(hd + 1, [700, 33, 0, 257], n_kv, hd, 16).device(torch), heads, [200, 33, 0, 1], step=7)


def test_prefill_of_a_mixed_step(ctx):
    """Single tokens behind long and short prefixes beside chunks and a request that brings nothing."""
    import torch
    c = Case(71, [3000, 300, 60, 1500, 1], 2, 64, 64).device(torch)
    _check_rows(ctx, torch, c, 14, [1, 200, 0, 7, 1], step=11)
    _check_prefill(ctx, torch, c, 14, [1, 0, 60, 1, 1], 100, 4)
