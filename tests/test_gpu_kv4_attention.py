"""Attention over the 4-bit cache against the 64-bit model on the cache's own
values; the tolerance is the model's bound (serving_ref.attention).  Every slot
that no query sees holds NaN scales."""
import numpy as np
import pytest

import hacedle_cuda as hc
import serving_ref as R

pytestmark = pytest.mark.gpu


class Case:
    """A cache of requests with the given lengths, scattered pages, and NaN everywhere else."""

    def __init__(self, seed, lens, n_kv, hd, page, kscale=1.0):
        self.rng = rng = np.random.default_rng(seed)
        self.lens, self.n_kv, self.hd, self.page = list(lens), n_kv, hd, page
        held = [-(-n // page) for n in lens]
        self.pages = sum(held) + 3
        ids = rng.permutation(self.pages).astype(np.int32)
        self.tables = np.full((len(lens), max(held + [1]) + 2), -1, np.int32)
        shape = (self.pages, n_kv, page, hd)
        self.kq, self.vq = (rng.integers(0, 16, shape, dtype=np.uint8) for _ in range(2))
        d = [np.full((*shape[:3], hd // 32), np.nan, np.float16) for _ in range(2)]
        at = 0
        for r, (n, h) in enumerate(zip(lens, held)):
            self.tables[r, :h] = ids[at:at + h]
            at += h
            for j in range(n):
                pg = self.tables[r, j // page]
                for x, c in zip(d, (kscale, 1.0)):
                    x[pg, :, j % page] = R._bf16(rng.uniform(0.02, 0.3, (n_kv, hd // 32)).astype(np.float32) * c
                                                 * rng.choice([-1, 1], (n_kv, hd // 32)).astype(np.float32))
        self.kd, self.vd = d

    def hide(self, r, j):
        """Position j of request r becomes NaN."""
        pg = self.tables[r, j // self.page]
        self.kd[pg, :, j % self.page] = np.nan
        self.vd[pg, :, j % self.page] = np.nan

    def device(self, torch):
        self.cache = torch.from_numpy(R.pack(self.kq, self.kd, self.vq, self.vd)).cuda()
        self.t = torch.from_numpy(self.tables).cuda()
        self.l = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        return self

    def kv(self, r, n):
        ids = np.clip(self.tables[r, :-(-n // self.page)], 0, self.pages - 1)
        take = lambda q, d: R.values(q[ids], d[ids]).transpose(0, 2, 1, 3).reshape(-1, self.n_kv, self.hd)[:n]  # noqa: E731
        return take(self.kq, self.kd), take(self.vq, self.vd)

    def expect(self, r, q, i, window, sinks, scale=0.0, floor=2.0 ** -40):
        n = i + 1
        ok = R.seen(i, n, window, sinks)
        named = np.repeat((self.tables[r] >= 0) & (self.tables[r] < self.pages), self.page)[:n]
        k, v = self.kv(r, n)
        return R.attention(q.astype(np.float64), k, v, ok & named, scale or self.hd ** -0.5, floor)


def _close(got, ref, tol):
    off = np.abs(got - ref)
    at = np.unravel_index(np.argmax(off - tol), off.shape)
    assert off[at] <= tol[at], (at, got[at], ref[at], tol[at])


def _decode(ctx, torch, c, heads, window=0, sinks=0, scale=0.0, q=None, ws=None):
    q = c.rng.standard_normal((len(c.lens), heads, c.hd)).astype(np.float32) if q is None else q
    out = torch.full(q.shape, 7.0, device="cuda")
    ctx.kv4_attention_decode(torch.from_numpy(q).cuda(), c.cache, c.t, c.l, out, window=window, sinks=sinks, scale=scale, ws=ws)
    return q, out


def _check_decode(ctx, torch, c, heads, window=0, sinks=0, scale=0.0):
    q, out = _decode(ctx, torch, c, heads, window, sinks, scale)
    got = out.cpu().numpy()
    for r, n in enumerate(c.lens):
        n = max(0, min(n, c.tables.shape[1] * c.page))
        if n == 0:
            assert not got[r].any()
            continue
        _close(got[r], *c.expect(r, q[r], n - 1, window, sinks, scale))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("heads,n_kv", [(1, 1), (2, 2), (6, 2), (14, 2), (8, 1), (9, 1), (32, 2)])
def test_decode_head_layouts(ctx, hd, heads, n_kv):
    import torch
    _check_decode(ctx, torch, Case(heads + hd, [1, 2, 15, 16, 17, 0, 33, 63, 64, 65, 130, 257], n_kv, hd, 16).device(torch), heads)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 5), (1, 0), (1, 1), (7, 3), (16, 16), (100, 4), (129, 130), (500, 1)])
def test_decode_windows_and_sinks(ctx, page, window, sinks):
    import torch
    c = Case(page + window, [1, 8, 100, 101, 131, 300, 517], 2, 64, page)
    for r, n in enumerate(c.lens):
        for j in np.flatnonzero(~R.seen(n - 1, n, window, sinks)):
            c.hide(r, j)
    _check_decode(ctx, torch, c.device(torch), 14, window, sinks)


@pytest.mark.parametrize("lens", [[5000], [3001, 1], [1, 1, 1, 4097, 1], [1500] * 3 + [0] * 4 + [700]])
def test_decode_long_rows_split_over_the_machine(ctx, lens):
    import torch
    c = Case(len(lens), lens, 1, 128, 64).device(torch)
    _check_decode(ctx, torch, c, 7)
    _check_decode(ctx, torch, c, 7, window=900, sinks=40)


def test_decode_many_requests(ctx):
    import torch
    rng = np.random.default_rng(4)
    _check_decode(ctx, torch, Case(4, rng.integers(0, 90, 700), 2, 32, 16).device(torch), 4)


def test_decode_scales_and_large_scores(ctx):
    """Scores far apart, a scale of the caller's, and q over many orders of magnitude."""
    import torch
    c = Case(6, [300, 40, 77], 2, 64, 16, kscale=30.0).device(torch)
    _check_decode(ctx, torch, c, 8)
    _check_decode(ctx, torch, c, 8, scale=0.003)
    q = (c.rng.standard_normal((3, 8, 64)) * np.array([1e-30, 1e4, 1e-3])[:, None, None]).astype(np.float32)
    q[0, 0] = 0
    _, out = _decode(ctx, torch, c, 8, q=q, scale=1e-3)
    for r in range(3):
        _close(out.cpu().numpy()[r], *c.expect(r, q[r], c.lens[r] - 1, 0, 0, 1e-3))


def test_decode_bad_pages_are_not_seen(ctx):
    import torch
    c = Case(7, [200, 40, 64], 2, 64, 16)
    c.tables[0, 3], c.tables[0, 7], c.tables[1, :] = -1, c.pages, -5
    c.tables[2, 0] = 2 ** 31 - 1
    c.device(torch)
    q, out = _decode(ctx, torch, c, 4)
    got = out.cpu().numpy()
    assert not got[1].any()
    for r in (0, 2):
        _close(got[r], *c.expect(r, q[r], c.lens[r] - 1, 0, 0))


def test_decode_lengths_out_of_range(ctx):
    """A negative length sees nothing; one beyond the table sees what the table holds."""
    import torch
    c = Case(8, [64, 64], 1, 32, 16)
    c.tables = np.ascontiguousarray(c.tables[:, :4])
    c.lens = [-3, 70]
    c.device(torch)
    q, out = _decode(ctx, torch, c, 2)
    assert not out.cpu().numpy()[0].any()
    _close(out.cpu().numpy()[1], *c.expect(1, q[1], 63, 0, 0))


def test_decode_a_nan_stays_in_its_head(ctx):
    import torch
    c = Case(9, [50, 20], 2, 64, 16)
    c.vd[c.tables[1, 0], 1, 3, 1] = np.nan        # request 1, kv head 1, dimensions 32..63
    c.device(torch)
    q = c.rng.standard_normal((2, 8, 64)).astype(np.float32)
    q[0, 2, 5] = np.nan
    _, out = _decode(ctx, torch, c, 8, q=q)
    got = out.cpu().numpy()
    assert np.isnan(got[0, 2]).all() and not np.isnan(np.delete(got[0], 2, 0)).any()
    assert np.isnan(got[1, 4:, 32:]).all() and not np.isnan(got[1, 4:, :32]).any() and not np.isnan(got[1, :4]).any()


def test_decode_strided_q(ctx):
    import torch
    c = Case(10, [33, 90, 4], 2, 64, 16).device(torch)
    fused = torch.randn(3, 8 * 64 + 4 * 64, device="cuda")
    q = fused[:, :8 * 64].unflatten(1, (8, 64))
    a, b = torch.empty(3, 8, 64, device="cuda"), torch.empty(3, 8, 64, device="cuda")
    ctx.kv4_attention_decode(q, c.cache, c.t, c.l, a)
    ctx.kv4_attention_decode(q.contiguous(), c.cache, c.t, c.l, b)
    assert torch.equal(a, b)


def test_decode_is_repeatable_and_captured(ctx):
    """The same bits from call to call; captured graphs with a workspace each follow the lengths they find."""
    import torch
    c = Case(11, [4000, 31, 900, 2000], 2, 64, 16).device(torch)
    q, out = _decode(ctx, torch, c, 14)
    for _ in range(5):
        assert torch.equal(_decode(ctx, torch, c, 14, q=q)[1], out)
    n = ctx.kv4_workspace_bytes(14, 2, 64)
    ws = [torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    qd = torch.from_numpy(q).cuda()
    outs, graphs, streams, lens = [], [], [], [c.l.clone(), (c.l // 2 + 1)]
    before = torch.cuda.current_stream().cuda_stream
    try:
        for i in range(2):
            s = torch.cuda.Stream()
            ctx.set_stream(s.cuda_stream)
            outs.append(torch.zeros_like(out))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                ctx.kv4_attention_decode(qd, c.cache, c.t, lens[i], outs[i], ws=ws[i])
            graphs.append(g)
            streams.append(s)
    finally:
        ctx.set_stream(before)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], out)
    half = torch.empty_like(out)
    ctx.kv4_attention_decode(qd, c.cache, c.t, lens[1], half)
    assert torch.equal(outs[1], half)
    lens[0].copy_(lens[1])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], half)
    small = torch.zeros(max(0, n - 1), dtype=torch.uint8, device="cuda")
    with pytest.raises(hc.HdError) as e:
        ctx.kv4_attention_decode(qd, c.cache, c.t, c.l, half, ws=small)
    assert e.value.code == hc.HD_E_SHAPE


def test_decode_one_workspace_for_every_head_size(ctx):
    """Calls of different head sizes after one another in the same bytes, the caller's and the context's."""
    import torch
    cases = [Case(12 + hd, [2500, 3, 900], 1, hd, 32).device(torch) for hd in (32, 64, 128)]
    ws = torch.zeros(max(ctx.kv4_workspace_bytes(8, 1, hd) for hd in (32, 64, 128)), dtype=torch.uint8, device="cuda")
    qs = [c.rng.standard_normal((3, 8, c.hd)).astype(np.float32) for c in cases]
    want = [_decode(ctx, torch, c, 8, q=q, ws=torch.zeros_like(ws))[1] for c, q in zip(cases, qs)]
    for i in (0, 1, 2, 1, 0, 2, 0):
        for w in (ws, None):
            assert torch.equal(_decode(ctx, torch, cases[i], 8, q=qs[i], ws=w)[1], want[i])


def _prefill(ctx, torch, c, heads, new, window=0, sinks=0, pad=0, q=None):
    row0 = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = c.rng.standard_normal((row0[-1] + pad, heads, c.hd)).astype(np.float32) if q is None else q
    out = torch.full(q.shape, 7.0, device="cuda")
    ctx.kv4_attention_prefill(torch.from_numpy(q).cuda(), c.cache, c.t, c.l, torch.from_numpy(row0).cuda(), out, window=window,
                              sinks=sinks)
    return row0, q, out


def _check_prefill(ctx, torch, c, heads, new, window=0, sinks=0, pad=0):
    row0, q, out = _prefill(ctx, torch, c, heads, new, window, sinks, pad)
    got = out.cpu().numpy()
    assert np.all(got[row0[-1]:] == 7.0)          # rows behind the last request
    for r, n in enumerate(c.lens):
        for t in range(new[r]):
            i = n - new[r] + t
            if i < 0:
                assert not got[row0[r] + t].any()
            else:
                _close(got[row0[r] + t], *c.expect(r, q[row0[r] + t], i, window, sinks, floor=2.0 ** -32))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("heads,n_kv", [(1, 1), (6, 2), (14, 2), (9, 1), (16, 1)])
def test_prefill_head_layouts(ctx, hd, heads, n_kv):
    import torch
    lens, new = [1, 5, 16, 0, 40, 100, 77], [1, 5, 3, 0, 40, 1, 50]
    _check_prefill(ctx, torch, Case(hd, lens, n_kv, hd, 16).device(torch), heads, new, pad=3)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 3), (1, 0), (5, 2), (33, 64), (90, 1)])
def test_prefill_windows_and_sinks(ctx, page, window, sinks):
    import torch
    _check_prefill(ctx, torch, Case(page, [150, 260, 64], 2, 64, page).device(torch), 4, [150, 37, 2], window, sinks)


def test_prefill_hides_what_no_query_sees(ctx):
    """NaN in front of the window of the chunk's first query, behind the sinks."""
    import torch
    c = Case(21, [400], 1, 64, 16)
    for j in range(4, 400 - 60 - 50 + 1):
        c.hide(0, j)
    _check_prefill(ctx, torch, c.device(torch), 4, [60], window=50, sinks=4)


def test_prefill_more_rows_than_positions_and_bad_pages(ctx):
    import torch
    c = Case(22, [3, 0, 70], 2, 32, 16)
    c.tables[2, 1] = -1
    _check_prefill(ctx, torch, c.device(torch), 4, [6, 4, 70])


def test_prefill_long(ctx):
    """Several tiles of rows and of positions; sampled rows against the model."""
    import torch
    c = Case(23, [1100, 700], 1, 128, 64).device(torch)
    row0, q, out = _prefill(ctx, torch, c, 7, [600, 333])
    got = out.cpu().numpy()
    for row in [0, 1, 17, 18, 100, 299, 598, 599, 600, 731, 932]:
        r = int(row >= 600)
        i = c.lens[r] - (600, 333)[r] + row - row0[r]
        _close(got[row], *c.expect(r, q[row], i, 0, 0, floor=2.0 ** -32))
    again = _prefill(ctx, torch, c, 7, [600, 333], q=q)[2]
    assert torch.equal(again, out)


def test_prefill_of_single_tokens_equals_decode(ctx):
    import torch
    c = Case(24, [1, 33, 200, 517], 2, 64, 32).device(torch)
    _, q, a = _prefill(ctx, torch, c, 14, [1, 1, 1, 1])
    b = _decode(ctx, torch, c, 14, q=q)[1]
    for r, n in enumerate(c.lens):
        _, tol = c.expect(r, q[r], n - 1, 0, 0, floor=2.0 ** -32)
        assert np.all(np.abs(a[r].cpu().numpy() - b[r].cpu().numpy()) <= 2 * tol)


def test_prefill_a_nan_reaches_the_rows_that_see_it_and_no_other(ctx):
    """NaN in a value group and in a key of one position: earlier rows and other heads stay as they are."""
    import torch
    c = Case(25, [300], 2, 64, 16)
    pg = lambda j: c.tables[0, j // 16]  # noqa: E731
    c.vd[pg(150), 1, 150 % 16, 1] = np.nan        # kv head 1, dimensions 32..63
    c.kd[pg(200), 0, 200 % 16, 0] = np.nan        # kv head 0: every dimension of the rows that see it
    c.device(torch)
    _, q, out = _prefill(ctx, torch, c, 4, [300])
    got = out.cpu().numpy()
    assert np.isnan(got[150:, 2:, 32:]).all() and not np.isnan(got[150:, 2:, :32]).any()
    assert np.isnan(got[200:, :2]).all()
    assert not np.isnan(got[:150]).any() and not np.isnan(got[150:200, :2]).any()
    for row in (0, 149, 151, 299):
        ref, tol = c.expect(0, q[row], row, 0, 0, floor=2.0 ** -32)
        fine = ~np.isnan(got[row])
        assert np.all(np.abs(got[row] - ref)[fine] <= tol[fine])


def test_prefill_with_a_window_rows_outlive_a_nan(ctx):
    import torch
    c = Case(26, [400], 1, 32, 16)
    c.vd[c.tables[0, 100 // 16], 0, 100 % 16, 0] = np.nan
    c.device(torch)
    got = _prefill(ctx, torch, c, 2, [400], window=50, sinks=3)[2].cpu().numpy()
    assert np.isnan(got[100:150]).all() and not np.isnan(got[:100]).any() and not np.isnan(got[150:]).any()


@pytest.mark.parametrize("scale", [0.0, 0.5, 1e-3])
def test_prefill_large_scores_move_the_maximum(ctx, scale):
    """Keys that grow along the request: the running maximum moves far and often."""
    import torch
    c = Case(27, [700], 1, 64, 16)
    for j in range(700):
        c.kd[c.tables[0, j // 16], :, j % 16] *= np.float16(1 + j / 64)
    c.kd = R._bf16(c.kd.astype(np.float32)).astype(np.float16)
    c.device(torch)
    row0, q, out = _prefill(ctx, torch, c, 8, [700])
    if scale:
        out = torch.empty_like(out)
        ctx.kv4_attention_prefill(torch.from_numpy(q).cuda(), c.cache, c.t, c.l, torch.from_numpy(row0).cuda(), out, scale=scale)
    got = out.cpu().numpy()
    for row in (0, 1, 63, 64, 127, 128, 255, 300, 511, 640, 699):
        _close(got[row], *c.expect(0, q[row], row, 0, 0, scale, floor=2.0 ** -32))


def test_prefill_many_short_requests_and_strided_q(ctx):
    import torch
    rng = np.random.default_rng(28)
    lens = rng.integers(0, 60, 500)
    new = np.minimum(lens, rng.integers(0, 4, 500)).tolist()
    c = Case(28, lens, 2, 32, 16).device(torch)
    row0 = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    fused = torch.randn(row0[-1] + 9, 6 * 32 + 64, device="cuda")
    q = fused[:, :6 * 32].unflatten(1, (6, 32))
    a, b = torch.full((len(q), 6, 32), 7.0, device="cuda"), torch.full((len(q), 6, 32), 7.0, device="cuda")
    ctx.kv4_attention_prefill(q, c.cache, c.t, c.l, torch.from_numpy(row0).cuda(), a)
    ctx.kv4_attention_prefill(q.contiguous(), c.cache, c.t, c.l, torch.from_numpy(row0).cuda(), b)
    assert torch.equal(a, b) and bool((a[row0[-1]:] == 7).all())
    got, qh = a.cpu().numpy(), q.cpu().numpy()
    for r in range(0, 500, 7):
        for t in range(new[r]):
            _close(got[row0[r] + t], *c.expect(r, qh[row0[r] + t], int(lens[r]) - new[r] + t, 0, 0, floor=2.0 ** -32))
