"""The 4-bit KV cache: appended bytes and the values read back, equal to the
64-bit model's (both are exact: scales and nibbles are fixed by the rule, and a
value is one exact product)."""
import numpy as np
import pytest

import hacedle_cuda as hc
import serving_ref as R

pytestmark = pytest.mark.gpu


def _dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _expect(k, v, slots, cache, page):
    """The cache's bytes after the append."""
    pages, n_kv, tiles, width = cache.shape
    hd, out = width // 18, cache.copy()
    (kq, kd), (vq, vd) = R.quantize(k), R.quantize(v)
    for r, s in enumerate(slots):
        if not 0 <= s < pages * page:
            continue
        pg, tile, p = s // page, s % page // 16, s % 16
        for h in range(n_kv):
            t = out[pg, h, tile]
            for part, (q, d) in enumerate(((kq, kd), (vq, vd))):
                g = q[r, h].reshape(-1, 2, 16)
                t[8 * hd * part + p * hd // 2:][:hd // 2] = (g[:, 0] | g[:, 1] << 4).reshape(-1)
                t[16 * hd + hd * part + p * hd // 16:][:hd // 16] = np.ascontiguousarray(d[r, h]).view(np.uint8)
    return out


@pytest.mark.parametrize("rows,n_kv,hd,page", [(1, 1, 32, 16), (1, 2, 64, 16), (5, 3, 128, 32), (33, 2, 64, 1024),
                                               (100, 4, 128, 64), (257, 1, 32, 128)])
def test_append_and_read(ctx, rows, n_kv, hd, page):
    import torch
    rng = np.random.default_rng(rows + hd)
    pages = -(-rows // page) + 2
    k = (rng.standard_normal((rows, n_kv, hd)) * np.exp(rng.uniform(-6, 6, (rows, n_kv, 1)))).astype(np.float32)
    v = rng.standard_normal((rows, n_kv, hd)).astype(np.float32)
    slots = rng.permutation(pages * page)[:rows].astype(np.int32)
    if rows > 4:
        slots[1], slots[3] = -1, pages * page          # skipped
    before = rng.integers(0, 256, hc.kv4_cache_shape(pages, page, n_kv, hd), dtype=np.uint8)
    cache = _dev(torch, before)
    ctx.kv4_append(_dev(torch, k), _dev(torch, v), _dev(torch, slots), cache)
    want = _expect(k, v, slots, before, page)
    assert np.array_equal(cache.cpu().numpy(), want)   # and nothing else was written
    ko, vo = torch.full((rows, n_kv, hd), 7.0, device="cuda"), torch.full((rows, n_kv, hd), 7.0, device="cuda")
    ctx.kv4_read(cache, _dev(torch, slots), ko, vo)
    for x, o in ((k, ko), (v, vo)):
        ref = R.values(*R.quantize(x))
        ref[(slots < 0) | (slots >= pages * page)] = 0
        assert np.array_equal(o.cpu().numpy().astype(np.float64), ref)


def test_steps_at_a_border_ties_and_the_largest_value(ctx):
    """Values next to every rounding border, exact ties, groups of equal and of opposite extremes."""
    import torch
    rng = np.random.default_rng(3)
    rows, hd = 4096, 32
    k = np.empty((rows, 1, hd), np.float32)
    for r in range(rows):
        top = np.float32(rng.choice([-1, 1]) * np.exp(rng.uniform(-12, 9)))
        d = np.float64(R.quantize(np.full((1, 32), top, np.float32))[1][0, 0])
        b = (rng.integers(-9, 9, hd) + 0.5) * d                      # ties, exact in float32
        x = b.astype(np.float32)
        side = rng.integers(-1, 2, hd)
        x = np.where(side > 0, np.nextafter(x, np.float32(np.inf)), np.where(side < 0, np.nextafter(x, -np.float32(np.inf)), x))
        x[np.abs(x) > abs(top)] = 0
        x[rng.integers(0, hd)] = top
        if r % 3 == 0:
            x[rng.integers(0, hd)] = -top                            # the first of the two is the extreme
        k[r, 0] = x
    cache = torch.zeros(hc.kv4_cache_shape(rows // 16, 16, 1, hd), dtype=torch.uint8, device="cuda")
    slots = np.arange(rows, dtype=np.int32)
    ctx.kv4_append(_dev(torch, k), _dev(torch, k[::-1]), _dev(torch, slots), cache)
    want = _expect(k, k[::-1], slots, np.zeros(cache.shape, np.uint8), 16)
    assert np.array_equal(cache.cpu().numpy(), want)


def test_special_values(ctx):
    import torch
    inf, nan, tiny = np.inf, np.nan, np.float32(1e-40)
    rows = np.zeros((8, 1, 32), np.float32)
    rows[1, 0, 5] = nan
    rows[1, 0, 6] = inf
    rows[2, 0, :3] = [inf, -inf, 1e5]
    rows[3, 0, :3] = [-inf, 2.0, -7e4]
    rows[4, 0, :2] = [tiny, -tiny]
    rows[5, 0, :2] = [3e-7, -1e-7]               # a subnormal f16 scale
    rows[6, 0, :3] = [3e38, -3e38, 65000.0]
    rows[7, 0, :] = -0.0
    cache = torch.zeros(hc.kv4_cache_shape(1, 16, 1, 32), dtype=torch.uint8, device="cuda")
    slots = _dev(torch, np.arange(8, dtype=np.int32))
    ctx.kv4_append(_dev(torch, rows), _dev(torch, rows), slots, cache)
    k, v = torch.empty(8, 1, 32, device="cuda"), torch.empty(8, 1, 32, device="cuda")
    ctx.kv4_read(cache, slots, k, v)
    k = k.cpu().numpy()
    assert np.array_equal(k, v.cpu().numpy(), equal_nan=True)
    assert np.isnan(k[1]).all() and not np.isnan(np.delete(k, 1, 0)).any()
    assert k[2, 0, 0] == 65280 and k[2, 0, 1] == -57120 and k[2, 0, 2] == 65280 and not k[2, 0, 3:].any()
    assert k[3, 0, 0] == -65280 and k[3, 0, 1] == 0 and k[3, 0, 2] == -65280
    assert not k[0].any() and not k[4].any() and not k[7].any()
    assert np.array_equal(k[5].astype(np.float64), R.values(*R.quantize(rows[5])))
    assert k[6, 0, 0] == 65280 and k[6, 0, 1] == -57120


def test_strided_rows_and_no_rows(ctx):
    """k and v as slices of fused q|k|v rows."""
    import torch
    rng = np.random.default_rng(1)
    rows, n_kv, hd, page = 21, 2, 64, 16
    fused = _dev(torch, rng.standard_normal((rows, 4 * hd + 2 * n_kv * hd)).astype(np.float32))
    k = fused[:, 4 * hd:4 * hd + n_kv * hd].unflatten(1, (n_kv, hd))
    v = fused[:, 4 * hd + n_kv * hd:].unflatten(1, (n_kv, hd))
    cache = torch.zeros(hc.kv4_cache_shape(2, page, n_kv, hd), dtype=torch.uint8, device="cuda")
    slots = np.arange(rows, dtype=np.int32)
    ctx.kv4_append(k, v, _dev(torch, slots), cache)
    want = _expect(k.cpu().numpy(), v.cpu().numpy(), slots, np.zeros(cache.shape, np.uint8), page)
    assert np.array_equal(cache.cpu().numpy(), want)
    ctx.kv4_append(k[:0], v[:0], _dev(torch, slots[:0]), cache)
    assert np.array_equal(cache.cpu().numpy(), want)


def test_slots_beyond_32_bits_of_bytes(ctx):
    """The last slots of a cache of more than 2^32 bytes."""
    import torch
    n_kv, hd, page = 4, 128, 64
    pages = (1 << 32) // (n_kv * 4 * 18 * hd) + 3
    cache = torch.zeros(hc.kv4_cache_shape(pages, page, n_kv, hd), dtype=torch.uint8, device="cuda")
    assert cache.numel() > 1 << 32
    rng = np.random.default_rng(1)
    slots = np.array([pages * page - 1, 0, pages * page - 30], np.int32)
    k = rng.standard_normal((3, n_kv, hd)).astype(np.float32)
    ctx.kv4_append(_dev(torch, k), _dev(torch, k[::-1]), _dev(torch, slots), cache)
    ko, vo = torch.empty(3, n_kv, hd, device="cuda"), torch.empty(3, n_kv, hd, device="cuda")
    ctx.kv4_read(cache, _dev(torch, slots), ko, vo)
    assert np.array_equal(ko.cpu().numpy().astype(np.float64), R.values(*R.quantize(k)))
    assert np.array_equal(vo.cpu().numpy().astype(np.float64), R.values(*R.quantize(k[::-1])))
    assert int((cache[-1] != 0).sum()) > 0 and int(cache[1:-1].max()) == 0
