"""The 4-bit cache where byte offsets pass 32 bits: a pool of 4.8 GB, its first
and its last pages in use."""
import numpy as np
import pytest

import hacedle_cuda as hc
import serving_ref as R

pytestmark = pytest.mark.gpu


def test_pages_beyond_four_gigabytes(ctx):
    import torch
    rng = np.random.default_rng(3)
    pages, page, n_kv, hd, heads = 130_000, 64, 4, 128, 8
    cache = torch.zeros(hc.kv4_cache_shape(pages, page, n_kv, hd), dtype=torch.uint8, device="cuda")
    assert cache.numel() > 1 << 32
    table = np.array([[pages - 1, 0, 116_508, pages - 2]], np.int32)      # page 116508 holds byte 2^32
    n = 4 * page - 5
    j = np.arange(n)
    slots = torch.from_numpy((table[0, j // page] * page + j % page).astype(np.int32)).cuda()
    k, v = (rng.standard_normal((n, n_kv, hd)).astype(np.float32) for _ in range(2))
    kd, vd = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    ctx.kv4_append(kd, vd, slots, cache)
    kv, vv = R.values(*R.quantize(k)), R.values(*R.quantize(v))
    ko, vo = torch.empty_like(kd), torch.empty_like(vd)
    ctx.kv4_read(cache, slots, ko, vo)
    assert np.array_equal(ko.cpu().numpy(), kv) and np.array_equal(vo.cpu().numpy(), vv)
    used = torch.zeros(pages, dtype=torch.bool, device="cuda")
    used[torch.from_numpy(table[0]).long().cuda()] = True
    # (counted in parts: nothing was written to any other page)
    for part in range(0, pages, 20_000):
        rest = cache[part:part + 20_000][~used[part:part + 20_000]]
        assert not rest.any().item()
    t, lens = torch.from_numpy(table).cuda(), torch.tensor([n], dtype=torch.int32, device="cuda")
    q = rng.standard_normal((20, heads, hd)).astype(np.float32)
    qd, out = torch.from_numpy(q).cuda(), torch.empty(20, heads, hd, device="cuda")
    ctx.kv4_attention_prefill(qd, cache, t, lens, torch.tensor([0, 20], dtype=torch.int32, device="cuda"), out)
    one = torch.empty(1, heads, hd, device="cuda")
    ctx.kv4_attention_decode(qd[-1:], cache, t, lens, one)
    for row, got in ((0, out[0]), (11, out[11]), (19, out[19]), (19, one[0])):
        i = n - 20 + row
        ref, tol = R.attention(q[row].astype(np.float64), kv[:i + 1], vv[:i + 1], np.ones(i + 1, bool), hd ** -0.5)
        assert np.all(np.abs(got.cpu().numpy() - ref) <= tol)
