"""Layers of the library's own kernels around the paged 4-bit cache: embedding,
RMSNorm, quantized GEMVs, RoPE at the positions that the page assignment gives,
append, attention, SwiGLU, LM head and the draw whose index is the next step's
input.  Each stage is held to the oracle or the 64-bit model on the inputs that
the stage before left (4-bit rounding is not continuous, so errors may not pile
up), with the cache's contents from the model's own quantizer."""
import numpy as np
import pytest

import hacedle_cuda as hc
import serving_ref as R
from hacedle_cuda import synth as S
from oracle import oracle as O

pytestmark = pytest.mark.gpu

H, F, HEADS, N_KV, HD, VOCAB, LAYERS, EPS = 256, 512, 4, 2, 64, 320, 2, 1e-6


def _rel(a, b):
    return float(np.abs(a - b).max() / np.abs(b).max())


def test_a_model_on_the_paged_cache(ctx):
    import torch
    rng = np.random.default_rng(5)
    page, pages, width, reqs, max_rows = 16, 12, 4, 3, 16
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    host = lambda t: t.cpu().numpy()  # noqa: E731
    raws, weights = {}, {}

    def weight(name, kind, rows, cols, seed):
        raws[name] = (kind, S.gen_weight(kind, rows, cols, seed), rows, cols)
        weights[name] = ctx.weight(kind, raws[name][1], rows, cols)

    for i in range(LAYERS):
        for j, (n, kind, rows, cols) in enumerate((("q", S.GGML_Q5_0, HEADS * HD, H), ("k", S.GGML_Q8_0, N_KV * HD, H),
                                                   ("v", S.GGML_Q8_0, N_KV * HD, H), ("o", S.GGML_Q5_0, H, HEADS * HD),
                                                   ("gate", S.GGML_Q4_K, F, H), ("up", S.GGML_Q4_K, F, H), ("down", S.GGML_Q6_K, H, F))):
            weight((i, n), kind, rows, cols, 10 * i + j)
    weight("embed", S.GGML_Q8_0, VOCAB, H, 90)
    weight("head", S.GGML_Q8_0, VOCAB, H, 91)
    norm = rng.uniform(0.5, 1.5, H).astype(np.float32)
    norm_dev = up(norm)

    def gemv(name, x, residual=None):
        """The device's product of the device's x, held to the oracle's."""
        kind, raw, rows, cols = raws[name]
        y = torch.empty(len(x), rows, device="cuda")
        ctx.qgemv(weights[name], x, y, residual=residual)
        ref = O.qgemv(kind, raw, rows, cols, host(x)).reshape(len(x), rows) + (0 if residual is None else host(residual))
        assert _rel(host(y), ref) <= 1e-5, name
        return y

    def normed(x):
        y = torch.empty_like(x)
        ctx.rmsnorm(x, norm_dev, y, EPS)
        assert _rel(host(y), O.rmsnorm(host(x), norm, EPS)) <= 1e-5
        return y

    caches = [torch.full(hc.kv4_cache_shape(pages, page, N_KV, HD), 255, dtype=torch.uint8, device="cuda") for _ in range(LAYERS)]
    tables, free, n_free = i32(reqs, width) - 1, up(rng.permutation(pages).astype(np.int32)), i32(1) + pages
    lens, row0, slots, pos, st = i32(reqs), i32(reqs + 1), i32(max_rows), i32(max_rows), i32(1)
    kept = [[(np.zeros((0, N_KV, HD)), np.zeros((0, N_KV, HD))) for _ in range(reqs)] for _ in range(LAYERS)]
    tokens = [rng.integers(0, VOCAB, n).tolist() for n in (9, 4, 1)]      # the prompts, then the draws
    drawn = 0
    for step in range(20):
        new = np.array([len(t) for t in tokens], np.int32)
        total = int(new.sum())
        ctx.kv_pages_assign(lens, up(new), tables, page, pages, free, n_free, n_free, lens, row0, slots, pos, st)
        assert st.item() == 0
        at, n_cached = host(row0), host(lens)
        x = torch.empty(total, H, device="cuda")
        ctx.embed(weights["embed"], up(np.concatenate(tokens).astype(np.int32)), x)
        for i in range(LAYERS):
            xn = normed(x)
            q, k, v = (gemv((i, n), xn) for n in "qkv")
            p = host(pos)[:total]
            assert np.array_equal(p, np.concatenate([np.arange(n_cached[r] - new[r], n_cached[r]) for r in range(reqs)]))
            for t, heads in ((q, HEADS), (k, N_KV)):
                ref = np.stack([O.rope_neox(a, np.array([b]), HD).reshape(-1) for a, b in zip(host(t), p)])
                ctx.rope_neox(t, pos[:total], heads, HD)
                assert _rel(host(t), ref) <= 1e-5
            ctx.kv4_append(k.view(total, N_KV, HD), v.view(total, N_KV, HD), slots[:total], caches[i])
            out = torch.empty(total, HEADS, HD, device="cuda")
            if total == reqs:
                ctx.kv4_attention_decode(q.view(total, HEADS, HD), caches[i], tables, lens, out)
            else:
                ctx.kv4_attention_prefill(q.view(total, HEADS, HD), caches[i], tables, lens, row0, out)
            got, qh = host(out), host(q).reshape(total, HEADS, HD).astype(np.float64)
            for r in range(reqs):
                kk, vv = (R.values(*R.quantize(host(a)[at[r]:at[r + 1]].reshape(-1, N_KV, HD))) for a in (k, v))
                kept[i][r] = (np.concatenate([kept[i][r][0], kk]), np.concatenate([kept[i][r][1], vv]))
                for t in range(new[r]):
                    n = n_cached[r] - new[r] + t + 1
                    ref, tol = R.attention(qh[at[r] + t], kept[i][r][0][:n], kept[i][r][1][:n], np.ones(n, bool), HD ** -0.5)
                    assert np.all(np.abs(got[at[r] + t] - ref) <= tol), (step, i, r, t)
            x = gemv((i, "o"), out.view(total, -1), residual=x)
            xn = normed(x)
            g, u, a = gemv((i, "gate"), xn), gemv((i, "up"), xn), torch.empty(total, F, device="cuda")
            ctx.swiglu(g, u, a)
            assert _rel(host(a), O.swiglu(host(g), host(u))) <= 1e-5
            x = gemv((i, "down"), a, residual=x)
        logits = gemv("head", normed(x[(row0[1:] - 1).long()]))
        r01, idx = rng.random(reqs).astype(np.float32), i32(reqs)
        ctx.sample_filtered(logits, up(r01), idx, temperature=torch.full((reqs,), 0.8, device="cuda"), top_k=i32(reqs) + 30,
                            top_p=torch.full((reqs,), 0.9, device="cuda"))
        for r, row in enumerate(host(logits)):
            want, margin = R.sample(row, r01[r], t=np.float64(np.float32(0.8)), k=30, p=0.9)
            if margin > 1e-9:
                assert idx[r].item() == want
                drawn += 1
        tokens = [[int(t)] for t in idx.tolist()]
    assert drawn >= 20 * reqs - 2
    assert host(lens).tolist() == [9 + 19, 4 + 19, 1 + 19] and n_free.item() == pages - 6


@pytest.mark.parametrize("hd,rows", [(32, 16), (64, 16), (128, 16), (32, 64), (64, 64)])
def test_products_right_behind_a_prefill(ctx, hd, rows):
    """The output projection is launched while the prefill still runs, and both use tensor memory."""
    import torch
    rng = np.random.default_rng(hd + rows)
    heads, n_kv, n, page = 14, 2, 700, 16
    pages = -(-n // page)
    cache = torch.zeros(hc.kv4_cache_shape(pages, page, n_kv, hd), dtype=torch.uint8, device="cuda")
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    k, v = (up(rng.standard_normal((n, n_kv, hd)).astype(np.float32)) for _ in range(2))
    ctx.kv4_append(k, v, torch.arange(n, dtype=torch.int32, device="cuda"), cache)
    table, lens = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous(), torch.tensor([n], dtype=torch.int32, device="cuda")
    row0 = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    cols, kind, out_rows = heads * hd, S.GGML_Q8_0, 896
    raw = S.gen_weight(kind, out_rows, cols, 7)
    w = ctx.weight(kind, raw, out_rows, cols)
    q = up(rng.standard_normal((rows, heads, hd)).astype(np.float32))
    y, outs = torch.empty(rows, out_rows, device="cuda"), []
    x = torch.zeros(rows, cols, device="cuda")
    for _ in range(30):
        ctx.kv4_attention_prefill(q, cache, table, lens, row0, x.view(rows, heads, hd))
        (ctx.qgemv if rows <= 16 else ctx.qgemm)(w, x, y)
        outs.append(y.clone())
    ctx.check_device_errors()
    ref = O.qgemv(kind, raw, out_rows, cols, x.cpu().numpy()).reshape(rows, out_rows)
    for got in outs:
        assert _rel(got.cpu().numpy(), ref) <= 1e-5
