"""The serving operators together, as a server uses them: requests come and go,
each step places their tokens, stores keys and values in the 4-bit cache,
attends over it and draws the next token.  Every step's attention is held to
the 64-bit model over the values that the model's own quantizer keeps."""
import numpy as np
import pytest

import hacedle_cuda as hc
import serving_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,window,sinks", [(16, 0, 0), (32, 24, 3)])
def test_serving_steps(ctx, page, window, sinks):
    import torch
    rng = np.random.default_rng(page)
    reqs, heads, n_kv, hd, vocab, pages, width, max_rows = 5, 6, 2, 64, 500, 40, 12, 160
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    cache = torch.full(hc.kv4_cache_shape(pages, page, n_kv, hd), 255, dtype=torch.uint8, device="cuda")   # NaN scales
    tables, free, n_free = torch.full((reqs, width), -1, dtype=torch.int32, device="cuda"), up(rng.permutation(pages).astype(np.int32)), i32(1) + pages
    lens, row0, slots, pos, st = i32(reqs), i32(reqs + 1), i32(max_rows), i32(max_rows), i32(1)
    head = rng.standard_normal((heads * hd, vocab)).astype(np.float32)
    head_dev = up(head)
    model = [(np.zeros((0, n_kv, hd)), np.zeros((0, n_kv, hd))) for _ in range(reqs)]
    checked = drawn = 0
    for step in range(14):
        done = np.zeros(reqs, np.int32)
        if step in (5, 9):
            done[[step % reqs, 2]] = 1
            ctx.kv_pages_release(up(done), lens, tables, page, free, n_free, st)
            assert st.item() == 0
            for r in np.flatnonzero(done):
                model[r] = (np.zeros((0, n_kv, hd)), np.zeros((0, n_kv, hd)))
        new = np.array([int(rng.integers(1, 30)) if len(m[0]) == 0 else 1 for m in model], np.int32)
        ctx.kv_pages_assign(lens, up(new), tables, page, pages, free, n_free, n_free, lens, row0, slots, pos, st)
        assert st.item() == 0
        total = int(new.sum())
        x = (rng.standard_normal((max_rows, (heads + 2 * n_kv) * hd)) * 1.5).astype(np.float32)   # fused q|k|v, padded
        qkv = up(x)
        q = qkv[:, :heads * hd].unflatten(1, (heads, hd))
        k = qkv[:, heads * hd:(heads + n_kv) * hd].unflatten(1, (n_kv, hd))
        v = qkv[:, (heads + n_kv) * hd:].unflatten(1, (n_kv, hd))
        ctx.kv4_append(k, v, slots, cache)               # rows behind the last have slot -1
        out = torch.full((max_rows, heads, hd), 7.0, device="cuda")
        if (new == 1).all():
            ctx.kv4_attention_decode(q[:reqs], cache, tables, lens, out[:reqs], window=window, sinks=sinks)
        else:
            ctx.kv4_attention_prefill(q, cache, tables, lens, row0, out, window=window, sinks=sinks)
        got, at = out.cpu().numpy(), 0
        assert np.all(got[total:] == 7.0)
        for r in range(reqs):
            kk, vv = (R.values(*R.quantize(a.reshape(-1, n_kv, hd))) for a in
                      (x[at:at + new[r], heads * hd:(heads + n_kv) * hd], x[at:at + new[r], (heads + n_kv) * hd:]))
            model[r] = (np.concatenate([model[r][0], kk]), np.concatenate([model[r][1], vv]))
            for t in range(new[r]):
                i = len(model[r][0]) - new[r] + t
                ref, tol = R.attention(x[at + t, :heads * hd].reshape(heads, hd).astype(np.float64), model[r][0][:i + 1],
                                       model[r][1][:i + 1], R.seen(i, i + 1, window, sinks), hd ** -0.5, 2.0 ** -32)
                assert np.all(np.abs(got[at + t] - ref) <= tol), (step, r, t)
                checked += 1
            at += new[r]
        last = out[(row0[1:] - 1).long()].reshape(reqs, -1)
        logits = last @ head_dev
        u = rng.random(reqs).astype(np.float32)
        idx = i32(reqs)
        ctx.sample_filtered(logits, up(u), idx, top_k=i32(reqs) + 40, top_p=torch.full((reqs,), 0.9, device="cuda"))
        for r, (row, got_idx) in enumerate(zip(logits.cpu().numpy(), idx.tolist())):
            want, margin = R.sample(row, u[r], k=40, p=0.9)
            if margin > 1e-9:
                assert got_idx == want
                drawn += 1
    assert checked > 100 and drawn >= 14 * reqs - 2
    held = sum(-(-len(m[0]) // page) for m in model)
    assert n_free.item() == pages - held


def test_a_captured_step_follows_the_state(ctx):
    """One graph holds a whole step; replayed, it does what the calls do one by one, also once the pages run out."""
    import torch
    rng = np.random.default_rng(77)
    reqs, heads, n_kv, hd, page, pages, width, steps = 4, 8, 2, 64, 16, 9, 4, 24
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    free = up(rng.permutation(pages).astype(np.int32))
    one = torch.ones(reqs, dtype=torch.int32, device="cuda")

    def state():
        return {"cache": torch.zeros(hc.kv4_cache_shape(pages, page, n_kv, hd), dtype=torch.uint8, device="cuda"),
                "tables": i32(reqs, width) - 1, "n_free": i32(1) + pages, "lens": i32(reqs),
                "row0": i32(reqs + 1), "slots": i32(6), "pos": i32(6), "st": i32(1), "idx": i32(reqs),
                "out": torch.zeros(reqs, heads, hd, device="cuda")}

    qkv, u = torch.zeros(6, (heads + 2 * n_kv) * hd, device="cuda"), torch.zeros(reqs, device="cuda")
    ws = [torch.zeros(ctx.kv4_workspace_bytes(heads, n_kv, hd), dtype=torch.uint8, device="cuda") for _ in range(2)]
    top_p = torch.full((reqs,), 0.8, device="cuda")

    def step(s, w):
        k = qkv[:, heads * hd:(heads + n_kv) * hd].unflatten(1, (n_kv, hd))
        v = qkv[:, (heads + n_kv) * hd:].unflatten(1, (n_kv, hd))
        ctx.kv_pages_assign(s["lens"], one, s["tables"], page, pages, free, s["n_free"], s["n_free"], s["lens"], s["row0"],
                            s["slots"], s["pos"], s["st"])
        ctx.kv4_append(k, v, s["slots"], s["cache"])
        ctx.kv4_attention_decode(qkv[:reqs, :heads * hd].unflatten(1, (heads, hd)), s["cache"], s["tables"], s["lens"], s["out"],
                                 window=20, sinks=2, ws=w)
        ctx.sample_filtered(s["out"].view(reqs, -1), u, s["idx"], top_p=top_p)

    eager, graphed = state(), state()
    before, stream, g = torch.cuda.current_stream().cuda_stream, torch.cuda.Stream(), torch.cuda.CUDAGraph()
    step(state(), ws[0])                          # (shared memory limits are set outside the capture)
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(g, stream=stream):
            step(graphed, ws[1])
    finally:
        ctx.set_stream(before)
    codes = []
    for _ in range(steps * 2):
        qkv.copy_(torch.from_numpy(rng.standard_normal(tuple(qkv.shape)).astype(np.float32)))
        u.copy_(torch.from_numpy(rng.random(reqs).astype(np.float32)))
        step(eager, ws[0])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for n in eager:
            assert torch.equal(eager[n], graphed[n]), n
        codes.append(eager["st"].item())
    # 9 pages hold two for each of four requests and one more: the 33rd token does not fit
    assert codes == [0] * 32 + [1] * (steps * 2 - 32)
