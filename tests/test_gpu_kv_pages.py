"""Page tables and slot maps built on the device against a plain loop over the
requests: whole numbers, equal."""
import numpy as np
import pytest

import serving_ref as R

pytestmark = pytest.mark.gpu


def _i32(torch, a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _state(rng, reqs, page, lens, new, spare=3, rows_extra=0):
    held = [-(-n // page) for n in lens]
    need = sum(-(-(n + m) // page) - h for n, m, h in zip(lens, new, held))
    width = max([-(-(n + m) // page) for n, m in zip(lens, new)] + [1]) + 1
    pages = sum(held) + need + spare
    ids = rng.permutation(pages).astype(np.int32)
    tables = np.full((reqs, width), -1, np.int32)
    at = 0
    for r, h in enumerate(held):
        tables[r, :h] = ids[at:at + h]
        at += h
    return tables, ids[at:], pages, sum(new) + rows_extra


def _run(ctx, torch, page, pages, lens, new, tables, free, rows, n_free=None, in_place=False):
    d = {"lens": _i32(torch, lens), "new": _i32(torch, new), "tables": _i32(torch, tables), "free": _i32(torch, free),
         "n_free": _i32(torch, [len(free) if n_free is None else n_free]), "row0": _i32(torch, [7] * (len(lens) + 1)),
         "slots": _i32(torch, [7] * rows), "pos": _i32(torch, [7] * rows), "status": _i32(torch, [7])}
    d["n_free_out"] = d["n_free"] if in_place else _i32(torch, [7])
    d["lens_out"] = d["lens"] if in_place else _i32(torch, [7] * len(lens))
    ctx.kv_pages_assign(d["lens"], d["new"], d["tables"], page, pages, d["free"], d["n_free"], d["n_free_out"], d["lens_out"],
                        d["row0"], d["slots"], d["pos"], d["status"])
    return {k: v.cpu().numpy() for k, v in d.items()}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("reqs,page,max_len,max_new,extra", [
    (1, 16, 0, 1, 0), (1, 16, 16, 1, 5), (1, 1024, 1023, 2, 0), (3, 16, 40, 17, 2), (33, 32, 100, 1, 0), (511, 16, 300, 3, 9),
    (513, 64, 700, 40, 1), (1500, 16, 90, 30, 3), (8192, 16, 33, 2, 0), (2, 128, 5, 60000, 11), (40, 16, 0, 0, 4),
    (512, 32, 500, 1, 20000), (513, 32, 500, 1, 20000)])
def test_assign_matches_the_plain_loop(ctx, reqs, page, max_len, max_new, extra, in_place):
    import torch
    rng = np.random.default_rng(reqs + page)
    lens = rng.integers(0, max_len + 1, reqs).tolist()
    new = (rng.integers(0, max_new + 1, reqs) if reqs > 1 else np.array([max_new])).tolist()
    tables, free, pages, rows = _state(rng, reqs, page, lens, new, rows_extra=extra)
    got = _run(ctx, torch, page, pages, lens, new, tables, free, rows, in_place=in_place)
    t, left, n, row0, slots, pos = R.pages_assign(lens, new, tables, page, free)
    assert got["status"][0] == 0 and got["n_free_out"][0] == len(left)
    assert np.array_equal(got["tables"], t)
    assert np.array_equal(got["lens_out"], n) and np.array_equal(got["row0"], row0)
    assert np.array_equal(got["slots"][:len(slots)], slots) and np.all(got["slots"][len(slots):] == -1)
    assert np.array_equal(got["pos"][:len(pos)], pos) and np.all(got["pos"][len(pos):] == -1)
    assert len(set(slots)) == len(slots)          # no slot twice


@pytest.mark.parametrize("what,status", [("short", 1), ("negative_len", 2), ("negative_new", 2), ("too_long", 2), ("rows", 3),
                                         ("free_count", 2)])
def test_a_step_that_does_not_fit_changes_nothing(ctx, what, status):
    import torch
    rng = np.random.default_rng(5)
    lens, new = [20, 5, 31, 0], [14, 2, 40, 16]
    tables, free, pages, rows = _state(rng, 4, 16, lens, new, spare=0)
    n_free = len(free)
    if what == "short":
        n_free -= 1
    elif what == "negative_len":
        lens[1] = -1
    elif what == "negative_new":
        new[2] = -5
    elif what == "free_count":
        n_free = len(free) + 1               # more than the list holds
    elif what == "too_long":
        new[3] = 2 ** 31 - 1
    else:
        rows -= 1
    got = _run(ctx, torch, 16, pages, lens, new, tables, free, rows, n_free=n_free)
    assert got["status"][0] == status and got["n_free_out"][0] == n_free
    assert np.array_equal(got["tables"], tables) and np.array_equal(got["lens_out"], lens)
    assert not got["row0"].any() and np.all(got["slots"] == -1) and np.all(got["pos"] == -1)


def test_no_requests_and_bad_page_ids(ctx):
    import torch
    got = _run(ctx, torch, 16, 4, [], [], np.zeros((0, 3), np.int32), [2, 1], 3)
    assert got["status"][0] == 0 and got["n_free_out"][0] == 2 and np.all(got["slots"] == -1) and got["row0"][0] == 0
    # a held table entry that names no page: its rows get slot -1, the positions stay
    tables = np.array([[9, -1, -1]], np.int32)
    got = _run(ctx, torch, 16, 4, [10], [8], tables, [3], 8)
    assert np.array_equal(got["slots"], [-1] * 6 + [3 * 16, 3 * 16 + 1]) and np.array_equal(got["pos"], range(10, 18))


def test_release_gives_the_pages_back(ctx):
    import torch
    rng = np.random.default_rng(9)
    reqs, page = 700, 32
    lens = rng.integers(0, 200, reqs).tolist()
    tables, free, pages, _ = _state(rng, reqs, page, lens, [0] * reqs)
    done = (rng.random(reqs) < 0.4).astype(np.int32)
    stack = np.full(pages, -7, np.int32)
    stack[:len(free)] = free
    d = [_i32(torch, x) for x in (done, lens, tables, stack, [len(free)], [9])]
    ctx.kv_pages_release(d[0], d[1], d[2], page, d[3], d[4], d[5])
    _, l, t, f, n, st = [x.cpu().numpy() for x in d]
    want, expect_t = list(free), tables.copy()
    for r in range(reqs):
        if done[r]:
            h = -(-lens[r] // page)
            want += tables[r, :h].tolist()
            expect_t[r, :h] = -1
    assert st[0] == 0 and n[0] == len(want) and np.array_equal(f[:len(want)], want)
    assert np.array_equal(t, expect_t) and np.array_equal(l, np.where(done, 0, lens))
    # a stack without room, or a length out of range: nothing changes
    for cap_off, bad in ((1, False), (0, True)):
        lens2 = list(lens)
        if bad:
            lens2[int(np.flatnonzero(done)[0])] = -4
        room = len(want) - cap_off if not bad else pages
        d = [_i32(torch, x) for x in (done, lens2, tables, stack[:room], [len(free)], [9])]
        ctx.kv_pages_release(d[0], d[1], d[2], page, d[3], d[4], d[5])
        assert d[5].item() == (2 if bad else 1) and d[4].item() == len(free)
        assert np.array_equal(d[1].cpu().numpy(), lens2) and np.array_equal(d[2].cpu().numpy(), tables)
        assert np.array_equal(d[3].cpu().numpy(), stack[:room])


def test_assign_and_release_many_steps_keep_every_page(ctx):
    """A server's life in one captured graph pair: pages never leak and never serve two requests."""
    import torch
    rng = np.random.default_rng(2)
    reqs, page, pages, width, rows = 24, 16, 400, 20, 400
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, new, done, tables = i(reqs), i(reqs), i(reqs), torch.full((reqs, width), -1, dtype=torch.int32, device="cuda")
    free, n_free = torch.arange(pages, dtype=torch.int32, device="cuda"), _i32(torch, [pages])
    row0, slots, pos, st, st2 = i(reqs + 1), i(rows), i(rows), i(1), i(1)
    stream, before = torch.cuda.Stream(), torch.cuda.current_stream().cuda_stream
    ctx.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                ctx.kv_pages_release(done, lens, tables, page, free, n_free, st2)
                ctx.kv_pages_assign(lens, new, tables, page, pages, free, n_free, n_free, lens, row0, slots, pos, st)
            for step in range(40):
                now = lens.cpu().numpy()
                d = (now > 150) | (rng.random(reqs) < 0.05)
                done.copy_(_i32(torch, d.astype(np.int32)))
                new.copy_(_i32(torch, np.where(d | (now == 0), rng.integers(0, 30, reqs), 1)))
                graph.replay()
                stream.synchronize()
                assert st.item() == 0 and st2.item() == 0
                t, n = tables.cpu().numpy(), lens.cpu().numpy()
                held = np.concatenate([t[r, :-(-n[r] // page)] for r in range(reqs)] + [free.cpu().numpy()[:n_free.item()]])
                assert np.array_equal(np.sort(held), np.arange(pages)), step
    finally:
        ctx.set_stream(before)
