"""Release of requests whose tables hold entries that name no page (pages given
back early behind a window, or never there): they are taken out of the table
and do not go on to the free stack."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _i32(torch, a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("reqs,page,max_len,share", [(1, 16, 100, 0.5), (5, 64, 900, 0.3), (700, 32, 200, 0.05), (3, 16, 40000, 0.4),
                                                     (900, 16, 300, 1.0), (8192, 1024, 3000, 0.01)])
def test_entries_that_name_no_page_are_dropped(ctx, reqs, page, max_len, share):
    import torch
    rng = np.random.default_rng(reqs + page)
    lens = rng.integers(0, max_len + 1, reqs)
    held = -(-lens // page)
    pages = int(held.sum()) + 4
    width = int(held.max()) + 1
    ids = rng.permutation(pages).astype(np.int32)
    tables = np.full((reqs, width), -1, np.int32)
    tables[np.arange(width) < held[:, None]] = ids[:held.sum()]
    # -1, other negative numbers, and ids of which no cache of fewer than 2^31 slots has that many
    bad = (rng.random(tables.shape) < share) & (np.arange(width) < held[:, None])
    tables[bad] = rng.choice(np.array([-1, -1, -7, -2 ** 31, 2 ** 31 - 1, 2 ** 31 // page], np.int64), int(bad.sum())).astype(np.int32)
    done = (rng.random(reqs) < 0.7).astype(np.int32)
    done[0] = 1
    stack = np.full(pages, -7, np.int32)
    stack[:4] = ids[held.sum():]
    d = [_i32(torch, a) for a in (done, lens, tables, stack, [4], [9])]
    ctx.kv_pages_release(d[0], d[1], d[2], page, d[3], d[4], d[5])
    _, l, t, f, n, st = [a.cpu().numpy() for a in d]
    want, expect = list(stack[:4]), tables.copy()
    for r in np.flatnonzero(done):
        want += [i for i, b in zip(tables[r, :held[r]], bad[r]) if not b]
        expect[r, :held[r]] = -1
    assert st[0] == 0 and n[0] == len(want)
    assert np.array_equal(f[:len(want)], want) and np.all(f[len(want):] == -7)
    assert np.array_equal(t, expect) and np.array_equal(l, np.where(done, 0, lens))


def test_room_is_counted_in_pages(ctx):
    """Three held entries of which one names a page fit a stack with room for one, and not one without."""
    import torch
    for room, status in ((3, 0), (2, 1)):
        d = [_i32(torch, a) for a in ([1], [40], [[-1, 5, -1]], [8, 9, -7][:room], [2], [9])]
        ctx.kv_pages_release(d[0], d[1], d[2], 16, d[3], d[4], d[5])
        assert d[5].item() == status and d[4].item() == (3 if status == 0 else 2)
        assert d[3].tolist() == ([8, 9, 5] if status == 0 else [8, 9])
        assert d[2].tolist() == ([[-1, -1, -1]] if status == 0 else [[-1, 5, -1]]) and d[1].item() == (0 if status == 0 else 40)


def test_tokens_after_such_a_release_have_slots(ctx):
    """What the release gives back is dealt again: no request gets an entry that names no page."""
    import torch
    page, pages = 16, 6
    tables = _i32(torch, [[-1, 0, 1, -1], [2, 3, -1, -1]])
    lens, n_free, st = _i32(torch, [48, 20]), _i32(torch, [2]), _i32(torch, [9])
    free = _i32(torch, [4, 5, -7, -7, -7, -7])
    ctx.kv_pages_release(_i32(torch, [1, 0]), lens, tables, page, free, n_free, st)
    assert st.item() == 0 and n_free.item() == 4
    row0, slots, pos = _i32(torch, [0] * 3), _i32(torch, [0] * 64), _i32(torch, [0] * 64)
    ctx.kv_pages_assign(lens, _i32(torch, [50, 12]), tables, page, pages, free, n_free, n_free, lens, row0, slots, pos, st)
    assert st.item() == 0 and n_free.item() == 0
    got = slots.cpu().numpy()[:62]
    assert np.all(got >= 0) and len(set(got.tolist())) == 62
