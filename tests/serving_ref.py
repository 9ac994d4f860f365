"""Plain 64-bit models of the serving operators: page tables, the 4-bit KV
cache, attention over it and filtered sampling (numpy only)."""
import numpy as np


def pages_assign(lens, new, tables, page, free):
    """(tables, free left, lens, row0, slots, pos) after placing new[r] tokens of each request."""
    tables, free = tables.copy(), list(free)
    row0, slots, pos = [0], [], []
    for r, (n, m) in enumerate(zip(lens, new)):
        held = -(-n // page)
        for k in range(held, -(-(n + m) // page)):
            tables[r, k] = free.pop()
        for p in range(n, n + m):
            slots.append(int(tables[r, p // page]) * page + p % page)
            pos.append(p)
        row0.append(row0[-1] + m)
    return tables, free, [n + m for n, m in zip(lens, new)], row0, slots, pos


def _bf16(x):
    """x rounded to bfloat16's 8 significant bits, ties to even (finite x)."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    b = (b + 0x7FFF + ((b >> 16) & 1)) >> 16 << 16
    return b.astype(np.uint32).view(np.float32)


def quantize(x):
    """(nibbles uint8, scales float16) of float32 x [..., hd], groups of 32."""
    x = np.asarray(x, np.float32)
    g = x.reshape(-1, 32)
    a = np.abs(g)
    at = np.where(np.isnan(a), np.inf, a).argmax(1)
    top = g[np.arange(len(g)), at]
    nan = np.isnan(g).any(1)
    with np.errstate(all="ignore"):
        d = np.clip(_bf16(np.where(nan, 0, top) * np.float32(-0.125)).astype(np.float64), -8160, 8160).astype(np.float16)
        dd = d.astype(np.float64)[:, None]
        q = np.where(dd != 0, np.rint(g.astype(np.float64) / np.where(dd != 0, dd, 1)), 0)
    q = np.clip(q, -8, 7)
    d = np.where(nan, np.float16(np.nan), d)
    q = np.where(nan[:, None], 0, q) + 8
    return q.astype(np.uint8).reshape(x.shape), d.reshape(*x.shape[:-1], -1)


def values(q, d):
    """What nibbles and scales stand for, in float64."""
    return (q.astype(np.float64) - 8) * np.repeat(d.astype(np.float64), 32, -1)


def pack(kq, kd, vq, vd):
    """Cache bytes [pages, n_kv, page/16, 18 hd] of nibbles [pages, n_kv, page, hd] and scales."""
    pages, n_kv, page, hd = kq.shape
    parts = []
    for q in (kq, vq):
        g = q.reshape(pages, n_kv, page // 16, 16, hd // 32, 2, 16)
        parts.append((g[..., 0, :] | (g[..., 1, :] << 4)).reshape(pages, n_kv, page // 16, 8 * hd))
    for d in (kd, vd):
        parts.append(np.ascontiguousarray(d.reshape(pages, n_kv, page // 16, hd // 2)).view(np.uint8))
    return np.concatenate(parts, -1)


def seen(i, n, window, sinks):
    """Which of positions 0..n-1 the query at position i sees."""
    j = np.arange(n)
    ok = j <= i
    if window:
        ok &= (j > i - window) | (j < sinks)
    return ok


def attention(q, k, v, ok, scale, floor=2.0 ** -40):
    """q [heads, hd], k and v [n, n_kv, hd] float64 -> (out [heads, hd], bound on a float32 kernel's error).

    The bound: a score is a dot product of hd float32 products, so it is off by
    at most (hd + 8) 2^-24 sum |q k| scale (the 8: the two-part operands, the
    scaling and the exponent's argument); a softmax weight is then off by twice
    the largest such error relative, plus 2^-21 for exp; and the output's sum
    of n terms in float32 by n / 4 + 64 roundings (partial sums of at least
    four parallel accumulators, then their merge) of 2^-24 of sum p |v|, for
    the numerator and for the denominator.  A weight enters its product in two
    f16 parts after a scaling of the largest to 2^15 (decode) or to between 2^7
    and 2^15 (prefill, which follows the maximum lazily); f16 has no bit below
    2^-24, so besides its relative error each weight is off by up to half of
    that, `floor` = 2^-25 / 2^15 = 2^-40 (or 2^-25 / 2^7 = 2^-32) of the largest
    weight, times its |v|: what a dimension shows whose heavy positions all
    hold a zero."""
    heads, hd = q.shape
    rep = heads // k.shape[1]
    out, tol = np.zeros((heads, hd)), np.zeros((heads, hd))
    if not ok.any():
        return out, tol
    for h in range(heads):
        kk, vv = k[ok, h // rep], v[ok, h // rep]
        s = kk @ q[h] * scale
        ds = (hd + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[h])).max() * scale + 2.0 ** -22 * np.abs(s).max()
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ vv
        tol[h] = (p @ np.abs(vv)) * (2 * ds + 2.0 ** -21 + 2 * (len(s) / 4 + 64) * 2.0 ** -24) \
            + floor * p.max() * np.abs(vv).sum(0)
    return out, tol


def sample(x, u, t=1.0, k=0, p=1.0, min_p=0.0):
    """(index, distance of the nearest decision to its border relative to the mass)."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    n, m = len(x), x.max()
    if m == -np.inf:
        return -1, 1.0
    if not t > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(all="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / t))
    w = np.where(np.isnan(w), 0.0, w)
    order = np.argsort(-x, kind="stable")
    if k <= 0 or k > n:
        k = n
    order = order[:k]
    margin = 1.0
    if p <= 0:
        order = order[:1]
    elif p < 1:
        c = np.cumsum(w[order])
        goal = np.float64(np.float32(p)) * c[-1]
        cut = int(np.searchsorted(c, goal, side="left")) + 1
        margin = min(margin, np.abs(c - goal).min() / c[-1])
        order = order[:cut]
    order = order[w[order] >= min(np.float64(np.float32(min_p)), 1.0)] if min_p > 0 else order
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    target = min(max(np.float64(np.float32(u)), 0.0), 1.0) * c[-1]
    margin = min(margin, np.abs(c[:-1] - target).min() / c[-1]) if len(c) > 1 else margin
    at = min(int(np.searchsorted(c, target, side="right")), int(np.flatnonzero(w[kept] > 0)[-1]))
    return int(kept[at]), margin
