"""The serving operators: page tables, the 4-bit KV cache, attention over it, and filtered sampling.

Each case is one operator at one size.  With `own` false, run() computes it in
elementary torch operations; with `own` true it makes the calls a user makes of
hacedle_cuda.  Both take what prepare() gives.

A 4-bit cache is bytes [pages][n_kv][page / 16] of tiles of 18 * head_dim
bytes, each 16 positions of one kv head: K quants [16][head_dim / 2], V quants
[16][head_dim / 2], K scales f16 [16][head_dim / 32], V scales the same.  Byte
j of a group of 32 values holds value j in its low and value j + 16 in its
high nibble; a value is (nibble - 8) * scale.
"""
import math
import os
import sys

import torch

own = False

VOCAB = 151936


def listed():
    return [
        # every step of a server that decodes 256 requests: one new token each, pages of 16
        {"name": "pages_decode_256", "op": "pages", "reqs": 256, "prefills": 0, "chunk": 1, "max_len": 4096, "page": 16},
        # a mixed step: 1024 requests, 96 of them bring a prompt chunk of up to 1024 tokens
        {"name": "pages_mixed_1024", "op": "pages", "reqs": 1024, "prefills": 96, "chunk": 1024, "max_len": 16384, "page": 64},
        # one layer's new keys and values of a 64-request decode step, the 0.5B shape
        {"name": "append_decode_64", "op": "append", "rows": 64, "n_kv": 2, "hd": 64, "page": 16},
        # one layer's keys and values of a 16383-token prefill, the 7B shape
        {"name": "append_prefill_16k", "op": "append", "rows": 16383, "n_kv": 4, "hd": 128, "page": 64},
        # a single chat in its first turns: the latency of one decode step's attention
        {"name": "decode_1x700", "op": "decode", "seqs": 1, "min_len": 700, "max_len": 700, "heads": 14, "n_kv": 2, "hd": 64,
         "page": 16, "window": 0, "sinks": 0},
        # a full batch of requests of very different ages, the 7B shape
        {"name": "decode_256_ragged", "op": "decode", "seqs": 256, "min_len": 64, "max_len": 4096, "heads": 28, "n_kv": 4,
         "hd": 128, "page": 64, "window": 0, "sinks": 0},
        # one request with a long document in its cache
        {"name": "decode_1x131k", "op": "decode", "seqs": 1, "min_len": 131001, "max_len": 131001, "heads": 28, "n_kv": 4,
         "hd": 128, "page": 64, "window": 0, "sinks": 0},
        # long streams that see their last 2048 tokens and 4 first ones
        {"name": "decode_32_window", "op": "decode", "seqs": 32, "min_len": 1000, "max_len": 30000, "heads": 14, "n_kv": 2,
         "hd": 64, "page": 32, "window": 2048, "sinks": 4},
        # prompt chunks of 12 requests, some of them with a cached prefix
        {"name": "prefill_12_ragged", "op": "prefill", "seqs": 12, "min_new": 1, "max_new": 500, "min_len": 3, "max_len": 2000,
         "heads": 14, "n_kv": 2, "hd": 64, "page": 16, "window": 0, "sinks": 0},
        # the second half of an 8192-token prompt, the 7B shape
        {"name": "prefill_1x4096", "op": "prefill", "seqs": 1, "min_new": 4096, "max_new": 4096, "min_len": 4096, "max_len": 4096,
         "heads": 28, "n_kv": 4, "hd": 128, "page": 64, "window": 0, "sinks": 0},
        # one chat's next token with every filter on
        {"name": "sample_1", "op": "sample", "rows": 1, "n": VOCAB, "spread": 3.0, "k": 50, "p": 0.9, "min_p": 0.02, "t": 0.7},
        # 256 requests' next tokens; each row has its own settings, some none
        {"name": "sample_256", "op": "sample", "rows": 256, "n": VOCAB, "spread": 2.5, "k": 0, "p": 0.95, "min_p": 0.0, "t": 1.0},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["pages", "append", "decode", "decode", "prefill", "sample"])
    if op == "pages":
        reqs = _log(rng, 1, 2000)
        return {"op": op, "reqs": reqs, "prefills": rng.randint(0, min(reqs, 60)), "chunk": _log(rng, 1, 1000),
                "max_len": _log(rng, 20, 16000), "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        hd = rng.choice([32, 64, 128])
        return {"op": op, "rows": _log(rng, 1, 12000), "n_kv": rng.randint(1, 4), "hd": hd, "page": rng.choice([16, 32, 64, 128])}
    n_kv = rng.randint(1, 4)
    heads, hd = n_kv * rng.choice([1, 2, 3, 4, 7, 8, 12, 16]), rng.choice([32, 64, 128])
    window = rng.choice([0, 0, _log(rng, 1, 3000)])
    tail = {"heads": heads, "n_kv": n_kv, "hd": hd, "page": rng.choice([16, 32, 64, 128]), "window": window,
            "sinks": rng.choice([0, 1, 4, 64]) if window else 0}
    if op == "decode":
        seqs = _log(rng, 1, 200)
        top = min(100000, 150000 // seqs)
        return {"op": op, "seqs": seqs, "min_len": _log(rng, 1, 100), "max_len": _log(rng, 101, top), **tail}
    if op == "prefill":
        seqs = _log(rng, 1, 30)
        most = min(3500, 98000 // heads) // seqs + 2
        return {"op": op, "seqs": seqs, "min_new": 1, "max_new": _log(rng, 2, most), "min_len": 0,
                "max_len": _log(rng, 2, 4000 // seqs + 2), **tail}
    return {"op": op, "rows": _log(rng, 1, 200), "n": _log(rng, 50, VOCAB), "spread": rng.choice([1.0, 2.0, 4.0]),
            "k": rng.choice([0, 1, _log(rng, 2, 2000)]), "p": rng.choice([1.0, 0.5, 0.8, 0.95]),
            "min_p": rng.choice([0.0, 0.0, 0.01, 0.1]), "t": rng.choice([0.6, 1.0, 1.5])}


# ------------------------------------------------------------------ inputs
def _ceil(a, b):
    return -(-a // b)


def _spread(n, low, high):
    """n whole numbers spread from low to high evenly in their logarithm; the same ones for every seed."""
    if n == 1:
        return [high]
    a, b = math.log(low + 1), math.log(high + 1)
    return [int(round(math.exp(a + (b - a) * i / (n - 1)))) - 1 for i in range(n)]


def _lengths(case):
    """(tokens cached before, new tokens) of each request, before their order is shuffled."""
    if case["op"] == "pages":
        chunks = _spread(case["prefills"], 1, case["chunk"]) if case["prefills"] else []
        return _spread(case["reqs"], 1, case["max_len"]), chunks + [1] * (case["reqs"] - case["prefills"])
    if case["op"] == "decode":
        return [n - 1 for n in _spread(case["seqs"], case["min_len"], case["max_len"])], [1] * case["seqs"]
    return _spread(case["seqs"], case["min_len"], case["max_len"]), _spread(case["seqs"], case["min_new"], case["max_new"])


def _visible(case):
    """(pairs a query sees, cached positions that any query sees), summed over the requests."""
    pairs = seen = 0
    w, s = case["window"], case["sinks"]
    for old, new in zip(*_lengths(case)):
        n = old + new
        if not w:
            pairs += new * old + new * (new + 1) // 2
            seen += n
            continue
        pairs += sum(min(i + 1, w + min(s, max(0, i + 1 - w))) for i in range(old, n))
        first = max(0, old - w + 1)
        seen += n - first + min(s, first)
    return pairs, seen


def _keys_values(g, shape):
    """Keys with a few channels much larger than the others, as trained models have them, and plain values."""
    k = torch.randn(shape, generator=g, device="cuda")
    k[..., ::21] *= 6.0
    return k, torch.randn(shape, generator=g, device="cuda")


def _quantize(x):
    """(nibbles as they are held, scales) of x [..., head_dim]."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    at = x.abs().argmax(-1, keepdim=True)
    d = (x.gather(-1, at) * -0.125).to(torch.bfloat16).float().clamp(-8160.0, 8160.0).half()
    dd = d.double()
    q = torch.where(dd != 0, torch.round(x.double() / dd), torch.zeros((), dtype=torch.float64, device=x.device))
    return (q.clamp(-8, 7) + 8).to(torch.uint8), d


def _encode(k, v):
    """Cache bytes [pages][n_kv][page / 16][18 * head_dim] of k, v [pages][n_kv][page][head_dim]."""
    pages, n_kv, page, hd = k.shape
    out = torch.empty(pages, n_kv, page // 16, 18 * hd, dtype=torch.uint8, device=k.device)
    (kq, kd), (vq, vd) = _quantize(k), _quantize(v)
    out[..., :8 * hd] = (kq[..., :16] | (kq[..., 16:] << 4)).reshape(pages, n_kv, page // 16, 8 * hd)
    out[..., 8 * hd:16 * hd] = (vq[..., :16] | (vq[..., 16:] << 4)).reshape(pages, n_kv, page // 16, 8 * hd)
    out[..., 16 * hd:17 * hd] = kd.reshape(pages, n_kv, page // 16, hd // 2).view(torch.uint8)
    out[..., 17 * hd:] = vd.reshape(pages, n_kv, page // 16, hd // 2).view(torch.uint8)
    return out


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "sample":
        rows, n = case["rows"], case["n"]
        s["logits"] = torch.randn(rows, n, generator=g, device="cuda") * case["spread"]
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        # a row's request may ask for less than the case does: every fourth asks for another temperature, every fifth for no top-p
        i = torch.arange(rows, device="cuda")
        s["t"] = torch.where(i % 4 == 3, 0.8, case["t"]).float()
        s["p"] = torch.where(i % 5 == 4, 1.0, case["p"]).float()
        s["k"] = torch.where(i % 8 == 7, 40, case["k"]).int()
        s["min_p"] = torch.full((rows,), case["min_p"], device="cuda")
        s["idx"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        return s
    if op == "append":
        rows, n_kv, hd, page = case["rows"], case["n_kv"], case["hd"], case["page"]
        pages = _ceil(rows, page) + 3
        s["k"], s["v"] = _keys_values(g, (rows, n_kv, hd))
        s["slots"] = torch.randperm(pages * page, generator=cpu)[:rows].int().cuda()
        s["cache"] = torch.zeros(pages, n_kv, page // 16, 18 * hd, dtype=torch.uint8, device="cuda")
        s["k_out"], s["v_out"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    old, new = _lengths(case)
    old = [old[i] for i in torch.randperm(len(old), generator=cpu).tolist()]
    new = [new[i] for i in torch.randperm(len(new), generator=cpu).tolist()]
    page, reqs, rows = case["page"], len(old), sum(new)
    have = [_ceil(o, page) for o in old]
    need = [_ceil(o + n, page) for o, n in zip(old, new)]
    pages = sum(need) + 7
    ids = torch.randperm(pages, generator=cpu).int()
    width = _ceil(max(old) + max(new), page) + 2
    filled = have if op == "pages" else need
    tables = torch.full((reqs, width), -1, dtype=torch.int32)
    tables[torch.arange(width)[None] < torch.tensor(filled)[:, None]] = ids[:sum(filled)]
    s["tables"], s["most_pages"], s["rows"], s["pages"] = tables.cuda(), max(need), rows, pages
    if op == "pages":
        s["lens"], s["new"] = _ints(old), _ints(new)
        s["free"] = ids[sum(have):].cuda()
        s["n_free"] = _ints([pages - sum(have)])
        s["out"] = {"n_free": _ints([0]), "lens": _ints(old), "row0": _ints([0] * (reqs + 1)), "status": _ints([0]),
                    "slots": torch.zeros(rows, dtype=torch.int32, device="cuda"),
                    "pos": torch.zeros(rows, dtype=torch.int32, device="cuda")}
        return s
    n_kv, hd = case["n_kv"], case["hd"]
    s["cache"] = _encode(*_keys_values(g, (pages, n_kv, page, hd)))
    s["lens"] = _ints([o + n for o, n in zip(old, new)])
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["row0"], s["max_new"] = _ints(starts), max(new)
    s["q"] = torch.randn(rows, case["heads"], hd, generator=g, device="cuda") * 1.5
    s["out"] = torch.zeros_like(s["q"])
    return s


# ------------------------------------------------------------------ plain forms
def _decode_bytes(tiles, hd):
    """K and V f32 [..., 16, head_dim] of cache tiles [..., 18 * head_dim]."""
    lead = tiles.shape[:-1]

    def values(quants, scales):
        b = quants.reshape(*lead, 16, hd // 32, 16)
        q = torch.cat((b & 15, b >> 4), -1).float() - 8.0
        return (q * scales.contiguous().view(torch.float16).reshape(*lead, 16, hd // 32, 1).float()).reshape(*lead, 16, hd)

    return (values(tiles[..., :8 * hd], tiles[..., 16 * hd:17 * hd]), values(tiles[..., 8 * hd:16 * hd], tiles[..., 17 * hd:]))


def _gathered(s):
    """K and V f32 [request][n_kv][position][head_dim] through the page tables."""
    c = s["case"]
    tiles = s["cache"][s["tables"][:, :s["most_pages"]].clamp(min=0).long()]
    k, v = _decode_bytes(tiles.transpose(1, 2), c["hd"])
    shape = (tiles.shape[0], c["n_kv"], s["most_pages"] * c["page"], c["hd"])
    return k.reshape(shape), v.reshape(shape)


def _seen(case, at, positions):
    """Which cached positions the queries at positions `at` see."""
    i, j = at[..., None], positions
    ok = j <= i
    if case["window"]:
        ok = ok & ((j > i - case["window"]) | (j < case["sinks"]))
    return ok


def _attention(s, kind):
    c = s["case"]
    heads, n_kv, hd = c["heads"], c["n_kv"], c["hd"]
    reqs, most = s["lens"].numel(), s["max_new"]
    k, v = (x.to(kind) for x in _gathered(s))
    n_new = s["row0"][1:] - s["row0"][:-1]
    t = torch.arange(most, device="cuda")
    rows = s["row0"][:-1, None] + t                     # the row of each request's t-th new token
    real = t < n_new[:, None]
    q = s["q"].to(kind)[torch.where(real, rows, 0).long()]  # [request][t][heads][hd]
    q = q.reshape(reqs, most, n_kv, heads // n_kv, hd).permute(0, 2, 3, 1, 4).reshape(reqs, n_kv, -1, hd)
    x = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(hd)
    at = (s["lens"] - n_new)[:, None] + t
    ok = _seen(c, at, torch.arange(k.shape[2], device="cuda"))
    x = x.reshape(reqs, n_kv, heads // n_kv, most, -1).masked_fill(~ok[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul((x / x.sum(-1, keepdim=True)).reshape(reqs, n_kv, (heads // n_kv) * most, -1), v)
    o = o.reshape(reqs, n_kv, heads // n_kv, most, hd).permute(0, 3, 1, 2, 4).reshape(reqs, most, heads, hd)
    return o[real].float() if kind == torch.float32 else o[real]


def _plain_pages(s):
    c, page = s["case"], s["case"]["page"]
    lens, new = s["lens"].long(), s["new"].long()
    row0 = torch.cat((new.new_zeros(1), new.cumsum(0)))
    have, need = (lens + page - 1) // page, (lens + new + page - 1) // page
    page0 = (need - have).cumsum(0) - (need - have)
    taken = (need - have).sum()
    col = torch.arange(s["tables"].shape[1], device="cuda")
    fresh = (col >= have[:, None]) & (col < need[:, None])
    place = s["n_free"].long() - 1 - (page0[:, None] + col - have[:, None])
    tables = torch.where(fresh, s["free"][place.clamp(0, s["free"].numel() - 1)], s["tables"])
    req = torch.searchsorted(row0[1:].contiguous(), torch.arange(s["rows"], device="cuda"), right=True)
    pos = lens[req] + torch.arange(s["rows"], device="cuda") - row0[req]
    slots = tables[req, pos // page].long() * page + pos % page
    return {"tables": tables, "n_free": (s["n_free"] - taken).int(), "lens": (lens + new).int(), "row0": row0.int(),
            "slots": slots.int(), "pos": pos.int(), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _plain_append(s):
    """The values the cache holds for each row's keys and values."""
    (kq, kd), (vq, vd) = _quantize(s["k"]), _quantize(s["v"])
    return ((kq.float() - 8.0) * kd.float()).reshape(s["k"].shape), ((vq.float() - 8.0) * vd.float()).reshape(s["v"].shape)


def _plain_sample(s):
    x = torch.where(s["logits"].isnan(), -math.inf, s["logits"])
    n = x.shape[1]
    y, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((y.double() - y[:, :1].double()) / s["t"].double()[:, None])
    k = torch.where(s["k"] <= 0, n, s["k"])[:, None]
    w = torch.where(torch.arange(n, device="cuda") < k, w, 0.0)
    before = w.cumsum(-1) - w
    p = s["p"].double()[:, None]
    keep = (before < p * w.sum(-1, keepdim=True)) | (p >= 1)
    keep[:, 0] = True
    w = torch.where(keep & (w >= s["min_p"].double()[:, None]), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)       # back in the vocabulary's order
    run_sum = w.cumsum(-1)
    target = s["u"].double()[:, None] * run_sum[:, -1:]
    last = torch.where(w > 0, torch.arange(n, device="cuda"), 0).amax(-1)
    return torch.minimum((run_sum <= target).sum(-1), last).int()


# ------------------------------------------------------------------ the framework's calls
_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "hace-fem-hacedle_b200", "python"))
        import hacedle_cuda

        _ctx = hacedle_cuda.Context(torch.cuda.current_device())
    return _ctx


def _own(s):
    c, ctx = s["case"], _context()
    op = c["op"]
    if op == "pages":
        o = s["out"]
        ctx.kv_pages_assign(s["lens"], s["new"], s["tables"], c["page"], s["pages"], s["free"], s["n_free"], o["n_free"],
                            o["lens"], o["row0"], o["slots"], o["pos"], o["status"])
        return {"tables": s["tables"], **o}
    if op == "append":
        ctx.kv4_append(s["k"], s["v"], s["slots"], s["cache"])
        ctx.kv4_read(s["cache"], s["slots"], s["k_out"], s["v_out"])
        return s["k_out"], s["v_out"]
    if op == "sample":
        ctx.sample_filtered(s["logits"], s["u"], s["idx"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["min_p"])
        return s["idx"]
    if op == "decode":
        ctx.kv4_attention_decode(s["q"], s["cache"], s["tables"], s["lens"], s["out"], window=c["window"], sinks=c["sinks"])
    else:
        ctx.kv4_attention_prefill(s["q"], s["cache"], s["tables"], s["lens"], s["row0"], s["out"], window=c["window"],
                                  sinks=c["sinks"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "pages":
        return _plain_pages(state)
    if op == "append":
        return _plain_append(state)
    if op == "sample":
        return _plain_sample(state)
    return _attention(state, torch.float32)


def work(case):
    op = case["op"]
    if op == "sample":
        # the logits, and about 25 operations of each weight in 64 bits
        return {"bytes": 4 * case["rows"] * (case["n"] + 6), "flops": 25 * case["rows"] * case["n"]}
    if op == "append":
        values = 2 * case["rows"] * case["n_kv"] * case["hd"]
        # each value read in 32 bits, written in 4 (and its group's scale), and given back
        return {"bytes": 4 * values + 2 * values * 18 // 32 + 4 * values + 8 * case["rows"], "flops": 4 * values}
    if op == "pages":
        old, new = _lengths(case)
        got = sum(_ceil(o + n, case["page"]) - _ceil(o, case["page"]) for o, n in zip(old, new))
        return {"bytes": 16 * case["reqs"] + 8 * sum(new) + 8 * got, "flops": 10 * sum(new)}
    pairs, seen = _visible(case)
    rows = sum(_lengths(case)[1])
    return {"bytes": seen * case["n_kv"] * 18 * case["hd"] // 16 + 8 * rows * case["heads"] * case["hd"],
            "flops": 4 * pairs * case["heads"] * case["hd"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_append(x):
    import numpy as np

    x = x.cpu().numpy().reshape(-1, 32)
    top = x[np.arange(len(x)), np.abs(x).argmax(1)]
    d = torch.from_numpy(top / np.float32(-8)).to(torch.bfloat16).double().clamp(-8160, 8160).to(torch.float16).double().numpy()[:, None]
    steps = np.divide(x.astype(np.float64), d, out=np.zeros(x.shape), where=d != 0)
    return np.clip(np.rint(steps), -8, 7) * d


def _exact_attention(s, c):
    """One request and kv head at a time, each query's softmax over the positions it sees alone."""
    hd, rep, page = c["hd"], c["heads"] // c["n_kv"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens, row0 = s["lens"].tolist(), s["row0"].tolist()
    signed = torch.arange(16, device="cuda", dtype=torch.float64) - 8
    for r, n in enumerate(lens):
        a, b = row0[r], row0[r + 1]
        if a == b:
            continue
        ids = s["tables"][r, :_ceil(n, page)].long()
        for h in range(c["n_kv"]):
            t = s["cache"][ids, h].reshape(-1, 18 * hd)
            kv = []
            for part in (0, 1):
                b8 = t[:, 8 * hd * part:8 * hd * (part + 1)].reshape(-1, hd // 32, 16)
                d = t[:, 16 * hd + hd * part:17 * hd + hd * part].contiguous().view(torch.float16).double().reshape(-1, hd // 32, 1)
                x = torch.empty(b8.shape[0], hd // 32, 32, dtype=torch.float64, device="cuda")
                x[..., :16] = signed[(b8 % 16).long()] * d
                x[..., 16:] = signed[(b8 // 16).long()] * d
                kv.append(x.reshape(-1, hd)[:n])
            for t0 in range(a, b, 512):
                t1 = min(b, t0 + 512)
                i = torch.arange(n - b + t0, n - b + t1, device="cuda")[:, None]
                j = torch.arange(n, device="cuda")[None]
                hide = j > i
                if c["window"]:
                    hide |= (j <= i - c["window"]) & (j >= c["sinks"])
                q = s["q"][t0:t1, h * rep:(h + 1) * rep].double()
                z = torch.einsum("thd,jd->htj", q, kv[0]) * hd ** -0.5
                z[:, hide] = -math.inf
                out[t0:t1, h * rep:(h + 1) * rep] = torch.einsum("htj,jd->thd", torch.softmax(z, -1), kv[1])
    return out


def exact(case, seed):
    if case["op"] in ("pages", "sample"):  # whole numbers
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        return tuple(torch.from_numpy(_exact_append(x)).reshape(x.shape) for x in (s["k"], s["v"]))
    return _exact_attention(s, case)
