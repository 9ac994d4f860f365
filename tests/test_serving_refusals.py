"""What the serving entry points refuse, without a GPU: the library checks its
arguments before it looks at the context, and the binding checks tensors
before it calls the library."""
import ctypes as C

import pytest

import hacedle_cuda as hc

P = 4096       # a non-null, 16-byte aligned address that is never read
OK = None


def assign(reqs=4, width=8, page=16, pages=32, rows=64, cap=32, **null):
    a = {n: P for n in ("lens", "new", "tables", "free", "n_free", "n_free_out", "lens_out", "row0", "slots", "pos", "status")}
    a.update({n: None for n in null})
    return hc.lib().hd_kv_pages_assign(None, a["lens"], a["new"], reqs, a["tables"], width, page, pages, a["free"],
                                       a["n_free"], cap, a["n_free_out"], a["lens_out"], a["row0"], a["slots"], a["pos"], rows,
                                       a["status"])


def release(reqs=4, width=8, page=16, cap=32, status=P):
    return hc.lib().hd_kv_pages_release(None, P, P, reqs, P, width, page, P, P, cap, status)


def append(k=P, v=P, kld=0, vld=0, slots=P, rows=4, n_kv=2, hd=64, cache=P, pages=8, page=16):
    return hc.lib().hd_kv4_append(None, k, v, kld, vld, slots, rows, n_kv, hd, cache, pages, page)


def read(cache=P, pages=8, page=16, slots=P, rows=4, n_kv=2, hd=64, k=P, v=P):
    return hc.lib().hd_kv4_read(None, cache, pages, page, slots, rows, n_kv, hd, k, v)


def decode(q=P, ld=0, cache=P, pages=8, page=16, tables=P, width=4, lens=P, seqs=2, heads=4, n_kv=2, hd=64, window=0,
           sinks=0, scale=0.0, out=P):
    return hc.lib().hd_kv4_attention_decode(None, q, ld, cache, pages, page, tables, width, lens, seqs, heads, n_kv, hd,
                                            window, sinks, C.c_float(scale), out, None, 0)


def prefill(q=P, ld=0, cache=P, pages=8, page=16, tables=P, width=4, lens=P, row0=P, seqs=2, rows=5, heads=4, n_kv=2, hd=64,
            window=0, sinks=0, scale=0.0, out=P):
    return hc.lib().hd_kv4_attention_prefill(None, q, ld, cache, pages, page, tables, width, lens, row0, seqs, rows, heads,
                                             n_kv, hd, window, sinks, C.c_float(scale), out)


def sample(x=P, ld=0, rows=2, n=100, u=P, idx=P):
    return hc.lib().hd_sample_filtered(None, x, ld, rows, n, None, None, None, None, u, idx)


@pytest.mark.parametrize("call", [assign, release, append, read, decode, prefill, sample])
def test_a_good_call_without_a_context_is_refused(call):
    assert call() == hc.HD_E_ARG


@pytest.mark.parametrize("call,kw,code", [
    (assign, {"lens": 1}, hc.HD_E_ARG), (assign, {"status": 1}, hc.HD_E_ARG), (assign, {"free": 1}, hc.HD_E_ARG),
    (assign, {"slots": 1}, hc.HD_E_ARG), (assign, {"reqs": -1}, hc.HD_E_SHAPE), (assign, {"width": 0}, hc.HD_E_SHAPE),
    (assign, {"page": 8}, hc.HD_E_SHAPE), (assign, {"page": 48}, hc.HD_E_SHAPE), (assign, {"page": 2048}, hc.HD_E_SHAPE),
    (assign, {"reqs": 8193}, hc.HD_E_UNSUPPORTED), (assign, {"width": 1 << 27}, hc.HD_E_SHAPE),
    (assign, {"rows": -1}, hc.HD_E_SHAPE), (assign, {"cap": -1}, hc.HD_E_SHAPE), (assign, {"rows": 1 << 31}, hc.HD_E_SHAPE),
    (assign, {"pages": 1 << 27}, hc.HD_E_SHAPE),
    (release, {"page": 24}, hc.HD_E_SHAPE), (release, {"cap": -1}, hc.HD_E_SHAPE), (release, {"status": None}, hc.HD_E_ARG),
    (append, {"k": None}, hc.HD_E_ARG), (append, {"cache": None}, hc.HD_E_ARG), (append, {"hd": 80}, hc.HD_E_UNSUPPORTED),
    (append, {"n_kv": 0}, hc.HD_E_SHAPE), (append, {"n_kv": 1 << 26, "rows": 1}, hc.HD_E_SHAPE), (append, {"page": 0}, hc.HD_E_SHAPE), (append, {"pages": 1 << 27}, hc.HD_E_SHAPE),
    (append, {"kld": 64}, hc.HD_E_SHAPE), (append, {"vld": 129}, hc.HD_E_ARG), (append, {"k": P + 4}, hc.HD_E_ARG),
    (append, {"cache": P + 8}, hc.HD_E_ARG), (append, {"rows": -1}, hc.HD_E_SHAPE), (append, {"rows": 1 << 33}, hc.HD_E_SHAPE),
    (read, {"slots": None}, hc.HD_E_ARG), (read, {"v": P + 4}, hc.HD_E_ARG), (read, {"hd": 96}, hc.HD_E_UNSUPPORTED),
    (read, {"rows": -3}, hc.HD_E_SHAPE),
    (decode, {"heads": 5}, hc.HD_E_SHAPE), (decode, {"heads": 34}, hc.HD_E_SHAPE), (decode, {"window": -1}, hc.HD_E_ARG),
    (decode, {"sinks": -1}, hc.HD_E_ARG), (decode, {"scale": -1.0}, hc.HD_E_ARG), (decode, {"scale": float("nan")}, hc.HD_E_ARG),
    (decode, {"scale": float("inf")}, hc.HD_E_ARG), (decode, {"q": P + 4}, hc.HD_E_ARG), (decode, {"ld": 128}, hc.HD_E_SHAPE),
    (decode, {"ld": 258}, hc.HD_E_ARG), (decode, {"width": 0}, hc.HD_E_SHAPE), (decode, {"lens": None}, hc.HD_E_ARG),
    (decode, {"seqs": -1}, hc.HD_E_SHAPE), (prefill, {"seqs": 1 << 30}, hc.HD_E_SHAPE), (decode, {"hd": 256}, hc.HD_E_UNSUPPORTED), (decode, {"cache": P + 8}, hc.HD_E_ARG),
    (prefill, {"row0": None}, hc.HD_E_ARG), (prefill, {"rows": -1}, hc.HD_E_SHAPE), (prefill, {"rows": 1 << 31}, hc.HD_E_SHAPE),
    (prefill, {"out": None}, hc.HD_E_ARG), (prefill, {"page": 20}, hc.HD_E_SHAPE),
    (sample, {"u": None}, hc.HD_E_ARG), (sample, {"idx": None}, hc.HD_E_ARG), (sample, {"n": 0}, hc.HD_E_SHAPE),
    (sample, {"n": 1 << 31}, hc.HD_E_SHAPE), (sample, {"ld": 99}, hc.HD_E_SHAPE), (sample, {"rows": -1}, hc.HD_E_SHAPE),
])
def test_refused(call, kw, code):
    assert call(**kw) == code


def test_cache_bytes():
    assert hc.lib().hd_kv4_cache_bytes(10, 64, 4, 128) == 10 * 4 * 4 * 18 * 128
    assert hc.kv4_cache_shape(10, 64, 4, 128) == (10, 4, 4, 18 * 128)
    # 18 bytes for 32 values of K and of V
    assert hc.lib().hd_kv4_cache_bytes(1, 16, 1, 32) * 32 == 2 * 16 * 32 * 18
    # a byte count beyond 32 bits
    assert hc.lib().hd_kv4_cache_bytes(1 << 21, 64, 8, 128) == (1 << 21) * 8 * 4 * 18 * 128
    for bad in ((-1, 16, 1, 32), (1, 15, 1, 32), (1, 16, 0, 32), (1, 16, 1, 48)):
        assert hc.lib().hd_kv4_cache_bytes(*bad) == 0
    with pytest.raises(ValueError):
        hc.kv4_cache_shape(4, 16, 2, 80)


def test_the_binding_refuses_tensors_that_do_not_fit():
    import torch
    ctx = hc.Context.__new__(hc.Context)   # no handle: the checks come before any library call
    ctx.h = None
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    cache = torch.zeros(hc.kv4_cache_shape(8, 16, 2, 64), dtype=torch.uint8)
    q, out = torch.zeros(3, 4, 64), torch.zeros(3, 4, 64)
    bad = [
        lambda: ctx.kv4_append(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), i32(4), cache),
        lambda: ctx.kv4_append(torch.zeros(4, 2, 64).half(), torch.zeros(4, 2, 64), i32(4), cache),
        lambda: ctx.kv4_append(torch.zeros(4, 64, 2).transpose(1, 2), torch.zeros(4, 2, 64), i32(4), cache),
        lambda: ctx.kv4_append(torch.zeros(4, 2, 64), torch.zeros(4, 2, 64), i32(4).long(), cache),
        lambda: ctx.kv4_append(torch.zeros(4, 2, 64), torch.zeros(4, 2, 64), i32(4), cache.float()),
        lambda: ctx.kv4_read(cache, i32(4), torch.zeros(4, 2, 64), torch.zeros(5, 2, 64)),
        lambda: ctx.kv4_attention_decode(q, cache, i32(2, 4), i32(3), out),
        lambda: ctx.kv4_attention_decode(q, cache, i32(3, 4), i32(3), out[:2]),
        lambda: ctx.kv4_attention_decode(q.double(), cache, i32(3, 4), i32(3), out),
        lambda: ctx.kv4_attention_decode(q, cache[:, :, ::1, :17], i32(3, 4), i32(3), out),
        lambda: ctx.kv4_attention_decode(q, cache[..., :0], i32(3, 4), i32(3), out),
        lambda: ctx.kv4_attention_prefill(q, cache, i32(2, 4), i32(2), i32(2), out),
        lambda: ctx.sample_filtered(torch.zeros(2, 50), torch.zeros(3), i32(2)),
        lambda: ctx.sample_filtered(torch.zeros(2, 50), torch.zeros(2), i32(2), top_k=torch.zeros(2)),
        lambda: ctx.kv4_attention_decode(q[:1].expand(3, 4, 64), cache, i32(3, 4), i32(3), out),
        lambda: ctx.kv4_append(torch.zeros(1, 2, 64).expand(4, 2, 64), torch.zeros(4, 2, 64), i32(4), cache),
        lambda: ctx.sample_filtered(torch.zeros(1, 50).expand(2, 50), torch.zeros(2), i32(2)),
        lambda: ctx.sample_filtered(torch.zeros(50, 2).t(), torch.zeros(2), i32(2)),
        lambda: ctx.kv_pages_assign(i32(2), i32(2), i32(3, 4), 16, 8, i32(8), i32(1), i32(1), i32(3), i32(4), i32(5), i32(5), i32(1)),
        lambda: ctx.kv_pages_release(i32(2), i32(3), i32(3, 4), 16, i32(8), i32(1), i32(1)),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
