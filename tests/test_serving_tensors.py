"""What the binding of the serving calls refuses before it hands an address to
a kernel: tensors of another device than the context's, and empty outputs."""
import pytest

import hacedle_cuda as hc


def _ctx(device=0):
    ctx = hc.Context.__new__(hc.Context)   # no handle: a call that came through would be refused by the library, as HdError
    ctx.h, ctx.device = None, device
    return ctx


def calls(ctx, device="cpu", wrong=None):
    """name -> (a call whose tensors fit one another, the number of its tensors).  wrong: the index of the tensor to
    put on another device (None: none)."""
    import torch

    class On:
        """Makes tensors on `device`, the `wrong`-th of them elsewhere."""
        def __init__(self):
            self.n = 0

        def __call__(self, *shape, dtype=torch.float32):
            self.n += 1
            other = "meta" if device != "meta" else "cpu"
            return torch.zeros(*shape, dtype=dtype, device=other if wrong == self.n - 1 else device)

        def i(self, *shape):
            return self(*shape, dtype=torch.int32)

    cache = lambda f: f(*hc.kv4_cache_shape(8, 16, 2, 64), dtype=torch.uint8)  # noqa: E731
    made = {
        "sample": lambda f: ctx.sample_filtered(f(3, 50), f(3), f.i(3), temperature=f(3), top_k=f.i(3), top_p=f(3), min_p=f(3)),
        "sample_plain": lambda f: ctx.sample_filtered(f(3, 50), f(3), f.i(3)),
        "assign": lambda f: ctx.kv_pages_assign(f.i(3), f.i(3), f.i(3, 4), 16, 8, f.i(8), f.i(1), f.i(1), f.i(3), f.i(4), f.i(5), f.i(5), f.i(1)),
        "release": lambda f: ctx.kv_pages_release(f.i(3), f.i(3), f.i(3, 4), 16, f.i(8), f.i(1), f.i(1)),
        "append": lambda f: ctx.kv4_append(f(4, 2, 64), f(4, 2, 64), f.i(4), cache(f)),
        "read": lambda f: ctx.kv4_read(cache(f), f.i(4), f(4, 2, 64), f(4, 2, 64)),
        "decode": lambda f: ctx.kv4_attention_decode(f(3, 4, 64), cache(f), f.i(3, 4), f.i(3), f(3, 4, 64), ws=f(1 << 20, dtype=torch.uint8)),
        "decode_own": lambda f: ctx.kv4_attention_decode(f(3, 4, 64), cache(f), f.i(3, 4), f.i(3), f(3, 4, 64)),
        "prefill": lambda f: ctx.kv4_attention_prefill(f(7, 4, 64), cache(f), f.i(3, 4), f.i(3), f.i(4), f(7, 4, 64)),
    }
    return {name: (On, call) for name, call in made.items()}


NUMBER = {"sample": 7, "sample_plain": 3, "assign": 11, "release": 6, "append": 4, "read": 4, "decode": 6, "decode_own": 5, "prefill": 6}


@pytest.mark.parametrize("name", NUMBER)
def test_host_tensors_are_refused(name):
    on, call = calls(_ctx())[name]
    f = on()
    with pytest.raises(ValueError, match="device"):
        call(f)
    assert f.n == NUMBER[name]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NUMBER)
def test_each_tensor_on_another_device_is_refused(name):
    for i in range(NUMBER[name]):
        on, call = calls(_ctx(), "cuda", wrong=i)[name]
        with pytest.raises(ValueError, match="device"):
            call(on())
    on, call = calls(_ctx(device=1), "cuda")[name]     # the tensors' device is not the context's
    with pytest.raises(ValueError, match="device"):
        call(on())
    on, call = calls(_ctx(), "cuda")[name]             # all of them where they belong: on to the library, which wants a handle
    with pytest.raises(hc.HdError):
        call(on())


@pytest.mark.gpu
def test_outputs_without_an_entry_are_refused(ctx):
    """n_free, n_free_out and status are used at their first entry; an empty tensor's address is null, which the
    library refuses, also where the tensor is a part of one that has entries."""
    import torch
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    for none in (i32(0), i32(4)[2:2]):
        for empty in range(3):
            one = [none if k == empty else i32(1) for k in range(3)]
            with pytest.raises(hc.HdError, match="null argument"):
                ctx.kv_pages_assign(i32(3), i32(3), i32(3, 4), 16, 8, i32(8), one[0], one[1], i32(3), i32(4), i32(5), i32(5), one[2])
        for empty in range(2):
            one = [none if k == empty else i32(1) for k in range(2)]
            with pytest.raises(hc.HdError, match="null argument"):
                ctx.kv_pages_release(i32(3), i32(3), i32(3, 4), 16, i32(8), one[0], one[1])
