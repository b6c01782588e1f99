"""What the Python binding passes on and what it refuses, on a context that records its calls (no GPU)."""
import numpy as np
import pytest
import torch

from mpc_amd import MpcxError
from mpc_amd.lib import Context, DeviceArray


class Calls(dict):
    """In the place of the foreign functions: every call is written down and succeeds."""

    def __init__(self):
        self.seen = []

    def get(self, key):
        return lambda h, *words: self.seen.append((key[0], words)) or 0


@pytest.fixture()
def ctx():
    c = object.__new__(Context)
    c.h, c.device, c._fns, c.lib = 1, 0, Calls(), None
    return c


@pytest.mark.parametrize("name,at,args", [("h2d", 1, 3), ("d2h", 0, 3), ("h2d_bits", 1, 3), ("d2h_bits", 0, 3), ("h2d_u16", 1, 3),
                                          ("d2h_u16", 0, 3), ("prg_state_at_pop", 3, 4)])
def test_host_tensors_where_a_host_address_is_taken(ctx, name, at, args):
    host = torch.zeros(16, dtype=torch.int64)
    a = [4096] * args
    a[at] = host
    ctx.call(name, *a)
    assert ctx._fns.seen == [(name, tuple(host.data_ptr() if i == at else 4096 for i in range(args)))]
    a[at], a[(at + 1) % args] = 4096, host  # and nowhere else
    with pytest.raises(MpcxError, match="context on device 0"):
        ctx.call(name, *a)


def test_device_arrays_of_another_device_are_refused(ctx):
    other = object.__new__(Context)
    other.h, other.device = None, 1
    here, there = DeviceArray(ctx, np.int64, 4, ptr=4096), DeviceArray(other, np.int64, 4, ptr=8192)

    class Derived(DeviceArray):
        pass

    for bad in (there, Derived(other, np.int64, 4, ptr=8192), there.view(1, 2), [there, there], [here, there], (here, None, there.view(0, 4))):
        with pytest.raises(MpcxError, match="an array on device 1 was passed to a context on device 0"):
            ctx.call("xor_bools", here, bad, here, 4)
    ctx.call("xor_bools", Derived(ctx, np.int64, 4, ptr=4096), here.view(1, 2), None, 4)
    assert ctx._fns.seen == [("xor_bools", (4096, 4104, 0, 4))]


# ---- what the language-model operators' arguments have to hold
I64 = lambda *s: torch.zeros(*s, dtype=torch.int64)
F32 = lambda *s: torch.zeros(*s, dtype=torch.float32)
BYTES = lambda n: torch.zeros(n, dtype=torch.uint8)


@pytest.fixture()
def host(ctx):
    """The context takes tensors in host memory (device -1), so that whole calls can be made; the scratch sizes are the library's."""
    from mpc_amd.lib import load_library
    ctx.device, ctx.lib = -1, load_library()

    class Both(Calls):
        def get(self, key):
            return dict.get(self, key) if key[1] == "scratch" else Calls.get(self, key)

    ctx._fns = Both()
    return ctx


def right_calls(ctx):
    V, D, n, R, k, top = 5, 4, 3, 2, 2, 3
    sc = lambda name, *s: BYTES(ctx.scratch_bytes(name, *s))
    X0, X1 = [I64(2, 3), I64(7)], [I64(6), I64(9)]  # the last one is longer than it is said to be
    return {
        "ring_embed": [I64(V, D), I64(V, D), V, D, I64(n), n, 1, 0, I64(n, D), I64(n, D)],
        "ring_embed_grad": [I64(n, D), I64(n, D), I64(n), n, V, D, 1, 0, 0, sc("ring_embed_grad", n, V, D), I64(V, D), I64(V, D)],
        "aby3_sqnorm_local": [X0, X1, [6, 7], 2, 1, 0, 2, 0, sc("aby3_sqnorm", 2), I64(1)],
        "aby3_clip_local": [1, X0, X1, [6, 7], 2, I64(1), I64(1), I64(1), 1 << 16, 16, 3, 0, I64(13), I64(1)],
        "reveal_logprobs": [I64(R, V), I64(R, V), I64(R, V), R, V, 16, I64(R, k), k, top, sc("reveal_logprobs", R, V, top), F32(R, k),
                            F32(R), I64(R, top), F32(R, top), I64(R), F32(R)],
        "reveal_logprobs_grad": [I64(R, V), I64(R, V), I64(R, V), R, V, 16, I64(R, k), k, F32(R, k), F32(R), I64(R), F32(R), F32(R),
                                 F32(R, V), I64(R, V), 16],
    }


def wrong(x):
    """Tensors that must not pass in the place of x: too short, of another type, not contiguous."""
    n = x.numel()
    yield torch.zeros(n - 1, dtype=x.dtype), "where the sizes ask for"
    if x.dtype == torch.uint8:  # scratch memory has no type
        return
    for t in (torch.int32, torch.float64, torch.float16, torch.int64, torch.float32):
        if t != x.dtype:
            yield torch.zeros(2 * n, dtype=t), "in the place of"
    yield torch.zeros(1, dtype=x.dtype).expand(n) if n > 1 else torch.zeros(4, dtype=x.dtype)[::2], "not contiguous"
    if x.dim() == 2 and n > 1:
        yield torch.zeros(x.shape[1], x.shape[0], dtype=x.dtype).t(), "not contiguous"


@pytest.mark.parametrize("name", ["ring_embed", "ring_embed_grad", "aby3_sqnorm_local", "aby3_clip_local", "reveal_logprobs",
                                  "reveal_logprobs_grad"])
def test_arguments_of_the_language_model_operators(host, name):
    args = right_calls(host)[name]
    host.call(name, *args)
    (_, words), = host._fns.seen
    for a, w in zip(args, words):
        assert isinstance(a, list) or w == (a.data_ptr() if isinstance(a, torch.Tensor) else a)
    lists = [i for i, a in enumerate(args) if isinstance(a, list) and isinstance(a[0], torch.Tensor)]
    places = [(i, None) for i, a in enumerate(args) if isinstance(a, torch.Tensor)] + [(i, j) for i in lists for j in (0, 1)]
    for i, j in places:
        x = args[i] if j is None else args[i][j]
        size = {0: 6, 1: 7}[j] if j is not None else x.numel()
        for bad, text in wrong(x.reshape(-1)[:size].view(x.shape) if x.numel() == size else x[:size]):
            a = list(args)
            a[i] = bad if j is None else [bad if q == j else e for q, e in enumerate(args[i])]
            with pytest.raises(MpcxError, match=f"mpcx_{name}: .*{text}"):
                host.call(name, *a)
    for i, a in enumerate(args):
        if isinstance(a, list):  # a list that is shorter than the count
            b = list(args)
            b[i] = a[:1]
            with pytest.raises(MpcxError, match=f"mpcx_{name}: 1 (counts )?of 2 tensors"):
                host.call(name, *b)
    with pytest.raises(TypeError):  # one argument too few
        host.call(name, *args[:-1])
    assert len(host._fns.seen) == 1


def test_arrays_and_addresses_of_the_language_model_operators(host):
    """DeviceArrays are checked like tensors; addresses, numpy sizes and a second share that is not there are taken."""
    D = lambda dt, n: DeviceArray(host, dt, n, ptr=4096)
    ok = [D(np.int64, 20), None, np.int64(5), 4, D(np.uint64, 3), 3, 1, 0, 8192, None]
    host.call("ring_embed", *ok)
    assert host._fns.seen == [("ring_embed", (4096, 0, 5, 4, 4096, 3, 1, 0, 8192, 0))]
    for at, bad in ((0, D(np.int64, 19)), (0, D(np.int32, 40)), (4, D(np.float64, 3)), (0, [I64(20)]), (8, I64(11))):
        a = list(ok)
        a[at] = bad
        with pytest.raises(MpcxError, match="mpcx_ring_embed: "):
            host.call("ring_embed", *a)
    host.call("aby3_sqnorm_local", [D(np.int64, 3), 4096, None], (D(np.int64, 3), I64(9), None), (3, 9, 0), 3, 1, 0, 2, 0, 8192, D(np.int64, 1))
    with pytest.raises(MpcxError, match="3 elements where the sizes ask for 4"):
        host.call("aby3_sqnorm_local", [D(np.int64, 3)], [D(np.int64, 4)], [4], 1, 1, 0, 2, 0, 8192, D(np.int64, 1))
    # party 0 reads the first shares only, party 2 none: what stands in their place is not looked at
    z, y = D(np.int64, 1), D(np.int64, 4)
    host.call("aby3_clip_local", 0, [D(np.int64, 4)], None, [4], 1, z, z, z, 1, 16, 0, 0, y, z)
    host.call("aby3_clip_local", 2, None, None, [4], 1, z, z, z, 1, 16, 0, 0, y, z)
    with pytest.raises(MpcxError, match="4 elements where the sizes ask for 5"):
        host.call("aby3_clip_local", 2, None, None, [5], 1, z, z, z, 1, 16, 0, 0, y, z)
