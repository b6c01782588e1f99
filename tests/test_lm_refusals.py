"""What the language-model entry points refuse: shapes and pointers are checked on the host before anything is launched, so
these run without a GPU (no context)."""
import ctypes

import numpy as np
import pytest

U = ctypes.c_uint64
P = ctypes.c_void_p
I = ctypes.c_int
L = ctypes.c_int64
X = P(4096)  # never read: the call is refused, or there is nothing to do
N = P(0)


@pytest.fixture(scope="module")
def lib():
    from mpc_amd.lib import load_library
    return load_library()


def refused(lib, name, args, text):
    assert getattr(lib, name)(N, *args) != 0
    assert text in lib.mpcx_last_error(None).decode(), lib.mpcx_last_error(None).decode()


def host(*v):
    return (ctypes.c_uint64 * max(len(v), 1))(*v)


@pytest.mark.parametrize("args,text", [
    ((X, N, U(1 << 40), U(1 << 40), X, U(1), L(1), I(0), X, N), "too large"),
    ((X, N, U(4), U(1 << 40), X, U(1 << 40), L(1), I(0), X, N), "too large"),
    ((X, N, U(4), U(4), X, U(1), L(1), I(64), X, N), "out of range"),
    ((X, N, U(4), U(4), X, U(1), L(1), I(-1), X, N), "out of range"),
    ((X, X, U(4), U(4), X, U(1), L(1), I(0), X, N), "second share"),
    ((X, N, U(4), U(4), X, U(1), L(1), I(0), X, X), "second share"),
    ((X, X, U(4), U(4), X, U(1), L(1), I(16), X, X), "not truncated locally"),
    ((N, N, U(4), U(4), X, U(1), L(1), I(0), X, N), "NULL"),
    ((X, N, U(4), U(4), N, U(1), L(1), I(0), X, N), "NULL"),
    ((X, N, U(4), U(4), X, U(1), L(1), I(0), N, N), "NULL"),
])
def test_embed(lib, args, text):
    refused(lib, "mpcx_ring_embed", args, text)


def test_nothing_to_do_is_no_error(lib):
    assert lib.mpcx_ring_embed(N, X, N, U(4), U(4), X, U(0), L(1), I(0), X, N) == 0
    assert lib.mpcx_ring_embed(N, X, N, U(4), U(0), X, U(3), L(1), I(0), X, N) == 0
    assert lib.mpcx_ring_embed_grad(N, X, N, X, U(3), U(0), U(4), L(1), I(0), I(0), X, X, N) == 0
    assert lib.mpcx_reveal_logprobs(N, X, N, N, U(0), U(5), I(16), X, U(1), U(1), X, X, N, X, X, N, N) == 0
    assert lib.mpcx_reveal_logprobs_grad(N, X, N, N, U(0), U(5), I(16), X, U(1), X, N, X, X, N, X, N, I(0)) == 0


@pytest.mark.parametrize("args,text", [
    ((X, N, X, U(1), U(1 << 40), U(1 << 40), L(1), I(0), I(0), X, X, N), "too large"),
    ((X, N, X, U(1 << 33), U(4), U(4), L(1), I(0), I(0), X, X, N), "too large"),
    ((X, N, X, U(1), U(1 << 33), U(4), L(1), I(0), I(0), X, X, N), "too large"),
    ((X, N, X, U(1), U(4), U(4), L(1), I(64), I(0), X, X, N), "out of range"),
    ((X, X, X, U(1), U(4), U(4), L(1), I(0), I(0), X, X, N), "second share"),
    ((X, N, X, U(1), U(4), U(4), L(1), I(0), I(0), X, X, X), "second share"),
    ((X, X, X, U(1), U(4), U(4), L(1), I(3), I(0), X, X, X), "not truncated locally"),
    ((N, N, X, U(1), U(4), U(4), L(1), I(0), I(0), X, X, N), "NULL"),
    ((X, N, N, U(1), U(4), U(4), L(1), I(0), I(0), X, X, N), "NULL"),
    ((X, N, X, U(1), U(4), U(4), L(1), I(0), I(0), N, X, N), "NULL"),
    ((X, N, X, U(1), U(4), U(4), L(1), I(0), I(0), X, N, N), "NULL"),
])
def test_embed_grad(lib, args, text):
    refused(lib, "mpcx_ring_embed_grad", args, text)


@pytest.mark.parametrize("args,text", [
    ((host(4096), host(4096), host(8), U(1), U(1), U(0), U(2), U(0), N, X), "NULL"),
    ((host(4096), host(4096), host(8), U(1), U(1), U(0), U(2), U(0), X, N), "NULL"),
    ((N, host(4096), host(8), U(1), U(1), U(0), U(2), U(0), X, X), "NULL"),
    ((host(4096), host(4096), N, U(1), U(1), U(0), U(2), U(0), X, X), "NULL"),
    ((host(4096, 0), host(4096, 4096), host(8, 8), U(2), U(1), U(0), U(2), U(0), X, X), "tensor 1: NULL"),
    ((host(4096, 4096), host(0, 4096), host(8, 8), U(2), U(1), U(0), U(2), U(0), X, X), "tensor 0: NULL"),
    ((host(4096), host(4096), host(1 << 60), U(1), U(1), U(0), U(2), U(0), X, X), "too long"),
])
def test_sqnorm(lib, args, text):
    refused(lib, "mpcx_aby3_sqnorm_local", args, text)


def clip(party=0, X0=None, X1=None, lens=None, count=1, z=(X, X, X), max_norm=1 << 16, number=16, Y0=X, coef=X):
    return (I(party), X0 if X0 is not None else host(4096), X1 if X1 is not None else host(4096), lens or host(8), U(count), *z,
            U(max_norm), I(number), U(2), U(0), Y0, coef)


@pytest.mark.parametrize("args,text", [
    (clip(party=3), "party 3"), (clip(party=-1), "party -1"),
    (clip(number=32), "fractional bits"), (clip(number=-1), "fractional bits"),
    (clip(max_norm=1 << 46), "max_norm"),
    (clip(z=(N, X, X)), "NULL"), (clip(z=(X, N, X)), "NULL"), (clip(z=(X, X, N)), "NULL"),
    (clip(Y0=N), "NULL"), (clip(coef=N), "NULL"), (clip(X0=host(0)), "NULL"), (clip(party=1, X1=host(0)), "NULL"), (clip(X0=N), "NULL"),
    (clip(lens=host(1 << 60)), "too long"),
])
def test_clip(lib, args, text):
    refused(lib, "mpcx_aby3_clip_local", args, text)


def lp(a=X, b=X, c=X, rows=3, vocab=5, frac=16, ids=X, per_row=1, top=2, scratch=X, logp=X, top_ids=X, top_logp=X):
    return (a, b, c, U(rows), U(vocab), I(frac), ids, U(per_row), U(top), scratch, logp, X, top_ids, top_logp, X, X)


@pytest.mark.parametrize("args,text", [
    (lp(vocab=0), "vocabulary"), (lp(vocab=1 << 31), "vocabulary"), (lp(rows=1 << 60), "too large"),
    (lp(rows=1 << 20, per_row=1 << 50), "too large"), (lp(frac=63), "fractional"), (lp(frac=-1), "fractional"),
    (lp(top=33, vocab=100), "alternatives"), (lp(top=6), "alternatives"), (lp(b=N), "third share"),
    (lp(a=N), "NULL"), (lp(ids=N), "NULL"), (lp(logp=N), "NULL"), (lp(scratch=N), "NULL"), (lp(top_ids=N), "NULL"),
    (lp(top_logp=N), "NULL"),
])
def test_logprobs(lib, args, text):
    refused(lib, "mpcx_reveal_logprobs", args, text)


def lg(a=X, b=X, c=X, rows=3, vocab=5, frac=16, ids=X, per_row=1, d_logp=X, d_entropy=X, row_max=X, log_sum=X, entropy=X,
       grad=X, words=X, grad_frac=16):
    return (a, b, c, U(rows), U(vocab), I(frac), ids, U(per_row), d_logp, d_entropy, row_max, log_sum, entropy, grad, words,
            I(grad_frac))


@pytest.mark.parametrize("args,text", [
    (lg(vocab=0), "vocabulary"), (lg(vocab=1 << 31), "vocabulary"), (lg(rows=1 << 60), "too large"), (lg(frac=63), "fractional"),
    (lg(grad_frac=63), "fractional"), (lg(grad_frac=-1), "fractional"), (lg(b=N), "third share"), (lg(a=N), "NULL"),
    (lg(ids=N), "NULL"), (lg(d_logp=N), "NULL"), (lg(row_max=N), "NULL"), (lg(log_sum=N), "NULL"), (lg(entropy=N), "NULL"),
    (lg(grad=N, words=N), "NULL"),
])
def test_logprobs_grad(lib, args, text):
    refused(lib, "mpcx_reveal_logprobs_grad", args, text)


class Sized:
    def __init__(self, n):
        self.size = n


def test_backend_refuses_arrays_that_do_not_fit_the_shapes():
    """The Python backends know the lengths of their arrays and check them before anything is uploaded."""
    from mpc_amd.backends import GpuBackend
    be = object.__new__(GpuBackend)  # without a context
    A = Sized
    calls = [
        lambda: be.ring_embed(A(11), None, 3, 4, A(2)),
        lambda: be.ring_embed(A(12), A(13), 3, 4, A(2)),
        lambda: be.ring_embed_grad(A(9), None, A(2), 3, 4),
        lambda: be.ring_embed_grad(A(8), A(7), A(2), 3, 4),
        lambda: be.aby3_sqnorm_local([A(3)], [A(4)], 1, 0, 2, 0),
        lambda: be.aby3_sqnorm_local([A(3)], [A(3), A(1)], 1, 0, 2, 0),
        lambda: be.aby3_clip_local(0, [A(3)], [A(2)], A(1), A(1), A(1), 1, 16, 1, 0),
        lambda: be.aby3_clip_local(0, [A(3)], [A(3)], A(1), A(2), A(1), 1, 16, 1, 0),
        lambda: be.reveal_logprobs(A(12), A(12), A(11), 3, 4, 16, A(3)),
        lambda: be.reveal_logprobs(A(12), None, None, 3, 4, 16, A(4)),
        lambda: be.reveal_logprobs_grad(A(12), None, None, 3, 4, 16, A(3), A(2), None, A(3), A(3), None, 16),
        lambda: be.reveal_logprobs_grad(A(12), None, None, 3, 4, 16, A(3), A(3), None, A(3), A(2), None, 16),
        lambda: be.reveal_logprobs_grad(A(12), None, None, 3, 4, 16, A(3), A(3), A(3), A(3), A(3), A(1), 16),
    ]
    for k, f in enumerate(calls):
        with pytest.raises(ValueError, match="elements where|first shares"):
            f()


def test_binding_refuses_tensors_of_another_device():
    import torch
    from mpc_amd import MpcxError
    from mpc_amd.lib import _word
    host = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(MpcxError, match="context on device 0"):
        _word(host, 0, [])
    with pytest.raises(MpcxError, match="context on device 0"):
        _word([host, host], 0, [])
    with pytest.raises(TypeError):
        _word(1.5, 0, [])
    keep = []
    assert _word(-3, 0, keep) == -3 and _word(None, 0, keep) == 0 and not keep
    _word([1, 2, -1], 0, keep)
    assert list(keep[0]) == [1, 2, 2 ** 64 - 1]
    _word((), 0, keep), _word([None, 2 ** 64 - 1, np.int64(5)], 0, keep)
    assert list(keep[1]) == [0] and list(keep[2]) == [0, 2 ** 64 - 1, 5]
    _word([host, host[1:]], -1, keep)
    assert list(keep[3]) == [host.data_ptr(), host.data_ptr() + 8]
    for wrong in ([host], [host, 7], [7, host[:1]], [host[:1], None], [torch.nn.Parameter(host.double()), host]):
        with pytest.raises(MpcxError, match="context on device 0"):  # one word of a tensor is never taken for a number
            _word(wrong, 0, [])


def test_logits_without_rows_are_no_error_whatever_their_columns(lib):
    for vocab, top in ((0, 0), (0, 3), (2, 3)):
        assert lib.mpcx_reveal_logprobs(N, X, N, N, U(0), U(vocab), I(16), X, U(1), U(top), X, X, N, X, X, N, N) == 0
    assert lib.mpcx_reveal_logprobs_grad(N, X, N, N, U(0), U(0), I(16), X, U(1), X, N, X, X, N, X, N, I(0)) == 0
    for args in (lp(rows=0, top=33), lp(rows=0, frac=63), lp(rows=0, vocab=1 << 31)):
        assert lib.mpcx_reveal_logprobs(N, *args) != 0


def test_scratch_sizes_of_calls_that_are_refused():
    """The sizes can be asked for whatever the numbers are (in a process of its own: it must not end by a signal)."""
    import os
    import subprocess
    import sys
    numbers = (0, 1, 255, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 56, 2 ** 63, 2 ** 64 - 2048, 2 ** 64 - 1)
    code = ("import ctypes, itertools\nfrom mpc_amd.lib import load_library\nlib = load_library()\n"
            "for name, k in (('ring_embed_grad', 3), ('aby3_sqnorm', 1), ('reveal_logprobs', 3)):\n"
            "    fn = getattr(lib, f'mpcx_{name}_scratch')\n"
            f"    for v in itertools.product({numbers}, repeat=k): fn(*map(ctypes.c_uint64, v))\n")
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
    assert subprocess.run([sys.executable, "-c", code], cwd=root, timeout=100).returncode == 0
