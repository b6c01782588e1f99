"""ctypes binding of libmpcx.so (the C ABI in include/mpcx.h).  Device memory is either owned by a
:class:`DeviceArray` (mpcx_malloc) or borrowed from a torch tensor via its ``data_ptr()``."""
import array
import ctypes
import operator
import os
import sys

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("MPCX_LIBRARY") or os.path.join(_HERE, "libmpcx.so")  # override: A/B runs of two builds

_lib = None


class MpcxError(RuntimeError):
    pass


def load_library():
    """Loads libmpcx.so.  There is no fallback: a missing library is an error."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise MpcxError(f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                            "(hipcc --offload-arch=gfx950); there is no CPU fallback")
        # A process that also uses PyTorch must bring torch's bundled HIP runtime up first: once this library (linked
        # against the system ROCm) has initialised HIP, torch no longer finds the device.
        torch = sys.modules.get("torch")
        if torch is not None and torch.cuda.is_available():
            torch.cuda.init()
        _lib = ctypes.CDLL(LIB_PATH)
        _lib.mpcx_last_error.restype = ctypes.c_char_p
        _lib.mpcx_last_error.argtypes = [ctypes.c_void_p]
        _lib.mpcx_get_stream.restype = ctypes.c_void_p
    return _lib


def exported_symbols():
    """Names declared in include/mpcx.h (parsed from the header text)."""
    import re
    hdr = open(os.path.join(os.path.dirname(_HERE), "include", "mpcx.h")).read()
    return sorted(set(re.findall(r"\b(mpcx_[a-z0-9_]+)\s*\(", hdr)))


class DeviceArray:
    """A typed device buffer.  ``ptr`` is the raw device address."""

    def __init__(self, ctx, dtype, n, ptr=None, owner=None):
        self.ctx, self.dtype, self.n = ctx, np.dtype(dtype), int(n)
        self.nbytes = self.n * self.dtype.itemsize
        self._own = ptr is None
        self._owner = owner  # keeps a borrowed allocation (e.g. a torch tensor) alive
        if ptr is None:
            p = ctypes.c_void_p()
            ctx._call("mpcx_malloc", ctypes.c_uint64(max(self.nbytes, 8)), ctypes.byref(p))
            ptr = p.value
        self.ptr = ptr

    @property
    def size(self):
        return self.n

    def view(self, offset_elems, n, dtype=None):
        dt = np.dtype(dtype) if dtype is not None else self.dtype
        return DeviceArray(self.ctx, dt, n, ptr=self.ptr + offset_elems * self.dtype.itemsize, owner=self)

    def to_host(self):
        out = np.empty(self.n, dtype=self.dtype)
        if self.n:
            self.ctx._call("mpcx_d2h", ctypes.c_void_p(out.ctypes.data), ctypes.c_void_p(self.ptr),
                           ctypes.c_uint64(self.nbytes))
        return out

    def free(self):
        if self._own and self.ptr:
            if self.ctx.h:  # a closed context has already released every block it handed out
                self.ctx._call("mpcx_free", ctypes.c_void_p(self.ptr))
            self.ptr = 0

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


# entry points that take the address of host memory, and in which arguments
_HOST_ARGS = {"h2d": (1,), "d2h": (0,), "h2d_bits": (1,), "d2h_bits": (0,), "h2d_u16": (1,), "d2h_u16": (0,),
              "prg_state_at_pop": (3,)}


def _word(x, device, keep):
    """One argument of the C ABI as the 64-bit word that carries it: an address, a size, or an int (whose callee reads the
    low half).  `keep` holds what must outlive the call."""
    t = type(x)
    if t is int:
        return x
    if x is None:
        return 0
    if t is DeviceArray:
        if x.ctx.device != device:
            raise MpcxError(f"an array on device {x.ctx.device} was passed to a context on device {device}")
        return x.ptr
    if hasattr(x, "data_ptr"):  # torch tensor: kernels can take neither host memory nor another device's
        if x.get_device() != device:
            raise MpcxError(f"a tensor on {x.device} was passed to a context on device {device}")
        return x.data_ptr()
    if isinstance(x, (int, np.integer)):
        return int(x)
    if isinstance(x, DeviceArray):  # of a derived class
        return _word(DeviceArray(x.ctx, x.dtype, x.n, ptr=x.ptr), device, keep)
    if isinstance(x, (list, tuple)):  # a host array: of device addresses (arrays, tensors) or of counts
        kinds, host = set(map(type, x)), None
        kind = kinds.pop() if len(kinds) == 1 else None
        if kind is int:  # the short ways: all counts, or all tensors on the device
            try:
                host = array.array("Q", x)
            except OverflowError:
                pass
        elif hasattr(kind, "data_ptr") and set(map(kind.get_device, x)) == {device}:
            host = array.array("Q", list(map(kind.data_ptr, x)))
        if host is None:
            host = array.array("Q", [_word(e, device, keep) & 0xFFFFFFFFFFFFFFFF for e in x] or [0])
        keep.append(host)
        return host.buffer_info()[0]
    raise TypeError(f"cannot pass {t} to the C ABI")


# ---- The language-model operators say what their arguments have to hold, and it is checked: contiguous arrays of the right
# type with as many elements as the sizes ask for (raw addresses are taken as they are).  A tensor that is right passes by
# four questions, so that short calls stay short; everything else goes the long way, which finds the words for what is wrong.
_I64 = _F32 = None  # torch's types, once an argument is a tensor


def _array(x, kind, need, device):
    """The address of one array of at least `need` elements: "w" 64-bit words, "f" 32-bit floats, "s" bytes of any type."""
    global _I64, _F32
    if x is None or isinstance(x, (int, np.integer)):
        return _word(x, device, [])
    word = _word(x, device, [])  # refuses what is no array, and other devices
    if isinstance(x, DeviceArray):
        right, have = x.dtype in (np.int64, np.uint64) if kind == "w" else x.dtype == np.float32, x.n
    elif isinstance(x, (list, tuple)):
        raise MpcxError("a list in the place of an array")
    else:
        torch = sys.modules["torch"]
        _I64, _F32 = torch.int64, torch.float32
        if not x.is_contiguous():
            raise MpcxError(f"a tensor of shape {tuple(x.shape)} and strides {x.stride()} that is not contiguous")
        right, have = x.dtype in ((_I64, torch.uint64) if kind == "w" else (_F32,)), x.numel()
    if kind == "s":
        have = x.nbytes
    elif not right:
        raise MpcxError(f"an array of {x.dtype} in the place of {'64-bit words' if kind == 'w' else '32-bit floats'}")
    if have < need:
        raise MpcxError(f"an array of {have} {'bytes' if kind == 's' else 'elements'} where the sizes ask for {need}")
    return word


def _w(x, need, device):
    if x is None:
        return 0
    if getattr(x, "dtype", 0) is _I64 and x.numel() >= need and x.get_device() == device and x.is_contiguous():
        return x.data_ptr()
    return _array(x, "w", need, device)


def _f(x, need, device):
    if x is None:
        return 0
    if getattr(x, "dtype", 0) is _F32 and x.numel() >= need and x.get_device() == device and x.is_contiguous():
        return x.data_ptr()
    return _array(x, "f", need, device)


def _counts(lens, count, keep):
    """The address of the word counts of a call's tensors."""
    if isinstance(lens, (list, tuple)) and len(lens) < count:
        raise MpcxError(f"{len(lens)} counts of {count} tensors")
    return _word(lens, None, keep)


def _tensors(xs, lens, count, device, keep):
    """The address of the addresses of `count` arrays of `lens` words each."""
    if not isinstance(xs, (list, tuple)) or not isinstance(lens, (list, tuple)):
        return _word(xs, device, keep)
    if len(xs) < count:
        raise MpcxError(f"{len(xs)} of {count} tensors")
    kinds = set(map(type, xs))
    kind = kinds.pop() if len(kinds) == 1 else None
    if (hasattr(kind, "data_ptr") and len(xs) == len(lens) == count and set(map(kind.dtype.__get__, xs)) == {_I64}
            and set(map(kind.get_device, xs)) == {device} and all(map(kind.is_contiguous, xs))
            and all(map(operator.ge, map(kind.numel, xs), lens))):
        host = array.array("Q", list(map(kind.data_ptr, xs)))
    else:
        host = array.array("Q", [_array(x, "w", n, device) & 0xFFFFFFFFFFFFFFFF for x, n in zip(xs[:count], lens)] or [0])
    keep.append(host)
    return host.buffer_info()[0]


def _ring_embed(ctx, keep, T0, T1, vocab, dim, ids, n, scale, shift, E0, E1):
    d, table, rows = ctx.device, vocab * dim, n * dim
    return _w(T0, table, d), _w(T1, table, d), vocab, dim, _w(ids, n, d), n, scale, shift, _w(E0, rows, d), _w(E1, rows, d)


def _ring_embed_grad(ctx, keep, G0, G1, ids, n, vocab, dim, scale, shift, accumulate, scratch, dT0, dT1):
    d, table, rows = ctx.device, vocab * dim, n * dim
    return (_w(G0, rows, d), _w(G1, rows, d), _w(ids, n, d), n, vocab, dim, scale, shift, accumulate,
            _array(scratch, "s", ctx.scratch_bytes("ring_embed_grad", n, vocab, dim), d), _w(dT0, table, d), _w(dT1, table, d))


def _aby3_sqnorm_local(ctx, keep, X0, X1, lens, count, seed_next, pop_next, seed_prev, pop_prev, scratch, z0):
    d = ctx.device
    return (_tensors(X0, lens, count, d, keep), _tensors(X1, lens, count, d, keep), _counts(lens, count, keep), count, seed_next,
            pop_next, seed_prev, pop_prev, _array(scratch, "s", ctx.scratch_bytes("aby3_sqnorm", count), d), _w(z0, 1, d))


def _aby3_clip_local(ctx, keep, party, X0, X1, lens, count, z_prev, z0, z1, max_norm, number, seed12, pop12, Y0, coef):
    d = ctx.device
    total = sum(lens[:count]) if isinstance(lens, (list, tuple)) else 0
    # party 0 does not read the second shares, party 2 none
    return (party, _tensors(X0, lens, count, d, keep) if party != 2 else 0, _tensors(X1, lens, count, d, keep) if party == 1 else 0,
            _counts(lens, count, keep), count, _w(z_prev, 1, d), _w(z0, 1, d), _w(z1, 1, d), max_norm, number, seed12, pop12,
            _w(Y0, total, d), _w(coef, 1, d))


def _reveal_logprobs(ctx, keep, a, b, c, rows, vocab, frac, ids, per_row, top, scratch, logp, entropy, top_ids, top_logp, row_max, log_sum):
    d, x, k, t = ctx.device, rows * vocab, rows * per_row, rows * top
    return (_w(a, x, d), _w(b, x, d), _w(c, x, d), rows, vocab, frac, _w(ids, k, d), per_row, top,
            _array(scratch, "s", ctx.scratch_bytes("reveal_logprobs", rows, vocab, top), d), _f(logp, k, d), _f(entropy, rows, d),
            _w(top_ids, t, d), _f(top_logp, t, d), _w(row_max, rows, d), _f(log_sum, rows, d))


def _reveal_logprobs_grad(ctx, keep, a, b, c, rows, vocab, frac, ids, per_row, d_logp, d_entropy, row_max, log_sum, entropy, grad,
                          grad_words, grad_frac):
    d, x, k = ctx.device, rows * vocab, rows * per_row
    return (_w(a, x, d), _w(b, x, d), _w(c, x, d), rows, vocab, frac, _w(ids, k, d), per_row, _f(d_logp, k, d), _f(d_entropy, rows, d),
            _w(row_max, rows, d), _f(log_sum, rows, d), _f(entropy, rows, d), _f(grad, x, d), _w(grad_words, x, d), grad_frac)


_CHECKED = {f.__name__[1:]: f for f in (_ring_embed, _ring_embed_grad, _aby3_sqnorm_local, _aby3_clip_local, _reveal_logprobs,
                                        _reveal_logprobs_grad)}


class Context:
    """One mpcx context (one HIP stream, one scratch workspace) on one GPU."""

    def __init__(self, device=0):
        self.lib = load_library()
        h = ctypes.c_void_p()
        rc = self.lib.mpcx_init(ctypes.c_int(device), ctypes.byref(h))
        if rc:
            raise MpcxError(self.lib.mpcx_last_error(None).decode())
        self.h = h
        self.device = device
        self._fns = {}  # (name, number of arguments) -> foreign function taking that many 64-bit words

    def close(self):
        if self.h:
            self.lib.mpcx_shutdown(self.h)
            self.h = None

    def _call(self, name, *args):
        if not self.h:
            raise MpcxError(f"{name}: the context is closed")
        rc = getattr(self.lib, name)(self.h, *args)
        if rc:
            raise MpcxError(f"{name}: {self.lib.mpcx_last_error(self.h).decode()}")

    def call(self, name, *args):
        """Calls ``mpcx_<name>(ctx, *args)``; DeviceArrays, tensors on the context's device, ints and lists of these are
        converted, and tensors in host memory where the entry point takes a host address.  Nothing is kept and nothing is
        ordered here: tensors have to be ready on the context's stream, and live until it has passed."""
        if not self.h:
            raise MpcxError(f"mpcx_{name}: the context is closed")
        fn = self._fns.get((name, len(args)))
        if fn is None:
            fn = self.lib["mpcx_" + name]  # an object of its own: its argument types do not touch the shared one's
            fn.argtypes = [ctypes.c_void_p] + [ctypes.c_uint64] * len(args)
            self._fns[name, len(args)] = fn
        keep = []
        host = _HOST_ARGS.get(name)
        if host is not None:  # the address of a tensor in host memory is an int like any other
            args = [x.data_ptr() if i in host and hasattr(x, "data_ptr") and x.get_device() < 0 else x for i, x in enumerate(args)]
        checked = _CHECKED.get(name)
        if checked is None:
            words = [_word(x, self.device, keep) for x in args]
        else:
            try:
                words = map(operator.index, checked(self, keep, *args))
            except MpcxError as e:
                raise MpcxError(f"mpcx_{name}: {e}") from None
        if fn(self.h, *words):
            raise MpcxError(f"mpcx_{name}: {self.lib.mpcx_last_error(self.h).decode()}")

    def scratch_bytes(self, name, *sizes):
        """Bytes of scratch memory that the caller of ``mpcx_<name>`` hands over (mpcx_<name>_scratch)."""
        fn = self._fns.get((name, "scratch"))
        if fn is None:
            fn = self.lib[f"mpcx_{name}_scratch"]
            fn.argtypes, fn.restype = [ctypes.c_uint64] * len(sizes), ctypes.c_uint64
            self._fns[name, "scratch"] = fn
        return fn(*map(operator.index, sizes))

    def sync(self):
        self._call("mpcx_sync")

    def stream(self):
        return self.lib.mpcx_get_stream(self.h)

    def empty(self, dtype, n):
        return DeviceArray(self, dtype, n)

    def to_device(self, arr, dtype=None):
        arr = np.ascontiguousarray(arr, dtype=dtype)
        d = DeviceArray(self, arr.dtype, arr.size)
        if arr.size:
            self._call("mpcx_h2d", ctypes.c_void_p(d.ptr), ctypes.c_void_p(arr.ctypes.data), ctypes.c_uint64(arr.nbytes))
        return d

    def wrap(self, tensor, dtype):
        """Borrows a torch CUDA tensor's storage as a DeviceArray of `dtype`."""
        nbytes = tensor.numel() * tensor.element_size()
        return DeviceArray(self, dtype, nbytes // np.dtype(dtype).itemsize, ptr=tensor.data_ptr(), owner=tensor)
