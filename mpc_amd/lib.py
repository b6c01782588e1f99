"""ctypes binding of libmpcx.so (the C ABI in include/mpcx.h).  Device memory is either owned by a
:class:`DeviceArray` (mpcx_malloc) or borrowed from a torch tensor via its ``data_ptr()``."""
import array
import ctypes
import os

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
        import sys
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
        converted, and tensors in host memory where the entry point takes a host address."""
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
        if fn(self.h, *[_word(x, self.device, keep) for x in args]):
            raise MpcxError(f"mpcx_{name}: {self.lib.mpcx_last_error(self.h).decode()}")

    def scratch_bytes(self, name, *sizes):
        """Bytes of scratch memory that the caller of ``mpcx_<name>`` hands over (mpcx_<name>_scratch)."""
        fn = getattr(self.lib, f"mpcx_{name}_scratch")
        fn.restype = ctypes.c_uint64
        return fn(*[ctypes.c_uint64(s) for s in sizes])

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
