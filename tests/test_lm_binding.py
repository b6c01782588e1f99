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
