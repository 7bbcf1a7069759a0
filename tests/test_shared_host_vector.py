"""rsp_shared_host_* / rsp_copy_to_host_async: one vector in POSIX shared memory that the rank processes of a node write
their slices into.  It is ordinary memory -- no page of it is locked -- so it opens on every machine, one without a GPU
included."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT
from rcppsparse_amd import capi

CHILD = """
import sys
sys.path.insert(0, {root!r})
from rcppsparse_amd import capi
v = capi.SharedHostVector({name!r}, {n}, create=False)
v.array[{lo}:{hi}] = range({lo}, {hi})
v.close()
"""


def _name(tag):
    return f"/rsp_test_{tag}_{os.getpid()}"


@pytest.mark.parametrize("n", [1, 511, 512, 513, 100_003])       # below, at and past a page of 512 doubles
def test_two_processes_write_one_vector(n):
    name, half = _name(f"two_{n}"), n // 2
    v = capi.SharedHostVector(name, n, create=True)
    try:
        assert v.array.shape == (n,) and not v.array.any()       # fresh shared memory is zero-filled
        v.array[:half] = np.arange(half)
        subprocess.run([sys.executable, "-c", CHILD.format(root=ROOT, name=name, n=n, lo=half, hi=n)], check=True, timeout=120)
        assert np.array_equal(v.array, np.arange(n))
    finally:
        v.close()
    assert not os.path.exists("/dev/shm" + name)                 # the creator unlinks the name


def test_a_reader_does_not_unlink_and_a_second_create_starts_afresh():
    name = _name("again")
    v = capi.SharedHostVector(name, 8, create=True)
    w = capi.SharedHostVector(name, 8, create=False)
    w.array[3] = 5.0
    assert v.array[3] == 5.0
    w.close()
    assert os.path.exists("/dev/shm" + name)
    u = capi.SharedHostVector(name, 8, create=True)              # replaces the name; the old mapping lives on by itself
    assert not u.array.any() and v.array[3] == 5.0
    for x in (u, v):
        x.close()
    assert not os.path.exists("/dev/shm" + name)


@pytest.mark.gpu
@pytest.mark.parametrize("n,offset", [(1, 0), (3, 7), (513, 511), (250_000, 1), (1_000_003, 12_345)])
def test_device_slices_arrive_and_nothing_else_is_written(n, offset):
    import torch
    assert torch.cuda.is_available(), "gpu-marked tests need a GPU"
    total = offset + n + 9
    v = capi.SharedHostVector(_name(f"dev_{n}"), total, create=True)
    try:
        v.array[:] = -1.0
        s = torch.cuda.Stream()
        for turn in range(3):
            src = torch.empty(n, dtype=torch.float64, device="cuda")
            with torch.cuda.stream(s):
                capi.gen_values_device(src, 42 + turn, 0, 0)     # the copy has to wait for the kernel in front of it
                v.copy_from_device(src, offset, stream=s)
            s.synchronize()
            assert np.array_equal(v.array[offset:offset + n], src.cpu().numpy())
            assert (v.array[:offset] == -1.0).all() and (v.array[offset + n:] == -1.0).all()
        torch.cuda.synchronize()
        assert float(torch.ones(4, device="cuda").sum()) == 4.0  # no error is left behind for the next call
    finally:
        v.close()


@pytest.mark.gpu
def test_page_locked_destinations_still_take_the_copy_kernel():
    import torch
    src = torch.arange(1001, dtype=torch.float64, device="cuda")
    dst = torch.full((1010,), -1.0, dtype=torch.float64, pin_memory=True)
    s = torch.cuda.current_stream()
    rc = capi.load().rsp_copy_to_host_async(ctypes.c_void_p(src.data_ptr()), ctypes.c_void_p(dst.data_ptr() + 8 * 4), 1001,
                                            ctypes.c_void_p(s.cuda_stream))
    assert rc == capi.RSP_OK
    s.synchronize()
    assert torch.equal(dst[4:1005], torch.arange(1001, dtype=torch.float64))
    assert (dst[:4] == -1).all() and (dst[1005:] == -1).all()
