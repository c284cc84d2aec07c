"""The handle of the operators on device memory: what it leaves behind when it goes, and what its status tells.  No GPU:
ops_engine.c built against stand-ins (fake_cuda_status.c)."""
import ctypes as C
import gc
import os
import subprocess
import types

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake") / "libfake_status.so")
    subprocess.run(["gcc", "-std=c11", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I/usr/local/cuda/include", "-w", "-o", so,
                    os.path.join(HERE, "fake_cuda_status.c"), os.path.join(ROOT, "fomoe_b200", "csrc", "ops_engine.c")], check=True)
    return C.CDLL(so)


@pytest.fixture
def make(fb, fake, monkeypatch):
    from fomoe_b200 import device_ops
    for name, (res, args) in device_ops.SIGS.items():
        f = getattr(fake, name)
        f.restype, f.argtypes = res, args
    monkeypatch.setattr(fb, "_lib", fake)

    def new():
        o = fb.DeviceOps(0)
        o.device = -1   # where CPU tensors are
        o._stream = lambda: 0
        return o
    return new


def product(o):
    q = torch.zeros(1, 16, dtype=torch.uint8).view(torch.float8_e4m3fn)
    o.f8_matmul(q, torch.zeros(1, 1), q, torch.zeros(1, 1))


def freed(fake):
    return C.c_int.in_dll(fake, "fake_freed").value


@pytest.mark.parametrize("how", ["close", "collected"])
def test_captured_calls_outlive_their_handle(make, fake, how):
    """A graph goes on storing into the status words of the handle that it was captured with."""
    o = make()
    product(o)
    n = freed(fake)
    if how == "close":
        o.close()
    del o
    gc.collect()
    assert freed(fake) == n
    fake.fake_goes_wrong(1)
    after = make()
    assert after.status() == 0   # and a later handle does not hear of it
    product(after)
    fake.fake_goes_wrong(1)
    assert after.status() == 1


def test_neither_fault_hides_the_other(make, fake):
    o = make()
    product(o)
    for order in ((1, 2), (2, 1)):
        for what in order:
            fake.fake_goes_wrong(what)
        assert [o.status() for _ in range(3)] == [2, 1, 0]


def test_a_handle_goes_without_touching_the_device(make):
    """Whoever drops it, wherever: a wait would end a capture of another thread or stream."""
    o = make()
    asked = []

    class Cuda(types.SimpleNamespace):
        def __getattr__(self, name):
            asked.append(name)
            return lambda *a: False
    o._t = types.SimpleNamespace(cuda=Cuda())
    del o
    gc.collect()
    assert asked == []
