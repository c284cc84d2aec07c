"""What the operators on device memory launch, and what they make of CUDA's errors.  No GPU: the library's own launchers over
stand-ins for the CUDA runtime (fake_cudart.c)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="module")
def fake(fb, tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake") / "libfake_launch.so")
    build = os.path.join(ROOT, "fomoe_b200", "csrc", "build")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-w", "-o", so, os.path.join(HERE, "fake_cudart.c")] +
                   [os.path.join(build, n + ".o") for n in ("ops_engine", "ops_rows", "ops_f8")] + ["-lstdc++", "-lm"], check=True)
    return C.CDLL(so)


@pytest.fixture
def ops(fb, fake, monkeypatch):
    from fomoe_b200 import device_ops
    for name, (res, args) in device_ops.SIGS.items():
        f = getattr(fake, name)
        f.restype, f.argtypes = res, args
    monkeypatch.setattr(fb, "_lib", fake)
    o = fb.DeviceOps(0)
    o.device = -1   # where CPU tensors are
    o._stream = lambda: 0
    o.fake = fake
    yield o
    for name, v in (("fake_launches", 0), ("fake_fail_at", -1), ("fake_last", 0)):
        C.c_int.in_dll(fake, name).value = v
    o.close()


def word(ops, name):
    return C.c_int.in_dll(ops.fake, name)


def launched(ops):
    """The kernels launched since the last call of this function, with their grids."""
    n = word(ops, "fake_launches").value
    names, grids = (C.c_char_p * 64).in_dll(ops.fake, "fake_name"), (C.c_uint * 192).in_dll(ops.fake, "fake_grid")
    word(ops, "fake_launches").value = 0
    return [(names[i].decode(), tuple(grids[3 * i:3 * i + 3])) for i in range(min(n, 64))]


def q8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def experts_call(ops, T, H=256, I=128, E=4, k=2, shared=True):
    R = E + shared
    raw = torch.empty(ops.f8_experts_workspace(T, H, I, E, k, shared) + 256, dtype=torch.uint8)   # (torch aligns CPU tensors to 64 bytes)
    return ops.f8_experts(q8(T, H), torch.zeros(T, H // 128), torch.zeros(T, k, dtype=torch.int32), torch.zeros(T, k), q8(R, 2 * I, H),
                          torch.zeros(R, 2 * I // 128, H // 128), q8(R, H, I), torch.zeros(R, H // 128, I // 128), shared=shared,
                          workspace=raw[-raw.data_ptr() % 256:][:raw.numel() - 256])


def product(ops, m, n=130, k=208):
    nb = (k + 127) // 128
    return ops.f8_matmul(q8(m, k), torch.zeros(m, nb), q8(n, k), torch.zeros((n + 127) // 128, nb))


CALLS = {"route": lambda o: o.route(torch.zeros(3, 64), 4), "norm": lambda o: o.norm(torch.zeros(3, 40), torch.ones(40)),
         "norm odd": lambda o: o.norm(torch.zeros(3, 41), torch.ones(41)), "quantize": lambda o: o.f8_quantize(torch.zeros(3, 200)),
         "quantize odd": lambda o: o.f8_quantize(torch.zeros(3, 203)), "few": lambda o: product(o, 5), "few 16": lambda o: product(o, 12),
         "product": lambda o: product(o, 40), "product large": lambda o: product(o, 2048, 2048, 2048),
         "experts few": lambda o: experts_call(o, 1), "experts": lambda o: experts_call(o, 300),
         "experts, bucket of many blocks": lambda o: experts_call(o, 5000)}
KERNELS = {"experts few": 2, "experts": 5, "experts, bucket of many blocks": 6}


@pytest.mark.parametrize("call", CALLS)
def test_an_error_that_was_there_before_is_not_this_call_s(ops, call):
    """An earlier call's error (600: a query that found its event not ready) is still the last one: the call does all of its
    work, succeeds, and leaves that error to whom it belongs."""
    word(ops, "fake_last").value = 600
    before = ops.kernel_launches()
    CALLS[call](ops)
    assert len(launched(ops)) == KERNELS.get(call, 1) == ops.kernel_launches() - before
    assert word(ops, "fake_last").value == 600


@pytest.mark.parametrize("call", CALLS)
def test_a_launch_that_fails_ends_the_call(ops, call):
    """Nothing is launched after it, the call says so, and its error is not left for others to find."""
    for at in range(KERNELS.get(call, 1)):
        word(ops, "fake_fail_at").value = at
        before = ops.kernel_launches()
        with pytest.raises(RuntimeError, match="launch failed"):
            CALLS[call](ops)
        assert len(launched(ops)) == at and ops.kernel_launches() == before
        assert word(ops, "fake_last").value == 0
