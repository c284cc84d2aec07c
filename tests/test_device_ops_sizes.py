"""Sizes that a C int does not hold are refused, not cut to their low 32 bits.  No GPU: ops_engine.c built against stand-ins
(fake_cuda.c); the tensors repeat a few values."""
import ctypes as C
import os
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
OVER = 1 << 32


@pytest.fixture
def ops(fb, tmp_path, monkeypatch):
    from fomoe_b200 import device_ops
    so = str(tmp_path / "libfake_ops.so")
    subprocess.run(["gcc", "-std=c11", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I/usr/local/cuda/include", "-w", "-o", so,
                    os.path.join(HERE, "fake_cuda.c"), os.path.join(ROOT, "fomoe_b200", "csrc", "ops_engine.c")], check=True)
    fake = C.CDLL(so)
    for name, (res, args) in device_ops.SIGS.items():
        f = getattr(fake, name)
        f.restype, f.argtypes = res, args
    monkeypatch.setattr(fb, "_lib", fake)
    o = fb.DeviceOps(0)
    o.device = -1   # where CPU tensors are
    o._stream = lambda: 0
    o.fake = fake
    yield o
    o.close()


def refused(ops, call):
    n = C.c_int.in_dll(ops.fake, "fake_launches")
    before = n.value
    with pytest.raises((ValueError, RuntimeError), match="rows|columns|2\\^31|top_k|n_group"):   # (not torch's out of memory)
        call()
    assert n.value == before


def many(rows, cols, dt=torch.float32):
    return torch.zeros(cols, dtype=dt).expand(rows, cols)


def test_rows_and_columns(ops):
    f8 = torch.float8_e4m3fn
    q = torch.zeros(1, 16, dtype=torch.uint8).view(f8)
    qs = torch.zeros(1, 1)
    for over in (OVER + 1, OVER + 2, (1 << 31) + 1):
        refused(ops, lambda: ops.route(many(over, 4), 2))
        refused(ops, lambda: ops.norm(many(over, 4), torch.ones(4)))
        refused(ops, lambda: ops.f8_quantize(many(over, 4)))
        refused(ops, lambda: ops.f8_matmul(q.expand(over, 16), many(over, 1), q, qs))
        refused(ops, lambda: ops.f8_matmul(q, qs, q.expand(over, 16), qs.expand(-(-over // 128), 1)))


def test_counts(ops):
    x = torch.zeros(3, 64)
    for over in (OVER + 2, -OVER + 2, 1 << 31):
        refused(ops, lambda: ops.route(x, over))
        refused(ops, lambda: ops.route(x, 2, n_group=over))
        refused(ops, lambda: ops.route(x, 2, n_group=4, topk_group=over))
        refused(ops, lambda: ops.route(x, 2, n_group=4, topk_group=2, group_best=over))
        for i in range(5):
            sizes = [3, 256, 128, 4, 2]
            assert ops.f8_experts_workspace(*sizes) > 0
            sizes[i] += over - over % 4
            assert ops.f8_experts_workspace(*sizes) == 0
