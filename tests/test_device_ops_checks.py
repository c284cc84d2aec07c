"""What the operators on device memory refuse, without a GPU: ops_engine.c built against stand-ins for the CUDA runtime and
the launchers (fake_cuda.c), called through the Python mirror with CPU tensors."""
import ctypes as C
import os
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake") / "libfake_ops.so")
    subprocess.run(["gcc", "-std=c11", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I/usr/local/cuda/include", "-w", "-o", so,
                    os.path.join(HERE, "fake_cuda.c"), os.path.join(ROOT, "fomoe_b200", "csrc", "ops_engine.c")], check=True)
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
    o.close()


def launches(ops):
    return C.c_int.in_dll(ops.fake, "fake_launches").value


def refused(ops, call, what=None, error=(RuntimeError, ValueError)):
    n = launches(ops)
    with pytest.raises(error, match=what):
        call()
    assert launches(ops) == n


def q8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def test_create_refuses_a_device_that_is_not_there(fb, fake, ops):
    with pytest.raises(RuntimeError):
        fb.DeviceOps(5)
    with pytest.raises(RuntimeError):
        fb.DeviceOps(-1)


def test_route(ops):
    x = torch.zeros(3, 64)
    ids, w = ops.route(x, 4)
    assert ids.shape == w.shape == (3, 4) and ids.dtype == torch.int32 and launches(ops) >= 1
    ops.route(x.bfloat16(), 16, score="sigmoid", bias=torch.zeros(64), n_group=8, topk_group=2, group_best=2,
              valid=torch.ones(3, dtype=torch.bool))
    ops.route(torch.zeros(5, 100)[:, 3:67], 4)   # strided rows
    n = launches(ops)
    assert ops.route(torch.zeros(0, 64), 4)[0].shape == (0, 4) and launches(ops) == n
    for kw in (dict(top_k=0), dict(top_k=17), dict(top_k=65), dict(top_k=4, n_group=7), dict(top_k=4, n_group=64),
               dict(top_k=4, n_group=0), dict(top_k=4, n_group=4, topk_group=5), dict(top_k=4, n_group=4, topk_group=0),
               dict(top_k=4, group_best=3), dict(top_k=4, score="relu"), dict(top_k=4, bias=torch.zeros(63)),
               dict(top_k=4, bias=torch.zeros(64).double()), dict(top_k=4, valid=torch.ones(2, dtype=torch.bool)),
               dict(top_k=-1)):
        refused(ops, lambda: ops.route(x, **kw))
    refused(ops, lambda: ops.route(torch.zeros(2, 8), 9), "top_k")
    refused(ops, lambda: ops.route(torch.zeros(2, 513), 4), "experts")
    refused(ops, lambda: ops.route(x.double(), 4), "logits", ValueError)
    refused(ops, lambda: ops.route(x.half(), 4), "logits", ValueError)
    refused(ops, lambda: ops.route(x.t(), 2), "contiguous", ValueError)
    refused(ops, lambda: ops.route(torch.zeros(1, 64).expand(3, 64), 4), "row_stride")


def test_norm(ops):
    x, blk, w = torch.zeros(3, 40), torch.zeros(3, 40).bfloat16(), torch.ones(40)
    for g in (torch.zeros(3, 40), torch.zeros(1, 40), torch.zeros(3, 1), torch.zeros(1, 1)):
        ops.norm(x, w, block=blk, post=w, gate=g.bfloat16(), out="f8")
    assert len(ops.norm(x, w, out="f8")) == 3 and len(ops.norm(x, w, block=blk)) == 2
    assert ops.norm(x, w, out="f32")[0] is x and ops.norm(x, block=blk, inplace=True)[0] is x
    assert ops.norm(x, block=blk)[1] is None
    n = launches(ops)
    ops.norm(torch.zeros(0, 40), w)
    assert launches(ops) == n
    refused(ops, lambda: ops.norm(x))
    refused(ops, lambda: ops.norm(x, w, out="f16"), "out", ValueError)
    refused(ops, lambda: ops.norm(x, w, post=w), "block", ValueError)
    refused(ops, lambda: ops.norm(x, w, gate=blk), "block", ValueError)
    refused(ops, lambda: ops.norm(x, w[:39]), "pre", ValueError)
    refused(ops, lambda: ops.norm(x, w.double()), "pre", ValueError)
    refused(ops, lambda: ops.norm(x, w, block=blk[:2]), "block", ValueError)
    refused(ops, lambda: ops.norm(x, w, block=blk, gate=torch.zeros(3, 40)), "gate", ValueError)
    refused(ops, lambda: ops.norm(x, w, block=blk, gate=torch.zeros(2, 40).bfloat16()), "gate", ValueError)
    refused(ops, lambda: ops.norm(torch.zeros(40), w), "x", ValueError)
    refused(ops, lambda: ops.norm(torch.zeros(2, 16385), torch.zeros(16385)), "columns")
    refused(ops, lambda: ops.norm(torch.zeros(1, 40).expand(3, 40), w), "x_stride")


def test_quantize_and_matmul(ops):
    x = torch.zeros(3, 200)
    q, s = ops.f8_quantize(x)
    assert q.shape == (3, 200) and s.shape == (3, 2)
    refused(ops, lambda: ops.f8_quantize(x.double()), "x", ValueError)
    refused(ops, lambda: ops.f8_quantize(x[0]), "x", ValueError)
    refused(ops, lambda: ops.f8_quantize(torch.zeros(3, 0)))
    a, sa, b, sb = q8(5, 208), torch.zeros(5, 2), q8(130, 208), torch.zeros(2, 2)
    assert ops.f8_matmul(a, sa, b, sb).dtype == torch.bfloat16 and ops.f8_matmul(a, sa, b, sb, out="f32").shape == (5, 130)
    ops.f8_matmul(q8(1, 208).as_strided((1, 208), (7, 1)), sa[:1], b, sb)   # one row: its stride means nothing
    n = launches(ops)
    assert ops.f8_matmul(q8(0, 208), torch.zeros(0, 2), b, sb).shape == (0, 130) and launches(ops) == n
    refused(ops, lambda: ops.f8_matmul(q8(5, 200), sa, q8(130, 200), sb), "multiple of 16")
    refused(ops, lambda: ops.f8_matmul(q8(5, 216)[:, :208], sa, b, sb), "strides")
    refused(ops, lambda: ops.f8_matmul(q8(5 * 224).as_strided((5, 208), (224, 1), 1), sa, b, sb), "aligned")
    refused(ops, lambda: ops.f8_matmul(a, sa, q8(130, 224), sb), "columns", ValueError)
    refused(ops, lambda: ops.f8_matmul(a, sa[:4], b, sb), "a_scales", ValueError)
    refused(ops, lambda: ops.f8_matmul(a, sa, b, sb[:1]), "b_scales", ValueError)
    refused(ops, lambda: ops.f8_matmul(a, sa, b, sb, out="f8"), "out", ValueError)
    refused(ops, lambda: ops.f8_matmul(a.float(), sa, b, sb), "a", ValueError)
    refused(ops, lambda: ops.f8_matmul(q8(1, 208).expand(5, 208), sa, b, sb), "below k")


def experts_args(T=3, H=256, I=128, E=4, k=2, shared=1):
    R = E + shared
    return dict(x=q8(T, H), x_scales=torch.zeros(T, H // 128), ids=torch.zeros(T, k, dtype=torch.int32),
                weights=torch.zeros(T, k), gate_up=q8(R, 2 * I, H), gate_up_scales=torch.zeros(R, 2 * I // 128, H // 128),
                down=q8(R, H, I), down_scales=torch.zeros(R, H // 128, I // 128), shared=bool(shared))


def test_experts(ops):
    a = experts_args()
    # (torch aligns CPU tensors to 64 bytes: the workspace of these tests is cut out at a multiple of 256)
    raw = torch.zeros(1 << 16, dtype=torch.uint8)
    ws = raw[-raw.data_ptr() % 256:][:1 << 15]
    assert ops.f8_experts(**a, workspace=ws).shape == (3, 256)
    n = launches(ops)
    assert ops.f8_experts(**experts_args(T=0), workspace=ws).shape == (0, 256) and launches(ops) == n
    assert ops.f8_experts_workspace(3, 256, 128, 4, 2, True) > 0
    for sizes in ((3, 200, 128, 4, 2), (3, 256, 100, 4, 2), (3, 256, 128, 513, 2), (3, 256, 128, 4, 17), (3, 256, 128, 4, 0),
                  (3, 256, 128, 0, 2), (-1, 256, 128, 4, 2), (3, 32768, 128, 4, 2), (1 << 22, 256, 128, 4, 2)):
        assert ops.f8_experts_workspace(*sizes) == 0
    refused(ops, lambda: ops.f8_experts(**a, workspace=ws[:1000]), "workspace")
    refused(ops, lambda: ops.f8_experts(**a, workspace=ws[16:]), "workspace")
    bad = [dict(ids=a["ids"].long()), dict(ids=a["ids"][:2]), dict(ids=a["ids"][0]), dict(weights=a["weights"].double()),
           dict(x_scales=torch.zeros(3, 1)), dict(gate_up=q8(4, 256, 256)), dict(down=q8(5, 256, 256)),
           dict(down_scales=torch.zeros(5, 2, 2)), dict(gate_up_scales=torch.zeros(5, 1, 2)), dict(x=q8(3, 128)),
           dict(x=torch.zeros(3, 256)), dict(gate_up=q8(5, 192, 256)), dict(gate_up=q8(5, 256, 512)[:, :, :256])]
    for b in bad:
        refused(ops, lambda: ops.f8_experts(**{**a, **b}, workspace=ws))
    refused(ops, lambda: ops.f8_experts(**{**a, "x": q8(3, 264)[:, :256]}, workspace=ws), "x_stride")


def test_other_device_is_current_again_and_a_failed_launch_is_reported(ops):
    dev = ops.fake.cudaSetDevice
    dev(1)
    ops.route(torch.zeros(2, 8), 2)
    got = C.c_int()
    ops.fake.cudaGetDevice(C.byref(got))
    assert got.value == 1 and C.c_int.in_dll(ops.fake, "fake_launch_device").value == 0
    fail = C.c_int.in_dll(ops.fake, "fake_fail")
    fail.value = 1
    before = ops.kernel_launches()
    with pytest.raises(RuntimeError, match="launch failed"):
        ops.route(torch.zeros(2, 8), 2)
    fail.value = 0
    ops.fake.cudaGetDevice(C.byref(got))
    assert got.value == 1 and ops.kernel_launches() == before
    dev(0)


def test_matmul_limits(ops):
    """The largest sizes whose coordinates fit, and the next ones (the launcher is a stand-in: nothing is read)."""
    from fomoe_b200.device_ops import F32, MatmulArgs

    def call(m, n, k):
        nb = (k + 127) // 128
        return ops._l.fomoe_b200_ops_f8_matmul(ops._h, MatmulArgs(m, n, k, 1 << 20, k, 1 << 20, nb, 1 << 20, k, 1 << 20, nb, 1 << 20,
                                                                 F32, n), None)
    assert call(32, 1 << 29, 16) == 0 and call(1 << 30, 16, 16) == 0 and call(1, 1, 1 << 30) == 0
    n = launches(ops)
    assert call(32, (1 << 29) + 1, 16) == -1 and call((1 << 30) + 1, 16, 16) == -1 and call(1, 1, (1 << 30) + 16) == -1
    assert launches(ops) == n
