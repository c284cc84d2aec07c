"""The operators on device memory at the ends of the ranges that they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops(fb):
    o = fb.DeviceOps(0)
    yield o
    torch.cuda.synchronize()
    assert o.status() == 0
    o.close()
    torch.cuda.empty_cache()


def test_widest_product_in_f32_without_alignment(ops):
    """2^29 columns of f32 are 2^31 bytes a row; rows that are not 16-byte aligned leave by plain stores.  (46 GB)"""
    from fomoe_b200.device_ops import F32, MatmulArgs
    M, N, K = 17, 1 << 29, 16
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("less than 60 GB free")
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    a = torch.randint(0, 0x60, (M, K), generator=g, device="cuda", dtype=torch.uint8)
    b = torch.randint(0, 0x60, (N, K), generator=g, device="cuda", dtype=torch.uint8)
    sa = torch.rand(M, 1, generator=g, device="cuda")
    sb = torch.rand(N // 128, 1, generator=g, device="cuda")
    out = torch.full((M * N + 1,), float("nan"), device="cuda")[1:].view(M, N)
    args = MatmulArgs(M, N, K, a.data_ptr(), K, sa.data_ptr(), 1, b.data_ptr(), K, sb.data_ptr(), 1, out.data_ptr(), F32, N)
    ops._ck(ops._l.fomoe_b200_ops_f8_matmul(ops._h, args, torch.cuda.current_stream().cuda_stream), "matmul")
    A = a.view(torch.float8_e4m3fn).double() * sa.double()
    for c in (0, 128, 1 << 20, (1 << 28) - 128, N - 640):
        n = slice(c, c + 640)
        want = A @ (b[n].view(torch.float8_e4m3fn).double() * sb[c // 128:c // 128 + 5].double().repeat_interleave(128, 0)).T
        # positive terms: 16 products and their sum, the scales' product and one more
        assert ((out[:, n].double() - want).abs() <= 20 * U * want).all(), c
    assert not any(bool(out[m].isnan().any()) for m in range(M))
