"""The operators on device memory at the ends of the ranges that they take."""
import pytest
import torch

from test_gpu_device_ops import experts64, make_experts, within

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


# ------------------------------------------------------------------ experts
@pytest.mark.parametrize("T,H,I,E,k,shared", [
    (1, 8320, 128, 4, 2, True), (2, 16384, 128, 3, 2, False),     # single pairs, more than 64 blocks of k in gate/up
    (1, 128, 16384, 6, 5, False), (1, 128, 16384, 6, 6, False), (1, 128, 8192, 16, 16, True),   # a token's activations: 80, 96, 136 KB
    (40, 16384, 128, 3, 2, True), (90, 256, 16384, 3, 3, False)])
def test_experts_widest(ops, T, H, I, E, k, shared):
    x, ids, w, gu, gus, dn, dns = make_experts(T + H + I, T, H, I, E, k, shared)
    xq, xs = ops.f8_quantize(x)
    out = ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns, shared=shared)
    want, tol = experts64(xq, xs, ids, w, gu, gus, dn, dns, shared)
    within(out, want, tol)


@pytest.mark.parametrize("shared", [False, True])
def test_experts_of_very_many_tokens(ops, shared):
    """264,000 pairs: buckets by runs of more than 4096 pairs a block, the sums by more than one launch (65,535 tokens in
    one).  A token's result does not depend on the others, to the bit."""
    T, H, I, E, k = 66000, 128, 128, 7, 4
    x, ids, w, gu, gus, dn, dns = make_experts(3, T, H, I, E, k, shared, 0.1)
    xq, xs = ops.f8_quantize(x)
    out = ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns, shared=shared)
    for t in (slice(0, 700), slice(32000, 33000), slice(65000, 66000)):
        part = ops.f8_experts(xq[t], xs[t], ids[t].contiguous(), w[t].contiguous(), gu, gus, dn, dns, shared=shared)
        assert (part == out[t]).all()
    want, tol = experts64(xq, xs, ids, w, gu, gus, dn, dns, shared)
    within(out, want, tol)


@pytest.mark.parametrize("T", [2, 50])
def test_experts_infinite_weights(ops, T):
    """An infinite weight makes its own token infinite or NaN; one of a slot that is left out does nothing."""
    x, ids, w, gu, gus, dn, dns = make_experts(T, T, 256, 128, 4, 2, False)
    xq, xs = ops.f8_quantize(x)
    clean = ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns)
    w[0, 1] = float("inf")
    out = ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns)
    assert not torch.isfinite(out[0]).any() and (out[1:] == clean[1:]).all()
    ids[0, 1] = -1
    assert torch.isfinite(ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns)).all()
