"""FP8 experts whose results can be written down: every step of them is exact in fp32, so there is no tolerance."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(fb):
    o = fb.DeviceOps(0)
    yield o
    torch.cuda.synchronize()
    assert o.status() == 0
    o.close()


def f8(t):
    q = t.to(torch.float8_e4m3fn)
    assert (q.float() == t).all()
    return q.cuda()


@pytest.mark.parametrize("T", [1, 300])
@pytest.mark.parametrize("H", [128, 640])
def test_outputs_of_experts_that_cancel(ops, T, H):
    """y_0 = 3584 + n % 8 and y_1 = 3584 with weights 1 and -1: what is left is n % 8.  silu(32) is 32 in fp32
    (exp(-32) < 2^-24), the activations are 448, 1 and zeros with scale 1, sums stay below 2^24."""
    I, E = 128, 2
    x = torch.zeros(T, H)
    x[:, 0] = 1.0
    gu = torch.zeros(E, 2 * I, H)
    gu[:, :I, 0] = 32.0
    gu[:, I, 0], gu[:, I + 1, 0] = 14.0, 2.0 ** -5
    dn = torch.zeros(E, H, I)
    dn[:, :, 0] = 8.0
    dn[0, :, 1] = torch.arange(H) % 8
    ones = lambda *s: torch.ones(*s, device="cuda")  # noqa: E731
    ids = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda").repeat(T, 1)
    w = torch.tensor([[1.0, -1.0]], device="cuda").repeat(T, 1)
    out = ops.f8_experts(f8(x), ones(T, H // 128), ids, w, f8(gu), ones(E, 2, H // 128), f8(dn), ones(E, H // 128, 1))
    assert (out.float().cpu() == (torch.arange(H) % 8).float()).all()


@pytest.mark.parametrize("T", [1, 300])
def test_activations_on_borders_go_to_even(ops, T):
    """Activations that lie exactly between two e4m3 numbers: act = 32 u, a block's largest is 448 s with s = m / 16, and
    act = t s with t = 17, 21, 25, 29, whose even neighbour is t - 1.  For these m the rounded 1 / s times act is above t."""
    ms, ts, H = [7, 13, 14, 26, 28, 52, 56], [17, 21, 25, 29], 128
    I, E = 128 * len(ms), 1
    digits = [2.0 ** 3, 1.0, 2.0 ** -3, 2.0 ** -6, 2.0 ** -9]
    x = torch.zeros(T, H)
    x[:, 0] = 1.0
    x[:, 1:6] = torch.tensor(digits)
    gu = torch.zeros(E, 2 * I, H)
    gu[:, :I, 0] = 32.0
    dn = torch.zeros(E, H, I)
    want = torch.zeros(H)
    for b, m in enumerate(ms):
        for r, v in enumerate([448] + ts):
            n = v * m   # act = n / 16, u = n / 512 in digits of base 8
            for k in range(5):
                gu[0, I + 128 * b + r, 1 + k] = (n >> (3 * (4 - k))) & 7
            assert n < 1 << 15
            if r:
                dn[0, 4 * b + r - 1, 128 * b + r] = 1.0
                want[4 * b + r - 1] = (v - 1) * m / 16
    s1 = lambda *s: torch.ones(*s, device="cuda")  # noqa: E731
    ids, w = torch.zeros(T, 1, dtype=torch.int32, device="cuda"), s1(T, 1)
    out = ops.f8_experts(f8(x), s1(T, 1), ids, w, f8(gu), s1(E, 2 * I // 128, 1), f8(dn), s1(E, 1, I // 128))
    assert (out.cpu() == want.bfloat16()).all()
