"""The operators on device memory against plain 64-bit implementations of their formulas.

Tolerances count roundings.  U = 2^-24 is half a step of fp32; sums of n terms by any order are off by at most n U times
the sum of the terms' magnitudes; an output in bf16 (e4m3) is off by half a step more, 2^-8 (2^-4) of its value."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -100
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ops(fb):
    o = fb.DeviceOps(0)
    yield o
    torch.cuda.synchronize()
    assert o.status() == 0
    o.close()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def within(got, want, tol, what=""):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(((got - want).abs() / tol).nan_to_num(1e9).max()))


# ------------------------------------------------------------------ routing
def route64(x, k, score="softmax", bias=None, n_group=1, topk_group=1, group_best=1, renorm=True, scale=1.0, valid=None):
    x = x.float().cpu().numpy().astype(np.float64)
    T, E = x.shape
    b = np.zeros(E) if bias is None else bias.cpu().numpy().astype(np.float64)
    ids, w = np.full((T, k), -1), np.zeros((T, k))
    for t in range(T):
        open_ = x[t] > -np.inf
        if valid is not None and not bool(valid[t]):
            open_[:] = False
        v = np.where(open_, np.minimum(x[t], np.finfo(np.float32).max), -np.inf)
        with np.errstate(all="ignore"):
            if score == "sigmoid":
                p = np.where(open_, 1 / (1 + np.exp(-v)), 0.0)
            else:
                p = np.where(open_, np.exp(v - v.max()), 0.0) if open_.any() else np.zeros(E)
                p = p / p.sum() if p.sum() > 0 else p
            c = p + b
        open_ &= c > -np.inf
        key = np.where(open_, v if bias is None else c, -np.inf)
        if n_group > 1:
            per = E // n_group
            gs = np.full(n_group, -np.inf)
            for g in range(n_group):
                m = np.sort(c[g * per:(g + 1) * per][open_[g * per:(g + 1) * per]])[::-1][:group_best]
                if m.size:
                    gs[g] = m.sum()
            stay = sorted(range(n_group), key=lambda g: (-gs[g], g))[:topk_group]
            for g in range(n_group):
                if g not in stay:
                    key[g * per:(g + 1) * per] = -np.inf
        best = [e for e in sorted(range(E), key=lambda e: (-key[e], e)) if key[e] > -np.inf][:k]
        ids[t, :len(best)] = best
        w[t, :len(best)] = p[best]
    if renorm:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return ids, w * scale


def check_route(ops, x, k, **kw):
    ids, w = ops.route(x, k, **kw)
    ri, rw = route64(x, k, **kw)
    assert (ids.cpu().numpy() == ri).all(), np.argwhere(ids.cpu().numpy() != ri)[:5]
    # p: an exp of a rounded argument (|x - max| U with |x - max| p below 0.4), 2 steps of exp, a sum of 16 terms a lane and
    # five levels, a quotient; then the sum over the slots, a quotient and the scale: under 64 U of a weight
    within(w.cpu(), torch.from_numpy(rw), 64 * U * torch.from_numpy(rw).abs() + 1e-37)


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 512, 10), (3, 33, 16), (67, 64, 6), (130, 257, 8), (515, 384, 8), (9, 16, 16)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_route(ops, T, E, k, score, bias, dt):
    g = gen(T * 1000 + E)
    x = (1.5 * randn(g, T, E)).to(dt)
    b = 0.1 * randn(g, E) if bias else None
    check_route(ops, x, k, score=score, bias=b, scale=2.5)
    check_route(ops, x, k, score=score, bias=b, renorm=False)


@pytest.mark.parametrize("T,E,G,kg,k", [(1, 256, 8, 4, 8), (77, 256, 8, 1, 8), (33, 96, 32, 3, 8), (50, 142, 2, 1, 16), (20, 64, 4, 4, 5), (31, 32, 32, 5, 5)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("bias", [False, True])
def test_route_groups(ops, T, E, G, kg, k, score, best, bias):
    g = gen(T * 100 + E + best)
    x = 1.5 * randn(g, T, E)
    x[torch.rand(T, E, generator=g, device="cuda") < 0.3] = float("-inf")
    check_route(ops, x, k, score=score, bias=0.3 * randn(g, E) if bias else None, n_group=G, topk_group=kg, group_best=best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n_group", [1, 4])
def test_route_closed_and_extreme(ops, score, bias, n_group):
    inf, nan, big = float("inf"), float("nan"), 3.4028234663852886e38
    x = torch.zeros(14, 64)
    x[0] = -inf
    x[1] = nan
    x[2, :] = -inf
    x[2, 7] = -big                                     # one open expert, the type's lowest value
    x[3, 5] = inf
    x[4, [3, 9]] = inf
    x[5, ::2] = nan
    x[6] = -big
    x[7] = -200.0                                      # sigmoid's fp32 value underflows
    x[8] = torch.arange(64) * 3.0                      # softmax underflows for most
    x[9, :] = 1.0                                      # all equal: lowest ids
    x[10] = torch.linspace(20, 40, 64)                 # sigmoid saturates
    x[11, 60:] = 5.0
    x[12] = torch.randn(64)
    x[13] = -torch.linspace(80, 110, 64)
    b = torch.zeros(64)
    if bias:
        b[11], b[12], b[13] = -inf, nan, 3.0
    valid = torch.ones(14, dtype=torch.uint8, device="cuda")
    valid[12] = 0
    with np.errstate(all="ignore"):
        check_route(ops, x.cuda(), 8, score=score, bias=b.cuda() if bias else None, n_group=n_group, topk_group=2 if n_group > 1 else 1,
                    group_best=2, valid=valid)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n_group", [1, 8])
def test_route_near_ties(ops, score, n_group):
    """Choices that differ by less than an fp32 step: the bias cancels the probabilities' differences."""
    g = gen(5)
    x = randn(g, 1, 128).repeat(200, 1)
    x += 1e-6 * randn(g, 200, 128)
    p = torch.softmax(x[0].double(), 0) if score == "softmax" else torch.sigmoid(x[0].double())
    check_route(ops, x, 8, score=score, bias=(0.7 - p).float(), n_group=n_group, topk_group=(n_group + 1) // 2, group_best=2)
    check_route(ops, x, 8, score=score, bias=torch.full((128,), 100.0, device="cuda"), n_group=n_group, topk_group=(n_group + 1) // 2)
    check_route(ops, x.bfloat16(), 8, score=score, n_group=n_group, topk_group=(n_group + 1) // 2)   # many equal logits
    check_route(ops, x.bfloat16(), 8, score=score, bias=torch.zeros(128, device="cuda"), n_group=n_group, topk_group=(n_group + 1) // 2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n_group", [1, 4])
def test_route_infinite_and_huge_bias(ops, score, n_group):
    g = gen(9)
    x = randn(g, 40, 64)
    x[torch.rand(40, 64, generator=g, device="cuda") < 0.2] = float("-inf")
    kw = dict(score=score, n_group=n_group, topk_group=min(2, n_group), group_best=2)
    for where, what in (([3, 9, 40], float("inf")), ([3, 9, 40], 1e30), (list(range(0, 64, 2)), 1e6), (list(range(64)), -1e6),
                        (list(range(1, 64)), float("-inf"))):
        b = 0.1 * randn(g, 64)
        b[where] = what
        check_route(ops, x, 6, bias=b, **kw)


def test_route_strided_rows_and_many_tokens(ops):
    g = gen(8)
    wide = randn(g, 300, 203)
    check_route(ops, wide[:, 3:131], 4, score="sigmoid")
    x = randn(g, 20011, 40)
    ids, w = ops.route(x, 3)
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    assert (ids == i[:, :3]).all()
    within(w, torch.softmax(v[:, :3].double(), 1), 64 * U)


# ------------------------------------------------------------------ norms
def rms64(v, w, eps, offset):
    return v / torch.sqrt(v.pow(2).mean(1, keepdim=True) + eps) * (w.double() + offset)


def step_e4m3(v):
    """The distance between e4m3 numbers around |v| (v: what is rounded, at most 448)."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)


def check_f8(q, s, want, tol):
    """q, s (from a kernel) stand for `want`, which its input's value may be off from by `tol`."""
    T, n = want.shape
    nb = (n + 127) // 128
    pad = lambda v: torch.nn.functional.pad(v, (0, nb * 128 - n)).view(T, nb, 128)  # noqa: E731
    sc = pad(want.abs()).amax(2).clamp(min=TINY) / 448
    within(s, sc, pad(tol).amax(2) / 448 + 4 * U * sc + 1e-45)
    s = s.double().repeat_interleave(128, 1)[:, :n]
    # half a step, the input's own error, and the quotient's and the scale's roundings
    within(q.double() * s, want, 0.5 * 1.001 * step_e4m3((want.abs() + tol) / s) * s + 1.1 * tol + 8 * U * want.abs())


SIZES = [(1, 1), (1, 128), (3, 7), (5, 64), (2, 130), (9, 256), (4, 264), (300, 512), (3, 1000), (2, 1024), (7, 2048),
         (2, 2050), (3, 2880), (1, 4096), (3, 5000), (2, 7177), (2, 8192), (2, 16383), (1, 16384), (1200, 2888), (1190, 4100), (1185, 3001)]


@pytest.mark.parametrize("T,n", SIZES)
@pytest.mark.parametrize("kind", range(6))
def test_norm(ops, T, n, kind):
    g = gen(T * 31 + n * 7 + kind)
    xt, bt = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
              (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)][kind]
    out = ["f32", "bf16", "f8", "f32", "f8", "f8"][kind]
    post = kind in (1, 2, 5)
    gate = [None, (T, n), (1, n), (T, 1), None, (1, 1)][kind]
    scale, offset, eps = (1.0, 0.5, 1.0, -2.0, 1.0, 0.25)[kind], (0.0, 1.0)[kind & 1], (1e-6, 1e-5)[kind & 1]
    x, blk = (3 * randn(g, T, n)).to(xt), randn(g, T, n).to(bt)
    wp, wq = 1 - offset + 0.1 * randn(g, n), 1 - offset + 0.1 * randn(g, n)
    gt = torch.sigmoid(randn(g, *gate)).to(bt) if gate else None
    r = ops.norm(x, wq, block=blk, post=wp if post else None, gate=gt, scale=scale, eps=eps, offset=offset, out=out)
    b = blk.double()
    if post:
        b = rms64(b, wp, eps, offset)
    if gt is not None:
        b = b * gt.double()
    x1 = x.double() + scale * b
    size = x.double().abs() + abs(scale) * b.abs()
    # a sum of n squares, at most n / 256 + 16 additions after one another, so half of that in the root; a dozen roundings
    rel = (n / 512 + 32) * U
    within(r[0], x1, rel * size + HALF[xt] * x1.abs() + 1e-40, "x")
    assert r[0].dtype == xt
    h = rms64(x1, wq, eps, offset)
    # sum over the row of x1's own error, relative to the row's norm, plus the element's
    inv = 1 / torch.sqrt(x1.pow(2).mean(1, keepdim=True) + eps)
    tol = rel * (size * inv * (wq.double() + offset).abs() + 2 * (size.pow(2).mean(1, keepdim=True).sqrt() * inv) * h.abs())
    if out == "f8":
        check_f8(r[1], r[2], h, tol)
    else:
        within(r[1], h, tol + HALF[r[1].dtype] * h.abs() + 1e-40, "h")


def test_norm_parts(ops):
    """Without a block x is left alone; without pre only x' is written; in place equals out of place; rows behind and
    columns beside strided rows stay as they were."""
    g = gen(3)
    x, blk, w = randn(g, 5, 320), randn(g, 5, 320).bfloat16(), torch.ones(320, device="cuda")
    keep = x.clone()
    x0, h = ops.norm(x, w, out="f32")
    assert x0 is x and (x == keep).all()
    within(h, rms64(x.double(), w, 1e-6, 0.0), 64 * U * h.double().abs())
    x1, none = ops.norm(x, block=blk, scale=0.3)
    assert none is None and (x == keep).all()
    x2, h2 = ops.norm(x, w, block=blk, scale=0.3, inplace=True)
    assert x2 is x and (x == x1).all()
    wide = randn(g, 6, 400)
    before = wide.clone()
    y = wide[:4, 8:328]
    want, _ = ops.norm(y.contiguous(), w, block=blk[:4])
    ops.norm(y, w, block=blk[:4], inplace=True)
    assert (y == want).all()
    wide[:4, 8:328] = before[:4, 8:328]
    assert (wide == before).all()
    odd = randn(g, 4, 331)[:, 3:323]   # rows that are not 16-byte aligned
    a, b = ops.norm(odd, w, block=blk[:4], out="f32"), ops.norm(odd.contiguous(), w, block=blk[:4], out="f32")
    assert (a[0] == b[0]).all() and (a[1] == b[1]).all()


def test_norm_extremes(ops):
    w = torch.ones(300, device="cuda")
    x = torch.zeros(4, 300, device="cuda")
    x[1, 5] = float("nan")
    x[2, 5] = float("inf")
    x[3] = 1e-30
    _, h = ops.norm(x, w, out="f32")
    assert (h[0] == 0).all() and h[1].isnan().all() and h[2, 5].isnan() and (h[2, :5] == 0).all()
    within(h[3], torch.full((300,), 1e-27, device="cuda"), 1e-32)
    _, q, s = ops.norm(x, w, out="f8")
    assert (q[0].float() == 0).all() and torch.isfinite(s[0]).all() and s[1].isnan().all()
    # an infinite gate against a block that is zero beside the row's end: nothing leaks from behind the row
    g = torch.full((4, 1), float("inf"), device="cuda")
    x1, _ = ops.norm(torch.ones(4, 300, device="cuda"), w, block=torch.ones(4, 300, device="cuda"), gate=g, out="f32")
    assert x1.isinf().all()


# ------------------------------------------------------------------ FP8
@pytest.mark.parametrize("T,n", [(1, 1), (1, 128), (3, 7), (2, 130), (33, 200), (5, 1000), (700, 2064), (1, 16384)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_quantize(ops, T, n, dt):
    g = gen(T + n)
    x = (torch.exp(3 * randn(g, T, 1)) * randn(g, T, n)).to(dt)
    q, s = ops.f8_quantize(x)
    nb = (n + 127) // 128
    b = torch.nn.functional.pad(x.float(), (0, nb * 128 - n)).view(T, nb, 128)
    amax = b.abs().amax(2).clamp(min=TINY)
    want = torch.div(amax, torch.full_like(amax, 448.0))
    assert (s == want).all()
    wq = torch.div(b, want[:, :, None]).to(torch.float8_e4m3fn).view(T, nb * 128)[:, :n]
    assert (q.float() == wq.float()).all()
    check_f8(q, s, x.double(), torch.zeros(T, n, device="cuda", dtype=torch.float64))
    wide = torch.cat([x, x], 1)[:, n:]   # strided, perhaps unaligned rows
    q2, s2 = ops.f8_quantize(wide)
    assert (q2.view(torch.uint8) == q.view(torch.uint8)).all() and (s2 == s).all()


def test_quotients_are_rounded_once(ops):
    """x / scale for many pairs, as IEEE division rounds it: the e4m3 numbers are the division's."""
    g = gen(77)
    x = (torch.exp2(40 * torch.rand(2000, 1, generator=g, device="cuda") - 20) * randn(g, 2000, 8192)).float()
    # values beside the borders between two e4m3 numbers: (m + 1/2) / 8 of a power of two times the scale
    q, s = ops.f8_quantize(x)
    b = x.view(2000, 64, 128)
    m = torch.randint(0, 240, b.shape, generator=g, device="cuda")
    edge = torch.exp2(torch.div(m, 16, rounding_mode="floor").float() - 7) * (1 + (2 * (m % 8) + 1).float() / 16) * s[:, :, None]
    step = torch.randint(-2, 3, b.shape, generator=g, device="cuda", dtype=torch.int32)
    edge = (edge.view(torch.int32) + step).view(torch.float32)
    edge[:, :, 0] = 448 * s                         # keeps the scale
    y = edge.view(2000, 8192)
    for v in (x, y):
        q, s = ops.f8_quantize(v)
        amax = v.view(2000, 64, 128).abs().amax(2).clamp(min=TINY)
        assert (s == torch.div(amax, torch.full_like(amax, 448.0))).all()
        want = torch.div(v.view(2000, 64, 128), s[:, :, None]).to(torch.float8_e4m3fn).view(2000, 8192)
        assert (q.view(torch.uint8) == want.view(torch.uint8)).all()


def test_quantize_extremes(ops):
    x = torch.zeros(6, 256, device="cuda")
    x[0, 3], x[0, 130] = float("nan"), 5.0
    x[1, 3] = float("inf")
    x[2, 3] = -float("inf")
    x[3, 3] = 3e38
    x[4] = 1e-42
    q, s = ops.f8_quantize(x)
    v = q.float() * s.repeat_interleave(128, 1)
    assert v[:3, :128].isnan().all() and (v[1:3, 128:] == 0).all() and v[0, 130] == 5.0
    within(v[3, 3], torch.tensor(3e38, device="cuda"), 3e38 * 2 * U)
    assert (v[4:] == 0).all() and torch.isfinite(s[3:]).all() and (s[3:] > 0).all()


def f8_table(g, *shape):
    rows, cols = shape[-2:]
    q = (60 * randn(g, *shape)).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.exp(0.3 * randn(g, *shape[:-2], -(-rows // 128), -(-cols // 128))) / (60 * cols ** 0.5)
    return q, s


def rows64(q, s):
    return q.double() * s.double().repeat_interleave(128, 1)[:, :q.shape[1]]


def mat64(q, s):
    return q.double() * s.double().repeat_interleave(128, -2).repeat_interleave(128, -1)[..., :q.shape[-2], :q.shape[-1]]


MNK = [(1, 1, 16), (1, 128, 128), (2, 130, 144), (3, 64, 2064), (7, 1000, 272), (8, 4096, 512), (9, 31, 128), (15, 513, 400),
       (16, 256, 1024), (17, 300, 640), (31, 128, 4096), (33, 257, 256), (64, 2048, 1040), (67, 1000, 2064), (127, 255, 384),
       (128, 256, 128), (129, 129, 160), (200, 1, 512), (255, 640, 2048), (513, 1152, 896), (1025, 520, 256),
       (640, 4001, 144), (1100, 4488, 176), (1281, 4096, 272)]


@pytest.mark.parametrize("M,N,K", MNK)
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_matmul(ops, M, N, K, out):
    g = gen(M * 7 + N * 3 + K)
    a, sa = ops.f8_quantize(randn(g, M, K))
    b, sb = f8_table(g, N, K)
    c = ops.f8_matmul(a, sa, b, sb, out=out)
    A, B = rows64(a, sa), mat64(b, sb)
    want, size = A @ B.T, A.abs() @ B.abs().T
    # a block's 128 products are exact and their sum takes at most 128 roundings; the block's two scales one, the sum of
    # the blocks one each
    tol = (K // 128 + 1 + 130) * U * size + HALF[c.dtype] * want.abs() + 1e-40
    within(c, want, tol)
    # and in the mean, where the roundings' signs differ, far less: the error of 2^-24 steps over sqrt(terms)
    if out == "f32" and M * N > 1000:
        assert float((c.double() - want).norm() / want.norm()) < 2e-6


def test_matmul_strides_and_neighbours(ops):
    """Strided operands; an output inside a larger buffer whose other values stay as they were (through the C entry)."""
    g = gen(12)
    M, N, K = 37, 200, 320
    a, sa = ops.f8_quantize(randn(g, M, K + 32))
    b, sb = f8_table(g, N, K + 64)
    for m in (1, 5, M):
        A, S = a[:m, 16:16 + K], sa[:m]      # (the scales go by column blocks of the slice)
        big = torch.full((m + 2, N + 8), 7.0, device="cuda")
        from fomoe_b200.device_ops import MatmulArgs
        o = big[1:1 + m, 3:3 + N]
        args = MatmulArgs(m, N, K, A.data_ptr(), A.stride(0), S.data_ptr(), S.stride(0), b.data_ptr(), b.stride(0), sb.data_ptr(),
                          sb.stride(0), o.data_ptr(), 0, o.stride(0))
        ops._ck(ops._l.fomoe_b200_ops_f8_matmul(ops._h, args, torch.cuda.current_stream().cuda_stream), "matmul")
        Av, Bv = rows64(A, S[:, :3]), mat64(b[:, :K], sb[:, :3])
        within(o, Av @ Bv.T, 140 * U * (Av.abs() @ Bv.abs().T))
        big[1:1 + m, 3:3 + N] = 7.0
        assert (big == 7.0).all()


def test_matmul_special_values(ops):
    """A NaN stays in its row (or column), an infinite scale in its row; a zero block is nothing."""
    g = gen(2)
    for M in (3, 40, 150):
        a, sa = ops.f8_quantize(randn(g, M, 256))
        b, sb = f8_table(g, 300, 256)
        clean = ops.f8_matmul(a, sa, b, sb, out="f32")
        a.view(torch.uint8)[1, 7] = 0x7f
        b.view(torch.uint8)[5, 200] = 0xff
        got = ops.f8_matmul(a, sa, b, sb, out="f32")
        assert got[1].isnan().all() and got[:, 5].isnan().all()
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[1], keep[:, 5] = False, False
        assert (got[keep] == clean[keep]).all()
        a.zero_()
        b.view(torch.uint8)[5, 200] = 0
        assert (ops.f8_matmul(a, sa, b, sb, out="f32") == 0).all()


# ------------------------------------------------------------------ experts
def experts64(x, xs, ids, w, gu, gus, dn, dns, shared):
    """-> (out, tolerance): the definition in 64 bits, and how far fp32 sums and e4m3 roundings of the activations that lie
    within those sums' error of a border may move it."""
    X = rows64(x, xs)
    T, H = X.shape
    I = gu.shape[1] // 2
    E = gu.shape[0] - int(shared)
    out, tol = torch.zeros(T, H, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e in range(gu.shape[0]):
        if e < E:
            t, j = torch.nonzero(ids == e, as_tuple=True)
            we = w[t, j].double()
        else:
            t, we = torch.arange(T, device="cuda"), torch.ones(T, dtype=torch.float64, device="cuda")
        if not t.numel():
            continue
        G, D = mat64(gu[e], gus[e]), mat64(dn[e], dns[e])
        z = X[t] @ G.T
        ez = (H // 128 + 131) * U * (X[t].abs() @ G.abs().T)
        s = 1 / (1 + torch.exp(-z[:, :I]))
        act = z[:, :I] * s * z[:, I:]
        # silu's slope is below 1.1; silu itself is a handful of roundings (the exp's argument |z| U, |z| silu' is bounded)
        ea = 1.1 * ez[:, :I] * z[:, I:].abs() + ez[:, I:] * (z[:, :I] * s).abs() + 16 * U * act.abs()
        nb = I // 128
        sc = act.view(-1, nb, 128).abs().amax(2).clamp(min=TINY) / 448
        esc = ea.view(-1, nb, 128).amax(2) / 448 + 4 * U * sc
        S, ES = sc.repeat_interleave(128, 1), esc.repeat_interleave(128, 1)
        v = act / S
        ev = ea / S + v.abs() * (ES / S) + 4 * U * v.abs()
        q = v.float().to(torch.float8_e4m3fn).double()
        unsure = ((v + ev).float().to(torch.float8_e4m3fn).double() != (v - ev).float().to(torch.float8_e4m3fn).double())
        eq = torch.where(unsure, step_e4m3(v.abs() + ev) + ev, torch.zeros_like(v))
        y = (q * S) @ D.T
        ey = ((eq * S + q.abs() * ES) @ D.abs().T) + (nb + 131) * U * ((q * S).abs() @ D.abs().T)
        out.index_add_(0, t, we[:, None] * y)
        tol.index_add_(0, t, we.abs()[:, None] * (ey + (ids.shape[1] + 3) * U * y.abs()))
    return out, tol + 2.0 ** -8 * out.abs() + 1e-38


def make_experts(seed, T, H, I, E, k, shared, dropped=0.0, skew=0.7):
    g = gen(seed)
    R = E + int(shared)
    gu, gus = f8_table(g, R, 2 * I, H)
    dn, dns = f8_table(g, R, H, I)
    x = randn(g, T, H)
    lg = randn(g, T, E) + skew * randn(g, 1, E)
    v, ids = torch.topk(lg, k, dim=1) if T else (lg[:, :k], lg[:, :k].long())
    ids = torch.where(torch.rand(T, k, generator=g, device="cuda") < dropped, -1, ids).to(torch.int32)
    return x, ids, torch.softmax(v, 1).contiguous(), gu, gus, dn, dns


EXPERTS = [(1, 128, 128, 1, 1, False, 0.0), (1, 256, 128, 4, 2, True, 0.0), (1, 1024, 512, 32, 10, True, 0.0), (2, 512, 256, 16, 8, False, 0.3),
           (3, 640, 384, 7, 7, True, 0.2), (5, 256, 128, 512, 16, False, 0.0), (13, 384, 640, 9, 3, True, 0.1), (33, 512, 256, 3, 2, False, 0.0),
           (64, 256, 256, 64, 8, True, 0.2), (129, 512, 128, 5, 1, False, 0.0), (257, 384, 384, 4, 3, True, 0.4), (700, 256, 256, 10, 6, False, 0.1),
           (1500, 256, 128, 33, 4, True, 0.0), (2000, 128, 128, 70, 7, True, 0.1),
           (300, 384, 256, 200, 4, True, 0.1), (600, 256, 384, 400, 3, False, 0.3), (90, 128, 1024, 64, 4, True, 0.0)]


@pytest.mark.parametrize("T,H,I,E,k,shared,dropped", EXPERTS)
def test_experts(ops, T, H, I, E, k, shared, dropped):
    x, ids, w, gu, gus, dn, dns = make_experts(T + H + I + E, T, H, I, E, k, shared, dropped)
    xq, xs = ops.f8_quantize(x)
    out = ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns, shared=shared)
    want, tol = experts64(xq, xs, ids, w, gu, gus, dn, dns, shared)
    within(out, want, tol)
    again = ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns, shared=shared)
    assert (again == out).all()      # no order of arrival in the sums


@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_experts_odd_ids(ops, T):
    """No expert at all, one expert twice, everyone at one expert, ids outside the table."""
    x, ids, w, gu, gus, dn, dns = make_experts(T, T, 256, 256, 6, 3, True)
    xq, xs = ops.f8_quantize(x)
    ids[0] = -1
    if T > 1:
        ids[1] = torch.tensor([2, 2, 2], dtype=torch.int32)
    for shared in (True, False):
        tabs = [t if shared else t[:6].contiguous() for t in (gu, gus, dn, dns)]
        out = ops.f8_experts(xq, xs, ids, w, *tabs, shared=shared)
        want, tol = experts64(xq, xs, ids, w, *tabs, shared)
        within(out, want, tol)
        if not shared:
            assert (out[0] == 0).all()
    none = ops.f8_experts(xq, xs, torch.full_like(ids, -1), w, *[t[:6].contiguous() for t in (gu, gus, dn, dns)])
    assert (none == 0).all()
    ids.fill_(4)
    within(ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns, shared=True), *experts64(xq, xs, ids, w, gu, gus, dn, dns, True))
    ids.fill_(-1)
    within(ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns, shared=True), *experts64(xq, xs, ids, w, gu, gus, dn, dns, True))
    ids[T // 2, 1], ids[T - 1, 2] = 6, -7      # the shared record is no routed expert
    torch.cuda.synchronize()
    assert ops.status() == 0
    out = ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns, shared=True)
    within(out, *experts64(xq, xs, torch.full_like(ids, -1), w, gu, gus, dn, dns, True))
    torch.cuda.synchronize()
    assert ops.status() == 1 and ops.status() == 0


def test_experts_special_values(ops):
    """A NaN or an infinite weight stays with its tokens; what a left-out slot's weight holds does not matter."""
    for T in (2, 50):
        x, ids, w, gu, gus, dn, dns = make_experts(T, T, 256, 128, 4, 2, False)
        x[0] = float("nan")
        xq, xs = ops.f8_quantize(x)
        ids[1, 0] = -1
        w[1, 0] = float("nan")
        out = ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns)
        assert out[0].isnan().all() and torch.isfinite(out[1:]).all()
        x[0] = 0.0
        xq, xs = ops.f8_quantize(x)
        assert (ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns)[0] == 0).all()


def test_experts_workspace_contents_do_not_matter(ops):
    for T in (1, 20, 200):
        x, ids, w, gu, gus, dn, dns = make_experts(T, T, 384, 256, 5, 2, True, 0.2)
        xq, xs = ops.f8_quantize(x)
        n = ops.f8_experts_workspace(T, 384, 256, 5, 2, True)
        outs = []
        for fill in (0, 255, 127):
            ws = torch.full((n + 1024,), fill, dtype=torch.uint8, device="cuda")
            outs.append(ops.f8_experts(xq, xs, ids, w, gu, gus, dn, dns, shared=True, workspace=ws[:n]))
            assert (ws[n:] == fill).all()
        assert (outs[0] == outs[1]).all() and (outs[0] == outs[2]).all()


# ------------------------------------------------------------------ together
def moe_block(ops, x, blk, router, bias, table, W):
    """One FP8 MoE layer: norms with the attention block's output, router logits, routing, experts, norms of the next."""
    x1, q, s = ops.norm(x, W["pre"], block=blk, post=W["post"], out="f8")
    logits = ops.f8_matmul(q, s, *router, out="f32")
    ids, w = ops.route(logits, 4, score="sigmoid", bias=bias, n_group=4, topk_group=2, group_best=2, scale=2.5)
    y = ops.f8_experts(q, s, ids, w, *table, shared=True)
    x2, h = ops.norm(x1, W["pre2"], block=y, post=W["post2"], gate=W["gate"], scale=0.5, out="bf16")
    return x1, q, s, logits, ids, w, y, x2, h


@pytest.mark.parametrize("T", [1, 3, 24, 200])
def test_layer_together_eager_streams_and_graphs(ops, T):
    H, I, E = 512, 256, 32
    g = gen(T)
    table = (*f8_table(g, E + 1, 2 * I, H), *f8_table(g, E + 1, H, I))
    router = f8_table(g, E, H)
    bias = 0.05 * randn(g, E)
    W = {n: 1 + 0.1 * randn(g, H) for n in ("pre", "post", "pre2", "post2")}
    W["gate"] = torch.rand(1, H, generator=g, device="cuda").bfloat16()
    xs = [(randn(g, T, H), randn(g, T, H).bfloat16()) for _ in range(3)]
    eager = [moe_block(ops, x, b, router, bias, table, W) for x, b in xs]
    for (x, b), (x1, q, s, logits, ids, w, y, x2, h) in zip(xs, eager):
        ri, rw = route64(logits, 4, score="sigmoid", bias=bias, n_group=4, topk_group=2, group_best=2, scale=2.5)
        assert (ids.cpu().numpy() == ri).all()
        within(y, *experts64(q, s, ids, w, *table, True))
        want = x1.double() + 0.5 * W["gate"].double() * rms64(y.double(), W["post2"], 1e-6, 0.0)
        within(x2, want, 64 * U * (x1.double().abs() + want.abs() + (want - x1.double()).abs()))
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for (x, b), st in zip(xs, streams):
        with torch.cuda.stream(st):
            got.append(moe_block(ops, x, b, router, bias, table, W))
    torch.cuda.synchronize()
    for e, o in zip(eager, got):
        assert all((u.view(torch.uint8) == v.view(torch.uint8)).all() for u, v in zip(e, o))
    # two graphs, each with its own inputs, replayed at once and again with other inputs
    graphs = []
    for x, b in xs[:2]:
        cx, cb = x.clone(), b.clone()
        st = torch.cuda.Stream()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st):
            with torch.cuda.graph(gr, stream=st):
                o = moe_block(ops, cx, cb, router, bias, table, W)
        graphs.append((gr, cx, cb, o, st))
    for order in ((0, 1), (2, 0)):
        for i, (gr, cx, cb, o, st) in zip(order, graphs):
            cx.copy_(xs[i][0])
            cb.copy_(xs[i][1])
        torch.cuda.synchronize()
        for _ in range(3):
            for gr, cx, cb, o, st in graphs:
                with torch.cuda.stream(st):
                    gr.replay()
        torch.cuda.synchronize()
        for i, (gr, cx, cb, o, st) in zip(order, graphs):
            assert all((u.view(torch.uint8) == v.view(torch.uint8)).all() for u, v in zip(eager[i], o))


def test_tensors_elsewhere_are_refused(ops):
    with pytest.raises(ValueError):
        ops.route(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError):
        ops.f8_quantize(torch.zeros(2, 8))


def test_handle_dropped_while_capturing(ops, fb):
    """A handle that goes away while another's call is captured leaves the capture alone."""
    x = torch.arange(300, device="cuda").float().view(3, 100)
    ops.f8_quantize(x)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    other = fb.DeviceOps(0)
    with torch.cuda.graph(gr):
        q, s = ops.f8_quantize(x)
        del other
    gr.replay()
    torch.cuda.synchronize()
    want = ops.f8_quantize(x)
    assert (q.view(torch.uint8) == want[0].view(torch.uint8)).all() and (s == want[1]).all()


# sizes whose tiles two SMs share: the second without rows, with some, with all; odd columns, a last block of k that is short
@pytest.mark.parametrize("M,N,K", [(700, 3500, 2560), (630, 4001, 4080), (513, 4000, 4080), (2049, 1025, 4096)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_matmul_by_pairs(ops, M, N, K, out):
    from fomoe_b200.device_ops import MatmulArgs
    g = gen(M + N + K)
    a, sa = ops.f8_quantize(randn(g, M, K))
    b, sb = f8_table(g, N, K)
    c = ops.f8_matmul(a, sa, b, sb, out=out)
    A, B = rows64(a, sa), mat64(b, sb)
    want, size = A @ B.T, A.abs() @ B.abs().T
    # (test_matmul's bound)
    tol = (K // 128 + 1 + 130) * U * size + HALF[c.dtype] * want.abs() + 1e-40
    within(c, want, tol)
    if out == "f32":
        assert float((c.double() - want).norm() / want.norm()) < 2e-6
    # inside a larger buffer whose rows are not aligned: the same values, and nothing beside them
    big = torch.full((M + 2, N + 7), 7.0, device="cuda", dtype=c.dtype)
    o = big[1:1 + M, 3:3 + N]
    args = MatmulArgs(M, N, K, a.data_ptr(), K, sa.data_ptr(), sa.stride(0), b.data_ptr(), K, sb.data_ptr(), sb.stride(0),
                      o.data_ptr(), 1 if out == "bf16" else 0, o.stride(0))
    ops._ck(ops._l.fomoe_b200_ops_f8_matmul(ops._h, args, torch.cuda.current_stream().cuda_stream), "matmul")
    assert (o == c).all()
    o.fill_(7.0)
    assert (big == 7.0).all()


def test_matmul_on_streams_at_once(ops):
    """Products of every kind of tile on four streams at once, and replayed from two graphs at once: the bits of calls in turn."""
    g = gen(77)
    cases = []
    for M, N, K in [(700, 3500, 2560), (640, 4001, 144), (200, 1000, 512), (64, 2048, 1040), (8, 4096, 512), (2049, 1025, 4096)]:
        a, sa = ops.f8_quantize(randn(g, M, K))
        cases.append((a, sa, *f8_table(g, N, K)))
    want = [ops.f8_matmul(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for r in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                for j in range(len(cases)):
                    k = (i + j + r) % len(cases)
                    got.append((k, ops.f8_matmul(*cases[k])))
    torch.cuda.synchronize()
    for k, c in got:
        assert (c.view(torch.uint8) == want[k].view(torch.uint8)).all()
    graphs = []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.stream(streams[i]):
            with torch.cuda.graph(gr, stream=streams[i]):
                o = [ops.f8_matmul(*c) for c in (cases if i else cases[::-1])]
        graphs.append((gr, o if i else o[::-1]))
    for _ in range(3):
        for st, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for _, o in graphs:
        for c, w in zip(o, want):
            assert (c.view(torch.uint8) == w.view(torch.uint8)).all()


@pytest.mark.parametrize("ratio", [2.0 ** -10, 2.0 ** -18, 2.0 ** -30])
def test_experts_blocks_of_very_different_scales(ops, ratio):
    """Outputs that only small-scaled blocks of a row reach, beside a block whose scale is far larger: an expert's output is
    held to 2^-11 of itself or 2^-38 of the bound 128 448^2 sum |sa sb|, whichever is more."""
    T, H, I, E = 257, 256, 256, 3
    x, ids, w, gu, gus, dn, dns = make_experts(5, T, H, I, E, 1, False)
    dns = dns.clone()
    dns[:, :, 1] *= ratio
    dn.view(torch.uint8)[:, ::2, :128] = 0
    q, s = ops.f8_quantize(x)
    y = ops.f8_experts(q, s, ids, w, gu, gus, dn, dns)
    want, tol = experts64(q, s, ids, w, gu, gus, dn, dns, False)
    top = torch.zeros_like(want)
    for e in range(E):
        t = torch.nonzero(ids[:, 0] == e)[:, 0]
        z = rows64(q, s)[t] @ mat64(gu[e], gus[e]).T
        act = z[:, :I] / (1 + torch.exp(-z[:, :I])) * z[:, I:]
        sc = act.view(-1, 2, 128).abs().amax(2).clamp(min=TINY) / 448
        top[t] = (sc @ dns[e].double().T).repeat_interleave(128, 1) * 128 * 448 ** 2
    within(y, want, tol + w.double() * 2.0 ** -38 * top + 2.0 ** -11 * want.abs())
    if ratio > 2.0 ** -20:   # and so the small ones are there at all
        even = want[:, ::2]
        assert float((y.double()[:, ::2] - even).norm() / even.norm()) < 0.02
