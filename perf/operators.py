"""The operators on device memory -- routing, norms around a block, FP8 products with block scales, FP8 experts -- as
cases to time and compare: each in its plain form (elementary torch operations) and as the library's call.

A pass is one call as a serving program makes it: the routing of a step's tokens, the norms between two blocks, a
projection of bf16 activations (quantise, then multiply), the experts of one layer.  FP8 values are e4m3 with one fp32
scale for 128 values of a row (activations) or 128 x 128 values (weights)."""
import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_TINY = 2.0 ** -100  # the smallest amax a block's scale is made from
_handle = None


def _ops():
    """The handle that a program makes once and keeps."""
    global _handle
    if _handle is None:
        import fomoe_b200
        _handle = fomoe_b200.DeviceOps()
    return _handle


def listed():
    return [
        # one decode step of the 397B layer shape: 512 experts, softmax, ten of them
        dict(name="route one token", op="route", T=1, E=512, k=10, score="softmax", bias=False, n_group=1, topk_group=1,
             group_best=1, renorm=True, scale=1.0, logits="f32", closed=0.0, padded=False),
        # a padded decode batch with groups, some experts closed and some rows with none open
        dict(name="route padded groups", op="route", T=509, E=256, k=8, score="sigmoid", bias=True, n_group=8,
             topk_group=4, group_best=2, renorm=True, scale=2.5, logits="bf16", closed=0.2, padded=True),
        # a prefill chunk, balance bias, no groups
        dict(name="route prefill", op="route", T=16384, E=384, k=8, score="sigmoid", bias=True, n_group=1,
             topk_group=1, group_best=1, renorm=True, scale=2.5, logits="f32", closed=0.0, padded=False),
        # between two blocks of a decode step, hidden size of the 397B shape, FP8 for the experts
        dict(name="norm one token", op="norm", T=1, n=4096, x="f32", y="f32", post=False, gate="none", scale=1.0,
             offset=0.0, out="f8"),
        # a ragged chunk of a hidden size that ends inside a block, gated by token, sandwich norms
        dict(name="norm ragged", op="norm", T=777, n=2880, x="bf16", y="bf16", post=True, gate="token", scale=0.5,
             offset=1.0, out="f32"),
        # a prefill chunk, sandwich norms and a gate for every channel
        dict(name="norm prefill", op="norm", T=8192, n=4096, x="f32", y="bf16", post=True, gate="channel", scale=1.0,
             offset=0.0, out="f8"),
        # a projection in a decode step, of what the norm before it left in FP8
        dict(name="linear one token", op="linear", M=1, N=4096, K=4096, quantise=False, out="f32"),
        # odd sizes: ragged rows, columns and last block
        dict(name="linear odd", op="linear", M=67, N=1000, K=2064, quantise=True, out="bf16"),
        # a projection of a prefill chunk
        dict(name="linear prefill", op="linear", M=4096, N=8192, K=4096, quantise=True, out="bf16"),
        # the experts of one layer of the 397B shape, one token
        dict(name="experts one token", op="experts", T=1, H=4096, I=1024, E=512, k=10, shared=True, dropped=0.0),
        # a decode batch with experts that live elsewhere
        dict(name="experts decode batch", op="experts", T=61, H=2048, I=768, E=256, k=8, shared=False, dropped=0.2),
        # a prefill chunk of a wide layer
        dict(name="experts prefill", op="experts", T=8192, H=4096, I=1024, E=64, k=8, shared=True, dropped=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "norm", "linear", "experts"])
    if op == "route":
        n_group = rng.choice([1, 1, 2, 4, 8])
        per = _log(rng, 16, 512 // n_group)
        topk_group = rng.randint(1, n_group)
        return dict(op=op, T=_log(rng, 1, 12000), E=per * n_group, k=rng.randint(1, min(16, per)),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, n_group=n_group,
                    topk_group=topk_group, group_best=rng.choice([1, 2]), renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), logits=rng.choice(["f32", "bf16"]), closed=rng.choice([0.0, 0.1]),
                    padded=rng.random() < 0.3)
    if op == "norm":
        n = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        return dict(op=op, T=min(_log(rng, 1, 8192), 18_000_000 // n), n=n, x=rng.choice(["f32", "bf16"]),
                    y=rng.choice(["f32", "bf16"]), post=rng.random() < 0.5,
                    gate=rng.choice(["none", "channel", "token", "element"]), scale=rng.choice([1.0, 0.5]),
                    offset=rng.choice([0.0, 1.0]), out=rng.choice(["f32", "bf16", "f8"]))
    if op == "linear":
        K, N = 16 * _log(rng, 8, 256), _log(rng, 64, 8192)
        quantise = rng.random() < 0.5
        return dict(op=op, M=min(_log(rng, 1, 4096), 120_000_000_000 // (N * K)), N=N, K=K, quantise=quantise,
                    out="bf16" if quantise else rng.choice(["f32", "bf16"]))
    H, I = 128 * _log(rng, 4, 32), 128 * _log(rng, 2, 12)
    E = min(_log(rng, 8, 192), 900_000_000 // (3 * H * I))
    return dict(op=op, T=_log(rng, 1, 4096), H=H, I=I, E=E, k=rng.randint(1, min(8, E)), shared=rng.random() < 0.5,
                dropped=rng.choice([0.0, 0.2]))


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (1 << 62) + 17)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _f8_table(g, n, rows, cols):
    """n matrices [rows, cols] in e4m3 (values around 60) with a scale for each 128 x 128 block: together N(0, 1/cols)."""
    q = torch.empty(n, rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
    step = max(1, (1 << 28) // (rows * cols))
    for i in range(0, n, step):
        m = min(step, n - i)
        q[i:i + m] = (_randn(g, m, rows, cols) * 60.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = torch.exp(0.3 * _randn(g, n, -(-rows // 128), -(-cols // 128))) * (1.0 / (60.0 * cols ** 0.5))
    return q, s


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    if op == "route":
        T, E = case["T"], case["E"]
        x = 1.5 * _randn(g, T, E)
        if case["closed"]:
            x[torch.rand(T, E, generator=g, device="cuda") < case["closed"]] = float("-inf")
            x[torch.rand(T, generator=g, device="cuda") < 0.02] = float("-inf")
        s["x"] = x.to(_DT[case["logits"]])
        s["b"] = 0.1 * _randn(g, E) if case["bias"] else None
        s["valid"] = (torch.arange(T, device="cuda") < T - T // 5).to(torch.uint8) if case["padded"] else None
    elif op == "norm":
        T, n = case["T"], case["n"]
        s["res"] = (3.0 * _randn(g, T, n)).to(_DT[case["x"]])
        s["blk"] = _randn(g, T, n).to(_DT[case["y"]])
        w = 1.0 - case["offset"]
        s["w_pre"] = w + 0.1 * _randn(g, n)
        s["w_post"] = w + 0.1 * _randn(g, n) if case["post"] else None
        shape = {"none": None, "channel": (1, n), "token": (T, 1), "element": (T, n)}[case["gate"]]
        s["g"] = torch.sigmoid(_randn(g, *shape)).to(_DT[case["y"]]) if shape else None
    elif op == "linear":
        s["a"] = _randn(g, case["M"], case["K"]).to(torch.bfloat16)
        if not case["quantise"]:
            s["aq"], s["as"] = _quant(s["a"])
        w, ws = _f8_table(g, 1, case["N"], case["K"])
        s["w"], s["ws"] = w[0], ws[0]
    else:
        T, H, I, E, k = (case[v] for v in ("T", "H", "I", "E", "k"))
        recs = E + int(case["shared"])
        s["gu"], s["gus"] = _f8_table(g, recs, 2 * I, H)
        s["dn"], s["dns"] = _f8_table(g, recs, H, I)
        x, xs = _quant(_randn(g, T, H))
        s["xq"], s["xs"] = x, xs
        lg = _randn(g, T, E) + 0.7 * _randn(g, 1, E)  # some experts are asked for more often than others
        v, ids = torch.topk(lg, k, dim=1)
        s["wt"] = torch.softmax(v, dim=1)
        s["ids"] = torch.where(torch.rand(T, k, generator=g, device="cuda") < case["dropped"], -1, ids).to(torch.int32)
    return s


# ---------------------------------------------------------------- plain forms
def _quant(x):
    """Rows of x in blocks of 128 (the last may be shorter): scale = max(amax, tiny) / 448, value = e4m3(x / scale)."""
    T, n = x.shape
    nb = -(-n // 128)
    b = torch.nn.functional.pad(x.float(), (0, nb * 128 - n)).view(T, nb, 128)
    amax = b.abs().amax(dim=2).clamp(min=_TINY)
    s = torch.div(amax, torch.full_like(amax, 448.0))
    q = torch.div(b, s[:, :, None]).to(torch.float8_e4m3fn).view(T, nb * 128)
    return q[:, :n].contiguous(), s


def _unq_rows(q, s):
    return q.float() * s.repeat_interleave(128, dim=1)[:, :q.shape[1]]


def _unq_blocks(q, s):
    return q.float() * s.repeat_interleave(128, dim=-2).repeat_interleave(128, dim=-1)[..., :q.shape[-2], :q.shape[-1]]


def _route(s):
    x, k, E = s["x"], s["k"], s["E"]
    T = x.shape[0]
    ninf = float("-inf")
    shut = ~(x > ninf)
    if s["valid"] is not None:
        shut = shut | (s["valid"] == 0)[:, None]
    # which expert comes first is decided in 64 bits: values next to one another
    x = x.double().clamp(max=3.4028234663852886e38).masked_fill(shut, ninf)
    if s["score"] == "sigmoid":
        p = torch.reciprocal(1.0 + torch.exp(-x))
    else:
        top = x.amax(dim=1, keepdim=True)
        e = torch.exp(x - torch.where(top > ninf, top, torch.zeros_like(top)))
        p = e / e.sum(dim=1, keepdim=True).clamp(min=1e-300)
    # without a bias the probabilities rank as their logits do
    c = (p if s["b"] is None else p + s["b"].double()).masked_fill(shut, ninf)
    order = x if s["b"] is None else c
    if s["n_group"] > 1:
        G = s["n_group"]
        per = c.view(T, G, E // G)
        two = torch.sort(per, dim=2, descending=True).values[:, :, :s["group_best"]]
        gs = torch.where(two > ninf, two, torch.zeros_like(two)).sum(dim=2).masked_fill(two[:, :, 0] == ninf, ninf)
        keep = torch.sort(gs, dim=1, descending=True, stable=True).indices[:, :s["topk_group"]]
        out = torch.ones(T, G, dtype=torch.bool, device=x.device).scatter(1, keep, False)
        order = order.masked_fill(out.repeat_interleave(E // G, dim=1), ninf)
    v, i = torch.sort(order, dim=1, descending=True, stable=True)
    v, i = v[:, :k], i[:, :k]
    w = torch.gather(p, 1, i).masked_fill(v == ninf, 0.0)
    if s["renorm"]:
        w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    return {"ids": i.masked_fill(v == ninf, -1).to(torch.int32), "weights": (w * s["scale"]).float()}


def _rms(v, w, eps, offset):
    return v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + eps) * (w + offset)


def _norm(s):
    r = s["blk"].float()
    if s["w_post"] is not None:
        r = _rms(r, s["w_post"], 1e-6, s["offset"])
    if s["g"] is not None:
        r = r * s["g"].float()
    x = s["res"].float() + s["scale"] * r
    h = _rms(x, s["w_pre"], 1e-6, s["offset"])
    x = x.to(s["res"].dtype)
    if s["out"] == "f8":
        q, sc = _quant(h)
        return {"x": x, "q": q, "scales": sc}
    return {"x": x, "h": h.to(_DT[s["out"]])}


def _linear(s):
    q, sc = _quant(s["a"]) if s["quantise"] else (s["aq"], s["as"])
    out = (_unq_rows(q, sc) @ _unq_blocks(s["w"], s["ws"]).t()).to(_DT[s["out"]])
    return {"q": q, "scales": sc, "out": out} if s["quantise"] else {"out": out}


def _ffn(x, gu, gus, dn, dns, I):
    """x [n, C, H] through n experts."""
    z = torch.bmm(x, _unq_blocks(gu, gus).transpose(1, 2))
    a = z[..., :I] * torch.sigmoid(z[..., :I]) * z[..., I:]
    n, C = a.shape[:2]
    a = _unq_rows(*_quant(a.reshape(n * C, I))).view(n, C, I)
    return torch.bmm(a, _unq_blocks(dn, dns).transpose(1, 2))


def _experts(s):
    T, H, I, E = s["T"], s["H"], s["I"], s["E"]
    k, w = s["k"], s["wt"]
    flat = s["ids"].long().reshape(-1)
    tokens = _unq_rows(s["xq"], s["xs"])
    x = tokens[torch.arange(T * k, device=flat.device) // k]
    if T * k <= E and T * k * H * I < 1 << 29:  # few pairs: each with its own expert's matrices
        e = flat.clamp(min=0)
        y = _ffn(x[:, None], s["gu"].view(torch.uint8)[e].view(torch.float8_e4m3fn), s["gus"][e],
                 s["dn"].view(torch.uint8)[e].view(torch.float8_e4m3fn), s["dns"][e], I)[:, 0]
    else:  # each expert with the pairs that ask for it, in rows of one length
        key = torch.where(flat < 0, E, flat)
        order = torch.argsort(key, stable=True)
        count = torch.bincount(key, minlength=E + 1)
        at = torch.arange(T * k, device=flat.device) - (torch.cumsum(count, 0) - count)[key[order]]
        C = max(1, int(count[:E].max()))
        slot = torch.empty_like(at)
        slot[order] = torch.where(key[order] < E, key[order] * C + at, E * C)
        rows = torch.zeros(E * C + 1, H, device=x.device)
        rows[slot] = x
        y = _ffn(rows[:-1].view(E, C, H), s["gu"][:E], s["gus"][:E], s["dn"][:E], s["dns"][:E], I).reshape(E * C, H)
        y = torch.cat([y, torch.zeros(1, H, device=y.device)])[slot]
    y = torch.where((flat < 0)[:, None], torch.zeros_like(y), y).view(T, k, H)
    out = (w[:, :, None] * y).sum(dim=1)
    if s["shared"]:
        out = out + _ffn(tokens[None], s["gu"][E:], s["gus"][E:], s["dn"][E:], s["dns"][E:], I)[0]
    return {"out": out.to(torch.bfloat16)}


def run(s):
    op = s["op"]
    if not own:
        return {"route": _route, "norm": _norm, "linear": _linear, "experts": _experts}[op](s)
    ops = _ops()
    if op == "route":
        ids, w = ops.route(s["x"], s["k"], score=s["score"], bias=s["b"], n_group=s["n_group"], topk_group=s["topk_group"],
                           group_best=s["group_best"], renorm=s["renorm"], scale=s["scale"], valid=s["valid"])
        return {"ids": ids, "weights": w}
    if op == "norm":
        r = ops.norm(s["res"], s["w_pre"], block=s["blk"], post=s["w_post"], gate=s["g"], scale=s["scale"], eps=1e-6,
                     offset=s["offset"], out=s["out"])
        return {"x": r[0], "q": r[1], "scales": r[2]} if s["out"] == "f8" else {"x": r[0], "h": r[1]}
    if op == "linear":
        if not s["quantise"]:
            return {"out": ops.f8_matmul(s["aq"], s["as"], s["w"], s["ws"], out=s["out"])}
        q, sc = ops.f8_quantize(s["a"])
        return {"q": q, "scales": sc, "out": ops.f8_matmul(q, sc, s["w"], s["ws"], out=s["out"])}
    return {"out": ops.f8_experts(s["xq"], s["xs"], s["ids"], s["wt"], s["gu"], s["gus"], s["dn"], s["dns"],
                                  shared=s["shared"])}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2, "f8": 1}
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": T * E * size[case["logits"]] + 8 * T * k + (4 * E if case["bias"] else 0) + (T if case["padded"] else 0),
                "flops": 6 * T * E}
    if op == "norm":
        T, n = case["T"], case["n"]
        gate = {"none": 0, "channel": n, "token": T, "element": T * n}[case["gate"]] * size[case["y"]]
        per = 2 * size[case["x"]] + size[case["y"]] + size[case["out"]]
        sc = 4 * T * -(-n // 128) if case["out"] == "f8" else 0
        return {"bytes": T * n * per + gate + 4 * n * (2 if case["post"] else 1) + sc, "flops": 10 * T * n}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        nb = -(-K // 128)
        rows = M * K * (3 if case["quantise"] else 1) + 4 * M * nb
        return {"bytes": rows + N * K + 4 * -(-N // 128) * nb + M * N * size[case["out"]],
                "flops": 2 * M * N * K}
    T, H, I, E, k = (case[v] for v in ("T", "H", "I", "E", "k"))
    live = k * (1.0 - case["dropped"])
    hit = E * (1.0 - (1.0 - live / E) ** T) + int(case["shared"])  # experts that some token asks for, on average
    per = 3 * H * I + 4 * 3 * (H // 128) * (I // 128)
    return {"bytes": hit * per + T * (H + H // 32 + 8 * k + 2 * H), "flops": 6 * T * (live + int(case["shared"])) * H * I}


# ---------------------------------------------------------------- the definitions in 64 bits
def _quant64(h):
    nb = (h.shape[1] + 127) // 128
    sc = torch.zeros(h.shape[0], nb, dtype=torch.float64, device=h.device)
    for b in range(nb):
        sc[:, b] = torch.maximum(h[:, 128 * b:128 * b + 128].abs().max(dim=1).values, torch.full((), _TINY, dtype=torch.float64, device=h.device)) / 448.0
    col = torch.arange(h.shape[1], device=h.device) // 128
    q = (h / sc[:, col]).to(torch.float32).to(torch.float8_e4m3fn)
    return q, sc, q.double() * sc[:, col]


def _mat64(q, s):
    r = torch.arange(q.shape[0], device=q.device) // 128
    c = torch.arange(q.shape[1], device=q.device) // 128
    return q.double() * s.double()[r][:, c]


def _exact_route(s):
    x = s["x"].float().cpu().numpy().astype(np.float64)
    T, E, k, G = s["T"], s["E"], s["k"], s["n_group"]
    shut = ~(x > -np.inf)
    if s["valid"] is not None:
        shut |= s["valid"].cpu().numpy()[:, None] == 0
    x = np.where(shut, -np.inf, np.minimum(x, np.finfo(np.float32).max))
    with np.errstate(all="ignore"):
        if s["score"] == "sigmoid":
            p = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
        else:
            p = np.exp(x - np.max(x, axis=1, keepdims=True))
            p = np.where(shut, 0.0, p)
            p = np.where(p.sum(1, keepdims=True) > 0, p / np.maximum(p.sum(1, keepdims=True), 1e-300), 0.0)
        c = np.where(shut, -np.inf, p + (s["b"].cpu().numpy().astype(np.float64) if s["b"] is not None else 0.0))
        if G > 1:
            v = -np.sort(-c.reshape(T, G, E // G), axis=2)
            score = v[:, :, 0].copy()
            if s["group_best"] == 2:
                score = score + np.where(v[:, :, 1] > -np.inf, v[:, :, 1], 0.0)
            best = np.zeros((T, G), bool)
            left = score.copy()
            left[np.isneginf(left)] = -1e300
            for _ in range(s["topk_group"]):
                a = np.argmax(left, axis=1)
                best[np.arange(T), a] = True
                left[np.arange(T), a] = -np.inf
            c = np.where(np.repeat(best, E // G, axis=1), c, -np.inf)
            shut = shut | ~np.repeat(best, E // G, axis=1)
        key = np.where(shut, -np.inf, x) if s["b"] is None else c
        w = np.zeros((T, k))
        for j in range(k):
            a = np.argmax(key, axis=1)
            some = key[np.arange(T), a] > -np.inf
            w[:, j] = np.where(some, p[np.arange(T), a], 0.0)
            key[np.arange(T), a] = -np.inf
    if s["renorm"]:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return {"ids": None, "weights": w * s["scale"]}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        return _exact_route(s)
    if op == "norm":
        r = s["blk"].double()
        if s["w_post"] is not None:
            r = r / torch.sqrt(r.pow(2).sum(1) / case["n"] + 1e-6)[:, None] * (s["w_post"].double() + case["offset"])
        if s["g"] is not None:
            r = r * s["g"].double()
        x = s["res"].double() + case["scale"] * r
        h = x / torch.sqrt(x.pow(2).sum(1) / case["n"] + 1e-6)[:, None] * (s["w_pre"].double() + case["offset"])
        if case["out"] == "f8":
            q, sc, _ = _quant64(h)
            return {"x": x, "q": q, "scales": sc}
        return {"x": x, "h": h}
    if op == "linear":
        if not case["quantise"]:
            col = torch.arange(case["K"], device="cuda") // 128
            return {"out": (s["aq"].double() * s["as"].double()[:, col]) @ _mat64(s["w"], s["ws"]).T}
        q, sc, a = _quant64(s["a"].double())
        return {"q": q, "scales": sc, "out": a @ _mat64(s["w"], s["ws"]).T}
    I = case["I"]
    nb = torch.arange(case["H"], device="cuda") // 128
    x = s["xq"].double() * s["xs"].double()[:, nb]
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
    for e in range(s["gu"].shape[0]):
        if e < case["E"]:
            t, j = torch.nonzero(s["ids"] == e, as_tuple=True)
            w = s["wt"][t, j].double()
        else:
            t = torch.arange(case["T"], device="cuda")
            w = torch.ones(case["T"], dtype=torch.float64, device="cuda")
        if t.numel():
            z = x[t] @ _mat64(s["gu"][e], s["gus"][e]).T
            a = z[:, :I] / (1.0 + torch.exp(-z[:, :I])) * z[:, I:]
            out.index_add_(0, t, w[:, None] * (_quant64(a)[2] @ _mat64(s["dn"][e], s["dns"][e]).T))
    return {"out": out}
