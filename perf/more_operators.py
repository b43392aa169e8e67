"""Operators of a routed layer on rows of atoms, as cases that can be timed: the root-mean-square norm before the router
(with the residual's addition, and with rows of 8 bits), the experts' products, and the step that trains them.

``run`` makes the framework's calls where ``own`` is true and computes the same in elementary torch operations where it
is not; ``exact`` restates each operator in 64 bits.  Atom counts, channels and degrees are those of the framework's
workloads (1,024-atom alloy, 12,288-atom water box, 101,306-atom bcc Fe; 64, 128 or 256 channels in irreps 0 .. L); the
wider rows are generic.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16, "float16": torch.float16}
E4M3 = torch.float8_e4m3fn
MASK32 = 0xFFFFFFFF
BLOCK = 256    # elements that share a scale of 8-bit states
LR, BETAS, EPS, DECAY = 2e-4, (0.9, 0.999), 1e-8, 0.01
NORM_EPS = 1e-6


# ------------------------------------------------------------------- cases ----
def listed():
    return [
        # scalar features of a small alloy cell, one training step's norm: latency
        dict(name="norm_alloy", kind="norm", rows=1024, C=128, L=0, dtype="float32", residual=True, out="same"),
        # the water box's features, every degree of an atom by its own mean square
        dict(name="norm_water", kind="norm", rows=12288, C=128, L=3, dtype="float32", residual=True, out="same"),
        # the large cell in 16 bits, evaluated: rows of 8 bits for the experts behind it
        dict(name="norm_iron_e4m3", kind="norm", rows=101306, C=256, L=0, dtype="bfloat16", residual=True, out="e4m3"),
        # wide rows in training
        dict(name="norm_wide_bf16", kind="norm", rows=8191, C=4096, L=0, dtype="bfloat16", residual=False,
             out="same"),
        # two of eight experts on the alloy's scalars, a training step: latency
        dict(name="experts_alloy", kind="experts", tokens=1024, k=2, experts=8, K=128, N=128, L=0, dtype="float32",
             drop=0.0),
        # the water box's features, degrees 0 .. 3 each with its own weights
        dict(name="experts_water", kind="experts", tokens=12288, k=1, experts=8, K=128, N=128, L=3, dtype="float32",
             drop=0.0),
        # the large cell in 16 bits, a tenth of the choices dropped (experts over capacity)
        dict(name="experts_iron_bf16", kind="experts", tokens=101306, k=2, experts=16, K=256, N=512, L=0,
             dtype="bfloat16", drop=0.1),
        # a wide layer in training: bound by its products
        dict(name="experts_wide_bf16", kind="experts", tokens=16384, k=2, experts=8, K=1024, N=2048, L=0,
             dtype="bfloat16", drop=0.0),
        # serving: a few tokens at once, bound by reading the experts' weights of 8 bits
        dict(name="experts_e4m3", kind="experts8", tokens=24, k=2, experts=16, K=1024, N=4096, gather=True),
        # the small cell's model: 60 tensors, latency and many launches
        dict(name="adam_alloy", kind="adam", tensors=60, largest=131072, dtype="float32", bits=32, clip=True),
        # the weights of all experts of a large layer
        dict(name="adam_experts", kind="adam", tensors=120, largest=4194304, dtype="float32", bits=32, clip=True),
        # weights of 16 bits with 32-bit masters and 8-bit states
        dict(name="adam_bf16_e4m3", kind="adam", tensors=120, largest=2097152, dtype="bfloat16", bits=8, clip=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "experts", "experts", "experts8", "adam", "adam"))
    dtype = rng.choice(("float32", "float32", "bfloat16", "bfloat16", "float16", "float64"))
    if kind == "norm":
        out = "e4m3" if dtype != "float64" and rng.random() < 0.4 else "same"
        if rng.random() < 0.5:
            C, L = rng.choice((32, 64, 100, 128, 256)), rng.randint(0, 3)
        else:
            C, L = _log_int(rng, 16, 8192), 0
        size = DTYPES[dtype].itemsize * C * (L + 1) ** 2
        return dict(kind=kind, rows=min(_log_int(rng, 64, 200000), 60000000 // size + 1), C=C, L=L, dtype=dtype,
                    residual=rng.random() < 0.6, out=out)
    if kind == "experts":
        experts = _log_int(rng, 2, 89)
        k = min(experts, rng.choice((1, 2, 2, 4)))
        L = rng.choice((0, 0, 1, 3))
        wide = 300 if dtype == "float64" or L else 1500
        K, N = _log_int(rng, 16, wide), _log_int(rng, 16, wide)
        if rng.random() < 0.7:      # (a multiple of 16, as channels are)
            K, N = -(-K // 16) * 16, -(-N // 16) * 16
        per = k * (L + 1) ** 2 * max(K * N / (16 if dtype == "float64" else 1), 600 * (K + N))
        return dict(kind=kind, tokens=min(_log_int(rng, 16, 100000), int(3e10 / per) + 1), k=k, experts=experts, K=K,
                    N=N, L=L, dtype=dtype, drop=rng.choice((0.0, 0.0, 0.15)))
    if kind == "experts8":
        experts = _log_int(rng, 2, 89)
        K, N = 16 * _log_int(rng, 4, 128), 16 * _log_int(rng, 4, 128)
        return dict(kind=kind, tokens=_log_int(rng, 1, 8000), k=min(experts, rng.choice((1, 2, 4))), experts=experts,
                    K=K, N=N, gather=rng.random() < 0.6)
    bits = 8 if dtype != "float64" and rng.random() < 0.4 else 32
    tensors = _log_int(rng, 1, 150)
    return dict(kind=kind, tensors=tensors, largest=min(_log_int(rng, 64, 4000000), 200000000 // tensors), dtype=dtype,
                bits=bits, clip=rng.random() < 0.6)


def _sizes(case):
    """Elements of each tensor: most far below the largest, odd ones among them."""
    n, big = case["tensors"], case["largest"]
    return [max(1, int(big * 0.5 ** ((i % 7) * (i % 3))) - (i % 4)) for i in range(n)]


def _comps(case):
    return [2 * l + 1 for l in range(case["L"] + 1)]


def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)


def prepare(case, seed):
    g, c = _gen(seed), case
    s = dict(case=c)
    if c["kind"] == "norm":
        dt, comps = DTYPES[c["dtype"]], _comps(c)
        D = c["C"] * sum(comps)
        s["x"] = _normal(g, dt, c["rows"], D)
        s["residual"] = _normal(g, dt, c["rows"], D) * 3 if c["residual"] else None
        s["weight"] = (1 + 0.2 * _normal(g, torch.float64, len(comps), c["C"])).to(dt)
        if c["out"] == "same":
            s["gy"] = _normal(g, dt, c["rows"], D)
            s["gh"] = _normal(g, dt, c["rows"], D) if c["residual"] else None
    elif c["kind"] in ("experts", "experts8"):
        T, k, E, K, N = c["tokens"], c["k"], c["experts"], c["K"], c["N"]
        popular = torch.randn(E, generator=g, device=DEVICE)
        e = (torch.randn(T, E, generator=g, device=DEVICE) + popular).topk(k)[1].reshape(-1)
        if c["kind"] == "experts":
            e = torch.where(torch.rand(T * k, generator=g, device=DEVICE) < c["drop"], E, e)
        s["order"] = e.argsort(stable=True)
        s["place"] = torch.empty_like(s["order"]).scatter_(0, s["order"], torch.arange(T * k, device=DEVICE)).int()
        s["order"] = s["order"].int()
        s["rowptr"] = torch.cat([e.new_zeros(1), e.bincount(minlength=E + 1)[:E].cumsum(0)]).int()
        if c["kind"] == "experts":
            dt, comps = DTYPES[c["dtype"]], _comps(c)
            s["x"] = _normal(g, dt, T * k, K * sum(comps))
            s["weight"] = _normal(g, dt, E, len(comps), K, N)
            s["gout"] = _normal(g, dt, T * k, N * sum(comps))
            s["scale"] = 1 / math.sqrt(K)
        else:
            rows = T if c["gather"] else T * k
            s["q"], s["q_scale"] = _codes(_normal(g, torch.float32, rows, K))
            s["w"], s["w_scale"] = _codes(_normal(g, torch.float32, E, N, K) / math.sqrt(K))
    else:
        _prepare_adam(s, c, g, seed)
    return s


def _codes(x):
    scale = x.abs().amax(-1, keepdim=True) / 448
    return (x / scale).to(E4M3), scale.squeeze(-1)


def _prepare_adam(s, c, g, seed):
    """Every tensor is a piece of one storage, from a multiple of 256 elements on (what lies between is zero), as buckets
    of parameters and gradients are; the states are those of a run that has taken some steps."""
    sizes, dt = _sizes(c), DTYPES[c["dtype"]]
    wide = torch.float64 if dt == torch.float64 else torch.float32
    start = np.concatenate([[0], np.cumsum([-(-n // BLOCK) * BLOCK for n in sizes])])
    total = int(start[-1])
    s["sizes"], s["start"] = sizes, start
    at = torch.arange(total, device=DEVICE)
    ends = torch.tensor(start, device=DEVICE)
    which = torch.bucketize(at, ends[1:], right=True)
    inside = at - ends[which] < torch.tensor(sizes, device=DEVICE)[which]
    del at, which
    values = lambda size: torch.where(inside, torch.randn(total, generator=g, device=DEVICE) * size, 0.0)
    master = values(0.05).to(wide)
    s["p"] = master.to(dt)
    s["master"] = master if dt.itemsize == 2 else None
    spread = torch.exp(0.5 * torch.randn(total // BLOCK, 1, generator=g, device=DEVICE))
    s["g"] = (values(1e-3).view(-1, BLOCK) * spread).view(-1).to(dt)
    m = (values(4e-4).view(-1, BLOCK) * spread).view(-1)
    r = (values(3e-4).abs().add_(8e-4).mul_(inside).view(-1, BLOCK) * spread).view(-1)
    if c["bits"] == 8:
        sm, sr = (t.view(-1, BLOCK).abs().amax(1).div(448).clamp(min=1e-30) for t in (m, r))
        s["m"] = (m.view(-1, BLOCK) / sm.view(-1, 1)).view(-1).to(E4M3)
        s["s"] = (r.view(-1, BLOCK) / sr.view(-1, 1)).view(-1).to(E4M3)
        s["scales"] = torch.stack([sm, sr], 1)
    else:
        s["m"], s["s"], s["scales"] = m.to(wide), (r * r).to(wide), None
    s["counter"] = torch.tensor([100 + int(seed) % 50, 0], dtype=torch.int64, device=DEVICE)
    s["seed"] = int(seed) * 7919 + (12345 << 34)
    piece = lambda t: None if t is None else [t[a:a + n] for a, n in zip(start.tolist(), sizes)]
    s["lists"] = [piece(s[key]) for key in ("p", "g", "m", "s", "master")]
    s["lists"].append(None if s["scales"] is None else
                      [s["scales"][a // BLOCK:a // BLOCK - (-n // BLOCK)] for a, n in zip(start.tolist(), sizes)])


def _leaf(t):
    return t.detach().requires_grad_(True)


def run(s):
    c = s["case"]
    if not own:
        return {"norm": _plain_norm, "experts": _plain_experts, "experts8": _plain_experts8,
                "adam": _plain_adam}[c["kind"]](s, c)
    from tace_amd import ops

    if c["kind"] == "norm":
        comps = _comps(c)
        if c["out"] == "e4m3":
            return ops.rms_norm_e4m3(s["x"], s["weight"], NORM_EPS, residual=s["residual"], components=comps)
        x, w = _leaf(s["x"]), _leaf(s["weight"])
        if not c["residual"]:
            y = ops.rms_norm(x, w, NORM_EPS, components=comps)
            return [y, *torch.autograd.grad(y, (x, w), s["gy"])]
        res = _leaf(s["residual"])
        y, h = ops.rms_norm(x, w, NORM_EPS, residual=res, components=comps)
        return [y, h, *torch.autograd.grad((y, h), (x, res, w), (s["gy"], s["gh"]))]
    if c["kind"] == "adam":
        p, g, m, sq, master, scales = s["lists"]
        norm = ops.adamw_step(p, g, m, sq, s["counter"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                              scales=scales, masters=master, max_norm=1.0 if c["clip"] else None, seed=s["seed"])
        return [s["p"], s["master"], s["m"], s["s"], s["scales"], norm, s["counter"][0]]
    plan = ops.RoutePlan(s["rowptr"], s["order"], s["place"], c["tokens"], c["k"])
    if c["kind"] == "experts8":
        return ops.expert_linear_e4m3(s["q"], s["q_scale"], s["w"], s["w_scale"], plan, gather=c["gather"])
    x, w = _leaf(s["x"]), _leaf(s["weight"])
    y = ops.expert_linear(x, w, plan, scale=s["scale"], components=_comps(c))
    return [y, *torch.autograd.grad(y, (x, w), s["gout"])]


def work(case):
    c = case
    if c["kind"] == "norm":
        b, n = DTYPES[c["dtype"]].itemsize, c["rows"] * c["C"] * (c["L"] + 1) ** 2
        fwd = (b * 3 if c["residual"] else b) * n
        if c["out"] == "e4m3":
            return dict(bytes=fwd + n + 4 * c["rows"] * (c["L"] + 1), flops=6 * n)
        # forward: x, residual, h, y; backward: gy, gh, h and the gradient
        return dict(bytes=fwd + b * n + b * n * (4 if c["residual"] else 3), flops=16 * n)
    if c["kind"] == "experts8":
        T, k, E, K, N = c["tokens"], c["k"], c["experts"], c["K"], c["N"]
        used = min(E, T * k)
        rows = T if c["gather"] else T * k
        return dict(bytes=used * N * (K + 4) + rows * (K + 4) + 2 * T * k * N, flops=2 * T * k * K * N)
    if c["kind"] == "experts":
        b, R = DTYPES[c["dtype"]].itemsize, c["tokens"] * c["k"]
        M, W = R * (c["L"] + 1) ** 2, c["experts"] * (c["L"] + 1) * c["K"] * c["N"]
        # forward: x, w, y; backward: gout, x and w once more, both gradients
        return dict(bytes=b * (M * (3 * c["K"] + 2 * c["N"]) + 3 * W), flops=6 * M * c["K"] * c["N"])
    n, b = sum(_sizes(c)), DTYPES[c["dtype"]].itemsize
    state = 2 * (1 + 4 / BLOCK) if c["bits"] == 8 else 2 * max(b, 4)
    each = 2 * state + (3 * b if b > 2 else 2 * b + 8)   # (weights of 16 bits are written only: their masters are read)
    return dict(bytes=int(n * (each + (b if c["clip"] else 0))), flops=n * 20)


# ------------------------------------------------------------- plain forms ----
def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _blocks(x, comps, C):
    """The degree blocks of group-major rows, each [rows, components, C]."""
    n = x.shape[0]
    return [p.view(n, d, C) for p, d in zip(x.reshape(-1).split([n * d * C for d in comps]), comps)]


def _join(parts, like):
    return torch.cat([p.reshape(-1) for p in parts]).view(like.shape)


def _plain_norm(s, c):
    comps, x, C = _comps(c), s["x"], c["C"]
    h = x if s["residual"] is None else (_wide(x) + _wide(s["residual"])).to(x.dtype)
    hs, w = _blocks(_wide(h), comps, C), _wide(s["weight"])
    inv = [torch.rsqrt(b.square().mean((1, 2), keepdim=True) + NORM_EPS) for b in hs]
    ys = [b * i * w[l] for l, (b, i) in enumerate(zip(hs, inv))]
    if c["out"] == "e4m3":
        top = [y.abs().amax((1, 2)) for y in ys]
        q = [(y * torch.where(t > 0, 448 / t, 0.0).view(-1, 1, 1)).to(E4M3).reshape(-1).view(torch.uint8)
             for y, t in zip(ys, top)]
        out = [torch.cat(q).view(E4M3).view(x.shape), torch.stack(top, 1) / 448]
        return out if s["residual"] is None else out + [h]
    us = [g * w[l] for l, g in enumerate(_blocks(_wide(s["gy"]), comps, C))]
    dh = [i * (u - b * i * i * (u * b).mean((1, 2), keepdim=True)) for u, b, i in zip(us, hs, inv)]
    dw = torch.stack([(g * b * i).sum((0, 1)) for g, b, i in zip(_blocks(_wide(s["gy"]), comps, C), hs, inv)])
    dx = _join(dh, x)
    y = _join(ys, x).to(x.dtype)
    if s["residual"] is None:
        return [y, dx.to(x.dtype), dw.to(x.dtype)]
    dx = (dx + _wide(s["gh"])).to(x.dtype)
    return [y, h, dx, dx, dw.to(x.dtype)]


def _plain_experts(s, c):
    comps, R, K, N, dt = _comps(c), c["tokens"] * c["k"], c["K"], c["N"], s["x"].dtype
    ends = s["rowptr"].tolist()
    x, g, w = _wide(s["x"]).view(-1, K), _wide(s["gout"]).view(-1, N), _wide(s["weight"])
    y, dx, dw = torch.zeros_like(g), torch.zeros_like(x), torch.zeros_like(w)
    for b, d in enumerate(comps):
        base = R * sum(comps[:b])
        for e in range(c["experts"]):
            at = slice(base + d * ends[e], base + d * ends[e + 1])
            torch.mm(x[at], w[e, b], out=y[at])
            torch.mm(g[at], w[e, b].t(), out=dx[at])
            torch.mm(x[at].t(), g[at], out=dw[e, b])
    return [t.mul_(s["scale"]).to(dt).view(like.shape)
            for t, like in ((y, s["gout"]), (dx, s["x"]), (dw, s["weight"]))]


def _plain_experts8(s, c):
    ends = s["rowptr"].tolist()
    x = s["q"].float() * s["q_scale"].unsqueeze(1)
    if c["gather"]:
        x = x[(s["order"] // c["k"]).long()]
    y = torch.zeros(x.shape[0], c["N"], device=x.device)
    for e in range(c["experts"]):
        if ends[e + 1] > ends[e]:
            w = s["w"][e].float() * s["w_scale"][e].unsqueeze(1)
            torch.mm(x[ends[e]:ends[e + 1]], w.t(), out=y[ends[e]:ends[e + 1]])
    return y.to(torch.bfloat16)


def _draws(s, n4):
    """Two draws of 16 bits for each element: Philox-4x32 with 10 rounds (Salmon et al. 2011) on (position / 4, tensor,
    step), word position % 4, low half for the average and high half for the root."""
    ends = torch.tensor(s["start"] // 4, device=DEVICE)
    at = torch.arange(n4, device=DEVICE)
    c1 = torch.bucketize(at, ends[1:], right=True)
    c0 = at - ends[c1]
    t = s["counter"][0] + 1
    c2, c3 = (t & MASK32).expand_as(c0), ((t >> 32) & MASK32).expand_as(c0)
    k0, k1 = s["seed"] & MASK32, (s["seed"] >> 32) & MASK32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & MASK32) ^ c1 ^ k0, b & MASK32, ((a >> 32) & MASK32) ^ c3 ^ k1, a & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    words = torch.stack([c0, c1, c2, c3], 1).view(-1)
    return (words & 0xFFFF).float() / 65536, (words >> 16).float() / 65536


def _drawn_codes(x, u):
    """(e4m3 codes, scales) by blocks; a value between two codes goes up with the probability of its distance."""
    top = x.view(-1, BLOCK).abs().amax(1, keepdim=True)
    y = x.view(-1, BLOCK) * torch.where(top > 0, 448 / top, 0.0)
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp(min=-5) - 4)
    q = (torch.floor(y.abs() / step + u.view(-1, BLOCK)) * step).clamp(max=448)
    return torch.copysign(q, y), top / 448


def _plain_adam(s, c):
    b1, b2 = BETAS
    dt = s["p"].dtype
    p = s["p"] if s["master"] is None else s["master"]
    g, m, v, norm = s["g"].to(p.dtype), s["m"], s["s"], None
    if c["clip"]:
        norm = g.double().square().sum().sqrt()
        g = g * torch.clamp(1.0 / norm, max=1.0).to(g.dtype)
        norm = norm.to(p.dtype)
    t = (s["counter"][0] + 1).double()
    c1, c2 = (1 - b1 ** t).to(p.dtype), (1 - b2 ** t).sqrt().to(p.dtype)
    if c["bits"] == 8:
        sm, sr = s["scales"][:, :1], s["scales"][:, 1:]
        m = (m.float().view(-1, BLOCK) * sm).view(-1)
        v = (v.float().view(-1, BLOCK) * sr).view(-1).square()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    r = v.sqrt()
    p = p * (1 - LR * DECAY) - m / (r / c2 + EPS) * (LR / c1)
    if c["bits"] == 8:
        um, ur = _draws(s, len(m) // 4)
        m, sm = _drawn_codes(m, um)
        v, sr = _drawn_codes(r, ur)
        v = torch.where(r.view(-1, BLOCK) > 0, v.clamp(min=2.0 ** -9), v)
        m, v, s["scales"] = m.view(-1).to(E4M3), v.view(-1).to(E4M3), torch.cat([sm, sr], 1)
    if s["master"] is not None:
        s["master"] = p
    s["p"], s["m"], s["s"] = p.to(dt), m, v
    s["counter"] = s["counter"] + torch.tensor([1, 0], device=DEVICE)
    return [s["p"], s["master"], s["m"], s["s"], s["scales"], norm, s["counter"][0]]


# ------------------------------------------------------------ in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "experts": _exact_experts, "experts8": _exact_experts8,
            "adam": _exact_adam}[case["kind"]](s, case)


def _nearest_e4m3(y):
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp(min=-5) - 4)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_norm(s, c):
    """Degree by degree through torch's own differentiation, from the rounded sum on."""
    n, C, dt = c["rows"], c["C"], s["x"].dtype
    h = s["x"].double()
    if s["residual"] is not None:
        h = (h + s["residual"].double()).to(dt).double()
    flat, w = h.reshape(-1).requires_grad_(True), s["weight"].double().requires_grad_(True)
    outs, tops, at = [], [], 0
    for l in range(c["L"] + 1):
        row = flat[at:at + n * (2 * l + 1) * C].view(n, -1)
        at += row.numel()
        y = row / torch.sqrt((row * row).sum(1, keepdim=True) / row.shape[1] + NORM_EPS) * w[l].repeat(2 * l + 1)
        if c["out"] == "e4m3":
            tops.append(y.detach().abs().max(1)[0] / 448)
            y = _nearest_e4m3(y.detach() / tops[-1].clamp(min=1e-300).unsqueeze(1))
        outs.append(y.reshape(-1))
    y = torch.cat(outs).view(n, -1)
    if c["out"] == "e4m3":
        return [y, torch.stack(tops, 1)] + ([] if s["residual"] is None else [h])
    dx, dw = torch.autograd.grad(y, (flat, w), s["gy"].double())
    dx, y = dx.view(n, -1), y.detach()
    if s["residual"] is None:
        return [y, dx, dw]
    dx = dx + s["gh"].double()
    return [y, h, dx, dx, dw]


def _exact_experts(s, c):
    """Expert by expert, all degrees of its rows at once."""
    R, K, N, L = c["tokens"] * c["k"], c["K"], c["N"], c["L"]
    parts = lambda t, C: [p.view(R, -1, C) for p in t.double().view(-1).split([R * (2 * l + 1) * C for l in range(L + 1)])]
    xs, gs, w = parts(s["x"], K), parts(s["gout"], N), s["weight"].double() * s["scale"]
    ys, dxs = [torch.zeros_like(t) for t in gs], [torch.zeros_like(t) for t in xs]
    dw = torch.zeros_like(w)
    first = 0
    for e, end in enumerate(s["rowptr"].tolist()[1:]):
        for l in range(L + 1):
            x, g = xs[l][first:end].reshape(-1, K), gs[l][first:end].reshape(-1, N)
            ys[l][first:end] = (x @ w[e, l]).view(-1, 2 * l + 1, N)
            dxs[l][first:end] = (g @ w[e, l].T).view(-1, 2 * l + 1, K)
            dw[e, l] = x.T @ g * s["scale"]
        first = end
    flat = lambda ts: torch.cat([t.reshape(-1) for t in ts])
    return [flat(ys).view(R, -1), flat(dxs).view(R, -1), dw]


def _exact_experts8(s, c):
    """Slot by slot of the sorted order, the expert of each from the plan."""
    ends = s["rowptr"].cpu().numpy()
    of = torch.from_numpy(np.repeat(np.arange(c["experts"]), np.diff(ends))).to(DEVICE)
    token = torch.div(s["order"].long(), c["k"], rounding_mode="floor") if c["gather"] else torch.arange(len(of), device=DEVICE)
    y = torch.empty(len(of), c["N"], dtype=torch.float64, device=DEVICE)
    for e in torch.unique(of).tolist():
        slots = torch.nonzero(of == e).squeeze(1)
        rows = s["q"].double()[token[slots]] * s["q_scale"].double()[token[slots]].unsqueeze(1)
        y[slots] = rows @ (s["w"][e].double() * s["w_scale"][e].double().unsqueeze(1)).T
    return y


def _philox_words(block, tensor, step, seed):
    """uint32 words [blocks, 4], on the host."""
    lo, sh = np.uint64(MASK32), np.uint64(32)
    a, b = block, tensor
    d, e = np.full_like(block, step & MASK32), np.full_like(block, step >> 32)
    for r in range(10):
        key = [np.uint64((v + r * w) & MASK32) for v, w in ((seed & MASK32, 0x9E3779B9), ((seed >> 32) & MASK32, 0xBB67AE85))]
        p, q = a * np.uint64(0xD2511F53), d * np.uint64(0xCD9E8D57)
        a, b, d, e = (q >> sh) ^ b ^ key[0], q & lo, (p >> sh) ^ e ^ key[1], p & lo
    return np.stack([a, b, d, e], 1).astype(np.uint32)


def _exact_adam(s, c):
    b1, b2 = BETAS
    t = int(s["counter"][0]) + 1
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    if c["clip"] and float(norm) > 1.0:
        g = g / norm
    p = (s["p"] if s["master"] is None else s["master"]).double()
    if c["bits"] == 8:
        scale = s["scales"].double().repeat_interleave(BLOCK, 0)
        m, v = s["m"].double() * scale[:, 0], (s["s"].double() * scale[:, 1]) ** 2
    else:
        m, v = s["m"].double(), s["s"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    scales = None
    if c["bits"] == 8:
        pads = np.diff(s["start"]) // 4
        if len(g) > 300000000:
            return None
        block = np.concatenate([np.arange(n, dtype=np.uint64) for n in pads])
        words = _philox_words(block, np.repeat(np.arange(len(pads), dtype=np.uint64), pads), t, s["seed"])
        draws = torch.from_numpy(words.reshape(-1).view(np.int32)).to(DEVICE)
        out, tops = [], []
        for x, u in ((m, draws & 0xFFFF), (torch.sqrt(v), (draws >> 16) & 0xFFFF)):
            rows = x.view(-1, BLOCK)
            top = rows.abs().max(1)[0] / 448
            y = rows / top.clamp(min=1e-300).unsqueeze(1)
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            q = torch.floor(y.abs() / step + u.view(-1, BLOCK).double() / 65536) * step
            out.append((torch.sign(y) * q.clamp(max=448)).view(-1))
            tops.append(top)
        m, v = out[0], torch.where(v > 0, out[1].clamp(min=2.0 ** -9), out[1])
        scales = torch.stack(tops, 1)
    return [p, p if s["master"] is not None else None, m, v, scales, norm if c["clip"] else None, None]
