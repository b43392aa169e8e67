"""Operators on rows of atoms, as cases that can be timed: the species embedding and its gradient, rows sorted by
expert and back, and dropout whose mask is drawn from a counter.

``run`` makes the framework's calls where ``own`` is true and computes the same in elementary torch operations where
it is not; ``exact`` restates each operator in 64 bits.  Atom and edge counts, channels and degrees are those of the
framework's workloads (1,024-atom alloy, 12,288-atom water box, 101,306-atom bcc Fe, batches of up to 128 crystals
with 89 elements; 64, 128 or 256 channels in irreps 0 .. L).
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16, "float16": torch.float16}
MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------- cases ----
def listed():
    return [
        # one training step's species embedding of a small alloy cell: latency
        dict(name="embed_alloy", kind="embed", n=1024, vocab=4, C=128, dtype="float32", index="int64", pad=0.0,
             train=True),
        # a batch of crystals padded to a fixed size (padding atoms have token -1)
        dict(name="embed_crystals", kind="embed", n=12801, vocab=89, C=256, dtype="float32", index="int64", pad=0.05,
             train=True),
        # the large iron cell: every row one of two tokens, so sums of 50,000 rows
        dict(name="embed_iron_bf16", kind="embed", n=101306, vocab=2, C=128, dtype="bfloat16", index="int32", pad=0.0,
             train=True),
        # ordered element pairs of all edges of the water-box size, 89^2 tokens, the radial network's width
        dict(name="embed_pairs", kind="embed", n=1063830, vocab=7921, C=64, dtype="float32", index="int32", pad=0.0,
             train=True),
        # one expert a row without gradients, as a small cell is evaluated
        dict(name="route_small_f64", kind="route", tokens=343, k=1, experts=4, C=64, L=0, blocks=False,
             dtype="float64", drop=0.0, train=False),
        # two of eight experts for the alloy's features (degrees 0 .. 3), a training step
        dict(name="route_alloy", kind="route", tokens=1024, k=2, experts=8, C=128, L=3, blocks=True, dtype="float32",
             drop=0.0, train=True),
        # the same for the water box
        dict(name="route_water", kind="route", tokens=12288, k=2, experts=8, C=128, L=3, blocks=True, dtype="float32",
             drop=0.0, train=True),
        # the large cell in 16 bits, row-major rows, a tenth of the choices dropped (expert over capacity)
        dict(name="route_iron_bf16", kind="route", tokens=101306, k=2, experts=16, C=128, L=2, blocks=False,
             dtype="bfloat16", drop=0.1, train=True),
        # scalar features of the alloy, a training step: latency
        dict(name="drop_alloy", kind="drop", rows=1024, C=128, L=0, dtype="float32", p=0.1, residual=False,
             train=True),
        # attention weights of all edges, four heads
        dict(name="drop_attention", kind="drop", rows=1063830, C=4, L=0, dtype="float32", p=0.1, residual=False,
             train=True),
        # the water box's features, one draw per (atom, degree, channel), added to the residual stream
        dict(name="drop_water", kind="drop", rows=12288, C=128, L=3, dtype="float32", p=0.1, residual=True,
             train=True),
        # the large cell's features in 16 bits
        dict(name="drop_iron_bf16", kind="drop", rows=101306, C=128, L=2, dtype="bfloat16", p=0.2, residual=False,
             train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("embed", "route", "drop"))
    dtype = rng.choice(("float32", "float32", "bfloat16", "float16", "float64"))
    train = rng.random() < 0.8
    if kind == "embed":
        C = rng.choice((16, 48, 64, 100, 128, 256))
        n = min(_log_int(rng, 64, 1 << 20), 600000000 // (C * DTYPES[dtype].itemsize))
        return dict(kind=kind, n=n, vocab=_log_int(rng, 1, 8000), C=C, dtype=dtype,
                    index=rng.choice(("int32", "int64")), pad=rng.choice((0.0, 0.0, 0.1)), train=train)
    C, L = rng.choice((32, 64, 100, 128, 256)), rng.randint(0, 3)
    size = {"float64": 8, "float32": 4}.get(dtype, 2) * C * (L + 1) ** 2   # bytes a row
    if kind == "route":
        experts = _log_int(rng, 2, 89)
        k = min(experts, rng.choice((1, 2, 2, 4, 8)))
        return dict(kind=kind, tokens=min(_log_int(rng, 64, 100000), 350000000 // (size * k)), k=k, experts=experts,
                    C=C, L=L, blocks=rng.random() < 0.5, dtype=dtype, drop=rng.choice((0.0, 0.0, 0.15)), train=train)
    rows = min(_log_int(rng, 64, 1 << 20), 400000000 // size, 40000000 // (C * (L + 1)))
    return dict(kind=kind, rows=rows, C=C, L=L, dtype=dtype, p=round(rng.uniform(0.02, 0.6), 3),
                residual=rng.random() < 0.5, train=train)


def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)


def _tokens(gen, n, vocab):
    """Tokens as compositions have them: some common, most rare, in runs (a structure's atoms of one element)."""
    weight = 1.0 / (1.0 + torch.randperm(vocab, generator=gen, device=DEVICE))
    runs = torch.multinomial(weight, n // 4 + 1, replacement=True, generator=gen)
    t = runs.repeat_interleave(4)[:n].clone()
    lone = torch.rand(n, generator=gen, device=DEVICE) < 0.5
    return torch.where(lone, torch.multinomial(weight, n, replacement=True, generator=gen), t)


def _blocks(case):
    return [case["C"] * (2 * l + 1) for l in range(case["L"] + 1)]


def prepare(case, seed):
    g, dt, c = _gen(seed), DTYPES[case["dtype"]], case
    s = dict(case=c)
    if c["kind"] == "embed":
        t = _tokens(g, c["n"], c["vocab"])
        s["tokens"] = torch.where(torch.arange(c["n"], device=DEVICE) >= int(c["n"] * (1 - c["pad"])), -1, t).to(
            torch.int32 if c["index"] == "int32" else torch.int64)
        s["table"] = _normal(g, dt, c["vocab"], c["C"])
        s["scale"] = 1.0 / math.sqrt(c["vocab"])
        s["gout"] = _normal(g, dt, c["n"], c["C"]) if c["train"] else None
    elif c["kind"] == "route":
        T, k, E, D = c["tokens"], c["k"], c["experts"], c["C"] * (c["L"] + 1) ** 2
        popular = torch.randn(E, generator=g, device=DEVICE)
        score, e = (torch.randn(T, E, generator=g, device=DEVICE) + popular).topk(k)
        dropped = torch.rand(T, k, generator=g, device=DEVICE) < c["drop"]
        s["experts"] = torch.where(dropped, -1, e).to(torch.int32)
        s["weights"] = torch.softmax(score, 1).to(dt if dt == torch.float64 else torch.float32)
        s["widths"] = _blocks(c) if c["blocks"] else None
        s["x"], s["y"] = _normal(g, dt, T, D), _normal(g, dt, T * k, D)
        if c["train"]:
            s["gxs"], s["gout"] = _normal(g, dt, T * k, D), _normal(g, dt, T, D)
    else:
        rows, D = c["rows"], c["C"] * (c["L"] + 1) ** 2
        s["rng"] = torch.tensor([int(seed) * 7919 + (12345 << 34), 977 + (int(seed) << 33)], dtype=torch.int64,
                                device=DEVICE)
        s["x"] = _normal(g, dt, rows, D)
        s["residual"] = _normal(g, dt, rows, D) if c["residual"] else None
        s["gout"] = _normal(g, dt, rows, D) if c["train"] else None
    return s


def _leaf(t):
    return t.detach().requires_grad_(True)


def run(s):
    c = s["case"]
    if not own:
        return {"embed": _plain_embed, "route": _plain_route, "drop": _plain_drop}[c["kind"]](s, c)
    from tace_amd import ops

    if c["kind"] == "embed":
        if not c["train"]:
            return ops.embedding(s["table"], s["tokens"], s["scale"])
        table = _leaf(s["table"])
        out = ops.embedding(table, s["tokens"], s["scale"])
        return [out, *torch.autograd.grad(out, table, s["gout"])]
    if c["kind"] == "route":
        if not c["train"]:
            plan = ops.route_plan(s["experts"], c["experts"])
            return [plan.rowptr, ops.expert_dispatch(s["x"], plan, widths=s["widths"]),
                    ops.expert_combine(s["y"], plan, s["weights"], widths=s["widths"])]
        x, y, w = _leaf(s["x"]), _leaf(s["y"]), _leaf(s["weights"])
        plan = ops.route_plan(s["experts"], c["experts"])
        xs = ops.expert_dispatch(x, plan, widths=s["widths"])
        out = ops.expert_combine(y, plan, w, widths=s["widths"])
        gy, gw = torch.autograd.grad(out, (y, w), s["gout"])
        return [plan.rowptr, xs, out, *torch.autograd.grad(xs, x, s["gxs"]), gy, gw]
    comps = [2 * l + 1 for l in range(c["L"] + 1)]
    if not c["train"]:
        return ops.dropout(s["x"], c["p"], s["rng"], site=3, components=comps, residual=s["residual"])
    leaves = [_leaf(t) for t in (s["x"], s["residual"]) if t is not None]
    out = ops.dropout(leaves[0], c["p"], s["rng"], site=3, components=comps,
                      residual=leaves[1] if c["residual"] else None)
    return [out, *torch.autograd.grad(out, leaves, s["gout"])]


def _rows_moved(c):
    return c["tokens"] * c["k"]


def work(case):
    c = case
    b = DTYPES[c["dtype"]].itemsize
    if c["kind"] == "embed":
        ids = c["n"] * (4 if c["index"] == "int32" else 8)
        fwd = ids + b * c["C"] * (min(c["vocab"], c["n"]) + c["n"])
        return dict(bytes=fwd + (b * c["C"] * (c["n"] + c["vocab"]) if c["train"] else 0),
                    flops=c["n"] * c["C"] * (2 if c["train"] else 1))
    D = c["C"] * (c["L"] + 1) ** 2
    if c["kind"] == "route":
        T, n = c["tokens"], _rows_moved(c)
        small = 4 * n + 4 * (c["experts"] + 1) + n * (8 if b == 8 else 4)
        one = b * D * (T + n)                       # rows once on each side
        if not c["train"]:
            return dict(bytes=small + 2 * one, flops=2 * n * D)
        # dispatch, its gradient, combine; the combine's gradient reads gout and y and writes gy (and the weights')
        return dict(bytes=small + 3 * one + b * D * (T + 2 * n) + n * (8 if b == 8 else 4), flops=8 * n * D)
    n = c["rows"] * D
    draws = c["rows"] * c["C"] * (c["L"] + 1)
    streams = (3 if c["residual"] else 2) + (2 if c["train"] else 0)
    return dict(bytes=b * n * streams, flops=n * (2 if c["train"] else 1) + draws * (2 if c["train"] else 1) * 12)


# ------------------------------------------------------------- plain forms ----
def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _plain_embed(s, c):
    t, table = s["tokens"].long(), s["table"]
    V = table.shape[0]
    ok = ((t >= 0) & (t < V)).unsqueeze(1)
    out = torch.where(ok, _wide(table)[t.clamp(0, V - 1)] * s["scale"], 0.0).to(table.dtype)
    if not c["train"]:
        return out
    at = torch.where(ok.squeeze(1), t, V)
    if V <= 128:   # few tokens: the product with their one-hot rows
        hot = torch.nn.functional.one_hot(at, V + 1)[:, :V].to(_wide(table).dtype)
        grad = hot.t() @ _wide(s["gout"])
    elif table.dtype != torch.float64:
        grad = torch.zeros(V + 1, c["C"], device=t.device).index_add_(0, at, s["gout"].float())[:V]
    else:          # rows sorted by token (padding last), each token's range summed
        key, order = at.sort(stable=True)
        end = torch.searchsorted(key, torch.arange(V + 1, device=key.device))
        grad = torch.segment_reduce(s["gout"][order], "sum", offsets=end, axis=0, initial=0.0, unsafe=True)
    return [out, (grad * s["scale"]).to(table.dtype)]


def _to_rows(x, widths):
    """Group-major features (every block of all rows after the other) as ordinary rows."""
    if widths is None:
        return x
    parts = x.reshape(-1).split([x.shape[0] * w for w in widths])
    return torch.cat([p.view(x.shape[0], w) for p, w in zip(parts, widths)], 1)


def _from_rows(x, widths):
    if widths is None:
        return x
    return torch.cat([p.reshape(-1) for p in x.split(widths, 1)]).view(x.shape)


def _plain_route(s, c):
    T, k, E, dt, wd = c["tokens"], c["k"], c["experts"], s["x"].dtype, s["widths"]
    e = s["experts"].long().reshape(-1)
    kept = (e >= 0) & (e < E)
    key = torch.where(kept, e, E)
    order = key.argsort(stable=True)
    rowptr = torch.cat([key.new_zeros(1), key.bincount(minlength=E + 1)[:E].cumsum(0)]).int()
    place = torch.empty_like(order).scatter_(0, order, torch.arange(T * k, device=order.device))
    token, w, used = order // k, _wide(s["weights"]), kept[order].unsqueeze(1)
    xs = _from_rows(torch.where(used, _to_rows(s["x"], wd)[token], 0.0), wd)
    y = torch.where(kept.unsqueeze(1), _wide(_to_rows(s["y"], wd)[place]), 0.0).view(T, k, -1)
    out = _from_rows((y * w.unsqueeze(2)).sum(1).to(dt), wd)
    if not c["train"]:
        return [rowptr, xs, out]
    gxs = torch.where(kept.unsqueeze(1), _wide(_to_rows(s["gxs"], wd)[place]), 0.0).view(T, k, -1)
    gx = _from_rows(gxs.sum(1).to(dt), wd)
    g = _wide(_to_rows(s["gout"], wd))
    gw = (g.unsqueeze(1) * y).sum(2).to(w.dtype)
    gy = _from_rows(torch.where(used, g[token] * w.reshape(-1)[order].unsqueeze(1), 0.0).to(dt), wd)
    return [rowptr, xs, out, gx, gy, gw]


def _keep(rng, site, count, p):
    """Philox-4x32 with 10 rounds (Salmon et al. 2011) on (index / 8, site, offset) under the key of the seed: eight
    draws of 16 bits a block, low half of each word first; true where a draw is at least round(65536 p)."""
    block = torch.arange((count + 7) // 8, device=rng.device)
    c0, c1 = block & MASK32, torch.full_like(block, site)
    c2, c3 = (rng[1] & MASK32).expand_as(block), ((rng[1] >> 32) & MASK32).expand_as(block)
    k0, k1 = rng[0] & MASK32, (rng[0] >> 32) & MASK32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & MASK32) ^ c1 ^ k0, b & MASK32, ((a >> 32) & MASK32) ^ c3 ^ k1, a & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    words = torch.stack([c0, c1, c2, c3], 1)
    return (torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:count] >= round(65536 * p))


def _plain_drop(s, c):
    x, C, n = s["x"], c["C"], c["rows"]
    comps = [2 * l + 1 for l in range(c["L"] + 1)]
    keep = _keep(s["rng"], 3, n * len(comps) * C, c["p"]).view(n, len(comps), 1, C)
    scale = 65536.0 / (65536 - round(65536 * c["p"]))

    def masked(t):
        parts = t.reshape(-1).split([n * d * C for d in comps])
        return torch.cat([torch.where(keep[:, b], _wide(q.view(n, d, C)) * scale, 0.0).reshape(-1)
                          for b, (q, d) in enumerate(zip(parts, comps))]).view(t.shape)

    out = masked(x)
    if s["residual"] is not None:
        out = out + _wide(s["residual"])
    out = out.to(x.dtype)
    if not c["train"]:
        return out
    return [out, masked(s["gout"]).to(x.dtype)] + ([s["gout"]] if c["residual"] else [])


# ------------------------------------------------------------ in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "route": _exact_route, "drop": _exact_drop}[case["kind"]](s, case)


def _exact_embed(s, c):
    t, table = s["tokens"].long(), s["table"].double()
    rows = torch.nonzero((t >= 0) & (t < c["vocab"])).squeeze(1)
    out = torch.zeros(c["n"], c["C"], dtype=torch.float64, device=t.device)
    out[rows] = table.index_select(0, t[rows]) * s["scale"]
    if not c["train"]:
        return out
    grad = torch.zeros_like(table).index_put_((t[rows],), s["gout"].double()[rows], accumulate=True)
    return [out, grad * s["scale"]]


def _exact_route(s, c):
    """Row by row of the sorted order, made on the host."""
    T, k, E, D, wd = c["tokens"], c["k"], c["experts"], s["x"].shape[1], s["widths"]
    dev = s["x"].device
    e = s["experts"].cpu().numpy().reshape(-1)
    slots = np.concatenate([np.flatnonzero(e == q) for q in range(E)])
    rowptr = np.concatenate([[0], np.cumsum([(e == q).sum() for q in range(E)])])
    R = len(slots)
    tok, slot = torch.from_numpy(slots // k).to(dev), torch.from_numpy(slots).to(dev)
    w = s["weights"].double().reshape(-1)[slot].unsqueeze(1)
    zero = torch.zeros(T * k, D, dtype=torch.float64, device=dev)

    def rows(t):
        return _to_rows(t.double(), wd)

    y = rows(s["y"])[:R]
    xs = zero.clone()
    xs[:R] = rows(s["x"])[tok]
    out = torch.zeros(T, D, dtype=torch.float64, device=dev).index_add_(0, tok, w * y)
    ptr = torch.from_numpy(rowptr.astype(np.int32))
    if not c["train"]:
        return [ptr, _from_rows(xs, wd), _from_rows(out, wd)]
    gx = torch.zeros(T, D, dtype=torch.float64, device=dev).index_add_(0, tok, rows(s["gxs"])[:R])
    g = rows(s["gout"])[tok]
    gw = torch.zeros(T * k, dtype=torch.float64, device=dev)
    gw[slot] = (g * y).sum(1)
    gy = zero
    gy[:R] = w * g
    return [ptr, _from_rows(xs, wd), _from_rows(out, wd), _from_rows(gx, wd), _from_rows(gy, wd), gw.view(T, k)]


def _exact_drop(s, c):
    n, C, comps = c["rows"], c["C"], [2 * l + 1 for l in range(c["L"] + 1)]
    seed, offset = (int(v) & (2 ** 64 - 1) for v in s["rng"].tolist())
    block = np.arange((n * len(comps) * C + 7) // 8, dtype=np.uint64)
    lo, sh = np.uint64(MASK32), np.uint64(32)
    a, b = block, np.full_like(block, 3)
    d, e = np.full_like(block, offset & MASK32), np.full_like(block, offset >> 32)
    for r in range(10):
        key = [np.uint64((v + r * w) & MASK32) for v, w in ((seed & MASK32, 0x9E3779B9), (seed >> 32, 0xBB67AE85))]
        p, q = a * np.uint64(0xD2511F53), d * np.uint64(0xCD9E8D57)
        a, b, d, e = (q >> sh) ^ b ^ key[0], q & lo, (p >> sh) ^ e ^ key[1], p & lo
    words = np.stack([a, b, d, e], 1).astype(np.uint32)
    draws = np.ascontiguousarray(words).view(np.uint16).reshape(-1)[:n * len(comps) * C]   # (little endian)
    thr = round(65536 * c["p"])
    keep = torch.from_numpy(draws >= thr).to(s["x"].device).view(n, len(comps), C).double() * (65536.0 / (65536 - thr))
    factor = torch.cat([keep[:, l].repeat_interleave(2 * l + 1, 0).reshape(-1) for l in range(c["L"] + 1)]).view(n, -1)
    out = s["x"].double() * factor
    if s["residual"] is not None:
        out = out + s["residual"].double()
    if not c["train"]:
        return out
    return [out, s["gout"].double() * factor] + ([s["gout"].double()] if c["residual"] else [])
