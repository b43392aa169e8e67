"""What the tests of the row operators share: bounds on rounding, Philox and 64-bit restatements (CPU tensors)."""

import torch

TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def sum_step(dt):
    """Half a step of the sums' type."""
    return 2.0 ** -53 if dt == torch.float64 else 2.0 ** -24


def rounded(value, dt):
    """How far a value (64 bits) may be off by one rounding to dt: half a step, and half the least subnormal."""
    f = torch.finfo(dt)
    return value.abs() * half_step(dt) + f.smallest_normal * f.eps / 2


def assert_within(got, want, bound, what=""):
    err = (got.detach().cpu().double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), err[bad].max().item(), bound.expand_as(err)[bad].max().item())


def philox(counter, key):
    """Philox-4x32, 10 rounds, on Python integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def draws(count, seed, offset, site):
    """The first `count` 16-bit draws of (seed, offset, site)."""
    s, o = seed % 2 ** 64, offset % 2 ** 64
    out = []
    for block in range((count + 7) // 8):
        for word in philox((block, site, o & 0xFFFFFFFF, o >> 32), (s & 0xFFFFFFFF, s >> 32)):
            out += [word & 0xFFFF, word >> 16]
    return torch.tensor(out[:count], dtype=torch.int64)


def keep_factor(rows, C, comps, p, seed, offset, site):
    """[rows, sum(comps) C] in group-major order: 0 where dropped, else the scale (64 bits)."""
    thr = round(65536 * p)
    keep = (draws(rows * len(comps) * C, seed, offset, site) >= thr).view(rows, len(comps), 1, C)
    scale = 0.0 if thr == 65536 else 65536.0 / (65536 - thr)
    parts = [(keep[:, b].double() * scale).expand(rows, d, C).reshape(-1) for b, d in enumerate(comps)]
    return torch.cat(parts).view(rows, sum(comps) * C) if parts else None


def to_rows(x, widths):
    """Group-major features as ordinary rows."""
    n = x.shape[0]
    return torch.cat([p.view(n, w) for p, w in zip(x.reshape(-1).split([n * w for w in widths]), widths)], 1)


def from_rows(x, widths):
    return torch.cat([p.reshape(-1) for p in x.split(list(widths), 1)]).view(x.shape)


class Route:
    """The sorted order of `experts` [T, k], on the host."""

    def __init__(self, experts, E):
        flat = experts.reshape(-1).long()
        self.k = experts.shape[1]
        self.kept = (flat >= 0) & (flat < E)
        self.order = torch.where(self.kept, flat, torch.full_like(flat, E)).argsort(stable=True)
        self.place = torch.empty_like(self.order)
        self.place[self.order] = torch.arange(len(flat))
        counts = torch.stack([(flat == e).sum() for e in range(E)]) if E else torch.zeros(0, dtype=torch.int64)
        self.rowptr = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])

    def dispatch(self, x, w, widths):
        rows = to_rows(x, widths).repeat_interleave(self.k, 0)
        if w is not None:
            rows = rows * w.reshape(-1, 1)
        rows = torch.where(self.kept.view(-1, 1), rows, torch.zeros((), dtype=x.dtype))
        return from_rows(rows[self.order], widths)

    def combine(self, y, w, widths):
        rows = to_rows(y, widths)[self.place]
        if w is not None:
            rows = rows * w.reshape(-1, 1)
        rows = torch.where(self.kept.view(-1, 1), rows, torch.zeros((), dtype=y.dtype))
        return from_rows(rows.view(-1, self.k, rows.shape[1]).sum(1), widths)
