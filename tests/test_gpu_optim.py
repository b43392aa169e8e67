"""The step of AdamW against 64-bit restatements and torch's optimiser.

u: half a step of the sums' type.  m and v: the two rates and their complements are rounded once each, two products, one
sum, v's square; a clipped gradient is off by its norm's error (16 squares a thread in the sums' type: 9 u, and 3).
"""

import math

import pytest
import torch

from tace_amd import ops, optim

import _rows as R

pytestmark = pytest.mark.gpu

ids = lambda v: str(v).replace("torch.", "")
BLOCK = 256
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
SIZES = [(1,), (3,), (255,), (256,), (257,), (16, 33), (4095,), (4096,), (4097,), (0,), (3, 5000), (12289,), (40000,)]


def _rand(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale


class Case:
    """Lists for adamw_step and their values in 64 bits."""

    def __init__(self, cuda, dt, sizes, bits=32, masters=False, steps=6, offset=0):
        wide = torch.float64 if dt == torch.float64 else torch.float32
        def place(t):   # (offset: elements from an aligned address)
            flat = torch.zeros(t.numel() + offset, dtype=t.dtype, device=cuda)
            return flat[offset:].view(t.shape).copy_(t)
        self.w = [_rand(s, i, 0.3) for i, s in enumerate(sizes)]
        self.p = [place(t.to(dt)) for t in self.w]
        self.g = [place(_rand(s, 100 + i, 0.1).to(dt)) for i, s in enumerate(sizes)]
        self.masters = [place(t.float()) for t in self.w] if masters else None
        m = [_rand(s, 200 + i, 0.05) for i, s in enumerate(sizes)]
        r = [_rand(s, 300 + i, 0.05).abs() + 0.02 for i, s in enumerate(sizes)]
        self.scales = None
        if bits == 8:
            self.m, self.s, self.scales = [], [], []
            for a, b in zip(m, r):
                ca, sa = self._codes(a)
                cb, sb = self._codes(b)
                self.m.append(place(ca))
                self.s.append(place(cb))
                self.scales.append(torch.stack([sa, sb], 1).to(cuda))
        else:
            self.m, self.s = [place(t.to(wide)) for t in m], [place(t.square().to(wide)) for t in r]
        self.counter = torch.tensor([steps, 0], dtype=torch.int64, device=cuda)
        self.dt, self.bits, self.u = dt, bits, R.sum_step(dt)

    @staticmethod
    def _codes(t):
        flat = torch.zeros(-(-t.numel() // BLOCK) * BLOCK, dtype=torch.float64)
        flat[:t.numel()] = t.reshape(-1)
        s = (flat.view(-1, BLOCK).abs().amax(1) / 448).float()
        q = (flat.view(-1, BLOCK) / s.double().clamp(min=1e-30).unsqueeze(1)).float().to(torch.float8_e4m3fn)
        return q.view(-1)[:t.numel()].view(t.shape), s

    def _state(self, t, i, col):
        v = t[i].cpu().double()
        if self.bits != 8:
            return v
        s = self.scales[i][:, col].cpu().double().repeat_interleave(BLOCK)[:v.numel()].view(v.shape)
        return v * s

    def values(self):
        """(weights, gradients, m, v) in 64 bits."""
        w = self.masters if self.masters else self.p
        return ([t.cpu().double() for t in w], [t.cpu().double() for t in self.g],
                [self._state(self.m, i, 0) for i in range(len(self.p))],
                [self._state(self.s, i, 1) ** (2 if self.bits == 8 else 1) for i in range(len(self.p))])

    def step(self, **more):
        return ops.adamw_step(self.p, self.g, self.m, self.s, self.counter, scales=self.scales, masters=self.masters,
                              **{**HYPER, **more})


def _formula(w, g, m, v, t, clip, lr, betas, eps, weight_decay):
    b1, b2 = betas
    # 1 - b^t: written so, it loses up to 1 / (1 - b^t) half steps, 5e-13 for b = 0.9999 and t = 2
    c1, c2 = (-math.expm1(t * math.log(b)) if b else 1.0 for b in betas)
    g = g * clip
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    mag = b1 * m.abs() + (1 - b1) * g.abs()
    den = (v / c2).sqrt() + eps
    return w * (1 - lr * weight_decay) - lr / c1 * m / den, m, v, lr / c1 * (mag + m.abs()) / den


def _run(c, max_norm=None, **more):
    before, t = c.values(), int(c.counter[0]) + 1
    norm = c.step(max_norm=max_norm, **more)
    total = torch.cat([g.reshape(-1) for g in before[1]]).norm()
    clip = 1.0
    if max_norm is not None:
        R.assert_within(norm, total, total * 14 * c.u, "norm")
        clip = min(1.0, max_norm / float(total))
    assert c.counter.tolist() == [t, 0]
    hyper = {**HYPER, **{k: v for k, v in more.items() if k in HYPER}}
    u, ug = c.u, 16 * c.u    # the clipped gradient's relative error
    for i, (w, g, m, v) in enumerate(zip(*before)):
        b1, b2 = hyper["betas"]
        p1, m1, v1, moved = _formula(w, g, m, v, t, clip, **hyper)
        m_slack = (b1 * m.abs() * 4 + (1 - b1) * (g * clip).abs() * 4) * u + (1 - b1) * (g * clip).abs() * ug
        v_slack = (b2 * v * 5 + (1 - b2) * (g * clip) ** 2 * 5) * u + (1 - b2) * (g * clip) ** 2 * 2 * ug
        # the quotient: m's and half of v's error, the two corrections' (4 u each), 8 operations; p's own 3
        p_slack = w.abs() * 4 * u + moved * (4 * u + ug + 2.5 * u + ug + 16 * u)
        got = (c.masters if c.masters else c.p)[i]
        R.assert_within(got, p1, p_slack + R.rounded(p1.abs() + p_slack, got.dtype), "p")
        if c.masters:
            assert torch.equal(c.p[i], c.masters[i].to(c.dt))
        if c.bits == 8:
            for col, want, slack in ((0, m1, m_slack), (1, v1.sqrt(), v1.sqrt() * (3 * u + ug))):
                codes = (c.m, c.s)[col][i].cpu().float().double().reshape(-1)
                scale = c.scales[i][:, col].cpu().double()
                flat = torch.zeros(len(scale) * BLOCK, dtype=torch.float64)
                flat[:codes.numel()] = want.reshape(-1)
                top = flat.view(-1, BLOCK).abs().amax(1) / 448
                R.assert_within(scale, top, top * 24 * u + ug * top, "scale")
                unit = want.reshape(-1) / scale.clamp(min=1e-300).repeat_interleave(BLOCK)[:codes.numel()]
                step = torch.exp2(torch.floor(torch.log2(unit.abs().clamp(min=2.0 ** -6))) - 3)
                R.assert_within(codes, unit, step * (1 + 2.0 ** -10), "codes")   # one of the two beside the value
                if col:
                    assert bool((codes[want.reshape(-1) > 0] > 0).all())
        else:
            wide = c.m[i].dtype
            R.assert_within(c.m[i], m1, m_slack + R.rounded(m1.abs() + m_slack, wide), "m")
            R.assert_within(c.s[i], v1, v_slack + R.rounded(v1.abs() + v_slack, wide), "v")


@pytest.mark.parametrize("max_norm", [None, 0.5, 1e4])
@pytest.mark.parametrize("dt,bits,masters", [(torch.float64, 32, False), (torch.float32, 32, False), (torch.float32, 8, False),
                                             (torch.bfloat16, 32, False), (torch.bfloat16, 32, True), (torch.bfloat16, 8, True),
                                             (torch.float16, 8, False), (torch.float16, 32, True)], ids=ids)
@pytest.mark.parametrize("offset", [0, 1])
def test_step(cuda, dt, bits, masters, max_norm, offset):
    c = Case(cuda, dt, SIZES, bits, masters, offset=offset)
    for _ in range(2):
        _run(c, max_norm)


@pytest.mark.parametrize("steps", [0, 1, 999, 10 ** 7, 2 ** 33])
def test_first_and_late_steps(cuda, steps):
    c = Case(cuda, torch.float32, [(300,), (5000,)], steps=steps)
    _run(c, betas=(0.9, 0.999))
    _run(Case(cuda, torch.float64, [(300,), (5000,)], steps=steps), betas=(0.9, 0.9999))


def test_ends_of_the_arguments(cuda):
    _run(Case(cuda, torch.float32, [(700,)]), betas=(0.0, 0.0))
    _run(Case(cuda, torch.float32, [(700,)]), lr=0.0, weight_decay=0.0)
    for dt in (torch.float32, torch.float64):
        lr = torch.tensor([1e-2], dtype=dt, device=cuda)
        a, b = Case(cuda, torch.float32, [(700,)]), Case(cuda, torch.float32, [(700,)])
        a.step(lr=lr)
        b.step(lr=float(lr))
        assert torch.equal(a.p[0], b.p[0])


def test_many_tensors_and_large_ones(cuda):
    _run(Case(cuda, torch.float32, [(1 + 37 * i,) for i in range(130)]), 0.3)
    _run(Case(cuda, torch.bfloat16, [(2_000_001,), (7,), (1 << 20,)], 8, True), 0.3)


@pytest.mark.parametrize("before", [56, 84, 160, 330])
def test_empty_tensors_before_others(cuda, before):
    """(a launch's worth of tensors without an element)"""
    for dt, bits, masters in ((torch.float32, 32, False), (torch.bfloat16, 32, True), (torch.float32, 8, False)):
        _run(Case(cuda, dt, [(0,)] * before + [(5,), (0,), (300,)], bits, masters), 0.3)
    g = [torch.zeros(0, device=cuda)] * before + [torch.full((4,), 3.0, device=cuda)]
    assert float(ops.grad_norm(g)) == 6.0


def test_elements_past_32_bits(cuda):
    """A parameter of 2^31 + 4097 elements: those at its end are stepped as those of a small one."""
    n = 2 ** 31 + 4097
    p = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    g = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    m, s = (torch.zeros(n, dtype=torch.float8_e4m3fn, device=cuda) for _ in range(2))
    sc = torch.zeros(-(-n // BLOCK), 2, device=cuda)
    p[-5000:], g[-5000:] = 1.0, torch.arange(5000, device=cuda).bfloat16() + 1
    counter = torch.zeros(2, dtype=torch.int64, device=cuda)
    norm = ops.adamw_step([p], [g], [m], [s], counter, scales=[sc], max_norm=1e9, lr=0.125, weight_decay=0.0)
    assert counter.tolist() == [1, 0] and abs(float(norm) - float(g[-5000:].double().norm())) < 1e-5 * float(norm)
    assert torch.equal(p[-5000:], torch.full((5000,), 0.875, dtype=torch.bfloat16, device=cuda))   # first step: lr
    assert not p[:-5000].any() and not sc[:-22].any() and bool((sc[-20:] > 0).all())
    assert bool((s[-5000:].float() > 0).all()) and not s[2 ** 31 - 5000:2 ** 31 - 4000].float().any()


# ------------------------------------------------------------------ 8 bits ----
def test_codes_are_the_drawn_ones(cuda):
    """Every code from its draw: floor(value / step + draw / 65536) steps, but where the sum is next to a whole number."""
    seed, steps, sizes = 2 ** 40 + 977, 2 ** 34 + 5, [(700,), (1300,)]
    c = Case(cuda, torch.float32, sizes, 8, steps=steps)
    before = c.values()
    c.step(seed=seed)
    t = steps + 1
    for i, (w, g, m, v) in enumerate(zip(*before)):
        _, m1, v1, _ = _formula(w, g, m, v, t, 1.0, **HYPER)
        n = w.numel()
        words = [x for b in range(-(-n // 4)) for x in R.philox((b, i, t & 0xFFFFFFFF, t >> 32),
                                                                (seed & 0xFFFFFFFF, seed >> 32))]
        words = torch.tensor(words[:n], dtype=torch.int64)
        for col, want, draw in ((0, m1, words & 0xFFFF), (1, v1.sqrt(), words >> 16)):
            codes = (c.m, c.s)[col][i].cpu().float().double()
            unit = want / c.scales[i][:, col].cpu().double().repeat_interleave(BLOCK)[:n]
            step = torch.exp2(torch.floor(torch.log2(unit.abs().clamp(min=2.0 ** -6))) - 3)
            place = unit.abs() / step + draw.double() / 65536
            near = (place - place.round()).abs() < 16 * 2.0 ** -20    # (values of up to 16 steps, off by 2^-20)
            edge = (torch.log2(unit.abs()) - torch.log2(unit.abs()).round()).abs() < 2.0 ** -18
            expect = torch.sign(unit) * (torch.floor(place) * step).clamp(max=448)
            ok = (codes == expect) | near | edge
            assert bool(ok.all()) and float((near | edge).double().mean()) < 0.01


@pytest.mark.parametrize("dt,masters", [(torch.float32, False), (torch.bfloat16, True)], ids=ids)
def test_scales_are_those_of_single_operations(cuda, dt, masters):
    """Every product and sum rounded by itself: a largest element a last place off could draw another code."""
    c = Case(cuda, dt, [(BLOCK * 500 + 77,), (4096,)], 8, masters=masters)
    b1, b2 = (torch.tensor(b, dtype=torch.float64) for b in HYPER["betas"])
    want = []
    for g, m, s, sc in zip(c.g, c.m, c.s, c.scales):
        g, m, s, sc = g.cpu().float(), m.cpu().float(), s.cpu().float(), sc.cpu()
        sm, sr = (sc[:, k].repeat_interleave(BLOCK)[:g.numel()] for k in (0, 1))
        m, r = m * sm, s * sr
        m = m * b1.float() + g * (1 - b1).float()
        v = (r * r) * b2.float() + (g * g) * (1 - b2).float()
        flat = torch.zeros(2, sc.shape[0] * BLOCK)
        # (a root in 64 bits, rounded once: the host's float32 root is not always the nearest)
        flat[0, :g.numel()], flat[1, :g.numel()] = m.abs(), v.double().sqrt().float()
        want.append(flat.view(2, -1, BLOCK).amax(2).mul(torch.tensor(1 / 448)).t())
    c.step()
    for w, sc in zip(want, c.scales):
        assert torch.equal(w, sc.cpu())


def test_a_slow_average_moves_in_the_mean(cuda):
    """0.1 % of the way a step: codes to nearest would never move."""
    n, steps = 1 << 16, 60
    p, m = torch.zeros(n, device=cuda), torch.zeros(n, device=cuda)
    q = [torch.zeros(n, dtype=torch.float8_e4m3fn, device=cuda) for _ in range(2)]
    q[1] = torch.full((n,), 448.0, device=cuda).to(torch.float8_e4m3fn)
    sc = torch.full((n // BLOCK, 2), 1.0 / 448, device=cuda)
    sc[:, 0] = 0
    g = torch.full((n,), 0.5, device=cuda)
    g[::BLOCK] = 1.0     # keeps the block's scale
    counter = torch.zeros(2, dtype=torch.int64, device=cuda)
    for _ in range(steps):
        ops.adamw_step([p], [g], [q[0]], [q[1]], counter, scales=[sc], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, seed=9)
    root = (q[1].float() * sc[:, 1].repeat_interleave(BLOCK))
    want = (0.999 ** steps + (1 - 0.999 ** steps) * 0.25) ** 0.5
    got = root.view(-1, BLOCK)[:, 1:].double().mean()
    # unbiased: a step's deviation is at most half a code's step (1/14 of the value); 65,000 of them, 60 steps, 6 sigma,
    # and the curvature of the root: the variance of r is added to v each step
    assert abs(float(got) - want) < 6 * (steps ** 0.5) / 28 / (n ** 0.5) + steps * (1 / 28) ** 2 * 0.02


# ------------------------------------------------------------------- norms ----
@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
def test_grad_norm(cuda, dt):
    for sizes in ([(1,)], SIZES, [(5_000_003,), (1,)], [(i + 1,) for i in range(120)]):
        g = [_rand(s, i).to(dt).to(cuda) for i, s in enumerate(sizes)]
        # (summed exactly: a sum of 5 M doubles one after the other is itself 40 half steps off)
        want = torch.tensor(math.sqrt(math.fsum(v * v for t in g for v in t.cpu().double().reshape(-1).tolist())),
                            dtype=torch.float64)
        got = ops.grad_norm(g)
        assert got.dim() == 0 and got.dtype == (torch.float64 if dt == torch.float64 else torch.float32)
        # float64's outer sums count too: 2 units a thread, 9 levels of a workgroup, 4 workgroups a thread, 9 levels, so
        # half of 17 + 24 and the root; the squares of the sum above (half of 1) and its root
        R.assert_within(got, want, want * (12 if dt != torch.float64 else 24) * R.sum_step(dt), str(sizes))
        assert torch.equal(got, ops.grad_norm(g))
    assert float(ops.grad_norm([torch.zeros(0, device=cuda)])) == 0
    assert torch.isnan(ops.grad_norm([torch.full((9,), float("nan"), device=cuda)]))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_norm_that_is_no_number_changes_nothing(cuda, bits):
    for bad in (float("inf"), float("nan")):
        c = Case(cuda, torch.float32, [(300,), (5000,)], bits)
        c.g[1][77] = bad
        everything = [t for l in (c.p, c.m, c.s, c.scales or []) for t in l] + [c.counter]
        before = [t.clone() for t in everything]
        norm = c.step(max_norm=1.0)
        assert not torch.isfinite(norm)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, everything))
        c.g[1][77] = 0.0
        _run(c, 1.0)    # and the next step is a step


def test_gradients_of_other_layouts(cuda):
    c, d = (Case(cuda, torch.float32, [(64, 48), (33, 7)]) for _ in range(2))
    c.g[0] = c.g[0].t().contiguous().t()
    c.g[1] = torch.ones((), device=cuda).expand(33, 7)
    d.g[1] = torch.ones(33, 7, device=cuda)
    c.step(max_norm=1.0)
    d.step(max_norm=1.0)
    assert all(torch.equal(a, b) for a, b in zip(c.p, d.p))


# --------------------------------------------------------------- optimiser ----
def _params(cuda, dt, n=5, seed=0):
    return [_rand((17 * (i + 1), 9), seed + i).to(dt).to(cuda).requires_grad_(True) for i in range(n)]


def _set_grads(ps, step):
    for i, p in enumerate(ps):
        p.grad = (_rand(p.shape, 1000 * step + i) * 0.1).to(p.dtype).to(p.device)


def test_optimiser_is_torchs(cuda):
    """Thirty steps in float64, two groups, clipping over both, a changing rate."""
    a, b = _params(cuda, torch.float64), _params(cuda, torch.float64)
    groups = lambda ps: [dict(params=ps[:2], lr=1e-2), dict(params=ps[2:], lr=3e-3, weight_decay=0.0)]
    ours = optim.AdamW(groups(a), betas=(0.8, 0.99), max_norm=0.7)
    theirs = torch.optim.AdamW(groups(b), betas=(0.8, 0.99), foreach=False)
    for k in range(30):
        _set_grads(a, k)
        _set_grads(b, k)
        norm = torch.cat([p.grad.reshape(-1) for p in b]).norm()
        for p in b:
            p.grad *= torch.clamp(0.7 / norm, max=1.0)
        for o in (ours, theirs):
            o.param_groups[0]["lr"] = 1e-2 / (1 + k)
            o.step()
        assert abs(float(ours.norm) - float(norm)) < 1e-12 * float(norm)
    for p, q in zip(a, b):
        # 30 steps of a few roundings each of values of order 1
        assert torch.allclose(p, q, rtol=1e-13, atol=1e-13)


def test_parameters_without_a_gradient_keep_their_count(cuda):
    a, b = _params(cuda, torch.float64), _params(cuda, torch.float64)
    ours, theirs = optim.AdamW(a, lr=1e-2), torch.optim.AdamW(b, lr=1e-2, foreach=False)
    for k, missing in enumerate(([], [1], [1, 3], [], [0, 1, 2, 3, 4], [4], [])):
        for ps, o in ((a, ours), (b, theirs)):
            _set_grads(ps, k)
            for i in missing:
                ps[i].grad = None
            o.step()
    for p, q in zip(a, b):
        assert torch.allclose(p, q, rtol=1e-13, atol=1e-13)
    assert [int(ours.state[p]["step"][0]) for p in a] == [int(theirs.state[q]["step"]) for q in b]


@pytest.mark.parametrize("dt,bits", [(torch.float32, 32), (torch.float32, 8), (torch.bfloat16, 8), (torch.bfloat16, 32)], ids=ids)
def test_state_dict_goes_on_where_it_was(cuda, dt, bits, tmp_path):
    a, b = _params(cuda, dt), _params(cuda, dt)
    oa, ob = (optim.AdamW(ps, lr=1e-2, bits=bits, seed=4) for ps in (a, b))
    for k in range(3):
        _set_grads(a, k)
        oa.step()
    torch.save(oa.state_dict(), tmp_path / "o.pt")
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    ob.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    assert len({id(ob.state[p]["step"]) for p in b}) == 1
    for k in range(3, 6):
        _set_grads(a, k)
        _set_grads(b, k)
        oa.step()
        ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and int(ob.state[b[0]]["step"][0]) == 6
    other = optim.AdamW(_params(cuda, dt), bits=40 - bits)
    with pytest.raises(ValueError, match="AdamW"):
        other.load_state_dict(oa.state_dict())


def test_groups_of_equal_shapes(cuda):
    shapes = [(16, 8), (16, 8)]
    a = [torch.nn.Parameter(_rand(s, i).to(cuda)) for i, s in enumerate(shapes * 2)]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    groups = lambda ps: [dict(params=ps[:2], lr=1e-2), dict(params=ps[2:], lr=3e-3, weight_decay=0.2)]
    ours, theirs = optim.AdamW(groups(a), max_norm=0.5), torch.optim.AdamW(groups(b))
    for k in range(3):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = _rand(p.shape, 10 * k + i).to(cuda)
            q.grad = p.grad.clone()
        ours.step()
        torch.nn.utils.clip_grad_norm_(b, 0.5)
        theirs.step()
    for p, q in zip(a, b):   # (clipping there divides by the norm and 1e-6)
        assert torch.allclose(p, q, rtol=0, atol=1e-6)


def test_recorded_steps_count(cuda):
    c = Case(cuda, torch.bfloat16, [(5000,), (300,)], 8, True, steps=0)
    d = Case(cuda, torch.bfloat16, [(5000,), (300,)], 8, True, steps=0)
    lr = torch.tensor(1e-2, device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        Case(cuda, torch.bfloat16, [(5000,)], 8, True).step(max_norm=0.1)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = c.step(max_norm=0.1, lr=lr, seed=3)
    assert c.counter.tolist() == [0, 0]
    for k in range(4):
        for x, y in zip(c.g, d.g):
            x.copy_(_rand(x.shape, 50 + k) * 0.1)
            y.copy_(x)
        lr.fill_(1e-2 / (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        want = d.step(max_norm=0.1, lr=lr, seed=3)
        assert torch.equal(norm, want) and c.counter.tolist() == [k + 1, 0]
        for l, r in zip((*c.p, *c.m, *c.s, *c.scales, *c.masters), (*d.p, *d.m, *d.s, *d.scales, *d.masters)):
            assert torch.equal(l.view(torch.uint8), r.view(torch.uint8))


def test_writes_are_seen_by_autograd(cuda):
    """A backward that would use weights from before the step raises, as with torch's optimisers."""
    w = torch.ones(8, 8, device=cuda, requires_grad=True)
    x = torch.ones(2, 8, device=cuda, requires_grad=True)
    y = (x @ w).square().sum()
    w.grad = torch.ones_like(w)
    optim.AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(cuda):
    c = Case(cuda, torch.float32, [(300,), (20,)])
    def call(**over):
        a = dict(params=c.p, grads=c.g, exp_avgs=c.m, exp_avg_sqs=c.s, counter=c.counter, lr=1e-3)
        a.update(over)
        return ops.adamw_step(a.pop("params"), a.pop("grads"), a.pop("exp_avgs"), a.pop("exp_avg_sqs"), a.pop("counter"), **a)
    before = [t.clone() for t in c.p]
    for over, text in [
            (dict(params=[]), "no parameters"), (dict(grads=c.g[:1]), "different lengths"),
            (dict(params=[c.p[0], c.p[0]], grads=[c.g[0]] * 2, exp_avgs=[c.m[0]] * 2, exp_avg_sqs=[c.s[0]] * 2), "given twice"),
            (dict(params=[t.cpu() for t in c.p]), "GPU tensor"), (dict(params=[t.int() for t in c.p]), "dtype"),
            (dict(grads=[t.double() for t in c.g]), "grads"), (dict(grads=[c.g[0], c.g[0]]), "grads"),
            (dict(exp_avgs=[t.half() for t in c.m]), "exp_avgs"), (dict(exp_avg_sqs=[c.s[0], c.s[0]]), "exp_avg_sqs"),
            (dict(counter=c.counter[:1]), "counter"), (dict(counter=c.counter.int()), "counter"),
            (dict(counter=c.counter.cpu()), "counter"), (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1.0), "negative"),
            (dict(lr=-1.0), "negative"), (dict(weight_decay=-1.0), "negative"), (dict(max_norm=0.0), "max_norm"),
            (dict(norm=torch.ones((), device=cuda)), "without max_norm"), (dict(masters=c.p), "16 bits"),
            (dict(scales=[torch.zeros(2, 2, device=cuda)] * 2), "exp_avgs"), (dict(lr=torch.ones(2, device=cuda)), "lr"),
            (dict(params=[c.p[0][::2], c.p[1]]), "contiguous")]:
        with pytest.raises(ValueError, match=text):
            call(**over)
    assert all(torch.equal(a, b) for a, b in zip(before, c.p)) and c.counter.tolist() == [6, 0]
    f64 = [torch.ones(4, device=cuda, dtype=torch.float64, requires_grad=True)]
    f64[0].grad = torch.ones_like(f64[0])
    with pytest.raises(ValueError, match="float64"):
        optim.AdamW(f64, bits=8).step()


def test_recorded_steps_of_an_optimiser(cuda):
    """A step recorded with the optimiser's states goes on as eager ones; one that would make states is refused."""
    a, b = _params(cuda, torch.float32), _params(cuda, torch.float32)
    oa, ob = (optim.AdamW(ps, lr=1e-2, max_norm=0.5) for ps in (a, b))
    _set_grads(a, 0)
    scratch = torch.zeros(4, device=cuda)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        scratch.add_(1)
        with pytest.raises(RuntimeError, match="init_states"):
            oa.step()
    assert not oa.state
    _set_grads(b, 0)
    a[1].grad = b[1].grad = None
    for o in (oa, ob):
        o.init_states()
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        ob.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert [int(oa.state[p]["step"][0]) for p in a] == [4, 0, 4, 4, 4] == [int(ob.state[p]["step"][0]) for p in b]


def test_resumed_where_gradients_were_missing(cuda, tmp_path):
    """Parameters with counts of their own draw the same codes after a state has been loaded."""
    a, b = _params(cuda, torch.float32, 6), _params(cuda, torch.float32, 6)
    oa, ob = (optim.AdamW(ps, lr=1e-2, bits=8, seed=4, max_norm=0.5) for ps in (a, b))
    missing = [[], [1], [0, 3], [5], [], [2, 3], [5], []]   # (0, 1, 3 and 5 come to one count on three ways)
    def run(ps, o, k):
        _set_grads(ps, k)
        for i in missing[k]:
            ps[i].grad = None
        o.step()
    for k in range(4):
        run(a, oa, k)
    torch.save(oa.state_dict(), tmp_path / "o.pt")
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    ob.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    for k in range(4, 8):
        run(a, oa, k)
        run(b, ob, k)
        assert torch.equal(oa.norm, ob.norm)
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            for name in ("exp_avg", "exp_avg_sq", "scales"):
                assert torch.equal(oa.state[p][name].view(torch.uint8), ob.state[q][name].view(torch.uint8))


def test_places_of_the_draws(cuda):
    """A parameter's codes are those of its place, beside others or alone; lists of 130 make holes of several launches."""
    n, some = 130, [0, 1, 57, 58, 129]
    whole, parts = (Case(cuda, torch.float32, [(300 + i,) for i in range(n)], 8) for _ in range(2))
    for c in (whole, parts):
        c.counter.fill_(0)
    whole.step(seed=5)
    pick = lambda l: [l[i] for i in some]
    ops.adamw_step(*(pick(l) for l in (parts.p, parts.g, parts.m, parts.s)), parts.counter, scales=pick(parts.scales), seed=5,
                   places=some, **HYPER)
    for a, b in ((whole.p, parts.p), (whole.m, parts.m), (whole.s, parts.s), (whole.scales, parts.scales)):
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(pick(a), pick(b)))
    assert parts.counter.tolist() == whole.counter.tolist() and parts.counter[1] == 0
    for bad in ([0], [0, 0], [1, 0], [-1, 0], [0, 1 << 20]):
        with pytest.raises(ValueError, match="places"):
            ops.adamw_step(parts.p[:2], parts.g[:2], parts.m[:2], parts.s[:2], parts.counter, scales=parts.scales[:2], lr=0.1,
                           places=bad)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("size", [1e30, 1e-30])
def test_norms_whose_squares_have_no_float32(cuda, dt, size):
    g = [(_rand((n,), n) * size).to(dt).to(cuda) for n in (4096, 5000, 3)]
    want = torch.cat([t.cpu().double() for t in g]).norm()
    # squares and sums are doubles': the norm is rounded once
    R.assert_within(ops.grad_norm(g), want, want * (1 + 2.0 ** -20) * 2.0 ** -24, "norm")
    c = Case(cuda, torch.float32, [(4096,)])
    c.g[0].fill_(1e30)
    before = c.p[0].clone()
    assert torch.isfinite(c.step(max_norm=1.0)) and not torch.equal(before, c.p[0]) and torch.isfinite(c.p[0]).all()


def test_tensors_that_overlap_are_refused(cuda):
    c = Case(cuda, torch.float32, [(300,), (300,)])
    flat = torch.zeros(1000, device=cuda)
    def call(**over):
        a = {**dict(params=c.p, grads=c.g, exp_avgs=c.m, exp_avg_sqs=c.s), **over}
        return ops.adamw_step(*(a[k] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")), c.counter, lr=1e-3)
    pair = [flat[:300], flat[299:599]]
    for over in (dict(params=pair), dict(exp_avgs=pair), dict(exp_avg_sqs=pair), dict(exp_avgs=c.s), dict(exp_avgs=[c.m[0], c.m[0]]),
                 dict(exp_avg_sqs=c.p), dict(grads=[c.m[0], c.g[1]]), dict(params=[flat[:300], c.p[1]], grads=[flat[1:301], c.g[1]])):
        with pytest.raises(ValueError, match="overlap|given twice"):
            call(**over)
    assert c.counter.tolist() == [6, 0] and not flat.any()
    call(grads=[c.g[0], c.g[0]])                                       # (gradients are read only)
    call(params=[flat[:300], flat[300:600]], grads=[flat[600:900], flat[600:900]])
