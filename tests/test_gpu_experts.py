"""The experts' products against 64-bit restatements.

Bounds count half steps u of the sums' type: a sum of n products in any order is off by at most (n + 1) u of the sum of
magnitudes (float32's products are six of three bfloat16 terms: five more additions a product and 2^-22 for the terms left
out, so 6 n + 4); the scale and one rounding to the output's type follow.  Sums in parts add no more terms than there are.
"""

import pytest
import torch

from tace_amd import ops

import _rows as R

pytestmark = pytest.mark.gpu

ids = lambda v: str(v).replace("torch.", "")


def _rand(shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dt)


def _sizes(kind, rows, E, seed):
    """Rows of each expert, some dropped."""
    g = torch.Generator().manual_seed(seed)
    if kind == "one":       # all rows one expert's
        e = torch.full((rows,), E // 2)
    elif kind == "none":
        e = torch.full((rows,), -1)
    elif kind == "skewed":  # half of them one expert's, others empty
        e = torch.randint(0, max(1, E // 2), (rows,), generator=g) * 2 % E
        e[torch.rand(rows, generator=g) < 0.5] = E - 1
    else:
        e = torch.randint(0, E, (rows,), generator=g)
        if kind == "dropped":
            e[torch.rand(rows, generator=g) < 0.3] = E
    return e


def _plan(cuda, experts, E, k=1):
    return ops.route_plan(experts.view(-1, k).to(cuda), E)


def _count(n, dt):
    return (6 * n + 4 if dt == torch.float32 else n + 1) + 1


def _reference(x, w, rowptr, comps, scale, transposed=False):
    """(product, bound before the rounding) of sorted group-major rows by experts' w [E, B, K, N]."""
    R_, dt = x.shape[0], x.dtype
    k, n = (w.shape[3], w.shape[2]) if transposed else (w.shape[2], w.shape[3])
    out, mag, at = [], [], 0
    for b, d in enumerate(comps):
        blk = x.double().reshape(-1)[at:at + R_ * d * k].view(R_, d * k)
        at += blk.numel()
        o, m = torch.zeros(2, R_, d, n, dtype=torch.float64)
        for e, (i, j) in enumerate(zip(rowptr, rowptr[1:])):
            m_e = w[e, b].double().t() if transposed else w[e, b].double()
            o[i:j] = blk[i:j].view(-1, d, k) @ m_e
            m[i:j] = blk[i:j].view(-1, d, k).abs() @ m_e.abs()
        out.append(o.reshape(-1))
        mag.append(m.reshape(-1))
    f = lambda t: torch.cat(t).view(R_, -1) * scale
    slack = f(mag).abs() * _count(k, dt) * R.sum_step(dt)
    return f(out), slack


def _weight_reference(x, g, rowptr, comps, K, N, scale):
    R_, dt, E = x.shape[0], x.dtype, len(rowptr) - 1
    dw, mag = torch.zeros(2, E, len(comps), K, N, dtype=torch.float64)
    ax, ag = 0, 0
    for b, d in enumerate(comps):
        xb = x.double().reshape(-1)[ax:ax + R_ * d * K].view(R_, d * K)
        gb = g.double().reshape(-1)[ag:ag + R_ * d * N].view(R_, d * N)
        ax, ag = ax + xb.numel(), ag + gb.numel()
        for e, (i, j) in enumerate(zip(rowptr, rowptr[1:])):
            p, q = xb[i:j].reshape(-1, K), gb[i:j].reshape(-1, N)
            dw[e, b], mag[e, b] = p.t() @ q, p.abs().t() @ q.abs()
    n = torch.tensor([float(j - i) for i, j in zip(rowptr, rowptr[1:])]).view(-1, 1, 1, 1) * \
        torch.tensor([float(d) for d in comps]).view(1, -1, 1, 1)
    return dw * scale, mag * abs(scale) * _count(n, dt) * R.sum_step(dt)


def _close(got, want, slack, what):
    R.assert_within(got, want, slack + R.rounded(want.abs() + slack, got.dtype), what)


def _check(cuda, dt, experts, E, K, N, comps=(1,), scale=0.3, flat=False, seed=0):
    plan = _plan(cuda, experts, E)
    rows, D = plan.n_rows, sum(comps)
    rowptr = plan.rowptr.tolist()
    x, w, g = _rand((rows, D * K), dt, seed), _rand((E, len(comps), K, N), dt, seed + 1), _rand((rows, D * N), dt, seed + 2)
    want, slack = _reference(x, w, rowptr, comps, scale)
    lx, lw = x.to(cuda).requires_grad_(True), (w[:, 0] if flat else w).to(cuda).requires_grad_(True)
    y = ops.expert_linear(lx, lw, plan, scale, comps)
    assert y.dtype == dt and y.shape == (rows, D * N)
    _close(y, want, slack, "y")
    gx, gw = torch.autograd.grad(y, (lx, lw), g.to(cuda))
    assert gx.shape == x.shape and gw.shape == lw.shape
    _close(gx, *_reference(g, w, rowptr, comps, scale, True), "dx")
    dw, slack = _weight_reference(x, g, rowptr, comps, K, N, scale)
    _close(gw.view(dw.shape), dw, slack, "dw")


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["even", "dropped", "skewed"])
@pytest.mark.parametrize("rows,E,K,N", [(1, 1, 1, 1), (5, 3, 8, 16), (40, 7, 33, 17), (200, 4, 64, 64), (777, 9, 128, 96),
                                        (130, 2, 72, 200), (64, 90, 16, 40)])
def test_small(cuda, dt, kind, rows, E, K, N):
    _check(cuda, dt, _sizes(kind, rows, E, rows), E, K, N, flat=rows % 2 == 0)


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["even", "dropped", "one", "none"])
@pytest.mark.parametrize("rows,E,K,N,L", [(3000, 5, 32, 48, 3), (700, 3, 20, 12, 1)])
def test_degrees(cuda, dt, kind, rows, E, K, N, L):
    _check(cuda, dt, _sizes(kind, rows, E, 1), E, K, N, [2 * l + 1 for l in range(L + 1)])


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("rows,E,K,N", [(20000, 3, 128, 128), (9000, 2, 256, 384), (30000, 1, 65, 130), (2000, 20, 520, 264),
                                        (300, 3, 2000, 1032), (100, 6, 1024, 2048)])
def test_large(cuda, dt, rows, E, K, N):
    _check(cuda, dt, _sizes("skewed", rows, E, 3), E, K, N)


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("rows,E,K,N", [(66000, 5, 128, 128), (22000, 4, 264, 264), (33000, 3, 129, 130)])
def test_full_tiles(cuda, dt, rows, E, K, N):
    """Enough rows for the largest tiles, in each of the three products."""
    _check(cuda, dt, _sizes("dropped", rows, E, 4), E, K, N)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=ids)
def test_every_size_of_a_group_by_full_tiles(cuda, dt):
    e = torch.repeat_interleave(torch.arange(301), torch.arange(301))
    _check(cuda, dt, e, 301, 200, 264)


def test_many_tiles_for_each_workgroup(cuda):
    """More than the 64 that a wavefront looks up at once."""
    rows, E, K, N = 280_000, 3, 8, 2048
    plan = _plan(cuda, _sizes("dropped", rows, E, 6), E)
    x, w = _rand((rows, K), torch.bfloat16, 7), _rand((E, K, N), torch.bfloat16, 8)
    y = ops.expert_linear(x.to(cuda), w.to(cuda), plan)
    ends = plan.rowptr.tolist()
    assert not y[ends[-1]:].any()
    for e in range(E):
        at = torch.arange(ends[e], ends[e + 1], 499)
        want, slack = _reference(x[at], w[e:e + 1].unsqueeze(1), [0, len(at)], [1], 1.0)
        _close(y[at.to(cuda)], want, slack, "y")


def test_many_groups_for_each_workgroup(cuda):
    rows, E, K, N = 21_000, 700, 1024, 1024
    plan = _plan(cuda, _sizes("dropped", rows, E, 9), E)
    x, g = _rand((rows, K), torch.bfloat16, 10), _rand((rows, N), torch.bfloat16, 11)
    lw = torch.zeros(E, K, N, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    (gw,) = torch.autograd.grad(ops.expert_linear(x.to(cuda), lw, plan), lw, g.to(cuda))
    ends = plan.rowptr.tolist()
    for e in range(0, E, 53):
        i, j = ends[e], ends[e + 1]
        dw, slack = _weight_reference(x[i:j], g[i:j], [0, j - i], [1], K, N, 1.0)
        _close(gw[e], dw[0, 0], slack[0, 0], "dw")


def test_many_large_matrices(cuda):
    """300 experts of 4096 x 4096, most of them without a row."""
    rows, E, K, N = 90, 300, 4096, 4096
    plan = _plan(cuda, torch.arange(rows) * 3 % 200, E)
    x, g = _rand((rows, K), torch.bfloat16, 12), _rand((rows, N), torch.bfloat16, 13)
    lw = torch.zeros(E, K, N, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    (gw,) = torch.autograd.grad(ops.expert_linear(x.to(cuda), lw, plan), lw, g.to(cuda))
    ends = plan.rowptr.tolist()
    for e in (0, 1, 2, 3, 57, 150, 198, 199, 200, 298, 299):
        i, j = ends[e], ends[e + 1]
        dw, slack = _weight_reference(x[i:j], g[i:j], [0, j - i], [1], K, N, 1.0)
        _close(gw[e], dw[0, 0], slack[0, 0], "dw")
    assert int(gw.view(torch.int16).ne(0).any(2).any(1).sum()) == 90


def test_every_size_of_a_group(cuda):
    """Experts of 0 .. 150 rows, across the tiles' heights."""
    e = torch.repeat_interleave(torch.arange(151), torch.arange(151))
    for dt in (torch.bfloat16, torch.float32, torch.float64):
        _check(cuda, dt, e, 151, 24, 40)


def test_many_experts(cuda):
    _check(cuda, torch.float32, _sizes("dropped", 4000, 1500, 5), 1500, 16, 8)
    _check(cuda, torch.bfloat16, _sizes("even", 900, 300, 5), 300, 40, 24, [1, 3])


def test_rows_past_32_bits(cuda):
    """Elements past 2^31: the last rows are the small call's."""
    T, K, N = 70_001, 32768, 16
    experts = torch.zeros(T, dtype=torch.int64)
    experts[-700:] = 1
    plan = _plan(cuda, experts, 2)
    x = torch.zeros(T, K, dtype=torch.bfloat16, device=cuda)
    x[-700:] = _rand((700, K), torch.bfloat16, 1).to(cuda)
    w = _rand((2, K, N), torch.bfloat16, 2).to(cuda)
    y = ops.expert_linear(x, w, plan, 0.01)
    assert not y[:-700].any()
    want, slack = _reference(x[-700:].cpu(), w[1:].cpu().unsqueeze(1), [0, 700], [1], 0.01)
    _close(y[-700:], want, slack, "y")
    lw = w.clone().requires_grad_(True)
    (gw,) = torch.autograd.grad(ops.expert_linear(x, lw, plan, 0.01), lw, torch.ones_like(y))
    dw, slack = _weight_reference(x[-700:].cpu(), torch.ones(700, N).bfloat16(), [0, 700], [1], K, N, 0.01)
    _close(gw[1], dw[0, 0], slack[0, 0], "dw")
    assert not gw[0].any()


# ------------------------------------------------------------------- values ----
@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
def test_infinities_and_nan_stay_in_their_rows(cuda, dt):
    """As products of the type itself have them; nothing reaches other rows, experts or columns."""
    E, K, N = 3, 40, 72
    plan = _plan(cuda, torch.arange(90) % 4, E)      # (a quarter dropped)
    first = plan.rowptr.tolist()
    x, w = _rand((90, K), dt, 1).to(cuda), _rand((E, K, N), dt, 2).to(cuda)
    clean = ops.expert_linear(x, w, plan)
    x[first[1] + 2, 3] = float("inf")
    x[first[0] + 1, 5] = float("nan")
    x[first[3]:] = float("nan")                       # dropped rows
    w[2, 7, 9] = -float("inf")
    y = ops.expert_linear(x, w, plan)
    want = torch.cat([x[a:b].double() @ w[e].double() for e, (a, b) in enumerate(zip(first, first[1:]))])
    assert torch.equal(torch.isnan(y[:first[3]]), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(y[:first[3]]), inf) and torch.equal(y[:first[3]][inf].double(), want[inf])
    same = torch.isfinite(want)
    assert torch.equal(y[:first[3]][same], clean[:first[3]][same]) and not y[first[3]:].any()
    g = torch.ones(90, N, dtype=dt, device=cuda)
    g[first[3]:] = float("nan")
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(ops.expert_linear(lx, lw, plan), (lx, lw), g)
    assert not gx[first[3]:].any() and torch.isfinite(gw[2]).all()
    assert torch.isinf(gw[1, 3]).all() and torch.isfinite(gw[1, :3]).all() and torch.isnan(gw[0, 5]).all()
    assert torch.equal(torch.isinf(gx[first[2]:first[3], 7]), torch.ones(first[3] - first[2], dtype=torch.bool, device=cuda))


def test_large_and_small_float32(cuda):
    """Magnitudes at float32's ends: no term of the split overflows or is lost where float32's product is not."""
    plan = _plan(cuda, torch.zeros(64, dtype=torch.int64), 1)
    for a, b in ((3.3e38, 0.5), (1e30, 1e-30), (1e-20, 1e-15), (3.4e38, 1.0)):
        x, w = torch.full((64, 32), 0.0, device=cuda), torch.full((1, 32, 64), 0.0, device=cuda)
        x[:, 3], w[:, 3] = a, b
        y = ops.expert_linear(x, w, plan)
        want = torch.tensor(a).double() * torch.tensor(b).double()   # (of the float32 values)
        R.assert_within(y, want.expand(64, 64), want * 4 * 2.0 ** -24 + 2.0 ** -133, (a, b))


# --------------------------------------------------- layouts and derivatives ----
def test_strides_alignment_and_empty(cuda):
    plan = _plan(cuda, _sizes("dropped", 100, 4, 1), 4)
    base, w = _rand((100, 65), torch.bfloat16, 1).to(cuda), _rand((4, 32, 48), torch.bfloat16, 2).to(cuda)
    want = lambda x, w: ops.expert_linear(x.contiguous().clone(), w.contiguous().clone(), plan)
    for v in (base[:, 32:64], base[:, ::2][:, :32], base.t()[:32].t(), base.view(-1)[7:3207].view(100, 32)):
        assert torch.equal(ops.expert_linear(v, w, plan), want(v, w))
    odd = torch.empty(4 * 32 * 48 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(4, 32, 48).copy_(w)
    wt = _rand((4, 48, 32), torch.bfloat16, 3).to(cuda).transpose(1, 2)
    for u in (odd, wt):
        assert torch.equal(ops.expert_linear(base[:, :32], u, plan), want(base[:, :32], u))
    empty = _plan(cuda, torch.zeros(0, dtype=torch.int64), 4)
    x0, lw = torch.zeros(0, 32, dtype=torch.bfloat16, device=cuda).requires_grad_(True), w.clone().requires_grad_(True)
    y = ops.expert_linear(x0, lw, empty)
    gx, gw = torch.autograd.grad(y.sum(), (x0, lw))
    assert y.shape == (0, 48) and gx.shape == (0, 32) and not gw.any()
    nobody = _plan(cuda, torch.zeros(9, dtype=torch.int64), 0)       # no experts: all rows dropped
    assert not ops.expert_linear(base[:9, :32], w[:0], nobody).any()


@pytest.mark.parametrize("comps", [[1], [1, 3]])
def test_gradients_against_differences(cuda, comps):
    plan = _plan(cuda, torch.tensor([0, 2, 2, -1, 0, 2, 1]), 4)
    x = _rand((7, 3 * sum(comps)), torch.float64, 1).to(cuda).requires_grad_(True)
    w = _rand((4, len(comps), 3, 2), torch.float64, 2).to(cuda).requires_grad_(True)
    f = lambda a, b: ops.expert_linear(a, b, plan, 0.7, comps)
    assert torch.autograd.gradcheck(f, (x, w))
    assert torch.autograd.gradgradcheck(f, (x, w))


def test_third_derivatives(cuda):
    plan = _plan(cuda, torch.tensor([0, 1, 1, -1]), 2)
    x = _rand((4, 3), torch.float64, 1).to(cuda).requires_grad_(True)
    w = _rand((2, 3, 2), torch.float64, 2).to(cuda).requires_grad_(True)
    def second(a, b):
        y = ops.expert_linear(a, b, plan)
        ga, gb = torch.autograd.grad(y.square().sum(), (a, b), create_graph=True)
        return torch.autograd.grad(ga.square().sum() + gb.pow(3).sum(), (a, b), create_graph=True)
    assert torch.autograd.gradcheck(second, (x, w))


def test_plans_written_to_raise(cuda):
    plan = _plan(cuda, torch.tensor([0, 1, 1, 0]), 2)
    x = torch.ones(4, 8, device=cuda, requires_grad=True)
    y = ops.expert_linear(x, torch.ones(2, 8, 8, device=cuda), plan)
    plan.rowptr[1] = 3
    with pytest.raises(RuntimeError, match="plan.rowptr is at version"):
        y.sum().backward()


@pytest.mark.parametrize("rowptr", [[0, 50, 20, 100], [30, 40, 60, 100], [0, 400, 500, 600], [-5, 10, 20, 30], [100, 0, 0, 0]])
def test_orders_that_are_none_stay_inside_the_rows(cuda, rowptr):
    """Whatever rowptr holds, reads and writes stay in the tensors (guards around the output keep their values)."""
    x, w = _rand((100, 32), torch.bfloat16, 1).to(cuda), _rand((3, 32, 64), torch.bfloat16, 2).to(cuda)
    plan = ops.RoutePlan(torch.tensor(rowptr, dtype=torch.int32, device=cuda), torch.arange(100, dtype=torch.int32, device=cuda),
                         torch.arange(100, dtype=torch.int32, device=cuda), 100, 1)
    lx, lw = x.requires_grad_(True), w.requires_grad_(True)
    y = ops.expert_linear(lx, lw, plan)
    torch.autograd.grad(y, (lx, lw), torch.ones_like(y))
    torch.cuda.synchronize()


def test_repeats_bit_for_bit_and_on_other_streams(cuda):
    plan = _plan(cuda, _sizes("skewed", 30000, 5, 1), 5)
    x, w, g = (_rand(s, torch.float32, i).to(cuda) for i, s in enumerate(((30000, 96), (5, 96, 64), (30000, 64))))
    def once():
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = ops.expert_linear(a, b, plan)
        return [y.detach(), *torch.autograd.grad(y, (a, b), g)]
    first = once()
    for _ in range(3):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = once()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# ------------------------------------------------------------------ 8 bits ----
def _codes(x):
    s = (x.abs().amax(-1, keepdim=True) / 448).clamp(min=1e-30)
    return (x / s).to(torch.float8_e4m3fn), s.squeeze(-1)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32], ids=ids)
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("T,k,E,K,N", [(1, 1, 1, 16, 1), (1, 2, 8, 1024, 512), (7, 2, 5, 48, 33), (24, 2, 16, 256, 130),
                                       (300, 3, 4, 144, 64), (2000, 2, 8, 512, 384), (999, 1, 90, 80, 72), (5000, 2, 3, 128, 256)])
def test_codes(cuda, out, gather, T, k, E, K, N):
    experts = _sizes("dropped", T * k, E, T).view(T, k)
    plan = ops.route_plan(experts.to(cuda), E)
    rowptr, order = plan.rowptr.tolist(), plan.order.cpu().long()
    q, qs = _codes(_rand((T if gather else T * k, K), torch.float32, 1))
    w, ws = _codes(_rand((E, N, K), torch.float32, 2))
    got = ops.expert_linear_e4m3(q.to(cuda), qs.to(cuda).view(-1, 1), w.to(cuda), ws.to(cuda), plan, gather, out)
    assert got.dtype == out and got.shape == (T * k, N)
    x, xs = (q.float().double()[order // k], qs.double()[order // k]) if gather else (q.float().double(), qs.double())
    want, mag = torch.zeros(2, T * k, N, dtype=torch.float64)
    for e, (i, j) in enumerate(zip(rowptr, rowptr[1:])):
        f = xs[i:j, None] * ws[e].double()
        want[i:j], mag[i:j] = (x[i:j] @ w[e].float().double().t()) * f, (x[i:j].abs() @ w[e].float().double().abs().t()) * f
    slack = mag * (K + 4) * 2.0 ** -24
    R.assert_within(got, want, slack + R.rounded(want.abs() + slack, out), "y")
    assert not got[rowptr[-1]:].any()


def test_codes_views_and_special_values(cuda):
    plan = ops.route_plan(torch.tensor([0, 1, 1, 0], device=cuda), 2)
    q, qs = (t.to(cuda) for t in _codes(_rand((4, 65), torch.float32, 1)))
    w, ws = (t.to(cuda) for t in _codes(_rand((2, 24, 64), torch.float32, 2)))
    v = q[:, 1:]                       # one byte from an aligned address, rows of 65
    want = ops.expert_linear_e4m3(v.contiguous().clone(), qs, w, ws, plan)
    assert torch.equal(ops.expert_linear_e4m3(v, qs, w, ws, plan), want)
    assert torch.equal(ops.expert_linear_e4m3(v, qs.view(4, 1).expand(4, 2)[:, 0], w, ws, plan), want)
    nan = v.contiguous().clone()
    nan[plan.place[1].long(), 5] = float("nan")
    got = ops.expert_linear_e4m3(nan, qs, w, ws, plan)
    assert torch.isnan(got).all(1).sum() == 1 and torch.isfinite(got).all(1).sum() == 3
    none = ops.route_plan(torch.zeros(0, 2, dtype=torch.int64, device=cuda), 2)
    assert ops.expert_linear_e4m3(v[:0], qs[:0], w, ws, none, True).shape == (0, 24)


def test_layout_of_the_weights(cuda):
    weight = _rand((3, 48, 20), torch.bfloat16, 1).to(cuda)
    weight[1, :, 4] = 0
    codes, scales = ops.expert_weights_e4m3(weight, 0.5)
    want = (weight.double() * 0.5).transpose(1, 2)
    got = codes.float().double() * scales.double().unsqueeze(2)
    step = torch.exp2(torch.floor(torch.log2((want / scales.double().clamp(min=1e-30).unsqueeze(2)).abs().clamp(min=2.0 ** -6))) - 3)
    assert bool(((got - want).abs() <= step * scales.double().unsqueeze(2) * (0.5 + 2.0 ** -18)).all())
    assert codes.is_contiguous() and codes.shape == (3, 20, 48) and not codes[1, 4].float().any()


# ----------------------------------------------------------------- together ----
def _layer(x, res, nw, w1, w2, experts, weights, E):
    """A routed layer before its residual: norm, experts of two products, back."""
    h, s = ops.rms_norm(x, nw, residual=res)
    plan = ops.route_plan(experts, E)
    y = ops.expert_linear(ops.expert_dispatch(h, plan), w1, plan, w1.shape[1] ** -0.5)
    y = ops.expert_linear(torch.nn.functional.silu(y), w2, plan, w2.shape[1] ** -0.5)
    return s + ops.expert_combine(y, plan, weights), plan


def test_a_routed_layer_trains(cuda):
    """Norm, dispatch, experts, combine and a step, against torch's own differentiation in float64."""
    from tace_amd import optim

    T, k, E, C, H = 50, 2, 5, 24, 40
    make = lambda: [_rand(s, torch.float64, i).to(cuda).requires_grad_(True)
                    for i, s in enumerate(((C,), (E, C, H), (E, H, C)))]
    ours, theirs = make(), make()
    x, r = (_rand((T, C), torch.float64, 10 + i).to(cuda) for i in range(2))
    experts = _sizes("dropped", T * k, E, 3).view(T, k).to(cuda)
    weights = _rand((T, k), torch.float64, 12).to(cuda).abs()

    def plain(nw, w1, w2):
        s = x + r
        h = s * torch.rsqrt(s.square().mean(1, keepdim=True) + 1e-6) * nw
        out = s
        for j in range(k):
            e = experts[:, j].clamp(0, E - 1)
            y = torch.nn.functional.silu(torch.einsum("tc,tch->th", h, w1[e]) * C ** -0.5)
            y = torch.einsum("th,thc->tc", y, w2[e]) * H ** -0.5
            out = out + torch.where(((experts[:, j] >= 0) & (experts[:, j] < E)).unsqueeze(1), y * weights[:, j:j + 1], 0.0)
        return out

    a, b = optim.AdamW(ours, lr=1e-2, max_norm=1.0), torch.optim.AdamW(theirs, lr=1e-2, foreach=False)
    for _ in range(3):
        one = _layer(x, r, *ours, experts, weights, E)[0].square().sum()
        two = plain(*theirs).square().sum()
        assert abs(float(one) - float(two)) < 1e-11 * float(two)
        for loss, opt in ((one, a), (two, b)):
            opt.zero_grad()
            loss.backward()
        for p, q in zip(ours, theirs):
            assert torch.allclose(p.grad, q.grad, rtol=1e-9, atol=1e-11 * float(q.grad.abs().max()))
        torch.nn.utils.clip_grad_norm_(theirs, 1.0)
        a.step()
        b.step()
        for p, q in zip(ours, theirs):    # (torch adds 1e-6 to the norm it divides by)
            assert torch.allclose(p, q, rtol=1e-7, atol=1e-7)


def test_a_served_layer(cuda):
    """Norm to codes, codes through the plan, back: as the same codes in float64."""
    T, k, E, C, N = 40, 2, 6, 64, 48
    x, r, nw = (_rand(s, torch.bfloat16, i).to(cuda) for i, s in enumerate(((T, C), (T, C), (C,))))
    experts = _sizes("dropped", T * k, E, 3).view(T, k).to(cuda)
    weights = _rand((T, k), torch.float32, 12).to(cuda).abs()
    w, ws = ops.expert_weights_e4m3(_rand((E, C, N), torch.bfloat16, 4).to(cuda), C ** -0.5)
    plan = ops.route_plan(experts, E)
    q, s, h = ops.rms_norm_e4m3(x, nw, residual=r)
    y = ops.expert_linear_e4m3(q, s, w, ws, plan, gather=True)
    out = ops.expert_combine(y, plan, weights)
    deq, wd = q.float().double() * s.double(), w.float().double() * ws.double().unsqueeze(2)
    want, mag = torch.zeros(2, T, N, dtype=torch.float64, device=cuda)
    for j in range(k):
        e, kept = experts[:, j].clamp(0, E - 1), ((experts[:, j] >= 0) & (experts[:, j] < E)).unsqueeze(1)
        one = torch.where(kept, (wd[e] @ deq.unsqueeze(2)).squeeze(2), 0.0)
        big = torch.where(kept, (wd[e].abs() @ deq.abs().unsqueeze(2)).squeeze(2), 0.0)
        want += one * weights[:, j:j + 1].double()
        mag += weights[:, j:j + 1].double() * (big * (C + 8) * 2.0 ** -24 + one.abs() * 2.0 ** -8)   # y's rounding
    want, mag = want.cpu(), mag.cpu()
    R.assert_within(out, want, mag + R.rounded(want.abs() + mag, torch.bfloat16) * (1 + 2.0 ** -10), "out")


def test_recorded(cuda):
    """Plan, norm, experts and their gradients, recorded once, for other rows and other experts each time."""
    T, k, E, C = 200, 2, 4, 64
    x, w = _rand((T, C), torch.bfloat16, 1).to(cuda), _rand((E, C, C), torch.bfloat16, 2).to(cuda)
    g = _rand((T * k, C), torch.bfloat16, 3).to(cuda)
    experts = _sizes("dropped", T * k, E, 4).view(T, k).to(cuda)
    w8, ws = ops.expert_weights_e4m3(w, C ** -0.5)
    nw = torch.ones(C, dtype=torch.bfloat16, device=cuda)

    def once():
        plan = ops.route_plan(experts, E)
        a, b = (t.detach().requires_grad_(True) for t in (ops.expert_dispatch(x, plan), w))
        y = ops.expert_linear(a, b, plan, C ** -0.5)
        q, s = ops.rms_norm_e4m3(x, nw)
        return [y.detach(), *torch.autograd.grad(y, (a, b), g), ops.expert_linear_e4m3(q, s, w8, ws, plan, True)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for i in range(4):
        x.copy_(_rand((T, C), torch.bfloat16, 20 + i))
        experts.copy_(_sizes(("dropped", "skewed", "one", "none")[i], T * k, E, 30 + i).view(T, k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, once()))


def test_refusals(cuda):
    plan = _plan(cuda, torch.tensor([0, 1, 1, 0]), 2)
    x, w = torch.ones(4, 16, device=cuda), torch.ones(2, 16, 8, device=cuda)
    q, qs = (t.to(cuda) for t in _codes(torch.ones(4, 16)))
    w8, ws = (t.to(cuda) for t in _codes(torch.ones(2, 8, 16)))
    for call, text in [
            (lambda: ops.expert_linear(x.int(), w, plan), "dtype"), (lambda: ops.expert_linear(x, w.half(), plan), "weight"),
            (lambda: ops.expert_linear(x, w[:1], plan), "weight"), (lambda: ops.expert_linear(x, w[0], plan), "weight"),
            (lambda: ops.expert_linear(x[:3], w, plan), "x has shape"), (lambda: ops.expert_linear(x[:, :8], w, plan), "x has shape"),
            (lambda: ops.expert_linear(x, w, plan, components=[1, 3]), "weight"), (lambda: ops.expert_linear(x, w, plan, components=[]), "components"),
            (lambda: ops.expert_linear(x, w.cpu(), plan), "weight is on"),
            (lambda: ops.expert_linear(x.cpu(), w, plan), "GPU tensor"),
            (lambda: ops.expert_linear_e4m3(x, qs, w8, ws, plan), "q is"), (lambda: ops.expert_linear_e4m3(q, qs, w, ws, plan), "weight is"),
            (lambda: ops.expert_linear_e4m3(q, qs[:3], w8, ws, plan), "q_scale"), (lambda: ops.expert_linear_e4m3(q, qs, w8, ws[:, :4], plan), "w_scale"),
            (lambda: ops.expert_linear_e4m3(q[:, :8], qs, w8[:, :, :8], ws, plan), "multiple of 16"),
            (lambda: ops.expert_linear_e4m3(q, qs, w8, ws, plan, out_dtype=torch.float64), "out_dtype"),
            (lambda: ops.expert_linear_e4m3(q.cpu(), qs, w8, ws, plan), "GPU tensor")]:
        with pytest.raises(ValueError, match=text):
            call()


class Guarded:
    """A buffer between margins whose bytes are known; nothing in it is a number until it is written."""

    MARGIN = 1 << 16

    def __init__(self, cuda, shape, dt):
        n = torch.Size(shape).numel() * dt.itemsize
        self.whole = torch.full((n + 2 * self.MARGIN,), 255, dtype=torch.uint8, device=cuda)
        self.inner = self.whole[self.MARGIN:self.MARGIN + n].view(dt).view(shape)

    def ptr(self):
        return self.inner.data_ptr()

    def check(self, written=True):
        m = self.MARGIN
        assert bool((self.whole[:m] == 255).all()) and bool((self.whole[-m:] == 255).all())
        assert not written or not torch.isnan(self.inner).any()


NO_ORDERS = [[0, 50, 20, 100], [30, 40, 60, 100], [0, 400, 500, 600], [-5, 10, 20, 30], [100, 0, 0, 0],
             [7, 7, 7, 7], [99, -1, 200, 50]]


@pytest.mark.parametrize("rowptr", NO_ORDERS)
@pytest.mark.parametrize("dt,K,M,comps", [(torch.bfloat16, 32, 64, [1]), (torch.bfloat16, 33, 17, [1]), (torch.float32, 40, 24, [1, 3]),
                                          (torch.float32, 7, 9, [1]), (torch.float64, 20, 12, [1]), (torch.float16, 136, 72, [1, 3])],
                         ids=ids)
def test_orders_that_are_none_write_every_row_and_nothing_else(cuda, rowptr, dt, K, M, comps):
    import ctypes

    from tace_amd import _native as N

    rows, E, B, D = 100, 3, len(comps), sum(comps)
    x, w, g = (_rand(s, dt, i).to(cuda) for i, s in enumerate(((rows, D * K), (E, B, K, M), (rows, D * M))))
    ptr = torch.tensor(rowptr, dtype=torch.int32, device=cuda)
    c = (ctypes.c_int32 * B)(*comps)
    code = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2, torch.float16: 3}[dt]
    s = torch.cuda.current_stream().cuda_stream
    y, dx, dw = (Guarded(cuda, t.shape, dt) for t in (g, x, w))
    L = N.lib()
    need = L.tace_expert_linear_grad_work(code, rows, E, B, c, K, M)
    work = Guarded(cuda, (need,), torch.uint8)
    for rc in (L.tace_expert_linear(code, 0, x.data_ptr(), w.data_ptr(), ptr.data_ptr(), rows, E, B, c, K, M, 0.5, y.ptr(), s),
               L.tace_expert_linear(code, 1, g.data_ptr(), w.data_ptr(), ptr.data_ptr(), rows, E, B, c, K, M, 0.5, dx.ptr(), s),
               L.tace_expert_linear_grad(code, x.data_ptr(), g.data_ptr(), ptr.data_ptr(), rows, E, B, c, K, M, 0.5, dw.ptr(),
                                         work.ptr(), need, s)):
        assert rc == 0
    torch.cuda.synchronize()
    for t in (y, dx, dw):
        t.check()
    work.check(False)


@pytest.mark.parametrize("rowptr", NO_ORDERS)
@pytest.mark.parametrize("gather", [False, True])
def test_codes_of_orders_that_are_none(cuda, rowptr, gather):
    from tace_amd import _native as N

    T, k, E, K, M = 50, 2, 3, 48, 40
    q, qs = (t.to(cuda) for t in _codes(_rand((T if gather else T * k, K), torch.float32, 1)))
    w, ws = (t.to(cuda) for t in _codes(_rand((E, M, K), torch.float32, 2)))
    order = (torch.arange(T * k, dtype=torch.int32, device=cuda) - 20) * 1000003     # (few of them are slots)
    ptr = torch.tensor(rowptr, dtype=torch.int32, device=cuda)
    y = Guarded(cuda, (T * k, M), torch.bfloat16)
    assert N.lib().tace_expert_linear_e4m3(2, q.data_ptr(), qs.data_ptr(), order.data_ptr() if gather else None, k, w.data_ptr(),
                                           ws.data_ptr(), ptr.data_ptr(), T * k, E, K, M, y.ptr(),
                                           torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    y.check()


def _time(f):
    f()
    best = float("inf")
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def test_a_step_of_nan_takes_no_longer(cuda):
    """Float32 sums that are not finite are made again from the inputs: a diverged step must not stand still there (it took
    ninety times a step's time when each of a lane's sums ran by itself to its end)."""
    rows, E, C = 16384, 2, 512
    plan = _plan(cuda, torch.arange(rows) % E, E)
    x, w, g = (_rand(s, torch.float32, i).to(cuda) for i, s in enumerate(((rows, C), (E, C, C), (rows, C))))
    def step(a, b, c):
        la, lb = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        return torch.autograd.grad(ops.expert_linear(la, lb, plan), (la, lb), c)
    usual = _time(lambda: step(x, w, g))
    nan = torch.full_like(g, float("nan"))
    gx, gw = step(x, w, nan)
    assert torch.isnan(gx).all() and torch.isnan(gw).all()
    one = g.clone()
    one[rows // 2] = float("nan")     # half of an expert's sums are run through before they end
    far = g.clone()
    far[rows - E:] = float("inf")     # (those of one sign run to their end)
    # (infinities: 64 sums a lane, 512 terms each, four loads at a time of up to 1 us: 8 ms, forty times a step's 0.2)
    for name, most, args in (("gradient", 20, (x, w, nan)), ("rows", 20, (nan, w, g)), ("row", 20, (x, w, one)),
                             ("infinite rows", 50, (x.abs(), w, far))):
        took = _time(lambda: step(*args))
        print(name, took, "of", usual, "ms")
        assert took < most * usual, name


def test_tensors_without_axes_are_refused_by_name(cuda):
    plan = _plan(cuda, torch.tensor([0]), 1)
    one = torch.ones((), device=cuda)
    q, qs = (t.to(cuda) for t in _codes(torch.ones(1, 16)))
    w8, ws = (t.to(cuda) for t in _codes(torch.ones(1, 8, 16)))
    for call, text in [(lambda: ops.expert_linear(one.view(1, 1), one, plan), "weight is"),
                       (lambda: ops.expert_linear(one, one.view(1, 1, 1), plan), "x has shape"),
                       (lambda: ops.expert_linear_e4m3(q, one, w8, ws, plan), "q_scale is"),
                       (lambda: ops.rms_norm(one, one.view(1)), "x has shape"),
                       (lambda: ops.rms_norm(one.view(1), one), "weight is")]:
        with pytest.raises(ValueError, match=text):
            call()
