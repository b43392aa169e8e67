"""Row operators (table lookup, rows by expert, dropout) against 64-bit restatements.

Bounds count roundings: a sum of m terms in the sums' type is off by at most (m + 1) half steps of the sum of the
terms' magnitudes (m - 1 additions, a product and a scale), and one more rounding gives the output's type.
"""

import threading

import pytest
import torch

from tace_amd import model as pm
from tace_amd import ops

import _rows as R

pytestmark = pytest.mark.gpu

ids = lambda v: str(v).replace("torch.", "")


def _rand(shape, dt, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dt)


# -------------------------------------------------------------- embedding ----
def _tokens(kind, n, V, seed):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, (n,), generator=g)
    if kind == "one":
        t[:] = V - 1
    elif kind == "hub":
        t[torch.rand(n, generator=g) < 0.8] = V // 2
    elif kind == "sorted":
        t = t.sort()[0]
    elif kind == "outside":
        t[torch.rand(n, generator=g) < 0.3] = -1
        t[::5] = V
        t[3::11] = 2 ** 31 - 1
    elif kind == "none":
        t[:] = -1
    return t


def _embed_reference(table, tokens, scale, g):
    V = table.shape[0]
    ok = (tokens >= 0) & (tokens < V)
    out = torch.zeros(len(tokens), table.shape[1], dtype=torch.float64)
    out[ok] = table.double()[tokens[ok]] * scale
    grad, mag = torch.zeros(2, V, table.shape[1], dtype=torch.float64)
    grad.index_add_(0, tokens[ok], g.double()[ok])
    mag.index_add_(0, tokens[ok], g.double()[ok].abs())
    return out, grad * scale, mag * abs(scale), torch.bincount(tokens[ok], minlength=V).double().view(-1, 1)


def _check_embedding(cuda, table, tokens, scale, g, index=torch.int64, groups=False):
    dt = table.dtype
    want, wgrad, mag, m = _embed_reference(table, tokens, scale, g)
    leaf, t = table.to(cuda).requires_grad_(True), tokens.to(index).to(cuda)
    grp = ops.group_by_key(t, table.shape[0]) if groups else None
    out = ops.embedding(leaf, t, scale, grp)
    assert out.dtype == dt and out.shape == want.shape
    R.assert_within(out, want, want.abs() * 2 * R.sum_step(dt) + R.rounded(want, dt) * (1 + 2.0 ** -20), "rows")
    (grad,) = torch.autograd.grad(out, leaf, g.to(cuda))
    assert grad.dtype == dt and grad.shape == table.shape
    slack = (m + 2) * R.sum_step(dt) * mag
    R.assert_within(grad, wgrad, slack + R.rounded(wgrad.abs() + slack, dt), "gradient")


@pytest.mark.parametrize("kind", ["even", "one", "hub", "sorted", "outside", "none"])
@pytest.mark.parametrize("n,V,C", [(1, 1, 1), (7, 3, 4), (63, 89, 128), (4096, 1024, 8), (4097, 5, 64), (4096, 1025, 16),
                                   (5000, 89, 100), (20001, 2, 128), (9000, 7921, 64),
                                   (70000, 128, 40), (70000, 129, 40), (262145, 7, 12),
                                   (40000, 32640, 8), (40000, 32641, 8), (8193, 300, 68), (30000, 3000, 4)])
def test_embedding(cuda, kind, n, V, C):
    _check_embedding(cuda, _rand((V, C), torch.float32, 1), _tokens(kind, n, V, n + V), 0.37,
                     _rand((n, C), torch.float32, 2))


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=ids)
@pytest.mark.parametrize("n,V,C", [(100, 4, 3), (100, 4, 256), (6000, 89, 9), (6000, 300, 72), (5001, 3, 1003), (300, 2, 4100)])
def test_embedding_types_and_widths(cuda, dt, index, n, V, C):
    _check_embedding(cuda, _rand((V, C), dt, 3), _tokens("outside", n, V, C), 1.7, _rand((n, C), dt, 4), index,
                     groups=n > 4096)


@pytest.mark.parametrize("kind", ["even", "hub", "outside", "none"])
@pytest.mark.parametrize("n,V,C", [(4000, 7, 12), (70000, 2, 128), (70000, 3000, 20), (270000, 300, 8)])
def test_embedding_with_a_grouping(cuda, kind, n, V, C):
    _check_embedding(cuda, _rand((V, C), torch.float32, 1), _tokens(kind, n, V, n + V), 0.37,
                     _rand((n, C), torch.float32, 2), groups=True)


def test_embedding_long_sums(cuda):
    """A million rows of three tokens; and one piece after another without rows of some tokens."""
    n = 1 << 20
    _check_embedding(cuda, _rand((3, 8), torch.float32, 5), _tokens("hub", n, 3, 6), 1.0, _rand((n, 8), torch.float32, 7))
    t = torch.arange(300000) // 700 * 17
    _check_embedding(cuda, _rand((8000, 16), torch.bfloat16, 8), t, 2.0, _rand((300000, 16), torch.bfloat16, 9))


def test_embedding_repeats_bit_for_bit(cuda):
    t, g = _tokens("hub", 70000, 89, 1).to(cuda), _rand((70000, 64), torch.float32, 2).to(cuda)
    leaf = _rand((89, 64), torch.float32, 3).to(cuda).requires_grad_(True)
    grads = [torch.autograd.grad(ops.embedding(leaf, t), leaf, g)[0] for _ in range(3)]
    assert all(torch.equal(grads[0], x) for x in grads[1:])


def test_embedding_strides_shapes_and_empty(cuda):
    table = _rand((12, 40), torch.float32, 1).to(cuda)
    t = torch.randint(0, 6, (5, 7), device=cuda)
    big = _rand((12, 41), torch.float32, 2).to(cuda)
    for tab in (table[::2], table[:6], big[:6, 1:], table.t()[:6]):
        assert torch.equal(ops.embedding(tab, t, 1.0), tab[t])
    # unaligned storage, transposed tokens, a scalar token
    flat = _rand((97,), torch.float32, 3).to(cuda)[1:].view(12, 8)
    assert torch.equal(ops.embedding(flat, t.t()), flat[t.t()])
    assert torch.equal(ops.embedding(flat, t[0, 0]), flat[t[0, 0]])
    leaf = table.clone().requires_grad_(True)
    out = ops.embedding(leaf, t[:0])
    assert out.shape == (0, 7, 40)
    assert torch.equal(torch.autograd.grad(out.sum(), leaf)[0], torch.zeros_like(table))
    assert torch.equal(ops.embedding(table[:0], t), torch.zeros(5, 7, 40, device=cuda))
    # an expanded gradient and an unaligned one
    out = ops.embedding(leaf, t)
    (grad,) = torch.autograd.grad(out.sum(), leaf)
    assert torch.equal(grad, torch.bincount(t.reshape(-1), minlength=12).float().view(-1, 1).expand(12, 40))


def test_embedding_rows_hold_what_the_table_holds(cuda):
    """Infinities and NaN of other rows stay out of a row and of another token's gradient."""
    table = torch.ones(3, 8, device=cuda)
    table[1] = float("nan")
    t = torch.tensor([0, -1, 2, 0, 5], device=cuda)
    leaf = table.clone().requires_grad_(True)
    out = ops.embedding(leaf, t, 2.0)
    assert torch.equal(out, torch.tensor([2.0, 0, 2, 2, 0], device=cuda).view(-1, 1).expand(5, 8))
    g = torch.ones(5, 8, device=cuda)
    g[1], g[4] = float("nan"), float("inf")
    assert torch.equal(torch.autograd.grad(out, leaf, g)[0],
                       torch.tensor([4.0, 0, 2], device=cuda).view(-1, 1).expand(3, 8))


def test_embedding_differentiates_again(cuda):
    table = _rand((4, 3), torch.float64, 1).to(cuda).requires_grad_(True)
    t = torch.tensor([0, 3, 3, -1, 1, 4], device=cuda)
    f = lambda x: ops.embedding(x, t, 0.7) ** 3
    assert torch.autograd.gradcheck(f, table) and torch.autograd.gradgradcheck(f, table)


# ----------------------------------------------------------------- routing ----
# one workgroup and its last position; several, with 1 .. 8 positions a thread; the general grouping behind that
@pytest.mark.parametrize("n", [1, 64, 1023, 1025, 8191, 8192, 8193, 131072, 131073, 300001, 1048576, 1048577, 2000003])
@pytest.mark.parametrize("E", [1, 2, 7, 64, 127, 128, 254, 255, 256, 1000])
def test_route_plan_is_the_stable_sort(cuda, n, E):
    g = torch.Generator().manual_seed(n + E)
    e = torch.randint(-1, E + 1, (n,), generator=g)
    e[torch.rand(n, generator=g) < 0.5] = E // 2
    if n % 2:
        e = e.sort(descending=True)[0]
    wide = torch.stack([e, -e], 1).to(cuda)   # (read with a stride)
    for t in (wide[:, 0], wide[:, 0].int()):
        plan = ops.route_plan(t, E)
        key = torch.where((t >= 0) & (t < E), t, E)
        order = torch.argsort(key, stable=True)
        assert torch.equal(plan.order.long(), order)
        assert torch.equal(plan.place.long()[order], torch.arange(n, device=cuda))
        assert torch.equal(plan.rowptr.long(), torch.searchsorted(key[order], torch.arange(E + 1, device=cuda)))


def _experts(T, k, E, drop, seed):
    g = torch.Generator().manual_seed(seed)
    e = torch.rand(T, E, generator=g).argsort(1)[:, :k] if E >= k else torch.randint(0, max(E, 1), (T, k), generator=g)
    e = e.contiguous()
    e[torch.rand(T, k, generator=g) < drop] = -1
    if drop and T > 3:
        e[0], e[1, 0] = E, 2 ** 31 - 1   # a token without experts, one far outside
    return e


def _check_routing(cuda, T, k, E, widths, dt, wdt=None, drop=0.0, group_major=True):
    D = sum(widths)
    e = _experts(T, k, E, drop, T + k)
    ref = R.Route(e, E)
    plan = ops.route_plan(e.to(cuda), E)
    assert torch.equal(plan.order.cpu().long(), ref.order) and torch.equal(plan.place.cpu().long(), ref.place)
    assert torch.equal(plan.rowptr.cpu().long(), ref.rowptr)
    ranges = [(i, int(a), int(b)) for i, (a, b) in enumerate(zip(ref.rowptr, ref.rowptr[1:])) if b > a]
    last = ranges.pop() if ranges else (0, 0, 0)
    assert plan.ranges == ranges + [(last[0], last[1], T * k)]   # (the dropped rows go with the last)
    x, y, gxs, go = (_rand((r, D), dt, i) for i, r in enumerate((T, T * k, T * k, T)))
    # the rows behind the last expert's are never read
    bad = torch.arange(T * k) >= int(ref.rowptr[-1])
    for t in (y, gxs):
        rows = R.to_rows(t, widths).clone()
        rows[bad] = float("nan")
        t.copy_(R.from_rows(rows, widths))
    w = None if wdt is None else _rand((T, k), wdt, 9)
    if w is not None:
        w[~ref.kept.view(T, k)] = float("nan")
    xg, yg = x.to(cuda).requires_grad_(True), y.to(cuda).requires_grad_(True)
    wg = None if w is None else w.to(cuda).requires_grad_(True)
    kw = dict(widths=widths if group_major else None)
    s, w64 = R.sum_step(dt), None if w is None else w.double()
    clean = lambda t: torch.nan_to_num(t.double(), nan=0.0)
    aw = None if w is None else clean(w).abs()

    def near(got, want, mag, m, out_dt=dt):
        assert got.dtype == out_dt
        slack = mag * (m + 2) * s
        R.assert_within(got, want, slack + R.rounded(want.abs() + slack, out_dt))

    xs = ops.expert_dispatch(xg, plan, **kw)
    assert torch.equal(xs.detach().cpu(), ref.dispatch(x, None, widths))
    out = ops.expert_combine(yg, plan, wg, **kw)
    near(out, ref.combine(y.double(), w64, widths), ref.combine(clean(y).abs(), aw, widths), k)
    (gx,) = torch.autograd.grad(xs, xg, gxs.to(cuda))
    near(gx, ref.combine(gxs.double(), None, widths), ref.combine(clean(gxs).abs(), None, widths), k)
    wanted = [yg] if wg is None else [yg, wg]
    grads = torch.autograd.grad(out, wanted, go.to(cuda))
    near(grads[0], ref.dispatch(go.double(), w64, widths), ref.dispatch(go.double().abs(), aw, widths), 1)
    if w is not None:
        rows = lambda t: torch.where(ref.kept.view(-1, 1), R.to_rows(t, widths)[ref.place], torch.zeros(()).double())
        g64 = R.to_rows(go.double(), widths).repeat_interleave(k, 0)
        near(grads[1], (g64 * rows(y.double())).sum(1).view(T, k), (g64 * rows(y.double())).abs().sum(1).view(T, k), D, wdt)
        # weights applied on the way out, and both of its gradients
        xw = ops.expert_dispatch(xg, plan, wg, **kw)
        near(xw, ref.dispatch(x.double(), w64, widths), ref.dispatch(x.double().abs(), aw, widths), 1)
        gx, gw = torch.autograd.grad(xw, (xg, wg), gxs.to(cuda))
        near(gx, ref.combine(gxs.double(), w64, widths), ref.combine(clean(gxs).abs(), aw, widths), k)
        x64 = R.to_rows(x.double(), widths).repeat_interleave(k, 0)
        near(gw, (x64 * rows(gxs.double())).sum(1).view(T, k), (x64 * rows(gxs.double())).abs().sum(1).view(T, k), D, wdt)


@pytest.mark.parametrize("T,k,E,drop", [(1, 1, 1, 0.0), (2, 1, 1, 1.0), (5, 2, 3, 0.3), (343, 1, 4, 0.0), (64, 8, 8, 0.2),
                                        (1000, 2, 89, 0.1), (37, 9, 12, 0.3), (6000, 3, 7, 0.1), (4097, 2, 300, 0.0),
                                        (130, 5, 4, 0.2)])
def test_routing(cuda, T, k, E, drop):
    _check_routing(cuda, T, k, E, (64, 64 * 3), torch.float32, torch.float32, drop)


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("widths", [(1,), (7,), (8, 24), (100, 300, 500), (128, 384, 640, 896), (3, 5), (4, 4, 4, 4, 4, 4, 4, 4),
                                    (1001,)])
def test_routing_types_and_blocks(cuda, dt, widths):
    _check_routing(cuda, 200, 2, 5, widths, dt, torch.float64 if dt == torch.float64 else torch.float32, 0.2)


@pytest.mark.parametrize("dt,wdt", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, None),
                                    (torch.bfloat16, None)], ids=ids)
def test_routing_weight_types_and_plain_rows(cuda, dt, wdt):
    _check_routing(cuda, 90, 3, 6, (72,), dt, wdt, 0.1, group_major=False)


def test_routing_degenerate(cuda):
    # no tokens; no experts at all; int64 choices with strides
    x = torch.ones(0, 8, device=cuda)
    plan = ops.route_plan(torch.zeros(0, 2, dtype=torch.int32, device=cuda), 3)
    assert ops.expert_dispatch(x, plan).shape == (0, 8) and ops.expert_combine(x, plan).shape == (0, 8)
    assert plan.ranges == [] and plan.rowptr.tolist() == [0, 0, 0, 0]
    plan = ops.route_plan(torch.zeros(4, 2, dtype=torch.int32, device=cuda), 0)
    y = torch.full((8, 8), float("nan"), device=cuda)
    assert plan.ranges == [] and torch.equal(ops.expert_combine(y, plan), torch.zeros(4, 8, device=cuda))
    assert torch.equal(ops.expert_dispatch(torch.ones(4, 8, device=cuda), plan), torch.zeros(8, 8, device=cuda))
    e = torch.tensor([[1, 9, 0], [0, 9, 0], [2, 9, 1]], device=cuda)[:, ::2]
    plan = ops.route_plan(e, 3)
    assert plan.order.tolist() == [1, 2, 3, 0, 5, 4] and plan.ranges == [(0, 0, 3), (1, 3, 5), (2, 5, 6)]
    one = ops.route_plan(torch.tensor([1, 0, 1], device=cuda), 2)
    assert one.k == 1 and one.order.tolist() == [1, 0, 2]


def test_routing_strided_rows_and_weights(cuda):
    e = _experts(40, 2, 4, 0.0, 3)
    plan, ref = ops.route_plan(e.to(cuda), 4), R.Route(e, 4)
    x = _rand((80, 33), torch.float64, 1)
    for v in (x[::2], x[:40, 1:], x[:40]):
        assert torch.equal(ops.expert_dispatch(v.to(cuda), plan).cpu(), ref.dispatch(v.contiguous(), None, (v.shape[1],)))
    # one weight a token for both experts: its gradient sums over them
    w = _rand((40, 1), torch.float64, 2)
    wg = w.to(cuda).requires_grad_(True)
    y = _rand((80, 33), torch.float64, 3)
    out = ops.expert_combine(y.to(cuda), plan, wg.expand(40, 2))
    g = _rand((40, 33), torch.float64, 4)
    (gw,) = torch.autograd.grad(out, wg, g.to(cuda))
    rows = y[ref.place].view(40, 2, 33).sum(1)
    assert torch.allclose(gw.cpu(), (rows * g).sum(1, keepdim=True), rtol=1e-13, atol=1e-13)


def test_gradients_of_one_input_only(cuda):
    e = _experts(50, 2, 4, 0.2, 5)
    plan = ops.route_plan(e.to(cuda), 4)
    x, y = _rand((50, 12), torch.float64, 1).to(cuda), _rand((100, 12), torch.float64, 2).to(cuda)
    w, g = _rand((50, 2), torch.float64, 3).to(cuda), _rand((50, 12), torch.float64, 4).to(cuda)
    leaf = lambda t: t.clone().requires_grad_(True)
    both = [leaf(y), leaf(w)]
    want = torch.autograd.grad(ops.expert_combine(both[0], plan, both[1]), both, g)
    a, b = leaf(y), leaf(w)
    assert torch.equal(torch.autograd.grad(ops.expert_combine(a, plan, w), a, g)[0], want[0])
    assert torch.equal(torch.autograd.grad(ops.expert_combine(y, plan, b), b, g)[0], want[1])
    both = [leaf(x), leaf(w)]
    want = torch.autograd.grad(ops.expert_dispatch(both[0], plan, both[1]), both, y)
    a, b = leaf(x), leaf(w)
    assert torch.equal(torch.autograd.grad(ops.expert_dispatch(a, plan, w), a, y)[0], want[0])
    assert torch.equal(torch.autograd.grad(ops.expert_dispatch(x, plan, b), b, y)[0], want[1])
    r = leaf(g)
    out = ops.dropout(x, 0.3, (1, 2), residual=r)
    assert torch.equal(torch.autograd.grad(out, r, g)[0], g)
    both = leaf(x)   # the same tensor dropped and added
    assert torch.equal(torch.autograd.grad(ops.dropout(both, 0.3, (1, 2), residual=both), both, g)[0],
                       ops.dropout(g, 0.3, (1, 2)) + g)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_unaligned_rows(cuda, dt, shift):
    """Contiguous rows that start inside 16 bytes give what aligned ones give."""
    T, k, D = 40, 2, 24
    e = _experts(T, k, 4, 0.2, 5)
    plan = ops.route_plan(e.to(cuda), 4)
    off = lambda t: torch.cat([t.new_zeros(shift), t.reshape(-1)])[shift:].view(t.shape)
    x, y, g = (_rand((r, D), dt, i).to(cuda) for i, r in enumerate((T, T * k, T)))
    w = _rand((T, k), torch.float32, 5).to(cuda)

    def run(move):
        a, b, c = (move(t).detach().requires_grad_(True) for t in (x, y, w))
        xs, out = ops.expert_dispatch(a, plan, widths=(8, 16)), ops.expert_combine(b, plan, c, widths=(8, 16))
        t = torch.arange(T, device=cuda) % 7
        rows = ops.embedding(a[:7], t)
        return [xs, out, rows, *torch.autograd.grad(out, (b, c), move(g)), *torch.autograd.grad(xs, a, move(y)),
                torch.autograd.grad(rows, a, move(g))[0]]
    for p, q in zip(run(off), run(lambda t: t)):
        # (the dot products are summed in another order: D terms a slot)
        assert torch.equal(p, q) or (p - q).abs().max().item() <= 2 * D * 2.0 ** -24 * D * 16


def test_rows_past_32_bit_offsets(cuda):
    """2.3 G elements: 70,000 rows of 32,768 bfloat16."""
    n, C = 70000, 32768
    table = torch.randn(3, C, device=cuda).bfloat16()
    t = torch.arange(n, device=cuda) % 3
    rows = ops.embedding(table, t)
    for i in (0, 65535, 65536, n - 1):
        assert torch.equal(rows[i], table[i % 3])
    leaf = table.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(ops.embedding(leaf, t), leaf, torch.ones((), device=cuda).bfloat16().expand(n, C))
    counts = torch.bincount(t, minlength=3).bfloat16()
    assert torch.equal(grad, counts.view(3, 1).expand(3, C))
    plan = ops.route_plan(t.flip(0), 3)
    xs = ops.expert_dispatch(rows, plan)
    tok = plan.order.long()
    for i in (0, 65535, 65536, n - 1):
        assert torch.equal(xs[i], rows[tok[i]])
    del rows
    back = ops.expert_combine(xs, plan, torch.full((n,), 2.0, device=cuda))
    for i in (0, 65535, 65536, n - 1):
        assert torch.equal(back[i], 2 * table[i % 3])
    del back
    dropped = ops.dropout(xs, 0.5, (1, 2))
    at = 2 ** 31 + 12345   # (of the flat order)
    want = R.draws(16, 1, 2, 0)
    assert torch.equal((dropped.view(-1)[:16] != 0).cpu(), (want >= 32768) & (xs.view(-1)[:16] != 0).cpu())
    block = [w for b in (at // 8, at // 8 + 1) for v in R.philox((b, 0, 2, 0), (1, 0)) for w in (v & 0xFFFF, v >> 16)]
    first = at // 8 * 8
    assert torch.equal((dropped.view(-1)[first:first + 16] != 0).cpu(),
                       (torch.tensor(block) >= 32768) & (xs.view(-1)[first:first + 16] != 0).cpu())


def test_without_autograd(cuda):
    x = _rand((6, 8), torch.float32, 1).to(cuda)
    with torch.inference_mode():
        plan = ops.route_plan(torch.tensor([0, 1, 0, 1, 2, 2], device=cuda), 3)
        y = ops.expert_dispatch(ops.dropout(ops.embedding(x, plan.order), 0.5, (1, 2)), plan)
        z = ops.expert_combine(y, plan)
    plan = ops.route_plan(torch.tensor([0, 1, 0, 1, 2, 2], device=cuda), 3)
    leaf = x.clone().requires_grad_(True)
    with torch.no_grad():
        a = ops.expert_dispatch(ops.dropout(ops.embedding(leaf, plan.order), 0.5, (1, 2)), plan)
    assert torch.equal(a, y) and not a.requires_grad
    assert torch.equal(ops.expert_combine(y.clone(), plan), z)


def test_passes_from_two_threads(cuda):
    states = [_pass_inputs(cuda, 5000, s) for s in (1, 30)]
    want = [_training_pass(s) for s in states]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i].append(_training_pass(states[i]))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads], [t.join() for t in threads]
    for i in range(2):
        assert len(got[i]) == 10 and all(torch.equal(p, q) for r in got[i] for p, q in zip(r, want[i]))


def test_routing_differentiates_again(cuda):
    e = torch.tensor([[0, 2], [2, -1], [1, 0], [-1, -1], [2, 1]], device=cuda)
    plan = ops.route_plan(e, 3)
    x, w = _rand((5, 4), torch.float64, 1).to(cuda), _rand((5, 2), torch.float64, 2).to(cuda)
    x.requires_grad_(True), w.requires_grad_(True)

    def f(x, w):   # both directions, weighted in both, on two blocks
        xs = ops.expert_dispatch(x, plan, w, widths=(1, 3))
        return ops.expert_combine(xs ** 2, plan, w * w, widths=(1, 3))
    assert torch.autograd.gradcheck(f, (x, w)) and torch.autograd.gradgradcheck(f, (x, w))
    h = lambda x: ops.expert_combine(ops.expert_dispatch(x, plan) ** 3, plan)
    assert torch.autograd.gradcheck(h, x) and torch.autograd.gradgradcheck(h, x)


# ----------------------------------------------------------------- dropout ----
def _check_dropout(cuda, rows, C, comps, p, dt, residual=False, rng=(5, 9), site=2, as_tensor=False, shift=0):
    D = sum(comps) * C
    x, g, r = (_rand((rows * D + shift,), dt, i)[shift:].view(rows, D) for i in range(3))
    fac = R.keep_factor(rows, C, comps, p, *rng, site)
    dropped = fac == 0
    x[dropped], g[dropped] = float("nan"), float("inf")
    move = lambda t: torch.cat([torch.zeros(shift, dtype=dt), t.reshape(-1)]).to(cuda)[shift:].view(rows, D)
    xg = move(x).requires_grad_(True)
    rg = move(r).requires_grad_(True) if residual else None
    state = torch.tensor(rng, dtype=torch.int64, device=cuda) if as_tensor else rng
    out = ops.dropout(xg, p, state, site=site, components=comps, residual=rg)
    scaled = lambda t: torch.where(dropped, torch.zeros((), dtype=torch.float64), t.double() * fac)
    want = scaled(x) + (r.double() if residual else 0.0)
    # the scale and the product (and the addition) rounded in the sums' type, then once more
    slack = (scaled(x).abs() * 2 + want.abs()) * R.sum_step(dt)
    R.assert_within(out, want, slack + R.rounded(want.abs() + slack, dt))
    wanted = [xg, rg] if residual else [xg]
    grads = torch.autograd.grad(out, wanted, move(g))
    wg = scaled(g)
    slack = wg.abs() * 2 * R.sum_step(dt)
    R.assert_within(grads[0], wg, slack + R.rounded(wg.abs() + slack, dt))
    if residual:
        assert torch.equal(grads[1].cpu(), g)


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("rows,C,comps", [(1, 1, (1,)), (3, 5, (1,)), (64, 8, (1,)), (33, 4, (1,)), (7, 16, (1, 3, 5, 7)),
                                          (9, 5, (1, 3)), (11, 12, (3,)), (5, 24, (7, 1)), (1, 3, (2, 1, 1, 1, 1, 1, 1, 4))])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(cuda, dt, rows, C, comps, residual):
    _check_dropout(cuda, rows, C, comps, 0.3, dt, residual)


@pytest.mark.parametrize("rng,site", [((0, 0), 0), ((2 ** 64 - 1, -1), 2 ** 32 - 1), ((-2 ** 63, 2 ** 63 - 1), 1), ((1 << 40, 3 << 33), 7)])
@pytest.mark.parametrize("as_tensor", [False, True])
def test_dropout_seeds(cuda, rng, site, as_tensor):
    if as_tensor:
        rng = tuple(v - 2 ** 64 if v >= 2 ** 63 else v for v in rng)
    _check_dropout(cuda, 21, 16, (1, 3), 0.5, torch.float32, rng=rng, site=site, as_tensor=as_tensor)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -16, 0.1, 0.999, 1.0])
def test_dropout_probabilities(cuda, p):
    _check_dropout(cuda, 50, 16, (1, 3), p, torch.float32, residual=True)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_dropout_unaligned(cuda, dt, shift):
    _check_dropout(cuda, 13, 8, (1, 3), 0.4, dt, residual=True, shift=shift)
    _check_dropout(cuda, 13, 8, (1,), 0.4, dt, residual=True, shift=shift)


def test_dropout_rate_over_a_large_tensor(cuda):
    """8 M draws: the rate within six standard deviations of p, sites and offsets apart independent."""
    n, p = 1 << 23, 0.25
    x = torch.ones(n, device=cuda)
    masks = [ops.dropout(x, p, (3, o), site=s) != 0 for s, o in ((0, 0), (1, 0), (0, 1), (0, 1 << 32))]
    sd = (p * (1 - p) * n) ** 0.5
    for m in masks:
        assert abs(int((~m).sum()) - p * n) < 6 * sd
        assert m.float().view(-1, 8).mean(0).sub(1 - p).abs().max().item() < 6 * (p * (1 - p) * 8 / n) ** 0.5
    both = (p * p * (1 - p * p) * n) ** 0.5
    for i in range(4):
        for j in range(i):
            assert abs(int((~masks[i] & ~masks[j]).sum()) - p * p * n) < 6 * both


def test_dropout_differentiates_again(cuda):
    x = _rand((6, 8), torch.float64, 1).to(cuda).requires_grad_(True)
    r = _rand((6, 8), torch.float64, 2).to(cuda).requires_grad_(True)
    f = lambda x, r: ops.dropout(x ** 2, 0.4, (1, 2), components=(1, 3), residual=r) ** 2
    assert torch.autograd.gradcheck(f, (x, r)) and torch.autograd.gradgradcheck(f, (x, r))


def test_dropout_empty_and_strided(cuda):
    assert ops.dropout(torch.ones(0, 8, device=cuda), 0.5, (1, 2)).shape == (0, 8)
    x = _rand((32, 24), torch.float32, 1).to(cuda)
    assert torch.equal(ops.dropout(x.t(), 0.5, (1, 2)), ops.dropout(x.t().contiguous(), 0.5, (1, 2)))
    assert torch.equal(ops.dropout(x[::2], 0.5, (1, 2)), ops.dropout(x[::2].contiguous(), 0.5, (1, 2)))


# --------------------------------------------------------------- refusals ----
def test_refusals(cuda):
    x, t = torch.zeros(6, 8, device=cuda), torch.zeros(6, dtype=torch.int64, device=cuda)
    plan = ops.route_plan(t.view(3, 2), 4)
    cpu = torch.zeros(6, 8)
    bad = [
        lambda: ops.embedding(x.int(), t), lambda: ops.embedding(x, t.float()), lambda: ops.embedding(x[0], t),
        lambda: ops.embedding(x, t.cpu()), lambda: ops.embedding(x[:, :0], t), lambda: ops.embedding(cpu, t),
        lambda: ops.embedding(x.new_zeros(2, 40000), t),
        lambda: ops.embedding(x, t, 1.0, (t, t)), lambda: ops.embedding(x, t, 1.0, ops.group_by_key(t, 5)),
        lambda: ops.route_plan(x, 4), lambda: ops.route_plan(t.view(1, 2, 3), 4), lambda: ops.route_plan(t, -1),
        lambda: ops.route_plan(t.view(6, 1)[:, :0], 4),
        lambda: ops.expert_dispatch(x, plan), lambda: ops.expert_combine(x[:3], plan),
        lambda: ops.expert_dispatch(x[:3], plan, widths=(4, 5)), lambda: ops.expert_dispatch(x[:3], plan, widths=(8, 0)),
        lambda: ops.expert_dispatch(x[:3], plan, widths=(1,) * 9),
        lambda: ops.expert_dispatch(x[:3], plan, torch.zeros(2, 3, device=cuda)),
        lambda: ops.expert_dispatch(x[:3], plan, torch.zeros(3, 2, dtype=torch.int32, device=cuda)),
        lambda: ops.expert_combine(x, plan, torch.zeros(3, 2)), lambda: ops.expert_combine(cpu, plan),
        lambda: ops.dropout(x, -0.1, (1, 2)), lambda: ops.dropout(x, 1.5, (1, 2)), lambda: ops.dropout(x, 1e-7, (1, 2)),
        lambda: ops.dropout(x, 1 - 1e-7, (1, 2)), lambda: ops.dropout(x, float("nan"), (1, 2)),
        lambda: ops.dropout(x, 0.1, (1, 2 ** 64)), lambda: ops.dropout(x, 0.1, (1, 2), site=-1), lambda: ops.dropout(x, 0.1, (1, 2), site=2 ** 32),
        lambda: ops.dropout(x, 0.1, (1, 2), components=(3,)), lambda: ops.dropout(x, 0.1, (1, 2), components=(0, 1)),
        lambda: ops.dropout(x, 0.1, (1, 2), components=()), lambda: ops.dropout(x, 0.1, torch.zeros(2, device=cuda)),
        lambda: ops.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64)), lambda: ops.dropout(x, 0.1, (1, 2), residual=x[0]),
        lambda: ops.dropout(x, 0.1, (1, 2), residual=x.double()), lambda: ops.dropout(x.long(), 0.1, (1, 2)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted:", i)
    with pytest.raises(AttributeError):
        ops.expert_dispatch(x[:3], None)


def test_kernel_timer_sees_every_launch(cuda):
    """Forward and backward launches, the backward's from autograd's thread."""
    ops.TIMER = ops.KernelTimer()
    try:
        s = _pass_inputs(cuda, 5000, 3)
        _training_pass(s)
        seen = ops.TIMER.summary()
    finally:
        ops.TIMER = None
    assert {k: v[0] for k, v in seen.items()} == dict(
        embed_fwd=1, embed_grad=1, dropout=2, route_group=1, route_dispatch=1, route_combine=2, route_dots=1)
    assert all(ms > 0 for _, ms, _ in seen.values())


# ---------------------------------------------------------- graphs, streams ----
def _training_pass(s):
    """The operators as a routed layer uses them, forward and backward."""
    leaves = [s[k].detach().requires_grad_(True) for k in ("table", "w")]
    x = ops.embedding(leaves[0], s["tokens"], 0.5)
    x = ops.dropout(x, 0.25, s["rng"], components=(1, 3), residual=x)
    plan = ops.route_plan(s["experts"], 4)
    out = ops.expert_combine(ops.expert_dispatch(x, plan, widths=(16, 48)) ** 2, plan, leaves[1], widths=(16, 48))
    return [out.detach(), *torch.autograd.grad(out, leaves, s["g"])]


def _pass_inputs(cuda, n, seed):
    g = torch.Generator().manual_seed(seed)
    return dict(table=_rand((50, 64), torch.float32, seed).to(cuda), w=_rand((n, 2), torch.float32, seed + 1).to(cuda),
                tokens=torch.randint(-1, 50, (n,), generator=g).to(cuda), g=_rand((n, 64), torch.float32, seed + 2).to(cuda),
                experts=torch.randint(-1, 4, (n, 2), generator=g).to(cuda),
                rng=torch.tensor([seed, 3], dtype=torch.int64, device=cuda))


@pytest.mark.parametrize("n", [300, 9000])
def test_recorded_graphs_replay(cuda, n):
    """Two graphs recorded side by side, replayed in turn on changed inputs with eager passes between."""
    states = [_pass_inputs(cuda, n, 1), _pass_inputs(cuda, n, 20)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in states:
            _training_pass(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_training_pass(s))
        graphs.append(graph)
    for turn in range(4):
        for i, s in enumerate(states):
            for k, v in _pass_inputs(cuda, n, 40 + 2 * turn + i).items():
                s[k].copy_(v)
        for graph in graphs:
            graph.replay()
        want = [_training_pass(s) for s in states]
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_passes_on_two_streams(cuda):
    states = [_pass_inputs(cuda, 5000, s) for s in (1, 30)]
    want = [_training_pass(s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = []
    for _ in range(3):
        for st, s in zip(streams, states):
            with torch.cuda.stream(st):
                got.append(_training_pass(s))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(r, want[i % 2]))


def test_routed_layer_of_atoms_against_64_bits(cuda):
    """Embedding, dropout, routing, the experts' linears and the way back, energy-like loss: outputs and the gradients of
    the table, the experts' weights and biases and the router's weights; and of a gradient-norm loss (twice through)."""
    n, S, C, E, k = 257, 5, 16, 4, 2
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(-1, S, (n,), generator=g)
    e = _experts(n, k, E, 0.1, 2)
    lin = pm.e3nnElementLinear(f"{C}x0e+{C}x1o", f"{C}x0e+{C}x1o", E).double()
    with torch.no_grad():
        lin.bias.copy_(_rand(lin.bias.shape, torch.float64, 3))
    ref = R.Route(e, E)
    widths, comps = (C, 3 * C), (1, 3)
    rng = (11, 12)
    fac = R.keep_factor(n, C, comps, 0.2, *rng, 0)
    inputs = [_rand((S, 4 * C), torch.float64, 4), torch.softmax(_rand((n, k), torch.float64, 5), 1),
              lin.weight.detach(), lin.bias.detach()]
    go = _rand((n, 4 * C), torch.float64, 6)

    def run(dev, table, w, weight, bias):
        own = dev != "cpu"
        if own:
            x = ops.embedding(table, tokens.to(dev), S ** -0.5)
            x = ops.dropout(x, 0.2, rng, components=comps)
            plan = ops.route_plan(e.to(dev), E)
            xs = ops.expert_dispatch(x, plan, widths=widths)
            with ops.differentiable_twice():
                ys = torch.func.functional_call(lin.to(dev), {"weight": weight, "bias": bias}, (xs, plan))
            return ops.expert_combine(ys ** 2, plan, w, widths=widths)
        x = torch.where((tokens >= 0).view(-1, 1), table[tokens.clamp(min=0)], torch.zeros((), dtype=torch.float64)) * S ** -0.5
        xs = ref.dispatch(x * fac, None, widths)
        ranges = [(i, int(a), int(b)) for i, (a, b) in enumerate(zip(ref.rowptr, ref.rowptr[1:]))] + [
            (0, int(ref.rowptr[-1]), n * k)]
        ys = pm._linear_autograd(xs, weight, bias, lin.lay, ranges, 1.0)
        return ref.combine(ys ** 2, w, widths)

    results = []
    for dev in ("cpu", cuda):
        leaves = [t.to(dev).clone().requires_grad_(True) for t in inputs]
        out = run(dev, *leaves)
        loss = (out * go.to(dev)).sum()
        first = torch.autograd.grad(loss, leaves, create_graph=True)
        again = torch.autograd.grad(sum((f ** 2).sum() for f in first), leaves)
        results.append([t.detach().cpu() for t in (out, *first, *again)])
    for a, b in zip(*results):
        assert (a - b).abs().max().item() <= 1e-11 * max(a.abs().max().item(), 1.0)
