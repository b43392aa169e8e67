"""The row operators at the ends of their arguments, against restatements in 64 bits or on whole numbers (which every
type and order of a sum holds exactly)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

from tace_amd import _native as N
from tace_amd import configs, data, structures
from tace_amd import library
from tace_amd import model as pm
from tace_amd import ops
from tace_amd.so3 import Irreps

import _rows as R

pytestmark = pytest.mark.gpu

ids = lambda v: str(v).replace("torch.", "")
CODES = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2, torch.float16: 3}   # TACE_ROW_*


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("groups", [False, True])
@pytest.mark.parametrize("n,V,C", [(1, 2000, 1), (100, 2000, 1), (100, 2000, 2), (2049, 2000, 1), (1, 2, 1), (50, 7, 1),
                                   (100, 3, 2), (1000, 2000, 2)])
def test_gradient_of_narrow_tables(cuda, dt, groups, n, V, C):
    """Rows of one and two elements: first and second order."""
    gen = torch.Generator().manual_seed(n + V)
    t = torch.randint(-1, V, (n,), generator=gen)
    # eighths, in sums below 2^12: exact in float32, and rounded once
    table, g = (torch.randint(-8, 9, (r, C), generator=gen).to(dt) / 8 for r in (V, n))
    ok = t >= 0
    leaf, tc = table.to(cuda).requires_grad_(True), t.to(cuda)
    out = ops.embedding(leaf, tc, 1.0, ops.group_by_key(tc, V) if groups else None)
    want = torch.where(ok.view(-1, 1), table[t.clamp(min=0)], torch.zeros((), dtype=dt))
    assert torch.equal(out.detach().cpu(), want)
    gl = g.to(cuda).requires_grad_(True)
    (grad,) = torch.autograd.grad(out, leaf, gl, create_graph=True)
    sums = torch.zeros(V, C, dtype=torch.float64).index_add_(0, t[ok], g[ok].double())
    assert torch.equal(grad.detach().cpu(), sums.to(dt))
    (again,) = torch.autograd.grad(grad, gl, table.to(cuda))   # the rows of table again
    assert torch.equal(again.cpu(), want)


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("V,C", [(1, 1), (9, 5), (1025, 3), (5000, 64), (32641, 7), (300001, 33)])
def test_gradient_of_no_rows_is_zeros(cuda, dt, V, C):
    """Through the C entry, without a grouping, and through autograd; nothing behind the gradient is written."""
    grad = torch.full((V * C + 64,), float("nan"), dtype=dt, device=cuda)
    for index in (4, 8):
        grad.fill_(float("nan"))
        rc = N.lib().tace_embed_grad(CODES[dt], index, None, None, None, None, 0, V, C, 0.5, grad.data_ptr(), None,
                                     0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, N.lib().tace_last_error()
        assert not bool(grad[:V * C].any()) and bool(grad[V * C:].isnan().all())
    leaf = torch.ones(V, C, dtype=dt, device=cuda, requires_grad=True)
    out = ops.embedding(leaf, torch.zeros(0, dtype=torch.int64, device=cuda))
    assert torch.equal(torch.autograd.grad(out.sum(), leaf)[0], torch.zeros_like(leaf))


def test_half_a_grouping_is_refused(cuda):
    x, t = torch.zeros(6, 8, device=cuda), torch.zeros(6, dtype=torch.int64, device=cuda)
    rowptr, order = ops.group_by_key(t, 6)
    for groups in ((None, order), (rowptr, None)):
        with pytest.raises(ValueError, match="one of"):
            ops.embedding(x, t, 1.0, groups)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("k", [1, 2, 3])
@pytest.mark.parametrize("D", [5, 64])
def test_places_outside_the_rows_stay_inside(cuda, dt, k, D):
    """A plan whose places are not ``route_plan``'s: what lies outside the rows is taken for the last one."""
    T = 40
    n = T * k
    plan = ops.route_plan(torch.arange(n, device=cuda).view(T, k) % 5, 5)
    bad = plan.place.clone()
    # (the last row's own slot among them, so that the rows stay distinct but for it)
    slots = torch.cat([torch.tensor([0, n // 2, n - 2], device=cuda), (plan.place == n - 1).nonzero().view(-1)]).unique()
    values = torch.tensor([n, -1, 2 ** 31 - 1, -2 ** 31], device=cuda, dtype=torch.int32)[:len(slots)]
    bad[slots] = values
    mine = ops.RoutePlan(plan.rowptr, plan.order, bad, T, k)
    near = torch.where((bad < 0) | (bad >= n), n - 1, bad).long().cpu()
    gen = torch.Generator().manual_seed(k)
    x, y, g = (torch.randint(-4, 5, (r, D), generator=gen).to(dt) for r in (T, n, T))
    w = torch.randint(1, 4, (T, k), generator=gen).float()
    xs = ops.expert_dispatch(x.to(cuda), mine).cpu()
    rows = x.repeat_interleave(k, 0)
    sure = torch.ones(n, dtype=torch.bool)
    sure[slots.cpu()] = False
    assert torch.equal(xs[near[sure]], rows[sure])
    # every element of the last row is one of those that were sent there
    assert bool((xs[n - 1] == rows[slots.cpu()]).any(0).all())
    yc, wc = y.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
    out = ops.expert_combine(yc, mine, wc)
    picked = y.double()[near].view(T, k, D)
    assert torch.equal(out.detach().cpu(), (picked * w.double().unsqueeze(2)).sum(1).to(dt))   # (small whole numbers)
    gy, gw = torch.autograd.grad(out, (yc, wc), g.to(cuda))
    assert torch.equal(gw.cpu(), (picked * g.double().unsqueeze(1)).sum(2).float())
    sent = (g.double().unsqueeze(1) * w.double().unsqueeze(2)).view(n, D).to(dt)
    assert torch.equal(gy.cpu()[near[sure]], sent[sure])


def test_buffers_written_before_the_backward_are_noticed(cuda):
    """The grouping's and the plan's tensors, first and second order; what a backward does not read may be written to."""
    t = torch.arange(50, device=cuda) % 7
    table = torch.ones(7, 8, device=cuda, requires_grad=True)
    written = pytest.raises(RuntimeError, match="modified by an inplace operation")
    for i in (0, 1):
        groups = ops.group_by_key(t, 7)
        out = ops.embedding(table, t, 1.0, groups)
        groups[i].add_(0)
        with written:
            torch.autograd.grad(out.sum(), table)
    groups = ops.group_by_key(t, 7)
    g = torch.ones(50, 8, device=cuda, requires_grad=True)
    (grad,) = torch.autograd.grad(ops.embedding(table, t, 1.0, groups), table, g, create_graph=True)
    groups[1].add_(0)
    assert torch.equal(torch.autograd.grad(grad, g, torch.ones_like(grad))[0], torch.ones_like(g))   # (a lookup again)

    e = torch.tensor([[0, 1], [1, 2], [2, 0], [0, -1]], device=cuda)
    x, y = torch.ones(4, 8, device=cuda, requires_grad=True), torch.ones(8, 8, device=cuda, requires_grad=True)
    w = torch.ones(4, 2, device=cuda, requires_grad=True)
    for f, leaf in ((lambda p: ops.expert_dispatch(x, p), x), (lambda p: ops.expert_combine(y, p), y),
                    (lambda p: ops.expert_dispatch(x, p, w), w), (lambda p: ops.expert_combine(y, p, w), w)):
        for name in ("place", "rowptr"):
            plan = ops.route_plan(e, 3)
            out = f(plan)
            getattr(plan, name).add_(0)
            with written:
                torch.autograd.grad(out.sum(), leaf)
            plan = ops.route_plan(e, 3)
            (first,) = torch.autograd.grad((f(plan) ** 2).sum(), leaf, create_graph=True)
            getattr(plan, name).add_(0)
            with written:
                torch.autograd.grad(first.sum(), leaf)
        plan = ops.route_plan(e, 3)
        out = f(plan)
        plan.order.add_(0)   # (no pass reads it)
        torch.autograd.grad(out.sum(), leaf)


def test_plans_of_inference_mode_train(cuda):
    e = torch.tensor([[0, 1], [1, 2], [2, 0], [0, -1]], device=cuda)
    t = torch.arange(50, device=cuda) % 7
    with torch.inference_mode():
        plan, groups = ops.route_plan(e, 3), ops.group_by_key(t, 7)
    x, table = torch.ones(4, 8, device=cuda, requires_grad=True), torch.ones(7, 8, device=cuda, requires_grad=True)
    out = ops.expert_combine(ops.expert_dispatch(x, plan), plan)
    want = torch.tensor([2.0, 2, 2, 1], device=cuda).view(4, 1).expand(4, 8)
    assert torch.equal(out, want) and torch.equal(torch.autograd.grad(out.sum(), x)[0], want)
    out = ops.embedding(table, t, 1.0, groups)
    assert torch.equal(torch.autograd.grad(out.sum(), table)[0], torch.bincount(t).float().view(7, 1).expand(7, 8))


def test_written_buffers_are_noticed_while_timed(cuda):
    """The error leaves autograd's thread while a timed launch is open."""
    x = torch.ones(4, 8, device=cuda, requires_grad=True)
    ops.TIMER = ops.KernelTimer()
    try:
        plan = ops.route_plan(torch.tensor([0, 1, 2, 0], device=cuda), 3)
        out = ops.expert_dispatch(x, plan)
        plan.place.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), x)
        assert "route_dispatch" in ops.TIMER.summary()
    finally:
        ops.TIMER = None


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=ids)
def test_species_without_weights_are_refused(cuda, index):
    """The per-species linear of exported programs, forward and backward; all species known, or no atoms, pass."""
    lin = pm.e3nnElementLinear("4x0e+4x1o", "4x0e+4x1o", 3).to(cuda)
    args = "4x0e+4x1o", "4x0e+4x1o", 1.0
    x = torch.ones(5, 16, device=cuda)
    for bad in ([0, 1, 2, 3, 0], [0, 1, -1, 2, 0], [9, 9, 9, 9, 9], [0, 0, 0, 0, 2 ** 31 - 1]):
        species = torch.tensor(bad, device=cuda, dtype=index)
        with pytest.raises(ValueError, match="species are outside 0 .. 2"):
            library.element_linear(x, lin.weight, lin.bias, species, *args)
        with pytest.raises(ValueError, match="species are outside 0 .. 2"):
            library.element_linear_backward(x, lin.weight, species, x, *args)
    species = torch.tensor([2, 0, 2, 0, 0], device=cuda, dtype=index)   # (one species without atoms)
    assert library.element_linear(x, lin.weight, lin.bias, species, *args).shape == (5, 16)
    assert library.element_linear(x[:0], lin.weight, lin.bias, species[:0], *args).shape == (0, 16)
    assert library.element_linear_backward(x[:0], lin.weight, species[:0], x[:0], *args).shape == (0, 16)


def test_signs_of_negated_views(cuda):
    """Parts of conjugates are views whose sign is not in memory: one by one, as inputs and as gradients."""
    gen = torch.Generator().manual_seed(1)
    z = lambda *shape: torch.view_as_complex(torch.randint(-4, 5, (*shape, 2), generator=gen).float()).to(cuda)
    minus = lambda t: torch._neg_view(-t)   # t, by a view of -t
    e = torch.tensor([[0], [1], [0], [2]], device=cuda)
    plan, t = ops.route_plan(e, 3), torch.tensor([0, 3, 1, 1], device=cuda)
    x, w = z(4, 8).real.contiguous(), z(4, 1).imag.contiguous()
    fs = (lambda x, w: ops.embedding(x, t), lambda x, w: ops.expert_dispatch(x, plan, w), lambda x, w: ops.dropout(x, 0.5, (1, 2)),
          lambda x, w: ops.expert_combine(x, plan, w), lambda x, w: ops.dropout(w.expand(4, 8).contiguous(), 0.5, (1, 2), residual=x))
    for f in fs:
        want = f(x, w)
        for v in (minus(x), torch.complex(x, -x).conj().imag):
            assert v.is_neg() and torch.equal(v, x)
            assert torch.equal(f(v, w), want)
        assert torch.equal(f(x, minus(w)), want)
        leaf = x.clone().requires_grad_(True)
        out = f(leaf, w)
        g = torch.randint(-4, 5, out.shape, generator=gen).float().to(cuda)
        (want,) = torch.autograd.grad(out, leaf, g, retain_graph=True)
        assert torch.equal(torch.autograd.grad(out, leaf, minus(g))[0], want)
    assert torch.equal(ops.embedding(x, minus(t)), x[t])
    other = ops.route_plan(minus(e), 3)
    assert torch.equal(other.order, plan.order) and torch.equal(other.rowptr, plan.rowptr)
    one = z(1, 1)
    assert ops.dropout(one.conj().imag, 0.0, (1, 2)).item() == -one.imag.item()
    with pytest.raises(ValueError, match="rng"):
        ops.dropout(x, 0.5, minus(torch.tensor([1, 2], device=cuda)))
    rowptr, order = ops.group_by_key(t, 4)
    with pytest.raises(ValueError, match="groups"):
        ops.embedding(x, t, 1.0, (rowptr, minus(order)))


def _operators(cuda):
    """name -> (function of its float tensors, the tensors)"""
    t = torch.tensor([0, 3, 1, 1], device=cuda)
    plan = ops.route_plan(t, 4)
    x, w = torch.ones(4, 8, device=cuda), torch.full((4, 1), 0.5, device=cuda)
    return dict(
        embedding=(lambda x: ops.embedding(x, t), [x]),
        dispatch=(lambda x, w: ops.expert_dispatch(x, plan, w), [x, w]),
        combine=(lambda x, w: ops.expert_combine(x, plan, w), [x, w]),
        dropout=(lambda x, r: ops.dropout(x, 0.5, (1, 2), residual=r), [x, x]))


@pytest.mark.parametrize("name", ["embedding", "dispatch", "combine", "dropout"])
def test_forward_mode_and_transforms_are_refused(cuda, name):
    """There is no forward-mode derivative and no batching rule: an error for every input, never a wrong value."""
    f, inputs = _operators(cuda)[name]
    for i in range(len(inputs)):
        one = lambda v: f(*inputs[:i], v, *inputs[i + 1:])
        with fwd.dual_level(), pytest.raises(RuntimeError, match="jvp is not implemented"):
            one(fwd.make_dual(inputs[i], torch.ones_like(inputs[i])))
        with pytest.raises(RuntimeError, match="functorch"):
            torch.func.grad(lambda v: one(v).sum())(inputs[i])
        with pytest.raises((RuntimeError, ValueError)):
            torch.vmap(one)(torch.stack([inputs[i]] * 2))


@pytest.mark.parametrize("name", ["embedding", "dispatch", "combine", "dropout"])
def test_fake_tensors_are_refused(cuda, name):
    f, inputs = _operators(cuda)[name]
    mode = FakeTensorMode(allow_non_fake_inputs=True)
    for i in range(len(inputs)):
        with pytest.raises(ValueError, match="holds no memory"):
            f(*inputs[:i], mode.from_tensor(inputs[i]), *inputs[i + 1:])
    t = mode.from_tensor(torch.zeros(4, dtype=torch.int64, device=cuda))
    state = mode.from_tensor(torch.zeros(2, dtype=torch.int64, device=cuda))
    for call in (lambda: ops.embedding(inputs[0], t), lambda: ops.route_plan(t, 3),
                 lambda: ops.dropout(inputs[0], 0.5, state)):
        with pytest.raises(ValueError, match="holds no memory"):
            call()


def test_recording_notices_dropout_of_a_model(cuda):
    drop = pm.Dropout(0.2, 0.0, seed=1)
    drop.step_masks()
    x = torch.ones(4, device=cuda)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(RuntimeError, match="recorded into a graph"):
            drop.step_masks()
    x.fill_(2)
    graph.replay()
    assert y.tolist() == [3.0] * 4 and drop.step == 1


def test_masks_differ_between_members(cuda):
    x, irreps = torch.ones(500, 32, device=cuda), Irreps("8x0e+8x1o")
    masks = [pm.Dropout(0.5, 0.5, 3, member).step_masks() for member in (0, 1)]
    for draw in (lambda m: m.features(x, irreps, 1), lambda m: m.attention(x, 1)):
        a, b = (draw(m) != 0 for m in masks)
        # 8,000 draws at least, by block: a share of 0.5 agrees by chance, its standard deviation below 0.007
        assert 0.45 < (a == b).float().mean().item() < 0.55


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_unaligned_rows_hold_the_same_bits(cuda, dt, shift):
    """What is not a sum over a row's elements does not depend on where the rows start.  (float16: a product of an element
    and a float32 may be rounded once, or to float32 first, as the compiler has it for each width of a move.  Both lie
    within half a step, eps / 2, of float32 values that differ by at most four half steps, 2^-24 each, of terms of
    together less than 32: within a step of each other and 4 * 32 * 2^-24 = 2^-17.)"""
    T, k, D = 40, 2, 24
    gen = torch.Generator().manual_seed(shift)
    e = torch.randint(-1, 4, (T, k), generator=gen).to(cuda)
    plan, t = ops.route_plan(e, 4), (torch.arange(T, device=cuda) * 3) % 8 - 1
    off = lambda v: torch.cat([v.new_zeros(shift), v.reshape(-1)])[shift:].view(v.shape)
    x, y, g = (torch.randn(r, D, generator=gen, dtype=torch.float64).to(dt).to(cuda) for r in (T, T * k, T))
    w = torch.rand(T, k, generator=gen, dtype=torch.float64).to(cuda).requires_grad_(True)

    def run(move):
        a, b = (move(v).detach().requires_grad_(True) for v in (x, y))
        kw = dict(widths=(8, 16))
        xs, xw, out = ops.expert_dispatch(a, plan, **kw), ops.expert_dispatch(a, plan, w, **kw), ops.expert_combine(b, plan, w, **kw)
        rows, kept = ops.embedding(a, t, 0.7), ops.dropout(a, 0.4, (1, 2), components=(1, 2), residual=move(g))
        return [xs, xw, out, rows, kept, torch.autograd.grad(out, b, move(g), retain_graph=True)[0],
                torch.autograd.grad(out, (b, w), move(g))[0], torch.autograd.grad(xs, a, move(y))[0],
                torch.autograd.grad(xw, a, move(y))[0], torch.autograd.grad(kept, a, move(g))[0]]
    for i, (p, q) in enumerate(zip(run(off), run(lambda v: v))):
        if dt == torch.float16:
            p, q = p.double(), q.double()
            assert bool(((p - q).abs() <= torch.finfo(dt).eps * torch.maximum(p.abs(), q.abs()) + 2.0 ** -17).all()), i
        else:
            assert torch.equal(p, q), i


@pytest.mark.parametrize("model_zs,batch_zs", [([24, 26, 27, 28], [26]), ([26], [24, 26, 27, 28]), ([24, 26, 27, 28], [26, 27])])
def test_batches_of_other_elements_are_refused(cuda, model_zs, batch_zs):
    """A batch made for another list of elements than the model's has other columns: an error in training (where the
    species are looked up) as in evaluation."""
    s = structures.bcc_fe(reps=(2, 2, 2), seed=4)
    cfg = configs.model_cfg("tece", model_zs, 58.0, num_channel=16, num_head=2, edge_ace_hidden=8)
    m = pm.create_model(cfg).to(cuda)
    m.reset_target_property(["energy", "forces"])
    d = data.gpu_graph([s], batch_zs, 5.0, torch.float32, cuda)
    for mode in (True, False):
        with pytest.raises((RuntimeError, ValueError, IndexError)):
            m.train(mode)(d)
    m.train()(data.gpu_graph([s], model_zs, 5.0, torch.float32, cuda))
