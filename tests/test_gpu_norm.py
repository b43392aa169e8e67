"""Root-mean-square norm against 64-bit restatements.

Bounds count half steps u of the sums' type.  A row's sum: at most 32 terms in a lane, 6 levels of a wavefront, 16
wavefronts, and a product each: 55 u of the sum of magnitudes, so 28 u of q = 1 / sqrt(sum / n + eps) and 4 more for the
division, the addition, the root and its reciprocal.
"""

import pytest
import torch

from tace_amd import ops

import _rows as R

pytestmark = pytest.mark.gpu

ids = lambda v: str(v).replace("torch.", "")
SUM, FACTOR = 55, 32


def _rand(shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dt)


def _blocks(x, comps, C):
    n = x.shape[0]
    return [p.view(n, d * C) for p, d in zip(x.reshape(-1).split([n * d * C for d in comps]), comps)]


def _flat(parts, like):
    return torch.cat([p.reshape(-1) for p in parts]).view(like.shape)


class Reference:
    """y, h and, from gy and gh, the gradients and their bounds (64 bits; x, res, w as given, h rounded to x's type)."""

    def __init__(self, x, res, w, eps, comps, gy=None, gh=None):
        dt, C, u = x.dtype, w.shape[-1], R.sum_step(x.dtype)
        w = w.double().view(len(comps), C)
        self.h = x.double() if res is None else (
            (x + res) if dt == torch.float64 else (x.float() + res.float()).to(dt)).double()
        hs = _blocks(self.h, comps, C)
        self.q = [1 / torch.sqrt(b.square().mean(1, keepdim=True) + eps) for b in hs]
        ws = [w[i].repeat(d) for i, d in enumerate(comps)]
        self.parts = [b * q * v for b, q, v in zip(hs, self.q, ws)]
        self.y = _flat(self.parts, x)
        self.y_slack = self.y.abs() * (FACTOR + 2) * u
        self.y_bound = self.y_slack + R.rounded(self.y.abs() + self.y_slack, dt)
        if gy is None:
            return
        gs = _blocks(gy.double(), comps, C)
        dh, slack, dw, mag = [], [], [], []
        for g, b, q, v, d in zip(gs, hs, self.q, ws, comps):
            n = b.shape[1]
            dot, dot_mag = (g * v * b).sum(1, keepdim=True), (g * v * b).abs().sum(1, keepdim=True)
            dh.append(q * (g * v - b * q * q * dot / n))
            # u: 2 roundings; h k: the sum's (and a product), q^2's 2 x 32 and 4 more; both by q: 32 and 2
            slack.append(q * ((g * v).abs() * (FACTOR + 4) + b.abs() * q * q * dot_mag / n * (SUM + 1 + 3 * FACTOR + 6)) * u)
            t = g * b * q
            dw.append(t.view(-1, d, C).sum((0, 1)))
            # every term: q's error and 2 products; summed in some order
            mag.append(t.abs().view(-1, d, C).sum((0, 1)) * (b.shape[0] * d + FACTOR + 2) * u)
        self.dx, s = _flat(dh, x), _flat(slack, x)
        if gh is not None:
            self.dx = self.dx + gh.double()
            s = s + (self.dx.abs() + s) * u
        self.dx_bound = s + R.rounded(self.dx.abs() + s, dt)
        self.dw, self.dw_slack = torch.stack(dw), torch.stack(mag)


def _check(cuda, dt, rows, C, comps, residual, wide=False, eps=1e-6, grad=True):
    D = C * sum(comps)
    x, w = _rand((rows, D), dt, 1, 0.7), _rand((len(comps), C), dt, 2) + 1
    w = w.to(torch.float64 if dt == torch.float64 else torch.float32) if wide else w
    res = _rand((rows, D), dt, 3, 2.0) if residual else None
    gy, gh = _rand((rows, D), dt, 4), _rand((rows, D), dt, 5) if residual else None
    ref = Reference(x, res, w, eps, comps, gy, gh)
    leaves = [t.to(cuda).requires_grad_(grad) for t in (x, w, res) if t is not None]
    out = ops.rms_norm(leaves[0], leaves[1], eps, residual=leaves[2] if residual else None, components=comps)
    y, h = out if residual else (out, None)
    assert y.dtype == dt and y.shape == x.shape
    R.assert_within(y, ref.y, ref.y_bound, "y")
    if residual:
        assert torch.equal(h.detach().cpu().double(), ref.h)
    if not grad:
        return
    gs = torch.autograd.grad((y, h) if residual else y, leaves, (gy.to(cuda), gh.to(cuda)) if residual else gy.to(cuda))
    assert [g.dtype for g in gs] == [t.dtype for t in leaves]
    R.assert_within(gs[0], ref.dx, ref.dx_bound, "dx")
    R.assert_within(gs[1], ref.dw, ref.dw_slack + R.rounded(ref.dw.abs() + ref.dw_slack, w.dtype), "dw")
    if residual:
        assert torch.equal(gs[0], gs[2])


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 2), (100, 64), (77, 63), (1000, 128), (41, 1000), (9, 1003), (6, 4096),
                                    (5, 8200), (3, 16384), (2, 32768), (2, 32767)])
def test_rows(cuda, dt, rows, C):
    _check(cuda, dt, rows, C, [1], residual=rows % 2 == 1)


@pytest.mark.parametrize("dt", R.TYPES, ids=ids)
@pytest.mark.parametrize("rows,C,L,residual", [(1, 5, 1, False), (130, 16, 3, True), (33, 100, 2, True), (500, 128, 3, False),
                                               (64, 256, 3, True), (3, 4000, 3, True)])
def test_degrees(cuda, dt, rows, C, L, residual):
    _check(cuda, dt, rows, C, [2 * l + 1 for l in range(L + 1)], residual, wide=rows % 2 == 0)


@pytest.mark.parametrize("residual", [False, True])
def test_many_rows(cuda, residual):
    _check(cuda, torch.float32, 70001, 16, [1], residual)
    _check(cuda, torch.bfloat16, 20011, 64, [1, 3], residual)


def test_evaluation_gives_the_training_forward(cuda):
    x, w, r = (_rand(s, torch.float32, i).to(cuda) for i, s in enumerate(((50, 96), (96,), (50, 96))))
    leaf = x.clone().requires_grad_(True)
    with torch.no_grad():
        a = ops.rms_norm(leaf, w, residual=r)
    b = ops.rms_norm(leaf, w, residual=r)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and b[0].requires_grad and not a[0].requires_grad


# ------------------------------------------------------------------ 8 bits ----
def _e4m3_step(y):
    """The codes' distance at y (in units of the scale)."""
    return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("rows,C,comps,residual", [(1, 1, [1], False), (100, 128, [1], True), (37, 100, [1, 3], True),
                                                   (50, 256, [1, 3, 5, 7], False), (7, 1003, [1], True),
                                                   (5, 8192, [1], True), (3, 32768, [1], False)])
def test_codes(cuda, dt, rows, C, comps, residual):
    D, u = C * sum(comps), 2.0 ** -24
    x, w = _rand((rows, D), dt, 1), _rand((len(comps), C), dt, 2)
    x[0, :] = 0
    if rows > 1:
        x[1] *= 1e-4
    res = _rand((rows, D), dt, 3) if residual else None
    ref = Reference(x, res, w, 1e-6, comps)
    got = ops.rms_norm_e4m3(x.to(cuda), w.to(cuda), 1e-6, None if res is None else res.to(cuda), comps)
    q, s = got[0], got[1]
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and s.dtype == torch.float32 and s.shape == (rows, len(comps))
    if residual:
        assert torch.equal(got[2].cpu().double(), ref.h)
    qs = _blocks(q.cpu().float().double(), comps, C)
    for b, y in enumerate(ref.parts):
        want = y.abs().amax(1) / 448
        R.assert_within(s[:, b], want, want * (FACTOR + 4) * u, "scale")
        scale = s[:, b].cpu().double().unsqueeze(1)
        unit = torch.where(scale > 0, y / scale.clamp(min=1e-300), torch.zeros_like(y))
        # half a code's step of a value that is itself off by y's error and two factors'
        slack = unit.abs() * (2 * FACTOR + 8) * u
        R.assert_within(qs[b], unit, _e4m3_step(unit.abs() + slack) / 2 + slack, "codes")


def test_codes_of_extreme_rows(cuda):
    x = torch.ones(6, 64, device=cuda)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] = 1e-30
    q, s = ops.rms_norm_e4m3(x, torch.ones(64, device=cuda), 1e-6)
    assert s[0, 0] == torch.tensor(1.0, device=cuda) / (1 + 1e-6) ** 0.5 / 448 or abs(float(s[0, 0]) * 448 - 1) < 1e-5
    assert float(s[1, 0]) == 0 and not q[1].float().any()
    assert torch.isnan(s[2, 0]) and torch.isnan(s[3, 0])
    assert torch.isfinite(q[[0, 1, 4, 5]].float()).all() and q[5].float().eq(448).all()
    w = torch.full((64,), 1e-35, device=cuda)      # below 2^-100: zeros
    q, s = ops.rms_norm_e4m3(x[:1], w, 1e-6)
    assert float(s) == 0 and not q.float().any()


# --------------------------------------------------- layouts and derivatives ----
def test_strides_shapes_and_empty(cuda):
    base = _rand((40, 48), torch.float32, 1).to(cuda)
    w = _rand((24,), torch.float32, 2).to(cuda)
    want = lambda t: ops.rms_norm(t.contiguous().clone(), w)
    for v in (base[:, 24:], base[::3, :24], base.t()[:24].t(), base.view(-1)[3:3 + 24 * 7].view(7, 24)):
        assert torch.allclose(ops.rms_norm(v, w), want(v), rtol=1e-6, atol=0)
    assert torch.equal(ops.rms_norm(base.view(2, 20, 2, 24), w).view(-1, 24), want(base.view(-1, 24)))
    assert torch.equal(ops.rms_norm(base[0, :24], w), want(base[:1, :24])[0])
    odd = torch.empty(25, device=cuda)[1:].copy_(w)   # an unaligned weight
    assert torch.allclose(ops.rms_norm(base[:, :24], odd), want(base[:, :24]), rtol=1e-6, atol=0)
    z = torch.view_as_complex(base.view(40, 24, 2)).conj().imag   # values behind a sign
    assert torch.equal(ops.rms_norm(z, w), want(z.resolve_neg()))
    leaf, lw = base[:0, :24].clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = ops.rms_norm(leaf, lw)
    gx, gw = torch.autograd.grad(y.sum(), (leaf, lw))
    assert y.shape == (0, 24) and gx.shape == (0, 24) and torch.equal(gw, torch.zeros_like(w))
    q, s = ops.rms_norm_e4m3(base[:0, :24], w)
    assert q.shape == (0, 24) and s.shape == (0, 1)


def test_one_sided_gradients(cuda):
    x, w, r = (_rand(s, torch.float64, i).to(cuda).requires_grad_(True) for i, s in enumerate(((9, 32), (32,), (9, 32))))
    y, h = ops.rms_norm(x, w, residual=r)
    g = torch.ones_like(y)
    only_h = torch.autograd.grad(h, (x, r, w), g, retain_graph=True, allow_unused=True)
    assert torch.equal(only_h[0], g) and torch.equal(only_h[1], g) and not only_h[2].any()
    both = torch.autograd.grad((y, h), (x, w), (g, g), retain_graph=True)
    only_y = torch.autograd.grad(y, (x, w), g)
    assert torch.allclose(both[0], only_y[0] + g, rtol=1e-14, atol=1e-14) and torch.equal(both[1], only_y[1])
    frozen = ops.rms_norm(x, w.detach())                    # no gradient for the weight
    assert torch.allclose(torch.autograd.grad(frozen, x, g)[0],
                          torch.autograd.grad(ops.rms_norm(x, w), x, g)[0], rtol=0, atol=0)


@pytest.mark.parametrize("comps", [[1], [1, 3]])
@pytest.mark.parametrize("residual", [False, True])
def test_gradients_against_differences(cuda, comps, residual):
    D = 6 * sum(comps)
    x, w, r = (_rand(s, torch.float64, i).to(cuda).requires_grad_(True)
               for i, s in enumerate(((4, D), (len(comps), 6), (4, D))))
    f = (lambda a, b, c: ops.rms_norm(a, b, 1e-3, c, comps)) if residual else (lambda a, b: ops.rms_norm(a, b, 1e-3, None, comps))
    args = (x, w, r) if residual else (x, w)
    assert torch.autograd.gradcheck(f, args)
    assert torch.autograd.gradgradcheck(f, args)


def test_repeats_bit_for_bit_and_on_other_streams(cuda):
    x, w, g = (_rand(s, torch.bfloat16, i).to(cuda) for i, s in enumerate(((9000, 384), (384,), (9000, 384))))
    def once():
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = ops.rms_norm(a, b)
        return [y.detach(), *torch.autograd.grad(y, (a, b), g)]
    first = once()
    for k in range(3):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = once()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_recorded(cuda):
    x, w, r, g = (_rand(s, torch.float32, i).to(cuda) for i, s in enumerate(((300, 128), (128,), (300, 128), (300, 128))))
    def once():
        a, b, c = (t.detach().requires_grad_(True) for t in (x, w, r))
        y, h = ops.rms_norm(a, b, residual=c)
        q = ops.rms_norm_e4m3(x, w, residual=r)
        return [y.detach(), h.detach(), *torch.autograd.grad((y, h), (a, b), (g, g)), q[0], q[1]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for k in range(4):
        x.copy_(_rand((300, 128), torch.float32, 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, once()))


def test_refusals(cuda):
    x, w = torch.ones(4, 16, device=cuda), torch.ones(16, device=cuda)
    for call, text in [
            (lambda: ops.rms_norm(x.int(), w), "dtype"), (lambda: ops.rms_norm(x, w[:8]), "weight"),
            (lambda: ops.rms_norm(x, w.half()), "weight"), (lambda: ops.rms_norm(x, w.cpu()), "weight is on"),
            (lambda: ops.rms_norm(x, w, residual=x[:2]), "residual"), (lambda: ops.rms_norm(x, w, residual=x.half()), "residual"),
            (lambda: ops.rms_norm(x, w, components=[1, 3]), "weight"), (lambda: ops.rms_norm(x, w, components=[3]), "x has shape"),
            (lambda: ops.rms_norm(x, w, components=[]), "components"), (lambda: ops.rms_norm(x, w, -1.0), "eps"),
            (lambda: ops.rms_norm(torch.ones(2, 32769, device=cuda), torch.ones(32769, device=cuda)), "32768"),
            (lambda: ops.rms_norm_e4m3(x.double(), w.double()), "float32, bfloat16 or float16"),
            (lambda: ops.rms_norm_e4m3(x.clone().requires_grad_(True), w), "no gradient")]:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(RuntimeError):   # forward-mode derivatives
        import torch.autograd.forward_ad as fwd
        with fwd.dual_level():
            ops.rms_norm(fwd.make_dual(x, x), w)


@pytest.mark.parametrize("dt,wide", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, True), (torch.float32, False)],
                         ids=ids)
@pytest.mark.parametrize("C,comps", [(256, [1]), (100, [1, 3]), (64, [1, 3, 5])])
def test_codes_on_borders_go_to_even(cuda, dt, wide, C, comps):
    """A value between two codes is h w 448 / max |h w| of its row, whatever the row's factor was rounded to: products of a
    few bits lie exactly there, and nowhere else nearer than 2^-22, where no single rounding moves them across."""
    x = _rand((200, C * sum(comps)), torch.bfloat16, 1).to(dt)
    w = torch.ones(len(comps), C, dtype=dt) if wide else _rand((len(comps), C), torch.bfloat16, 2).to(dt)
    q, _ = ops.rms_norm_e4m3(x.to(cuda), (w.float() if wide else w).to(cuda), 1e-6, None, comps)
    borders = 0
    for i, (b, got) in enumerate(zip(_blocks(x.double(), comps, C), _blocks(q.cpu().float().double(), comps, C))):
        p = b * w[i].double().repeat(comps[i])
        unit = p * 448 / p.abs().amax(1, keepdim=True)
        steps = unit / _e4m3_step(unit)
        assert torch.equal(got, torch.round(steps) * _e4m3_step(unit))
        borders += int((steps.frac().abs() == 0.5).sum())
    assert borders > 0


def test_codes_of_the_largest_and_smallest_rows(cuda):
    """Rows at float32's ends: scales are max |y| / 448 as long as those are numbers of 2^-100 and more."""
    x = _rand((50, 72), torch.bfloat16, 1).float()
    for size in (2.0 ** 126, 1e37, 1.0, 1e-20, 2.0 ** -98):
        w = (_rand((72,), torch.float32, 2).abs() + 0.5).clamp(max=1.0) * size
        x = x / x.abs().amax(1, keepdim=True)
        x[:, 0], w[0] = 1.0, size               # (the largest |y|: size by a row's factor of 1 to 4)
        ref = Reference(x, None, w, 1e-6, [1])
        q, s = ops.rms_norm_e4m3(x.to(cuda), w.to(cuda), 1e-6)
        top = ref.y.abs().amax(1)
        held = top < 3.4e38
        R.assert_within(s[held.to(cuda), 0], (top / 448)[held], (top / 448 * (FACTOR + 4) * 2.0 ** -24)[held], size)
        unit = ref.y / (s.cpu().double())
        slack = unit.abs() * (2 * FACTOR + 8) * 2.0 ** -24
        R.assert_within(q[held.to(cuda)].float(), unit[held], (_e4m3_step(unit + slack) / 2 + slack)[held], size)
        assert int(held.sum()) >= 10
