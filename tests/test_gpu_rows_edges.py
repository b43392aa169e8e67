"""The row operators at the ends of their arguments, against restatements in 64 bits or on whole numbers (which every
type and order of a sum holds exactly)."""

import pytest
import torch

from tace_amd import ops

import _rows as R

pytestmark = pytest.mark.gpu

ids = lambda v: str(v).replace("torch.", "")


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
