"""The row operators at the ends of their arguments (CPU)."""

import pytest
import torch

from tace_amd import _native as N
from tace_amd import configs
from tace_amd import model as pm
from tace_amd import ops


@pytest.mark.parametrize("ty", range(4))
def test_workspace_is_asked_for_wherever_one_is_needed(ty):
    """0 bytes for the form that looks through all tokens, and only for it; rows of one or two elements need few."""
    L = N.lib()
    for n in (1, 100, 1000, 2049, 4096, 4097, 70000):
        for V in (1, 2, 128, 129, 1024, 1025, 2000):
            for C in (1, 2, 3, 64):
                assert L.tace_embed_grad_work(ty, n, V, C, 1) > 0
                none = n <= 4096 and V <= 1024
                if none or not L.tace_embed_grad_grouped(n, V):
                    assert (L.tace_embed_grad_work(ty, n, V, C, 0) == 0) == none


def test_no_rows_need_no_grouping():
    """A gradient of no rows takes neither a grouping nor a workspace, whatever the table's size."""
    L = N.lib()
    for V in (0, 1, 9, 128, 129, 1024, 1025, 32640, 32641, 2 ** 31 - 8193):
        assert L.tace_embed_grad_grouped(0, V) == 0, V
        assert L.tace_embed_grad_work(0, 0, V, 4, 0) == 0
    assert L.tace_embed_grad(0, 8, None, None, None, None, 0, 5000, 4, 1.0, None, None, 0, None) < 0
    assert b"null" in L.tace_last_error()   # (the gradient itself is what is missing)


def _plan(rowptr, tokens, k=1):
    return ops.RoutePlan(torch.tensor(rowptr, dtype=torch.int32), None, None, tokens, k)


def test_ranges_of_a_plan_that_is_none_are_refused():
    """Ranges reach the linears as row numbers."""
    assert _plan([0, 2, 2, 5], 5).ranges == [(0, 0, 2), (2, 2, 5)]
    assert _plan([0, 2, 2, 3], 3, 2).ranges == [(0, 0, 2), (2, 2, 6)]
    for rowptr in ([0, 5, 3, 6], [0, 2, 9], [1, 2, 6], [-1, 3, 6], [0, -4, 6]):
        with pytest.raises(ValueError, match="rowptr"):
            _plan(rowptr, 6).ranges


@pytest.mark.parametrize("double", [False, True])
def test_experts_take_the_rows_of_their_plan(double):
    """Rows that the plan does not have, or too few of them, are refused; so is a plan without experts."""
    lin = pm.e3nnElementLinear("4x0e+4x1o", "4x0e+4x1o", 3)
    with ops.differentiable_twice(double), torch.no_grad():
        if double:   # (the kernels' path takes GPU tensors)
            assert lin(torch.ones(6, 16), _plan([0, 2, 2, 5], 3, 2)).shape == (6, 16)
            assert lin(torch.ones(0, 16), _plan([0, 0, 0, 0], 0)).shape == (0, 16)
        for rows in (3, 5, 7, 12):
            with pytest.raises(ValueError, match="6 rows"):
                lin(torch.ones(rows, 16), _plan([0, 2, 2, 5], 3, 2))
        with pytest.raises(ValueError, match="no experts"):
            lin(torch.ones(6, 16), _plan([0], 6))


def test_masks_of_a_recorded_forward_are_refused(monkeypatch):
    drop = pm.Dropout(0.2, 0.0, seed=1)
    assert drop.step_masks().rng == (1, 1)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="recorded into a graph"):
        drop.step_masks()
    assert drop.step == 1   # (no forward was drawn for)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert drop.step_masks().rng == (1, 2)


def test_members_of_an_ensemble_draw_their_own_masks():
    make = lambda: pm.create_model(configs.model_cfg("tece", [26], 58.0, num_channel=16, num_head=2, edge_ace_hidden=8))
    both = torch.nn.ModuleList([make(), make()])
    assert pm.set_dropout(both, features=0.1, attention=0.1, seed=5) == 4
    drops = [m.readout_fn.dropout for m in both]
    sites = [d.site(layer, kind) for d in drops for layer in range(64) for kind in (0, 1)]
    assert len(set(sites)) == len(sites) and all(0 <= s < 2 ** 32 for s in sites)
    # a single network draws where it always did
    pm.set_dropout(both[1], features=0.1)
    assert [both[1].readout_fn.dropout.site(layer, kind) for layer in (0, 3) for kind in (0, 1)] == [0, 1, 6, 7]


def test_a_binding_of_another_version_is_refused(monkeypatch):
    """The torch binding has the version of the header it was compiled with, beside the library's own."""
    mod = N.rows()
    assert mod.BUILT_FOR == N.ROWS_ABI_VERSION == N.lib().tace_rows_abi_version()
    monkeypatch.setattr(N, "_rows_mod", None)
    monkeypatch.setattr(mod, "BUILT_FOR", N.ROWS_ABI_VERSION - 1)
    monkeypatch.setattr(N, "_load_rows", lambda path: mod)
    with pytest.raises(N.NativeError, match="built for row operators of version"):
        N.rows()
