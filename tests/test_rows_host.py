"""The row operators' boundary and refusals (CPU)."""

import ctypes
import os
import re

import pytest
import torch

from tace_amd import _native as N
from tace_amd import ops

from _rows import philox

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "tace_rows.h")


def test_header_bindings_and_library_agree():
    txt = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(tace_\w+)\s*\(", txt))
    lib = N.lib()
    assert declared == set(N.ROWS_EXPORTED)
    assert all(hasattr(lib, name) for name in declared)
    version = int(re.search(r"TACE_ROWS_ABI_VERSION (\d+)", txt).group(1))
    assert lib.tace_rows_abi_version() == version == N.ROWS_ABI_VERSION


def test_rows_of_another_version_are_refused(monkeypatch):
    monkeypatch.setattr(N, "_lib", None)
    monkeypatch.setattr(N, "ROWS_ABI_VERSION", N.ROWS_ABI_VERSION - 1)
    with pytest.raises(N.NativeError, match="row operators of version"):
        N.lib()


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))])
def test_restated_philox_has_the_published_values(counter, key, want):
    """The known answers published with the generator's paper."""
    assert tuple(philox(counter, key)) == want


def _refused(rc, text):
    assert rc < 0 and text in N.lib().tace_last_error(), N.lib().tace_last_error()


def test_entries_refuse_bad_arguments():
    """Before any device work."""
    L = N.lib()
    p = 4096   # (never read)
    w = (ctypes.c_int64 * 9)(*([4] * 9))
    one = (ctypes.c_int32 * 9)(*([1] * 9))
    _refused(L.tace_embed_fwd(9, 8, p, p, 4, 4, 4, 1.0, p, None), b"row type")
    _refused(L.tace_embed_fwd(0, 2, p, p, 4, 4, 4, 1.0, p, None), b"4 or 8 bytes")
    _refused(L.tace_embed_fwd(0, 8, p, p, 4, 4, 40000, 1.0, p, None), b"bad sizes")
    _refused(L.tace_embed_fwd(0, 8, p, p, 4, 2 ** 31, 4, 1.0, p, None), b"bad sizes")
    _refused(L.tace_embed_fwd(0, 8, None, p, 4, 4, 4, 1.0, p, None), b"null")
    assert L.tace_embed_fwd(0, 8, None, None, 0, 4, 4, 1.0, None, None) == 0
    _refused(L.tace_embed_grad(0, 8, p, p, None, None, 4096, 5000, 4, 1.0, p, None, 0, None), b"without a grouping")
    _refused(L.tace_embed_grad(0, 8, p, p, None, None, 5000, 4, 4, 1.0, p, None, 0, None), b"workspace")
    _refused(L.tace_embed_grad(0, 8, p, p, p, p, 5000, 4, 4, 1.0, p, p, 16, None), b"workspace")
    need = L.tace_embed_grad_work(0, 5000, 4, 4, 1)
    _refused(L.tace_embed_grad(0, 8, p, p, p, p, 5000, 4, 4, 1.0, p, p + 8, need, None), b"workspace")
    _refused(L.tace_embed_grad(0, 8, p, p, p, p, 2 ** 31, 4, 4, 1.0, p, p, need, None), b"bad sizes")
    for f in (L.tace_route_dispatch, L.tace_route_combine):
        _refused(f(4, p, None, p, p, 4, 2, 1, w, p, None), b"row type")
        _refused(f(0, p, None, p, p, 4, 0, 1, w, p, None), b"bad sizes")
        _refused(f(0, p, None, p, p, 2 ** 30, 2, 1, w, p, None), b"bad sizes")
        _refused(f(0, p, None, p, p, 4, 2, 9, w, p, None), b"blocks")
        _refused(f(0, p, None, p, p, 4, 2, 1, (ctypes.c_int64 * 1)(40000), p, None), b"32768")
        _refused(f(0, p, None, p, None, 4, 2, 1, w, p, None), b"null")
        assert f(0, None, None, None, None, 0, 2, 1, w, None, None) == 0
    _refused(L.tace_route_dots(0, p, p, None, p, p, 4, 2, 1, w, None, None, None), b"null")
    _refused(L.tace_route_group(4, None, 1, 4, 4, p, p, p, p, None), b"null")
    _refused(L.tace_route_group(3, p, 1, 4, 4, p, p, p, p, None), b"4 or 8 bytes")
    _refused(L.tace_route_group(4, p, 1, 2 ** 31, 4, p, p, p, p, None), b"bad sizes")
    _refused(L.tace_dropout(0, p, None, None, 0, 0, 0, 65537, 4, 4, 1, one, p, None), b"threshold")
    _refused(L.tace_dropout(0, p, None, None, 0, 0, 0, 5, 4, 4, 9, one, p, None), b"bad sizes")
    _refused(L.tace_dropout(0, p, None, None, 0, 0, 0, 5, 2 ** 34, 2, 1, one, p, None), b"2^34")
    _refused(L.tace_dropout(0, p, None, None, 0, 0, 0, 5, 4, 4, 1, (ctypes.c_int32 * 1)(0), p, None), b"components")
    _refused(L.tace_dropout(0, None, None, None, 0, 0, 0, 5, 4, 4, 1, one, p, None), b"null")


def test_operators_take_no_cpu_tensors():
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.embedding(x, t), lambda: ops.route_plan(t, 4), lambda: ops.dropout(x, 0.1, (1, 2))):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()


def test_workspace_covers_every_workgroup():
    """Two sums of a row for each workgroup's sorted positions: at most 512 of them, whatever the size."""
    L = N.lib()
    for n in (1, 31, 257, 4097, 131072, 131073, 1063830, 2 ** 31 - 8193):
        for ty, size in ((0, 4), (1, 8), (2, 4)):
            for C in (1, 7, 100, 128, 4096, 32768):
                nbytes = L.tace_embed_grad_work(ty, n, 7, C, 1)
                assert nbytes % (2 * C * size) == 0
                assert 1 <= nbytes // (2 * C * size) <= 512
                # ungrouped: a sum for each of 128 tokens and at least 256 rows
                nbytes = L.tace_embed_grad_work(ty, n, 128, C, 0)
                assert nbytes <= 16 + (n / 256 + 1) * 128 * (C * size + 4)
    assert [L.tace_embed_grad_grouped(*a) for a in ((4096, 1024), (4097, 128), (4097, 129), (4096, 1025), (0, 9),
                                                         (8193, 8192), (8193, 8193), (40000, 32640), (40000, 32641),
                                                         (2 ** 22, 999), (2 ** 22 + 1, 999))] == [
        0, 0, 0, 1, 0, 0, 1, 0, 1, 0, 1]
    _refused(L.tace_embed_grad(0, 8, 4096, 4096, 4096, 4096, 0, 4, 4, 1.0, 4096, 4096, 16, None), b"no rows")


def test_set_dropout_arguments():
    from tace_amd import configs, model as pm

    m = pm.create_model(configs.model_cfg("tece", [26], 58.0, num_channel=16, num_head=2, edge_ace_hidden=8))
    before = set(m.state_dict())
    assert pm.set_dropout(m, features=0.1) == 2 and pm.set_dropout(m, attention=0.1) == 1   # (layer 0 has none)
    assert m.readout_fn.dropout.attention == 0.1 and set(m.state_dict()) == before
    for bad in (dict(features=-0.1), dict(features=1.0), dict(attention=1e-7), dict(features=float("nan"))):
        with pytest.raises(ValueError, match="dropout of"):
            pm.set_dropout(m, **bad)
    with pytest.raises(ValueError, match="TensorModel"):
        pm.set_dropout(torch.nn.Linear(2, 2), 0.1)
    assert pm.set_dropout(m) == 0 and m.readout_fn.dropout is None
