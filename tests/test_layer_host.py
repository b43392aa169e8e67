"""The routed layer's operators: boundary and refusals (CPU)."""

import copy
import ctypes
import io
import random

import pytest
import torch

from tace_amd import _native as N
from tace_amd import ops, optim

P = 4096   # an address that is never read


def _refused(rc, text):
    assert rc < 0 and text in N.lib().tace_last_error(), N.lib().tace_last_error()


def _ints(*v):
    return (ctypes.c_int32 * len(v))(*v)


def test_norm_entries_refuse_bad_arguments():
    L = N.lib()
    fwd = lambda ty=0, x=P, r=None, w=P, rows=4, C=8, blocks=1, comps=_ints(1), h=None, y=P, s=None: L.tace_rms_norm_fwd(
        ty, x, r, w, 0, rows, C, blocks, comps, 1e-6, h, y, s, None, None)
    _refused(fwd(ty=4), b"row type")
    _refused(fwd(rows=-1), b"bad sizes")
    _refused(fwd(C=0), b"bad sizes")
    _refused(fwd(blocks=9, comps=_ints(*[1] * 9)), b"bad sizes")
    _refused(fwd(comps=_ints(0)), b"components")
    _refused(fwd(C=32769), b"32768")
    _refused(fwd(C=16385, comps=_ints(2)), b"32768")
    _refused(fwd(rows=2 ** 31 - 1), b"bad sizes")
    _refused(fwd(x=None), b"null")
    _refused(fwd(r=P), b"null")          # a residual without a place for the sum
    _refused(fwd(h=P), b"null")
    _refused(fwd(ty=1, s=P), b"8 bits")
    assert fwd(rows=0, x=None, y=None) == 0
    bwd = lambda ty=0, gy=P, rows=4, dw=None, work=None, nbytes=0: L.tace_rms_norm_bwd(
        ty, gy, None, P, P, 0, P, rows, 8, 1, _ints(1), P, dw, work, nbytes, None)
    _refused(bwd(gy=None), b"null")
    _refused(bwd(rows=0), b"no rows")
    _refused(bwd(dw=P), b"workspace")
    need = L.tace_rms_norm_bwd_work(0, 4, 8, 1, _ints(1))
    _refused(bwd(dw=P, work=P, nbytes=need - 1), b"workspace")
    _refused(bwd(dw=P, work=P + 8, nbytes=need), b"workspace")
    _refused(L.tace_rms_norm_bwd_work(7, 4, 8, 1, _ints(1)), b"row type")


def test_norm_workspace_is_bounded():
    """A row of sums for each of about 1,024 workgroups (or one a row, if they are fewer)."""
    L = N.lib()
    for ty, size in ((0, 4), (1, 8), (2, 4), (3, 4)):
        for rows in (1, 7, 1000, 10 ** 6):
            for C, comps in ((1, (1,)), (63, (1, 3)), (128, (1, 3, 5, 7)), (4096, (1,)), (32768, (1,)), (32767, (1,))):
                nbytes = L.tace_rms_norm_bwd_work(ty, rows, C, len(comps), _ints(*comps))
                assert C * len(comps) * size <= nbytes <= min(1024 + 8, rows * len(comps)) * C * max(comps) * size


class Row(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ("p", "g", "m", "s", "master", "scales")] + [("n", ctypes.c_int64)]


def test_adamw_entries_refuse_bad_arguments():
    L = N.lib()
    row = lambda **over: Row(**{**dict(p=P, g=P, m=P, s=P, n=5), **over})

    def step(ty=0, eight=0, rows=(row(),), counter=P, b1=0.9, b2=0.99, eps=1e-8):
        t = (Row * max(1, len(rows)))(*rows)
        return L.tace_adamw(ty, eight, t, len(rows), counter, 1e-3, None, 0, b1, b2, eps, 0.0, None, 0.0, 0, None)

    _refused(step(ty=9), b"row type")
    _refused(step(counter=None), b"null")
    _refused(step(rows=(row(), row(m=None))), b"null")
    _refused(step(rows=(row(g=None),)), b"null")
    _refused(step(eight=1), b"null")                                 # no scales
    _refused(step(ty=1, eight=1, rows=(row(scales=P),)), b"float64")
    _refused(step(rows=(row(master=P),)), b"masters")
    _refused(step(rows=(row(n=-1),)), b"2^34")
    _refused(step(rows=(row(n=2 ** 34 + 1),)), b"2^34")
    for bad in (dict(b1=1.0), dict(b2=-0.1), dict(b1=float("nan")), dict(eps=-1.0)):
        _refused(step(**bad), b"betas")
    assert step(rows=()) == 0 and step(rows=(Row(n=0),)) == 0
    t = (Row * 2)(row(n=10 ** 9), row())
    need = L.tace_grad_norm_work(t, 2)
    assert need == 8 * 1024
    norm = lambda count=2, ticket=P, out=P, work=P, nbytes=need: L.tace_grad_norm(0, t, count, ticket, out, work, nbytes, None)
    _refused(norm(count=0), b"no gradients")
    for bad in (dict(ticket=None), dict(out=None), dict(work=None), dict(work=P + 4), dict(nbytes=need - 1)):
        _refused(norm(**bad), b"workspace")


def test_operators_take_no_cpu_tensors():
    x, w = torch.ones(4, 8), torch.ones(8)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_e4m3(x, w), lambda: ops.grad_norm([x]),
                 lambda: ops.adamw_step([x], [x], [x], [x], torch.zeros(2, dtype=torch.int64), lr=0.1)):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
    with pytest.raises(ValueError, match="no gradients"):
        ops.grad_norm([])
    with pytest.raises(ValueError, match="64 bits"):
        ops.adamw_step([x], [x], [x], [x], x, lr=0.1, seed=2 ** 64)


def test_optimiser_arguments():
    p = [torch.ones(3, requires_grad=True)]
    for bad, text in ((dict(bits=16), "bits"), (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1.0), "negative"),
                      (dict(lr=-1.0), "negative"), (dict(weight_decay=-0.1), "negative"), (dict(max_norm=0.0), "max_norm")):
        with pytest.raises(ValueError, match=text):
            optim.AdamW(p, **bad)
    o = optim.AdamW(p, max_norm=1.0)
    o.step()                                  # nothing has a gradient
    assert o.norm is None and not o.state[p[0]]
    o.init_states()
    assert o.state[p[0]]["step"].tolist() == [0, 0] and o.state[p[0]]["exp_avg"].dtype == torch.float32


def test_expert_entries_refuse_bad_arguments():
    L = N.lib()
    one = _ints(1)

    def rows(ty=0, x=P, w=P, ptr=P, n=4, E=2, blocks=1, comps=one, K=8, M=8, out=P):
        return L.tace_expert_linear(ty, 0, x, w, ptr, n, E, blocks, comps, K, M, 1.0, out, None)

    _refused(rows(ty=5), b"row type")
    for bad in (dict(n=-1), dict(n=2 ** 31 - 1), dict(E=-1), dict(E=2 ** 21), dict(blocks=0), dict(blocks=9), dict(K=0),
                dict(M=0), dict(K=65537), dict(M=65537), dict(comps=None)):
        _refused(rows(**bad), b"bad sizes")
    _refused(rows(comps=_ints(0)), b"components")
    for bad in (dict(x=None), dict(w=None), dict(ptr=None), dict(out=None)):
        _refused(rows(**bad), b"null")
    assert rows(n=0, x=None, w=None, out=None) == 0

    def grad(ty=0, x=P, g=P, ptr=P, n=100000, E=2, dw=P, work=P, nbytes=1 << 40, M=64):
        return L.tace_expert_linear_grad(ty, x, g, ptr, n, E, 1, one, M, M, 1.0, dw, work, nbytes, None)

    need = L.tace_expert_linear_grad_work(0, 100000, 2, 1, one, 64, 64)
    assert need > 0 and L.tace_expert_linear_grad_work(0, 100, 2, 1, one, 64, 64) == 0
    for bad in (dict(work=None), dict(work=P + 8), dict(nbytes=need - 1)):
        _refused(grad(**bad), b"workspace")
    for bad in (dict(x=None), dict(g=None), dict(dw=None), dict(ptr=None)):
        _refused(grad(**bad), b"null")
    _refused(grad(ty=4), b"row type")
    _refused(grad(E=70000, M=1024), b"bad sizes")
    assert grad(E=0, dw=None) == 0

    def codes(out=2, x=P, xs=P, order=None, k=1, w=P, ws=P, ptr=P, n=4, K=32, o=P):
        return L.tace_expert_linear_e4m3(out, x, xs, order, k, w, ws, ptr, n, 2, K, 8, o, None)

    _refused(codes(out=1), b"float32, bfloat16 or float16")
    _refused(codes(K=24), b"multiple of 16")
    _refused(codes(k=0), b"bad sizes")
    _refused(codes(order=P, k=3), b"bad sizes")
    for bad in (dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(ptr=None), dict(o=None)):
        _refused(codes(**bad), b"null")
    _refused(codes(x=P + 8), b"aligned")
    _refused(codes(w=P + 1), b"aligned")
    assert codes(n=0, x=None, o=None) == 0


def test_expert_workspace_covers_every_part():
    """Two pieces of every tile of [K, M] for each stretch of rows; stretches are no more than units of 128 rows and empty
    groups, and a stretch's workgroups, with one to four tiles each, all run at once."""
    L = N.lib()
    for ty, size in ((0, 4), (1, 8), (2, 4)):
        for rows in (1, 257, 5000, 300000):
            for E in (1, 7, 90):
                for comps in ((1,), (1, 3, 5, 7)):
                    for K, M in ((16, 8), (128, 128), (1024, 2048), (8192, 8192)):
                        nbytes = L.tace_expert_linear_grad_work(ty, rows, E, len(comps), _ints(*comps), K, M)
                        tiles = -(-K // 128) * -(-M // 128)
                        side = 64 if ty == 1 or min(K, M) <= 64 or (rows * sum(comps) // 128 * tiles < 512 and
                            len(comps) * E * (-(-K // 64) * -(-M // 64)) <= 65536) else 128
                        tiles = -(-K // side) * -(-M // side)
                        cuts, rest = divmod(nbytes, 2 * tiles * side * side * size)
                        assert rest == 0
                        if cuts:
                            assert 2 <= cuts <= rows * sum(comps) // 128 + len(comps) * E
                            assert cuts * -(-tiles // 4) <= (1024 if side == 64 else 512)
                        else:
                            assert rows * max(comps) <= 128 or tiles > 512 or rows * sum(comps) // 128 + E * len(comps) < 2


def _states(o):
    return [{k: (v.dtype, v.clone()) for k, v in o.state[p].items()} for g in o.param_groups for p in g["params"]]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_state_dict_changes_nothing(bits):
    make = lambda b, shapes=((300,), (5, 7)): optim.AdamW([torch.ones(s, requires_grad=True) for s in shapes], bits=b, lr=b / 100)
    o, other = make(bits), make(40 - bits)
    for x, v in ((o, 0.5), (other, 2.0)):
        x.init_states()
        for s in x.state.values():
            for k in s:
                s[k].copy_(torch.full(s[k].shape, v))
    wrong = other.state_dict(), make(bits, ((300,),)).state_dict(), make(bits, ((301,), (5, 7)))
    wrong[2].init_states()
    before = _states(o)
    for d in (wrong[0], wrong[1], wrong[2].state_dict(), {**o.state_dict(), "state": {0: {"step": torch.zeros(2)}}}):
        with pytest.raises(ValueError):
            o.load_state_dict(d)
        assert o.param_groups[0]["lr"] == bits / 100 and len(o.param_groups[0]["params"]) == 2
        for a, b in zip(before, _states(o)):
            assert list(a) == list(b)
            for k in a:
                assert a[k][0] == b[k][0] and torch.equal(a[k][1].view(torch.uint8), b[k][1].view(torch.uint8))


def test_state_dicts_pass_hooks():
    """What the hooks before a load make of it is loaded; those after it see the states as they are kept."""
    p = [torch.ones(9, requires_grad=True)]
    o, seen = optim.AdamW(p, bits=8), []
    o.init_states()
    d = o.state_dict()
    def double(opt, s):
        return {**s, "state": {i: {**v, "scales": v["scales"] + 2} for i, v in s["state"].items()}}
    o.register_load_state_dict_pre_hook(double)
    o.register_load_state_dict_post_hook(lambda opt: seen.append(opt.state[p[0]]["exp_avg"].dtype))
    o.load_state_dict(d)
    assert seen == [torch.float8_e4m3fn] and float(o.state[p[0]]["scales"][0, 0]) == 2
    o.load_state_dict(d)      # (hooks of a load leave with it)
    assert float(o.state[p[0]]["scales"][0, 0]) == 2


def _saved(o):   # (pickle alone has no tensors of 8 bits)
    f = io.BytesIO()
    torch.save(o, f)
    return torch.load(io.BytesIO(f.getvalue()), weights_only=False)


@pytest.mark.parametrize("copied", [copy.deepcopy, _saved])
def test_copies_of_an_optimiser_are_whole(copied):
    p = [torch.nn.Parameter(torch.ones(n)) for n in (300, 5)]
    o = optim.AdamW(p, bits=8, max_norm=2.0, masters=False, seed=77)
    o.init_states()
    c = copied(o)
    assert (c.bits, c.max_norm, c.masters, c.seed, c.norm) == (8, 2.0, False, 77, None)
    mine = [c.state[q] for q in c.param_groups[0]["params"]]
    assert mine[0]["step"] is mine[1]["step"] and mine[0]["step"] is not o.state[p[0]]["step"]
    c.step()                          # nothing has a gradient
    c.load_state_dict(o.state_dict())
    c.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(2))]))
    c.init_states()


class Recorder:
    """Stands in for the kernels: notes what they are given and counts steps."""

    def __init__(self, monkeypatch, norm=3.0):
        self.steps, self.norms = [], []

        def adamw_step(params, grads, ms, ss, counter, *, norm=None, max_norm=None, **more):
            assert len({(p.device, p.dtype) for p in (*params, *grads)}) == 1
            self.steps.append(dict(more, params=params, grads=grads, counter=counter, norm=norm))
            counter[0] += 1
            if max_norm is not None:
                return torch.tensor(1.0) if norm is None else norm

        def grad_norm(grads):
            assert len({(g.device, g.dtype) for g in grads}) == 1
            self.norms.append(list(grads))
            return torch.tensor(norm * len(self.norms), dtype=torch.float64 if grads[0].dtype == torch.float64 else torch.float32)

        monkeypatch.setattr(optim.ops, "adamw_step", adamw_step)
        monkeypatch.setattr(optim.ops, "grad_norm", grad_norm)


def _with_grads(*ps):
    for p in ps:
        p.grad = torch.ones_like(p)
    return list(ps)


def test_parameters_of_two_devices_are_clipped_together(monkeypatch):
    r = Recorder(monkeypatch)
    here = _with_grads(*(torch.ones(n, requires_grad=True) for n in (3, 4)))
    there = _with_grads(*(torch.ones(n, requires_grad=True, device="meta") for n in (5, 6)))
    o = optim.AdamW([here[0], there[0], here[1], there[1]], max_norm=1.0)
    o.step()
    assert [len(n) for n in r.norms] == [2, 2] and float(o.norm) == 45 ** 0.5 and len(r.steps) == 2
    for s in r.steps:      # each with the norm of all, where it is read
        assert s["norm"].device == s["params"][0].device and s["norm"].dtype == torch.float32


def test_recordings_that_a_replay_would_undo_are_refused(monkeypatch):
    """States made, or counts parted, inside a recording would be made again by every replay."""
    r, recording = Recorder(monkeypatch), [True]
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: recording[0])
    p = _with_grads(*(torch.ones(4, requires_grad=True) for _ in range(3)))
    o = optim.AdamW(p, max_norm=1.0)
    with pytest.raises(RuntimeError, match="init_states"):
        o.step()
    assert not o.state and not r.steps
    o.init_states()
    p[1].grad = None
    one = o.state[p[0]]["step"]
    with pytest.raises(RuntimeError, match="without a gradient"):
        o.step()
    assert not r.steps and all(o.state[q]["step"] is one for q in p)
    recording[0] = False
    o.step()                               # (parts them)
    recording[0] = True
    o.step()
    assert len(r.steps) == 2 and o.state[p[1]]["step"] is not one


def test_codes_are_drawn_by_parameters_not_by_launches(monkeypatch):
    r = Recorder(monkeypatch)
    p = [torch.ones(4, requires_grad=True, dtype=torch.bfloat16 if i in (1, 4) else torch.float32) for i in range(6)]
    o = optim.AdamW([dict(params=p[:5]), dict(params=p[5:])], bits=8, seed=3)
    _with_grads(*p)
    o.step()
    everywhere = [(s["seed"], s["places"]) for s in r.steps]
    assert everywhere == [(3000009, [0, 1, 2]), (3000010, [0, 1]), (3000009 + 8191, [0])]
    p[2].grad = p[4].grad = None
    o.step()
    assert [(s["seed"], s["places"]) for s in r.steps[3:]] == [(3000009, [0, 2]), (3000010, [0]), (3000009 + 8191, [0])]
    _with_grads(*p)
    o.step()
    assert {(s["seed"], i) for s in r.steps[6:] for i in s["places"]} == {(s, i) for s, l in everywhere for i in l}


def test_counts_that_are_equal_again_share_a_launch(monkeypatch):
    """Gradients missing in turns part the counts of steps; launches stay few, and each parameter's own count."""
    r = Recorder(monkeypatch)
    rng = random.Random(1)
    p = [torch.ones(4, requires_grad=True) for _ in range(60)]
    o = optim.AdamW([dict(params=p[:50]), dict(params=p[50:])])
    o.init_states()
    counts, most = [0] * len(p), 0
    for _ in range(40):
        for i, q in enumerate(p):
            q.grad = None if rng.random() < 0.2 else torch.ones_like(q)
            counts[i] += q.grad is not None
        before = len(r.steps)
        o.step()
        most = max(most, len(r.steps) - before)
        assert [int(o.state[q]["step"][0]) for q in p] == counts
        kinds = len({(i < 50, c) for i, c in enumerate(counts)})
        assert len(r.steps) - before <= max(32, 2 * kinds)
    assert most > 8          # (they did part)
    for g in o.param_groups:   # no count is of two groups
        mine = {id(o.state[q]["step"]) for q in g["params"]}
        assert not mine & {id(o.state[q]["step"]) for h in o.param_groups if h is not g for q in h["params"]}


def test_counts_of_a_recorded_step_stay_its_own(monkeypatch):
    """A graph goes on writing to the counters that it was recorded with."""
    Recorder(monkeypatch)
    p = _with_grads(*(torch.ones(4, requires_grad=True) for _ in range(80)))
    o = optim.AdamW(p)
    for i in range(80):       # every parameter alone
        for k, q in enumerate(p):
            q.grad = torch.ones_like(q) if k == i else None
        o._apart = 1000
        o.step()
    _with_grads(*p)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    o._apart = 1
    o.step()
    held = [o.state[q]["step"] for q in p]
    assert len({id(c) for c in held}) == 80
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    o.step()
    assert all(o.state[q]["step"] is c for q, c in zip(p, held))


def test_weights_of_8_bits_below_float32s_quotients_are_zeros():
    """448 / top overflows below 2^-118: codes were NaN. Such a column is zeros under scale 0, as a normed row is."""
    w = torch.zeros(2, 4, 3)
    w[0, 1:, 0], w[0, 2, 1], w[0, 3, 2] = 2.0 ** -125, -(2.0 ** -101), 2.0 ** -100
    w[1, 0, 0], w[1, :, 1] = float("nan"), float("inf")
    codes, scales = ops.expert_weights_e4m3(w)
    least = torch.tensor(2.0 ** -100 / 448).item()     # (rounded to float32, as scales are)
    assert not codes[0, :2].float().any() and scales[0].tolist() == [0, 0, least]
    assert codes[0, 2].float().tolist() == [0, 0, 0, 448]
    assert torch.isnan(codes[1, 0].float() * scales[1, 0]).all() and torch.isnan(codes[1, 1].float() * scales[1, 1]).all()
    assert not codes[1, 2].float().any() and scales[1, 2] == 0
