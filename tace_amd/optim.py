"""AdamW for models in training mode: one pass over the parameters a step.

``AdamW`` is a ``torch.optim.Optimizer`` (parameter groups, ``state_dict``,
schedulers, hooks) whose step is ``ops.adamw_step``: the parameters of a type in
few launches (56 to 84 of them each), the clipping norm in one for each 160,
states in 32 bits or in 8."""

from __future__ import annotations

from typing import Dict, List, Optional

import torch

from . import ops


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) on GPU parameters of float64, float32,
    bfloat16 or float16.

    ``bits``: 32, states in float32 (float64 for float64 parameters), or 8, e4m3
    codes with a float32 scale for each 256 (``exp_avg_sq`` then holds the codes of
    the root, drawn with its mean: the average of squares itself settles some 5 % high).
    Parameters of 16 bits are stepped as float32 masters kept with the states, unless
    ``masters`` is False; what is written to such a parameter elsewhere is lost at the
    next step.  ``max_norm``: the gradients of all groups together are scaled to this
    norm where it is exceeded, and a step whose norm is infinite or NaN changes
    nothing; ``norm`` is the last step's.  ``seed``: of the 8-bit states' rounding, a
    function of it, a parameter's place among the group's of its type, and its steps.
    ``lr`` of a group may be a tensor of one element on the GPU.

    A step can be recorded into a graph (its gradients' addresses are part of
    it) once the states are made, by a first step or ``init_states()``; a
    recording that would make states, or part the count of steps of parameters
    without a gradient from others', is refused.

    Parameters of a type in a group take one launch for each count of steps among
    them: those that miss gradients in turns have counts of their own, which are
    read back and joined again where a step takes more than 32 launches."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 bits: int = 32, max_norm: Optional[float] = None, masters: bool = True, seed: int = 0):
        if bits not in (8, 32):
            raise ValueError(f"AdamW: states of {bits} bits, expected 8 or 32")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"AdamW: betas {betas} are not in [0, 1)")
        if not (eps >= 0 and weight_decay >= 0 and (isinstance(lr, torch.Tensor) or lr >= 0)):
            raise ValueError("AdamW: lr, eps and weight_decay are not negative")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"AdamW: max_norm {max_norm} is not positive")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self.bits, self.max_norm, self.masters, self.seed = bits, max_norm, masters, int(seed)
        self.norm: Optional[torch.Tensor] = None

    def __getstate__(self):
        """What copies and pickles hold, the optimiser's own settings among it."""
        return {**super().__getstate__(), **{k: getattr(self, k) for k in ("bits", "max_norm", "masters", "seed", "norm")}}

    # Launches of a step before counters are looked through for equal ones (twice those that there
    # are at least), and whether a graph holds their addresses.
    _apart, _recorded = 32, False

    # ------------------------------------------------------------ states ----
    def _init(self, p: torch.Tensor, counter: torch.Tensor) -> Dict[str, torch.Tensor]:
        wide = torch.float64 if p.dtype == torch.float64 else torch.float32
        if self.bits == 8 and p.dtype == torch.float64:
            raise ValueError("AdamW: float64 parameters have no states of 8 bits")
        held = torch.float8_e4m3fn if self.bits == 8 else wide
        like = dict(dtype=held, device=p.device)
        s = {"step": counter, "exp_avg": torch.zeros(p.shape, **like), "exp_avg_sq": torch.zeros(p.shape, **like)}
        if self.bits == 8:
            s["scales"] = torch.zeros(-(-p.numel() // ops.ADAM_BLOCK), 2, dtype=torch.float32, device=p.device)
        if self.masters and p.dtype in (torch.bfloat16, torch.float16):
            s["master"] = p.detach().to(torch.float32, copy=True)
        return s

    def _init_of(self, params: List[torch.Tensor]) -> None:
        """States of those that have none; one counter for each type and device."""
        counters: Dict[tuple, torch.Tensor] = {}
        for p in params:
            if not self.state.get(p):
                key = (p.device, p.dtype)
                if key not in counters:
                    counters[key] = torch.zeros(2, dtype=torch.int64, device=p.device)
                self.state[p] = self._init(p, counters[key])

    def init_states(self) -> None:
        """Makes the states of all parameters that require a gradient now."""
        for group in self.param_groups:
            self._init_of([p for p in group["params"] if p.requires_grad])

    def _check_recording(self) -> None:
        """A recorded step makes no states and parts no counts: each replay would do so again."""
        for group in self.param_groups:
            states = [(p.grad is not None, self.state.get(p)) for p in group["params"]]
            if any(has and not s for has, s in states):
                raise RuntimeError("AdamW: a step is recorded before its parameters have states; call init_states() or step() "
                                   "first")
            moved = {id(s["step"]) for has, s in states if has}
            if any(s and id(s["step"]) in moved for has, s in states if not has):
                raise RuntimeError("AdamW: a recorded step has parameters without a gradient whose steps are counted with "
                                   "others'; step() once with the same gradients missing before")

    def _launches(self, group) -> List[List[torch.Tensor]]:
        """Parameters with gradients that take one launch: those of one counter
        (and so of one type).  A counter counts the steps of all that share it, so
        parameters without a gradient this time leave with a copy."""
        with_grad = [p for p in group["params"] if p.grad is not None]
        self._init_of(with_grad)
        sets: Dict[int, List[torch.Tensor]] = {}
        for p in with_grad:
            sets.setdefault(id(self.state[p]["step"]), []).append(p)
        if len(with_grad) < len(group["params"]):
            copies: Dict[int, torch.Tensor] = {}
            for p in group["params"]:
                s = self.state.get(p) if p.grad is None else None
                if s and id(s["step"]) in sets:
                    shared = s["step"]
                    if id(shared) not in copies:
                        copies[id(shared)] = shared.clone()
                    s["step"] = copies[id(shared)]
        return list(sets.values())

    def _rejoin(self) -> None:
        """Counters of a group's parameters of a type that are equal become one.  Reads them back:
        the one place where a step waits for the GPU, where more launches than ``_apart``
        would take longer."""
        held = {id(s["step"]): s["step"] for s in self.state.values() if s}
        count: Dict[int, int] = {}
        for device in {c.device for c in held.values()}:
            mine = [c for c in held.values() if c.device == device]
            count.update(zip(map(id, mine), torch.stack(mine)[:, 0].tolist()))
        shared: Dict[tuple, torch.Tensor] = {}
        for k, group in enumerate(self.param_groups):
            for p in group["params"]:
                s = self.state.get(p)
                if s:
                    s["step"] = shared.setdefault((k, p.device, p.dtype, count[id(s["step"])]), s["step"])

    def _places(self, group, ps: List[torch.Tensor]):
        """Where the group's first parameter like ``ps`` is, and the places of ``ps``
        among those like them: codes are drawn alike however launches divide them."""
        if self.bits != 8:
            return 0, None
        if len(ps) == len(group["params"]):
            return 0, list(range(len(ps)))
        alike = [(i, p) for i, p in enumerate(group["params"]) if p.dtype == ps[0].dtype and p.device == ps[0].device]
        place = {id(p): n for n, (_, p) in enumerate(alike)}
        return alike[0][0], [place[id(p)] for p in ps]

    # -------------------------------------------------------------- step ----
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            self._check_recording()
            self._recorded = True
        launches = [(k, group, ps) for k, group in enumerate(self.param_groups) for ps in self._launches(group)]
        if len(launches) > self._apart and not self._recorded:
            self._rejoin()
            launches = [(k, group, ps) for k, group in enumerate(self.param_groups) for ps in self._launches(group)]
            self._apart = max(AdamW._apart, 2 * len(launches))
        self.norm = None
        if self.max_norm is not None and len(launches) > 1:
            alike: Dict[tuple, List[torch.Tensor]] = {}   # (in the parameters' order, whatever the launches)
            for group in self.param_groups:
                for p in group["params"]:
                    if p.grad is not None:
                        alike.setdefault((p.device, p.dtype), []).append(p.grad)
            norms = [ops.grad_norm(g) for g in alike.values()]
            self.norm = norms[0] if len(norms) == 1 else torch.stack(
                [n.to(norms[0].device, torch.float64) for n in norms]).square().sum().sqrt()
        for k, group, ps in launches:
            states = [self.state[p] for p in ps]
            norm = self.norm
            if norm is not None:
                norm = norm.to(ps[0].device, torch.float64 if ps[0].dtype == torch.float64 else torch.float32)
            first, places = self._places(group, ps)
            got = ops.adamw_step(
                ps, [p.grad for p in ps], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                states[0]["step"], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                weight_decay=group["weight_decay"], scales=[s["scales"] for s in states] if self.bits == 8 else None,
                masters=[s["master"] for s in states] if "master" in states[0] else None, max_norm=self.max_norm,
                norm=norm, seed=(self.seed * 1000003 + k * 8191 + first) % 2 ** 64,
                places=places)
            if self.norm is None:
                self.norm = got
        return loss

    # ------------------------------------------------------------- state ----
    def _states_of(self, state_dict) -> Dict[torch.Tensor, Dict[str, torch.Tensor]]:
        """The states that ``state_dict`` holds, checked, for this optimiser's parameters."""
        groups, given = state_dict["param_groups"], state_dict["state"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("AdamW: the state's parameter groups are not the optimiser's")
        counters: Dict[tuple, torch.Tensor] = {}
        states = {}
        for k, (theirs, ours) in enumerate(zip(groups, self.param_groups)):
            for i, p in zip(theirs["params"], ours["params"]):
                if i not in given:
                    continue
                s = {}
                want = self._init(p, torch.zeros(2, dtype=torch.int64, device=p.device))
                for name, zero in want.items():
                    v = given[i].get(name)
                    if not isinstance(v, torch.Tensor):
                        raise ValueError(f"AdamW: the state of parameter {i} has no {name}; its states have other bits")
                    if v.dtype != zero.dtype or v.shape != zero.shape:
                        raise ValueError(f"AdamW: {name} of parameter {i} is {v.dtype} {tuple(v.shape)}, expected "
                                         f"{zero.dtype} {tuple(zero.shape)}")
                    s[name] = v.detach().to(p.device, copy=True, memory_format=torch.contiguous_format)
                key = (k, p.dtype, p.device, int(s["step"][0]))
                s["step"] = counters.setdefault(key, s["step"])
                states[p] = s
        return states

    def load_state_dict(self, state_dict) -> None:
        """As ``Optimizer.load_state_dict``, but states keep their types (masters
        and codes are not cast to the parameters' type) and parameters whose steps
        are equal share a counter again.  A state that is refused changes nothing."""
        made: Dict[torch.Tensor, Dict[str, torch.Tensor]] = {}
        # (between the caller's hooks: after those before the load, before those after it)
        before = self.register_load_state_dict_pre_hook(lambda _, given: made.update(self._states_of(given)))
        after = self.register_load_state_dict_post_hook(lambda _: self.state.update(made), prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            before.remove()
            after.remove()
