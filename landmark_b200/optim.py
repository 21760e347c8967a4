"""AdamW over many tensors at once (``gnr_adamw_step``), with optimiser states in 32 or in 8 bits.

The reference trains the planes, lines and network of a field with ``torch.optim.Adam`` over parameter groups; ``AdamW`` takes the
same groups.  A step is one launch for each parameter type of a group (per 400 tensors), whatever the tensors' sizes; with
``state_bits=8`` the states take 2 bytes a value instead of 8.

8-bit states: every 256 values of a tensor share two scales; the first moment is ``scale * code``, the second
``(scale * code) ** 2`` with float8_e4m3fn codes, rounded at random without bias (a hash of seed, step, tensor and place, so a
step repeats bit for bit); a second moment below the smallest code's, 2^-35.6 of the largest beside it, becomes that code, never 0.  A gradient
that is not finite spoils its own value only.

16-bit parameters can have a copy in fp32 (``masters``): the step updates the copy, the parameter is its rounded image.  Without
one, what a step changes by less than half a unit of the last place is lost.
"""

from __future__ import annotations

import ctypes as C
import operator
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import check, lib
from .embedding import _TYPES, _on, _raw_stream

BLOCK = _lib.ADAMW_BLOCK
_CODES = torch.float8_e4m3fn
_WORDS = C.sizeof(_lib.GnrAdamwTensor) // 8  # nine 64-bit words a tensor
_GRAD, _N = 1, 7
_step_of, _dtype_of = operator.itemgetter("step"), operator.attrgetter("dtype")
_version_of, _layout_of, _is_neg = operator.attrgetter("_version"), operator.attrgetter("layout"), torch.Tensor.is_neg
_address, _numel, _get_device, _is_contiguous = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous


def _versions(tensors) -> Optional[List[int]]:
    """How often autograd has counted a write of each (None: of inference tensors)."""
    try:
        return list(map(_version_of, tensors))
    except RuntimeError:
        return None


def state_blocks(numel: int) -> int:
    """Scales of a tensor's 8-bit state."""
    return -(-numel // BLOCK)


_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


def _no_capture():
    if _capturing():
        raise RuntimeError("an AdamW step cannot be captured into a CUDA graph: a replay would repeat this step's count and rates.  Capture "
                           "AdamWTensors.step_clocked() with an AdamWClock")


def _shared(ranges) -> Optional[tuple]:
    """Names of two of the ``ranges`` (address, bytes, name ...) that share memory, if any do."""
    ranges = sorted(ranges)
    for one, next_one in zip(ranges, ranges[1:]):
        if one[0] + one[1] > next_one[0]:
            return one[2:], next_one[2:]
    return None


class AdamWTensors:
    """Parameters and optimiser states that are stepped together: checked once, then stepped with new gradients.

    ``params``: dense CUDA tensors of one type (float32, float16, bfloat16) on one device; ``exp_avgs`` and ``exp_avg_sqs``: the
    moments, float32 of the same sizes, or float8_e4m3fn codes with ``exp_avg_scales`` and ``exp_avg_sq_scales`` (float32, one for
    every 256 values).  ``masters``: float32 copies of 16-bit parameters.  The tensors share no memory, with each other or with the gradients;
    they are updated in place where they were when this was made; a step with a parameter that was given other memory since is refused."""

    def __init__(self, params: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor],
                 exp_avg_scales: Optional[Sequence[torch.Tensor]] = None, exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
                 masters: Optional[Sequence[torch.Tensor]] = None):
        self.params = list(params)
        if not self.params:
            raise ValueError("no tensors to step")
        self.dtype, self.device = self.params[0].dtype, self.params[0].device
        if self.dtype not in _TYPES:
            raise TypeError(f"params must be float32, float16 or bfloat16, got {self.dtype}")
        if self.device.type != "cuda":
            raise ValueError(f"params must be on a CUDA device, got {self.device}")
        eight = len(exp_avgs) > 0 and exp_avgs[0].dtype == _CODES
        self.state_bits = 8 if eight else 32
        if eight != (exp_avg_scales is not None) or eight != (exp_avg_sq_scales is not None):
            raise ValueError("exp_avg_scales and exp_avg_sq_scales go with float8_e4m3fn states, and with no others")
        if masters is not None and self.dtype == torch.float32:
            raise ValueError("float32 parameters have no masters")
        self._index = self.device.index
        state = _CODES if eight else torch.float32
        sizes = [p.numel() for p in self.params]
        self._single = [k for k, n in enumerate(sizes) if n == 1]  # a view with its sign to come is contiguous only there
        blocks = [state_blocks(n) for n in sizes]
        self._tensors = {"params": (self.params, self.dtype, sizes), "exp_avgs": (list(exp_avgs), state, sizes),
                         "exp_avg_sqs": (list(exp_avg_sqs), state, sizes)}
        if eight:
            self._tensors["exp_avg_scales"] = (list(exp_avg_scales), torch.float32, blocks)
            self._tensors["exp_avg_sq_scales"] = (list(exp_avg_sq_scales), torch.float32, blocks)
        if masters is not None:
            self._tensors["masters"] = (list(masters), torch.float32, sizes)
        self.sizes = sizes
        table = np.zeros((len(sizes), _WORDS), dtype=np.int64)
        ranges = []
        for column, name in ((0, "params"), (2, "exp_avgs"), (3, "exp_avg_sqs"), (4, "exp_avg_scales"), (5, "exp_avg_sq_scales"), (6, "masters")):
            if name not in self._tensors:
                continue
            tensors, dtype, want = self._tensors[name]
            if len(tensors) != len(sizes):
                raise ValueError(f"{len(tensors)} {name} for {len(sizes)} params")
            if not self._as_wanted(tensors, dtype, want):
                for k, (t, n) in enumerate(zip(tensors, want)):
                    if not isinstance(t, torch.Tensor):
                        raise TypeError(f"{name}[{k}] must be a tensor, got {type(t).__name__}")
                    if not self._as_wanted([t], dtype, [n]):
                        raise ValueError(f"{name}[{k}] must be {n} contiguous values of {dtype} on {self.device}, got {tuple(t.shape)} of {t.dtype} "
                                         f"on {t.device}")
            addresses = list(map(_address, tensors))
            table[:, column] = addresses
            width = tensors[0].element_size()
            ranges += [(at, n * width, name, k) for k, (at, n) in enumerate(zip(addresses, want)) if n]
        shared = _shared(ranges)
        if shared:
            (first, i), (second, k) = shared
            raise ValueError(f"{second}[{k}] lies in the memory of another tensor of the step, {first}[{i}]")
        table[:, _N] = sizes
        table[:, _N + 1] = np.arange(len(sizes))
        self.starts = table[:, 0].tolist()  # addresses of the parameters
        self._words, self._bytes = C.c_int64 * table.size, table.tobytes()
        written = [t for tensors, _, _ in self._tensors.values() for t in tensors]
        # what autograd counts the writes of, so that a backward pass over what was computed from old values is an error: views share the
        # count of the tensor that they are views of
        self._written = list({id(t): t for t in (t if t._base is None else t._base for t in written)}.values())
        # the memory that the table names stays, whatever becomes of the tensors
        self._kept = [t.detach() for t in written]
        self._borrowed = False
        self.versions: Optional[List[int]] = None  # of the parameters, after the last step

    def _as_wanted(self, tensors, dtype, sizes) -> bool:
        try:
            return (list(map(_numel, tensors)) == sizes and set(map(_dtype_of, tensors)) == {dtype} and set(map(_get_device, tensors)) == {self._index}
                    and set(map(_layout_of, tensors)) == {torch.strided} and all(map(_is_contiguous, tensors)) and not any(map(_is_neg, tensors)))
        except (AttributeError, TypeError, RuntimeError):
            return False

    def _borrow_params(self):
        """From here on the parameters' memory is theirs alone: the owner asks ``_here`` before every step."""
        self._kept = self._kept[len(self.params):]
        self._borrowed = True

    def _here(self) -> bool:
        """Whether the parameters lie where and as they did when they were checked (their type is the owner's to watch)."""
        return (list(map(_address, self.params)) == self.starts and list(map(_numel, self.params)) == self.sizes
                and all(map(_is_contiguous, self.params)))

    def step(self, grads: Sequence[Optional[torch.Tensor]], *, step: int, lr: float, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
             weight_decay: float = 1e-2, seed: int = 0):
        """One step with the gradients ``grads`` (of one type, float32 or 16 bits; None leaves its tensor as it is); ``step``
        counts from 1.  ``seed``: of the random rounding of 8-bit states."""
        table, kind, kept = self._filled(grads)
        if kind is None:
            return
        index = self._index
        with _on(index):
            if not self._borrowed:  # (the owner has asked before it made the states)
                _no_capture()
            check(lib.gnr_adamw_step(table, len(self.sizes), _TYPES[self.dtype], _TYPES[kind], self.state_bits, step, lr, betas[0], betas[1],
                                     eps, weight_decay, seed & 0xFFFFFFFF, _raw_stream(index)), "gnr_adamw_step")
        increment_version(self._written if kept is grads else self._written_with(grads))

    def step_clocked(self, grads: Sequence[Optional[torch.Tensor]], clock: "AdamWClock"):
        """The step that ``clock`` stands at, for capture into a CUDA graph: replays read the gradients where they lay then.  A clock
        that has done no step yet (``advance`` comes first) changes nothing."""
        if clock.device != self.device:
            raise ValueError(f"clock on {clock.device}, parameters on {self.device}")
        table, kind, kept = self._filled(grads)
        if kind is None:
            return
        index = self._index
        with _on(index):
            check(lib.gnr_adamw_step_clocked(table, len(self.sizes), _TYPES[self.dtype], _TYPES[kind], self.state_bits, clock.memory.data_ptr(),
                                             _raw_stream(index)), "gnr_adamw_step_clocked")
        increment_version(self._written if kept is grads else self._written_with(grads))

    def _written_with(self, grads):
        return [t for tensors, _, _ in self._tensors.values() for t, g in zip(tensors, grads) if g is not None]

    def _filled(self, grads):
        """(a copy of the table with the gradients in it, their type or None where there are none, what has to stay until the launch)"""
        if len(grads) != len(self.sizes):
            raise ValueError(f"{len(grads)} gradients for {len(self.sizes)} tensors")
        if not self._borrowed and list(map(_address, self.params)) != self.starts:
            raise ValueError("a parameter has been given other memory since it was checked")
        table = self._words.from_buffer_copy(self._bytes)
        try:  # all there and as they should be
            kinds = {g.dtype for g in grads}
            if (list(map(_numel, grads)) == self.sizes and set(map(_get_device, grads)) == {self._index} and len(kinds) == 1
                    and all(map(_is_contiguous, grads)) and kinds <= _TYPES.keys() and not any([grads[k].is_neg() for k in self._single])):
                if len(grads) > 32:
                    np.frombuffer(table, dtype=np.int64)[_GRAD::_WORDS] = list(map(_address, grads))
                else:
                    for at, address in zip(range(_GRAD, len(table), _WORDS), map(_address, grads)):
                        table[at] = address
                return table, kinds.pop(), grads
        except (AttributeError, TypeError, RuntimeError):
            pass
        kept, kind = self._grads(grads, table)
        return table, kind, kept

    def _grads(self, grads, table):
        """Gradients one by one: some missing, not contiguous or wrong.  Returns what has to stay until the launch, and their type."""
        kept, kind = [], None
        for k, (g, n) in enumerate(zip(grads, self.sizes)):
            if g is None:
                table[k * _WORDS + _N] = 0
                continue
            if g.get_device() != self.device.index or g.layout is not torch.strided or g.numel() != n:
                raise ValueError(f"gradient {k} must be {n} dense values on {self.device}, got {tuple(g.shape)} on {g.device}")
            if kind is None:
                kind = g.dtype
            if g.dtype is not kind or kind not in _TYPES:
                raise TypeError(f"gradients must be of one type, float32, float16 or bfloat16: got {g.dtype} at {k}, {kind} before")
            g = g.contiguous().resolve_neg()
            kept.append(g)
            table[k * _WORDS + _GRAD] = g.data_ptr()
        return kept, kind


class AdamWClock:
    """Rates and count of steps on the device, for steps that are captured into a CUDA graph: capture ``advance()`` and one
    ``AdamWTensors.step_clocked(grads, clock)`` for every set of tensors; every replay is then the next step.  ``set`` changes rates (and the
    count) between replays, in the order of the stream it is called on."""

    def __init__(self, device, *, lr: float, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, step: int = 0,
                 seed: int = 0):
        self.memory = torch.zeros(_lib.ADAMW_CLOCK_BYTES, dtype=torch.uint8, device=device)
        self.device = self.memory.device
        if self.device.type != "cuda":
            raise ValueError(f"the clock must be on a CUDA device, got {self.device}")
        self._rates = {"lr": lr, "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay}
        self._seed = seed & 0xFFFFFFFF
        self.set(step=step)

    def set(self, *, step: Optional[int] = None, **rates):
        """New ``lr``, ``betas``, ``eps`` or ``weight_decay``; ``step``: the steps done so far (None: as many as there are)."""
        if rates.keys() - self._rates.keys():
            raise TypeError(f"a clock has {', '.join(self._rates)}, got {', '.join(rates)}")
        if step is not None and step < 0:
            raise ValueError(f"step {step}")
        new = {**self._rates, **rates}
        with _on(self.device.index):
            check(lib.gnr_adamw_clock_set(self.memory.data_ptr(), -1 if step is None else step, new["lr"], new["betas"][0], new["betas"][1], new["eps"],
                                          new["weight_decay"], self._seed, _raw_stream(self.device.index)), "gnr_adamw_clock_set")
        self._rates = new

    def advance(self):
        """One step further; once before the ``step_clocked`` calls of a step, which without it would be the step before once more."""
        with _on(self.device.index):
            check(lib.gnr_adamw_clock_advance(self.memory.data_ptr(), _raw_stream(self.device.index)), "gnr_adamw_clock_advance")


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step: int, lr: float, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, exp_avg_scales=None, exp_avg_sq_scales=None, masters=None, seed: int = 0):
    """One AdamW step over lists of tensors, in place (see ``AdamWTensors``, which checks the lists once for many steps)."""
    AdamWTensors(params, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, masters).step(
        grads, step=step, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, seed=seed)


def _check_group(group: dict):
    """Refuses what torch's optimisers have in their groups and a step here would not do."""
    for name in ("maximize", "amsgrad", "differentiable"):
        if group.get(name):
            raise ValueError(f"{name} is not offered")
    if group.get("decoupled_weight_decay") is False and group.get("weight_decay", 0):
        raise ValueError("coupled weight decay (decoupled_weight_decay=False, as of torch.optim.Adam) is not offered")


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` over dense CUDA parameters: groups, learning rate schedulers and ``state_dict`` as there.  Groups that
    ask for ``maximize``, ``amsgrad``, ``differentiable`` or coupled weight decay are refused.

    ``state_bits``: 32 or 8.  ``master_weights``: 16-bit parameters keep an fp32 copy in the state; what others write to a parameter
    between steps (weights that are loaded, not writes through ``.data``, which nothing counts) is taken over into the copy.  ``seed``: of
    the random rounding of 8-bit states."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32, master_weights: bool = True, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not lr >= 0 or not eps >= 1e-30 or not weight_decay >= 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError(f"lr {lr}, betas {betas}, eps {eps} (at least 1e-30), weight_decay {weight_decay}")
        self.state_bits, self.master_weights, self.seed = state_bits, master_weights, seed
        self._sets: dict = {}  # (group, device, type) -> (parameters, their states, these by name, AdamWTensors)
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay})

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):  # (what is not is refused by torch)
            _check_group({**self.defaults, **param_group})
        super().add_param_group(param_group)
        self._sets.clear()

    def load_state_dict(self, state_dict):
        """Restores what ``state_dict`` returned, every state in its own type (torch would give it the parameter's).  The state of a
        ``torch.optim.AdamW`` (or of an ``Adam`` without weight decay) with fp32 moments is taken as well."""
        def check(_, loaded):  # the last hook before and the first behind torch's own work: on what the user's hooks made of the dict
            for group in loaded["param_groups"]:
                _check_group(group)
            taken.append(loaded)

        def keep_types(_):
            self._sets.clear()
            saved = taken[0]["state"]
            ids = [i for group in taken[0]["param_groups"] for i in group["params"]]
            for i, p in zip(ids, [p for group in self.param_groups for p in group["params"]]):
                if i in saved:
                    self.state[p] = {k: int(v) if k == "step" else v.detach().to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                     for k, v in saved[i].items()}

        taken: list = []
        hooks = self.register_load_state_dict_pre_hook(check), self.register_load_state_dict_post_hook(keep_types, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "master_weights": self.master_weights, "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._sets = {}

    def _state_of(self, p: torch.Tensor) -> dict:
        """The state of ``p``; a new one, not yet entered, where it has none or a part is missing."""
        s = self.state.get(p)
        fresh = not s
        copied = self.master_weights and p.dtype != torch.float32 and (fresh or "master" not in s)
        if not fresh and not copied:
            return s
        s = dict(s or {})
        if fresh:
            s["step"] = 0
            kind = _CODES if self.state_bits == 8 else torch.float32
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.zeros(p.shape, dtype=torch.float32 if kind is torch.float32 else torch.uint8, device=p.device)
                if self.state_bits == 8:
                    s[name] = s[name].view(kind)
                    s[name + "_scale"] = torch.zeros(state_blocks(p.numel()), device=p.device)
        if copied:
            s["master"] = p.detach().float()
        return s

    @staticmethod
    def _kept(states, parts) -> bool:
        try:
            return all([all(map(operator.is_, map(operator.itemgetter(name), states), kept)) for name, kept in parts.items()])
        except KeyError:
            return False

    def _take_over(self, made: AdamWTensors, old):
        """Brings the fp32 copies of parameters that others have written since the last step (weights that were loaded, say) to what they
        hold now: a value that is still the copy's rounded image keeps its copy."""
        now = _versions(made.params)
        if now is None or (old is made and now == made.versions):
            return
        known = {} if old is None or old.versions is None else {id(p): at for p, *at in zip(old.params, old.starts, old.versions)}
        for p, at, version, master in zip(made.params, made.starts, now, made._tensors["masters"][0]):
            if known.get(id(p)) != [at, version]:
                master.copy_(torch.where(p == master.to(p.dtype), master, p.float()))

    def _tensors(self, key, params) -> Tuple[list, AdamWTensors]:
        """States of ``params`` and the checked set of them, made again where a parameter or state has been replaced."""
        old = self._sets.get(key)
        if old is not None:
            old_params, states, parts, made = old  # parts: of every state, by name
            if (len(old_params) == len(params) and all(map(operator.is_, old_params, params)) and made._here()
                    and all(map(operator.is_, map(self.state.get, params), states))
                    and self._kept(states, parts)):
                if "master" in parts:
                    self._take_over(made, made)
                return states, made
        states = [self._state_of(p) for p in params]
        parts = {n: [s.get(n) for s in states] for n in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master") if n in states[0]}
        made = AdamWTensors(params, parts["exp_avg"], parts["exp_avg_sq"], parts.get("exp_avg_scale"), parts.get("exp_avg_sq_scale"),
                            parts.get("master"))
        made._borrow_params()
        for p, state in zip(params, states):  # (only now: what is refused leaves no state behind)
            self.state[p] = state
        if "master" in parts:
            self._take_over(made, old[3] if old is not None else None)
        self._sets[key] = (params, states, parts, made)
        return states, made

    @torch.no_grad()
    def step(self, closure=None):
        if closure is not None and torch.cuda.is_initialized():
            _no_capture()
        for group in self.param_groups:
            _check_group(group)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        todo = []  # every set of every group: states are made, and refusals raised, before anything is stepped
        for number, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if len(set(map(_dtype_of, params))) == len(set(map(_get_device, params))) == 1:
                sets = {(number, params[0].device, params[0].dtype): params}
            else:
                sets = {}
                for p in params:
                    sets.setdefault((number, p.device, p.dtype), []).append(p)
            for k, (key, params) in enumerate(sets.items()):
                if key[1].type == "cuda":
                    with _on(key[1].index):
                        _no_capture()
                todo.append((number, group, k, params, *self._tensors(key, params)))
        if len(self._sets) > len(todo):  # sets of parameters that have moved, to another device say, are not looked up again
            used = {id(tensors) for *_, tensors in todo}
            self._sets = {key: kept for key, kept in self._sets.items() if id(kept[3]) in used or kept[3]._here()}
        for number, group, k, params, states, tensors in todo:
            counts = set(map(_step_of, states))
            for t in sorted(counts):  # one, unless a parameter had no gradient in some steps
                grads = [p.grad for p in params] if len(counts) == 1 else [p.grad if s["step"] == t else None for p, s in zip(params, states)]
                tensors.step(grads, step=int(t) + 1, lr=float(group["lr"]), betas=group["betas"], eps=group["eps"],
                             weight_decay=group["weight_decay"], seed=self.seed + 0x3C6EF372 * (2 * number + 1) + k)
            for s in states:
                s["step"] += 1
        for *_, tensors in todo:  # (behind all steps: parameters may share a count of writes)
            if "masters" in tensors._tensors:
                tensors.versions = _versions(tensors.params)
        return loss
