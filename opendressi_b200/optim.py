"""Optimisation of many tensors at once: ``AdamW`` and ``grad_norm``.

The counterpart, for a torch program, of the Adam inside the fused plans
(which steps one flat parameter): one kernel launch steps the vertices,
textures, material maps and network weights of a scene. The step runs on the
parameters' device and its current stream, reads nothing back and keeps its
counters on the device, so it can be captured in a CUDA graph. It is no
operator of a torch graph: make_fx and torch.jit.trace refuse it.
"""

from __future__ import annotations

import copy
import math

import torch

from . import _native as N
from .ops import binding, grad_norm

__all__ = ["AdamW", "grad_norm"]

_BLOCK = 256  # values of 8-bit state that share a scale
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _order(t) -> list:
    """The strides of a tensor, where they count."""
    return [s for s, n in zip(t.stride(), t.shape) if n != 1 and t.numel()]


class _Pack:
    """The state of one parameter group: a flat tensor of each kind, every
    parameter at a multiple of 256 values of it."""

    def __init__(self, params, state_bits: int, index: int):
        self.params = params
        self.flat = {}
        self.views = []
        self.rows = None
        if not params:
            return
        first = [0]
        for p in params:
            first.append(first[-1] - (-p.numel() // _BLOCK))
        total = first[-1]
        dev = params[0].device
        wide = dict(dtype=torch.float32, device=dev)
        code = dict(dtype=torch.float8_e4m3fn, device=dev)
        flat = {"step": torch.zeros(len(params), dtype=torch.int32,
                                    device=dev)}
        if state_bits == 32:
            kinds = ("exp_avg", "exp_avg_sq")
            for k in kinds:
                flat[k] = torch.zeros(total * _BLOCK, **wide)
        else:
            kinds = ("exp_avg", "root_avg_sq")
            for k in kinds:
                flat[k] = torch.zeros(total * _BLOCK, **code)
                flat[k + "_scale"] = torch.zeros(total, **wide)
        for i, p in enumerate(params):
            view = {}
            for k, t in flat.items():
                if k == "step":
                    view[k] = t[i]
                elif k.endswith("_scale"):
                    view[k] = t[first[i]:first[i + 1]]
                else:  # in the parameter's own order of memory
                    view[k] = t.as_strided(p.shape, p.stride(),
                                           first[i] * _BLOCK)
            self.views.append(view)
        self.flat = flat
        self.rows = binding().Pack(
            params, first[:-1], flat["step"], *(flat[k] for k in kinds),
            *(flat.get(k + "_scale") for k in kinds), index, state_bits)


class AdamW(torch.optim.Optimizer):
    """AdamW (Adam with decoupled weight decay) as one launch for all tensors
    of a parameter group and type.

        g *= min(1, max_norm / (norm of all gradients + 1e-6))   with max_norm
        m = m b1 + g (1 - b1);  v = v b2 + g g (1 - b2);  t = t + 1
        p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
        p = clamp(p, *clamp)                                     with clamp

    Parameters are float32, float16 or bfloat16 CUDA tensors of any dense
    layout, on one device; the arithmetic is in 32 bits. ``t`` counts the
    steps in which a tensor had a gradient, on the device. lr, betas, eps,
    weight_decay and clamp can differ between parameter groups; lr can be a
    0-dim float32 CUDA tensor, which a captured step reads anew.

    state_bits = 8 keeps both moments as e4m3 codes, a quarter of the memory,
    with a float32 scale for each 256 values; they are rounded up or down at
    random (repeatably: from `seed`, the step and the place) with the right
    mean, since a moving average moves too little in a step to survive
    rounding to the nearest code. The second moment is kept as its root. What
    is not finite is kept as NaN and does not touch its neighbours.

    A gradient that is not finite makes its parameter not finite, or with
    max_norm all of them, as the formula says.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32,
                 max_norm: float | None = None, clamp=None, seed: int = 0):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if max_norm is not None and not (0.0 < max_norm < math.inf):
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        self.state_bits = state_bits
        self.max_norm = None if max_norm is None else float(max_norm)
        self.seed = int(seed) & 0xFFFFFFFF
        self._packs: list[_Pack] = []
        self._device = None
        self._ticket = None
        #: with max_norm: the norm of the last step's gradients, before
        #: clipping (a 0-dim CUDA tensor that each step overwrites)
        self.last_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps,
                                      weight_decay=weight_decay, clamp=clamp))

    # ------------------------------------------------------------- groups

    @staticmethod
    def _check_options(g) -> None:
        lr = g["lr"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1:
                raise ValueError("lr must be a number or hold one")
            if lr.is_cuda and lr.dtype != torch.float32:
                raise ValueError("a CUDA lr must be float32")
            lr = 0.0 if lr.is_cuda else float(lr)  # no read from the device
        if not 0.0 <= lr < math.inf:
            raise ValueError(f"lr must be finite and not negative, got {lr}")
        if len(g["betas"]) != 2 or not all(0.0 <= b < 1.0
                                           for b in g["betas"]):
            raise ValueError(f"betas must be two of [0, 1), got {g['betas']}")
        for k in ("eps", "weight_decay"):
            if not 0.0 <= g[k] < math.inf:
                raise ValueError(f"{k} must be finite and not negative, got "
                                 f"{g[k]}")
        if g["clamp"] is not None:
            lo, hi = g["clamp"]
            if not lo <= hi:
                raise ValueError(f"clamp must be (low, high), got "
                                 f"{g['clamp']}")

    def add_param_group(self, param_group) -> None:
        group = dict(param_group)
        params = group["params"]
        params = [params] if isinstance(params, torch.Tensor) else list(params)
        group["params"] = params
        merged = {**self.defaults, **group}
        self._check_options(merged)
        seen = [p for g in self.param_groups for p in g["params"]]
        dev = self._device
        for p in params:
            if isinstance(p, tuple):
                raise TypeError("AdamW takes parameters without names")
            if not isinstance(p, torch.Tensor) or not p.is_cuda:
                raise N.DressiError(N.ERR_INVALID,
                                    "parameters must be CUDA tensors")
            if p.dtype not in _DTYPES:
                raise N.DressiError(N.ERR_INVALID, "parameters must be "
                                    "float32, float16 or bfloat16, got "
                                    f"{p.dtype}")
            dev = dev or p.device
            if p.device != dev:
                raise N.DressiError(N.ERR_INVALID,
                                    "parameters on several devices")
            if p.layout != torch.strided or not binding().dense(p):
                raise N.DressiError(N.ERR_INVALID, "a parameter's memory must "
                                    "be dense and not overlap itself")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() *
                        p.element_size()) for p in seen + params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters share memory")
        super().add_param_group(group)
        params = self.param_groups[-1]["params"]
        try:
            if dev is not None and self._device is None:
                self._ticket = torch.zeros(1, dtype=torch.int32, device=dev)
                if self.max_norm is not None:
                    self.last_norm = torch.zeros((), dtype=torch.float32,
                                                 device=dev)
            pack = _Pack(params, self.state_bits,
                         sum(len(q.params) for q in self._packs))
        except BaseException:  # groups and packs go together
            self.param_groups.pop()
            raise
        self._device = dev
        self._packs.append(pack)
        for p, view in zip(params, pack.views):
            self.state[p] = view

    def packed_state(self, group: int = 0) -> dict:
        """The state of a parameter group as a few flat tensors (the tensors
        of ``state`` are views of them): "step" [parameters], and "exp_avg",
        "exp_avg_sq", or with 8 bits "exp_avg", "exp_avg_scale",
        "root_avg_sq" and "root_avg_sq_scale" (value = code * scale), each
        parameter from a multiple of 256 values on. To be changed in place
        only."""
        return dict(self._packs[group].flat)

    # --------------------------------------------------------------- step

    def _numbers(self, group) -> tuple:
        """What a step takes from a group, as the binding wants it."""
        self._check_options(group)
        lr, lr_device = group["lr"], None
        if isinstance(lr, torch.Tensor):
            if lr.is_cuda and lr.device != self._device:
                raise N.DressiError(N.ERR_INVALID, "lr is on another device "
                                    "than the parameters")
            lr, lr_device = (0.0, lr) if lr.is_cuda else (float(lr), None)
        lo, hi = group["clamp"] or (-math.inf, math.inf)
        return (lr, lr_device, *group["betas"], group["eps"],
                group["weight_decay"], lo, hi)

    @torch.no_grad()
    def step(self, closure=None):
        """One step of every parameter that has a gradient. Returns the
        closure's loss, if there is a closure."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        packs, numbers = [], []
        for pack, group in zip(self._packs, self.param_groups):
            if pack.rows is not None:
                packs.append(pack.rows)
                numbers.append(self._numbers(group))
        if packs:
            binding().adamw_step(packs, numbers, self.max_norm or 0.0,
                                 self.last_norm if self.max_norm else None,
                                 self.seed, self._ticket)
        return loss

    # ---------------------------------------------------------- save / load

    def state_dict(self) -> dict:
        """torch's state_dict with this optimizer's own options under
        "adamw"."""
        sd = super().state_dict()
        sd["adamw"] = {"state_bits": self.state_bits, "seed": self.seed,
                       "max_norm": self.max_norm}
        return sd

    @staticmethod
    def _loaded_options(group, saved) -> dict:
        """A group's options with copies of the saved ones in their place."""
        options = {k: v.detach().clone() if isinstance(v, torch.Tensor)
                   else copy.deepcopy(v)
                   for k, v in saved.items() if k != "params"}
        return {**group, **options}

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """Copies a state_dict() of an optimizer over like parameters into
        this one's own tensors (a learning rate that is a tensor here among
        them, so that a captured step reads the loaded one). 8-bit moments
        need parameters in the same order of memory: their scales go by it."""
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            if changed is not None:
                state_dict = changed
        own = state_dict.get("adamw", {})
        if own.get("state_bits") != self.state_bits:
            raise ValueError("the state was kept in "
                             f"{own.get('state_bits')} bits, this optimizer "
                             f"keeps it in {self.state_bits}")
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != \
                [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the state has other parameter groups")
        pairs = []
        for old, pack in zip(groups, self._packs):
            for k, view in zip(old["params"], pack.views):
                got = state_dict["state"][k]
                for kind, t in view.items():
                    if kind not in got or got[kind].shape != t.shape or \
                            got[kind].dtype != t.dtype:
                        raise ValueError(f"the state's {kind} is not like "
                                         "this optimizer's")
                    if t.dtype not in (torch.int32, torch.float32) and \
                            _order(got[kind]) != _order(t):
                        raise ValueError("the state's codes have scales of "
                                         "another order of memory")
                    pairs.append((t, got[kind]))
        options = [self._loaded_options(g, old)
                   for g, old in zip(self.param_groups, groups)]
        for new in options:  # all of it is right before any is changed
            self._check_options({**new, "lr": float(new["lr"])})
        for group, new in zip(self.param_groups, options):
            lr = group["lr"]
            if isinstance(lr, torch.Tensor):
                lr.copy_(torch.as_tensor(new["lr"]).reshape(lr.shape))
                new["lr"] = lr
            elif isinstance(new["lr"], torch.Tensor) and new["lr"].is_cuda:
                new["lr"] = new["lr"].to(self._device, torch.float32)
            group.update(new)
        for t, got in pairs:
            t.copy_(got)
        self.seed = int(own.get("seed", self.seed))
        self.max_norm = own.get("max_norm", self.max_norm)
        if self.max_norm is not None and self.last_norm is None and \
                self._device is not None:
            self.last_norm = torch.zeros((), dtype=torch.float32,
                                         device=self._device)
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def __getstate__(self):
        raise TypeError("an AdamW holds device state: save its state_dict()")
