"""Optimisation of many tensors at once: ``AdamW`` and ``grad_norm``.

The counterpart, for a torch program, of the Adam inside the fused plans
(which steps one flat parameter): one kernel launch steps the vertices,
textures, material maps and network weights of a scene. The step runs on the
parameters' device and its current stream, reads nothing back and keeps its
counters on the device, so it can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes as C
import math
from array import array

import torch

from . import _native as N
from .ops import _DTYPES, _On, _stream_of, grad_norm

__all__ = ["AdamW", "grad_norm"]

_BLOCK = 256  # values of 8-bit state that share a scale


def _dense(t: torch.Tensor) -> bool:
    """Whether t's values fill its extent in memory, in some order, once."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size != 1:
            if stride != want:
                return False
            want *= size
    return True


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    return (a.is_contiguous() and b.is_contiguous()) or \
        a.stride() == b.stride()


class _Pack:
    """The state of one parameter group: a flat tensor of each kind, every
    parameter at a multiple of 256 values of it."""

    def __init__(self, params, state_bits: int, index: int):
        dev = params[0].device if params else None
        self.params = params
        self.numel = [p.numel() for p in params]
        self.dtype = [p.dtype for p in params]
        self.stride = [p.stride() for p in params]
        blocks = [-(-n // _BLOCK) for n in self.numel]
        first = [0]
        for b in blocks:
            first.append(first[-1] + b)
        total = first[-1]
        self.flat = {}
        if params:
            wide = dict(dtype=torch.float32, device=dev)
            code = dict(dtype=torch.float8_e4m3fn, device=dev)
            self.flat["step"] = torch.zeros(len(params), dtype=torch.int32,
                                            device=dev)
            if state_bits == 32:
                self.flat["exp_avg"] = torch.zeros(total * _BLOCK, **wide)
                self.flat["exp_avg_sq"] = torch.zeros(total * _BLOCK, **wide)
            else:
                for k in ("exp_avg", "root_avg_sq"):
                    self.flat[k] = torch.zeros(total * _BLOCK, **code)
                    self.flat[k + "_scale"] = torch.zeros(total, **wide)
        self.views = []
        for i, p in enumerate(params):
            view = {}
            for k, flat in self.flat.items():
                if k == "step":
                    view[k] = flat[i]
                elif k.endswith("_scale"):
                    view[k] = flat[first[i]:first[i + 1]]
                else:  # in the parameter's own order of memory
                    view[k] = flat.as_strided(p.shape, p.stride(),
                                              first[i] * _BLOCK)
            self.views.append(view)
        second = "exp_avg_sq" if state_bits == 32 else "root_avg_sq"
        size = 4 if state_bits == 32 else 1

        def at(kind, step):
            if kind not in self.flat:
                return [0] * len(params)
            base = self.flat[kind].data_ptr()
            return [base + f * step for f in first[:-1]]

        steps = self.flat["step"].data_ptr() if params else 0
        # what each parameter's state is called by in the C call
        self.rows = list(zip(
            self.numel, at("exp_avg", _BLOCK * size),
            at(second, _BLOCK * size), at("exp_avg_scale", 4),
            at(second + "_scale", 4),
            [steps + 4 * i for i in range(len(params))],
            range(index, index + len(params))))
        self.whole = self.columns(range(len(params)))

    def columns(self, which):
        """The C call's host arrays for the parameters `which`."""
        cols = list(zip(*(self.rows[i] for i in which))) or [()] * 7
        return [array("Q", c) for c in cols[:6]] + [array("I", cols[6])]


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
        elif not 0.0 <= lr < math.inf:
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
            if not _dense(p):
                raise N.DressiError(N.ERR_INVALID, "a parameter's memory must "
                                    "be dense and not overlap itself")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() *
                        p.element_size()) for p in seen + params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters share memory")
        super().add_param_group(group)
        params = self.param_groups[-1]["params"]
        if dev is not None and self._device is None:
            self._device = dev
            self._ticket = torch.zeros(1, dtype=torch.int32, device=dev)
            if self.max_norm is not None:
                self.last_norm = torch.zeros((), dtype=torch.float32,
                                             device=dev)
        pack = _Pack(params, self.state_bits,
                     sum(len(q.params) for q in self._packs))
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

    def _gradients(self, pack: _Pack) -> list:
        """Each parameter's gradient in the parameter's order of memory."""
        grads = []
        for p, n, dtype, stride in zip(pack.params, pack.numel, pack.dtype,
                                       pack.stride):
            g = p.grad
            if p.dtype is not dtype or p.numel() != n or \
                    p.stride() != stride or p.device != self._device:
                raise N.DressiError(N.ERR_INVALID, "a parameter changed its "
                                    "type, shape or device; make a new "
                                    "optimizer")
            if g is not None:
                if g.is_sparse or g.dtype is not dtype or \
                        g.shape != p.shape or g.device != self._device:
                    raise N.DressiError(N.ERR_INVALID, "a gradient must be "
                                        "dense and like its parameter")
                if not _same_order(g, p):
                    g = torch.empty_like(p).copy_(g)
            grads.append(g)
        return grads

    @torch.no_grad()
    def step(self, closure=None):
        """One step of every parameter that has a gradient. Returns the
        closure's loss, if there is a closure."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._device is None:
            return loss
        grads = [self._gradients(pack) for pack in self._packs]
        with _On(self._ticket):
            if self.max_norm is not None:
                grad_norm([g for gs in grads for g in gs if g is not None],
                          out=self.last_norm)
            for group, pack, gs in zip(self.param_groups, self._packs, grads):
                self._check_options(group)
                for dtype in dict.fromkeys(pack.dtype):
                    which = [i for i, g in enumerate(gs)
                             if g is not None and pack.dtype[i] is dtype]
                    if which:
                        self._launch(group, pack, gs, which, dtype)
        return loss

    def _launch(self, group, pack, grads, which, dtype) -> None:
        whole = len(which) == len(pack.params)
        numel, m, v, sm, sv, steps, index = (
            pack.whole if whole else pack.columns(which))
        ptrs = array("Q", [pack.params[i].data_ptr() for i in which])
        gptrs = array("Q", [grads[i].data_ptr() for i in which])
        lr = group["lr"]
        lr_device = None
        if isinstance(lr, torch.Tensor):
            if lr.is_cuda:
                if lr.device != self._device:
                    raise N.DressiError(N.ERR_INVALID, "lr is on another "
                                        "device than the parameters")
                lr, lr_device = 0.0, lr.data_ptr()
            else:
                lr = float(lr)
        lo, hi = group["clamp"] or (-math.inf, math.inf)
        clip = self.max_norm is not None
        d = N.AdamWDesc(
            C.sizeof(N.AdamWDesc), len(which), _DTYPES[dtype],
            self.state_bits, numel.buffer_info()[0], ptrs.buffer_info()[0],
            gptrs.buffer_info()[0], m.buffer_info()[0], v.buffer_info()[0],
            sm.buffer_info()[0], sv.buffer_info()[0], steps.buffer_info()[0],
            index.buffer_info()[0], lr, *group["betas"], group["eps"],
            group["weight_decay"], lr_device,
            self.max_norm if clip else 0.0,
            self.last_norm.data_ptr() if clip else None, lo, hi, self.seed,
            self._ticket.data_ptr())
        N.call("dressi_adamw_step", d, _stream_of(self._ticket))

    # ---------------------------------------------------------- save / load

    def state_dict(self) -> dict:
        """torch's state_dict with this optimizer's own options under
        "adamw"."""
        sd = super().state_dict()
        sd["adamw"] = {"state_bits": self.state_bits, "seed": self.seed,
                       "max_norm": self.max_norm}
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """Copies a state_dict() of an optimizer over like parameters into
        this one's own tensors."""
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
                    pairs.append((t, got[kind]))
        for group, old in zip(self.param_groups, groups):
            merged = {**group, **{k: v for k, v in old.items()
                                  if k != "params"}}
            self._check_options(merged)
            group.update(merged)
        for t, got in pairs:
            t.copy_(got)
        self.seed = int(own.get("seed", self.seed))
        self.max_norm = own.get("max_norm", self.max_norm)
        if self.max_norm is not None and self.last_norm is None and \
                self._device is not None:
            self.last_norm = torch.zeros((), dtype=torch.float32,
                                         device=self._device)

    def __getstate__(self):
        raise TypeError("an AdamW holds device state: save its state_dict()")
