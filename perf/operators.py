"""Cases that measure the learning operators: group normalisation with an
activation over channels-last images (forward, and forward + backward), the
AdamW step over many tensors (states in 32 or in 8 bits) and the norm over
many gradients. Each case runs in a plain form, elementary torch operations,
or -- where `own` is true -- through opendressi_b200's entry points."""

import math
import random

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_LR, _BETAS, _EPS, _DECAY = 1e-3, (0.9, 0.999), 1e-8, 1e-2
_SEED, _STEPS_DONE = 7, 100
_BLOCK = 256          # values that share a scale, and the padding of a tensor
_E4M3_MAX, _SCALE_FLOOR = 448.0, 2.0 ** -100
_M32 = 0xFFFFFFFF


def _norm(name, n, h, w, c, groups, dtype, act, train, affine=True):
    case = {"op": "group_norm", "n": n, "h": h, "w": w, "c": c,
            "groups": groups, "dtype": dtype, "act": act, "train": train,
            "affine": affine}
    return {"name": name, **case} if name else case


def _adamw(name, tensors, shortest, longest, lengths_seed, dtype, bits,
           max_norm):
    case = {"op": "adamw", "tensors": tensors, "shortest": shortest,
            "longest": longest, "lengths_seed": lengths_seed, "dtype": dtype,
            "bits": bits, "max_norm": max_norm}
    return {"name": name, **case} if name else case


def _grad_norm(name, tensors, shortest, longest, lengths_seed, dtype):
    case = {"op": "grad_norm", "tensors": tensors, "shortest": shortest,
            "longest": longest, "lengths_seed": lengths_seed, "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    texture = 2048 * 2048 * 3
    return [
        # the innermost level of a small decoder, one view: latency
        _norm("norm_tile_f32", 1, 16, 16, 32, 8, "f32", "silu", False),
        # eight rendered views in a decoder's middle level, as it is shown
        _norm("norm_views_bf16", 8, 256, 256, 64, 16, "bf16", "silu", False),
        # views of an odd resolution, channels per group that are no power of 2
        _norm("norm_odd_f16", 3, 127, 193, 96, 16, "f16", "relu", False),
        # training on small crops with few channels, odd in every extent
        _norm("norm_train_crops_f32", 3, 61, 47, 40, 10, "f32", "silu", True),
        # training on two full 1024^2 views at a decoder's widest level
        _norm("norm_train_views_bf16", 2, 1024, 1024, 64, 32, "bf16", "silu",
              True),
        # one icosphere's vertices (642 x 3) and a few tables: latency
        _adamw("adamw_mesh_f32", 4, 32, 1926, 1, "f32", 32, 0.0),
        # a decoder's weights and biases in bf16, clipped by their norm
        _adamw("adamw_decoder_bf16", 96, 16, 600000, 2, "bf16", 32, 1.0),
        # the textures of eight objects (2048^2 x 3)
        _adamw("adamw_textures_f32", 8, texture, texture, 3, "f32", 32, 0.0),
        # ragged decoder and scene tensors, states in 8 bits, clipped
        _adamw("adamw8_scene_f32", 150, 1, 600000, 4, "f32", 8, 1.0),
        # the textures of eight objects, states in 8 bits
        _adamw("adamw8_textures_f32", 8, texture, texture, 5, "f32", 8, 0.0),
        # the norm over a decoder's many small gradients
        _grad_norm("grad_norm_scene_bf16", 150, 1, 600000, 6, "bf16"),
        # the norm over the gradients of eight textures
        _grad_norm("grad_norm_textures_f32", 8, texture, texture, 7, "f32"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return min(high, max(low, int(round(math.exp(
        rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "adamw", "adamw",
                     "grad_norm"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "group_norm":
        most = 2 * 1024 * 1024 * 64 // (2 if dtype == "f32" else 1)
        groups = rng.choice([1, 2, 3, 4, 8, 16, 32])
        c = groups * _spread(rng, 1, max(1, min(64, 512 // groups)))
        n = _spread(rng, 1, 16)
        side = max(4, min(1024, math.isqrt(most // (n * c))))
        h, w = _spread(rng, 4, side), _spread(rng, 4, side)
        return _norm(None, n, h, w, c, groups, dtype,
                     rng.choice(["silu", "relu", "none"]),
                     rng.random() < 0.5, rng.random() < 0.85)
    tensors = _spread(rng, 1, 200)
    longest = _spread(rng, 16, min(2048 * 2048 * 3, 90000000 // tensors))
    shortest = min(longest, _spread(rng, 1, 4096))
    lengths_seed = rng.randrange(1 << 30)
    if op == "grad_norm":
        return _grad_norm(None, tensors, shortest, longest, lengths_seed,
                          dtype)
    return _adamw(None, tensors, shortest, longest, lengths_seed, dtype,
                  rng.choice([32, 8]), rng.choice([0.0, 1.0]))


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case):
    rng = random.Random(case["lengths_seed"])
    got = [_spread(rng, case["shortest"], case["longest"])
           for _ in range(case["tensors"])]
    got[0] = case["shortest"]
    got[-1] = case["longest"]
    return got


def _prepare_norm(case, seed):
    g = _generator(seed)
    dtype = _DTYPES[case["dtype"]]
    n, h, w, c = case["n"], case["h"], case["w"], case["c"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # features of what is seen, zeros where a view shows the background
    seen = (torch.rand((n, h, w, 1), generator=g, device="cuda") < 0.7)
    x = (normal(n, h, w, c) * (0.5 + normal(c).abs()) + normal(c)) * seen
    state = {"case": case, "x": x.to(dtype),
             "weight": 1.0 + 0.2 * normal(c) if case["affine"] else None,
             "bias": 0.2 * normal(c) if case["affine"] else None}
    if case["train"]:
        state["grad"] = (0.1 * normal(n, h, w, c)).to(dtype)
        state["x"].requires_grad_(True)
        if case["affine"]:
            state["weight"].requires_grad_(True)
            state["bias"].requires_grad_(True)
    return state


def _prepare_tensors(case, seed):
    """The tensors as views of one padded buffer each, so that all of a kind
    are returned as one."""
    g = _generator(seed)
    dtype = _DTYPES[case["dtype"]]
    lengths = _lengths(case)
    blocks = [-(-k // _BLOCK) for k in lengths]
    starts = [0]
    for b in blocks:
        starts.append(starts[-1] + b * _BLOCK)
    total = starts[-1]
    dev = torch.device("cuda")
    of_block = torch.repeat_interleave(
        torch.arange(len(lengths), device=dev),
        torch.tensor(blocks, device=dev))
    first = torch.tensor(starts[:-1], device=dev)[of_block]
    place = (torch.arange(len(of_block), device=dev) * _BLOCK - first)
    place = place[:, None] + torch.arange(_BLOCK, device=dev)
    real = place < torch.tensor(lengths, device=dev)[of_block][:, None]
    # texels and weights that no view reaches have no gradient
    reached = (torch.rand((len(of_block), 1), generator=g, device=dev) < 0.8)
    real_or_not = (real & reached).reshape(-1)

    def normal():
        return torch.randn(total, generator=g, device=dev)

    grad = (1e-2 * normal() * real_or_not).to(dtype)

    def split(flat):
        return [flat[s:s + k] for s, k in zip(starts, lengths)]

    state = {"case": case, "grad": grad, "grads": split(grad),
             "of_block": of_block, "place": place}
    if case["op"] == "grad_norm":
        return state
    param = (normal() * real.reshape(-1)).to(dtype)
    state["param"] = param
    state["step"] = torch.full((len(lengths),), _STEPS_DONE,
                               dtype=torch.int32, device=dev)
    if case["bits"] == 32:
        moments = {"exp_avg": 3e-3 * normal() * real_or_not,
                   "exp_avg_sq": 1e-4 * normal().square() * real_or_not}
    else:
        def code(x):
            return ((x * real_or_not).clamp(-_E4M3_MAX, _E4M3_MAX)
                    .to(torch.float8_e4m3fn))

        def scale(of):
            return of / _E4M3_MAX * torch.exp(0.3 * torch.randn(
                len(of_block), generator=g, device=dev))

        moments = {"exp_avg": code(100.0 * normal()),
                   "exp_avg_scale": scale(1e-2),
                   "root_avg_sq": code(20.0 + 100.0 * normal().abs()),
                   "root_avg_sq_scale": scale(4e-2)}
    state["moments"] = moments
    if own:
        from opendressi_b200 import optim
        params = [torch.nn.Parameter(p) for p in split(param)]
        for p, d in zip(params, state["grads"]):
            p.grad = d
        opt = optim.AdamW(params, lr=_LR, betas=_BETAS, eps=_EPS,
                          weight_decay=_DECAY, state_bits=case["bits"],
                          max_norm=case["max_norm"] or None, seed=_SEED)
        packed = opt.packed_state()
        packed["step"].copy_(state["step"])
        for k, v in moments.items():
            packed[k].copy_(v)
        state["optimizer"], state["packed"] = opt, packed
    return state


def prepare(case, seed):
    if case["op"] == "group_norm":
        return _prepare_norm(case, seed)
    return _prepare_tensors(case, seed)


# -------------------------------------------------------------- plain forms

def _sum32(t, dim):
    return t.sum(dim, keepdim=True)


def _plain_norm(state):
    case, eps = state["case"], 1e-5
    with torch.no_grad():
        n, c, groups = case["n"], case["c"], case["groups"]
        shape = (n, case["h"] * case["w"], groups, c // groups)
        x = state["x"].float().reshape(shape)
        count = shape[1] * shape[3]
        centred = x - _sum32(x, (1, 3)) / count
        rstd = torch.rsqrt(_sum32(centred * centred, (1, 3)) / count + eps)
        hat = centred * rstd
        z = hat
        if case["affine"]:
            weight = state["weight"].reshape(1, 1, groups, -1)
            z = hat * weight + state["bias"].reshape(1, 1, groups, -1)
        if case["act"] == "silu":
            s = 1.0 / (1.0 + torch.exp(-z))
            y, slope = z * s, s * (1.0 + z * (1.0 - s))
        elif case["act"] == "relu":
            y, slope = z.clamp(min=0.0), (z > 0).float()
        else:
            y, slope = z, None
        dtype = state["x"].dtype
        y = y.reshape(state["x"].shape).to(dtype)
        if not case["train"]:
            return y
        dz = state["grad"].float().reshape(shape)
        dz = dz if slope is None else dz * slope
        dhat = dz * weight if case["affine"] else dz
        mean_d = _sum32(dhat, (1, 3)) / count
        mean_dh = _sum32(dhat * hat, (1, 3)) / count
        dx = (rstd * (dhat - mean_d - hat * mean_dh)).reshape(y.shape)
        out = {"y": y, "dx": dx.to(dtype)}
        if case["affine"]:
            out["dweight"] = (dz * hat).sum((0, 1)).reshape(-1)
            out["dbias"] = dz.sum((0, 1)).reshape(-1)
        return out


def _mix(x):
    """Wang's integer hash of 32-bit values held in int64."""
    x = (x ^ 61) ^ (x >> 16)
    x = (x * 9) & _M32
    x = x ^ (x >> 4)
    x = (x * 0x27D4EB2D) & _M32
    return x ^ (x >> 15)


def _random_bits(state, step):
    """32 random bits for each value: what both roundings of the 8-bit states
    take as given, from the seed, the step, the tensor and the place in it."""
    step = _mix(step.to(torch.int64))
    index = torch.arange(step.numel(), device=step.device)
    key = _mix((_mix(step ^ _SEED) + index) & _M32)
    return _mix((key[state["of_block"]][:, None] + state["place"]) & _M32)


def _round_e4m3(a, bits16):
    """a in [0, 448] up or down to a neighbouring e4m3 value, up with the
    probability of its place between the two."""
    small = a < 2.0 ** -6
    a = torch.where(small, a + 2.0 ** -6, a)
    a = (a.view(torch.int32) + (bits16 << 4 | 8).to(torch.int32))
    a = (a & ~0xFFFFF).view(torch.float32)
    return torch.where(small, a - 2.0 ** -6, a).clamp(max=_E4M3_MAX)


def _plain_adamw(state):
    case, moments = state["case"], state["moments"]
    b1, b2 = _BETAS
    with torch.no_grad():
        step = state["step"].add_(1)
        t = step.double()
        size = (_LR / (1.0 - b1 ** t)).float()[state["of_block"]][:, None]
        root = torch.rsqrt(1.0 - b2 ** t).float()[state["of_block"]][:, None]
        g = state["grad"].float().reshape(-1, _BLOCK)
        if case["max_norm"]:
            norm = (g * g).sum(dtype=torch.float64).sqrt().float()
            g = g * (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        if case["bits"] == 32:
            m = moments["exp_avg"].reshape(-1, _BLOCK)
            v = moments["exp_avg_sq"].reshape(-1, _BLOCK)
        else:
            m = (moments["exp_avg"].float().reshape(-1, _BLOCK)
                 * moments["exp_avg_scale"][:, None])
            v = (moments["root_avg_sq"].float().reshape(-1, _BLOCK)
                 * moments["root_avg_sq_scale"][:, None])
            v = v * v
        m = m * b1 + g * (1.0 - b1)
        v = v * b2 + g * g * (1.0 - b2)
        p = state["param"].float().reshape(-1, _BLOCK) * (1.0 - _LR * _DECAY)
        p = p - size * (m / (v.sqrt() * root + _EPS))
        state["param"].copy_(p.reshape(-1))
        if case["bits"] == 32:
            moments["exp_avg"].copy_(m.reshape(-1))
            moments["exp_avg_sq"].copy_(v.reshape(-1))
        else:
            r = v.sqrt()
            bits = _random_bits(state, step)
            for kind, x, part in (("exp_avg", m, bits & 0xFFFF),
                                  ("root_avg_sq", r, bits >> 16)):
                top = x.abs().amax(1, keepdim=True).clamp(min=_SCALE_FLOOR)
                a = (x.abs() * (_E4M3_MAX / top)).clamp(max=_E4M3_MAX)
                a = _round_e4m3(a, part)
                if kind == "root_avg_sq":  # what is not 0 does not become 0
                    a = torch.where(x > 0, a.clamp(min=2.0 ** -9), a)
                a = torch.copysign(a, x).reshape(-1)
                moments[kind].copy_(a)
                moments[kind + "_scale"].copy_((top / _E4M3_MAX).reshape(-1))
    return {"param": state["param"], "step": step, **moments}


def _plain_grad_norm(state):
    g = state["grad"].float()
    return (g * g).sum(dtype=torch.float64).sqrt().float()


def run(state):
    case = state["case"]
    if not own:
        return {"group_norm": _plain_norm, "adamw": _plain_adamw,
                "grad_norm": _plain_grad_norm}[case["op"]](state)
    if case["op"] == "group_norm":
        from opendressi_b200 import torch_api as dr
        if not case["train"]:
            with torch.no_grad():
                return dr.group_norm(state["x"], case["groups"],
                                     state["weight"], state["bias"],
                                     activation=case["act"])
        y = dr.group_norm(state["x"], case["groups"], state["weight"],
                          state["bias"], activation=case["act"])
        if not case["affine"]:
            (dx,) = torch.autograd.grad(y, (state["x"],), state["grad"])
            return {"y": y, "dx": dx}
        dx, dw, db = torch.autograd.grad(
            y, (state["x"], state["weight"], state["bias"]), state["grad"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "grad_norm":
        from opendressi_b200 import optim
        return optim.grad_norm(state["grads"])
    state["optimizer"].step()
    packed = state["packed"]
    return {"param": state["param"], "step": packed["step"],
            **{k: packed[k] for k in state["moments"]}}


# --------------------------------------------------------------------- work

def work(case):
    size = _DTYPES[case["dtype"]].itemsize
    if case["op"] == "group_norm":
        values = case["n"] * case["h"] * case["w"] * case["c"]
        table = 4 * case["c"] * (2 if case["affine"] else 0)
        if case["train"]:  # x and dy in, y and dx out
            return {"bytes": 4 * values * size + 2 * table,
                    "flops": 40 * values}
        return {"bytes": 2 * values * size + table, "flops": 15 * values}
    values = sum(_lengths(case))
    if case["op"] == "grad_norm":
        return {"bytes": values * size + 4, "flops": 2 * values}
    # parameter in and out, gradient in, two states in and out
    state = 8 if case["bits"] == 32 else 2 + 8 / _BLOCK
    clip = 3 * values if case["max_norm"] else 0
    return {"bytes": values * (3 * size + 2 * state) + 8 * case["tensors"],
            "flops": values * (14 if case["bits"] == 32 else 40) + clip}


# -------------------------------------------------------- the definition, 64

def _exact_norm(case, state):
    x = state["x"].detach().double()
    n, c, groups = case["n"], case["c"], case["groups"]
    cols = torch.arange(c, device=x.device) // (c // groups)
    # moments of each channel, then of each group of channels
    count = case["h"] * case["w"]
    pool = torch.nn.functional.one_hot(cols, groups).double()
    share = pool / (count * (c // groups))
    mean = (x.sum((1, 2)) @ share)[:, cols][:, None, None, :]
    x = x - mean
    var = ((x ** 2).sum((1, 2)) @ share)[:, cols][:, None, None, :]
    deviation = (var + 1e-5) ** 0.5
    x = x / deviation
    w = b = None
    z = x
    if case["affine"]:
        w, b = state["weight"].detach().double(), state["bias"].detach().double()
        z = x * w + b
    if case["act"] == "silu":
        y = z * torch.sigmoid(z)
    elif case["act"] == "relu":
        y = torch.relu(z)
    else:
        y = z
    if not case["train"]:
        return y
    dz = state["grad"].double()
    if case["act"] == "silu":
        s = torch.sigmoid(z)
        dz = dz * (s + y * (1 - s))
    elif case["act"] == "relu":
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    sums, products = dz.sum((1, 2)), (dz * x).sum((1, 2))
    gain = w if w is not None else torch.ones(c, device=x.device).double()
    lift = ((sums * gain) @ share)[:, cols][:, None, None, :]
    tilt = ((products * gain) @ share)[:, cols][:, None, None, :]
    out = {"y": y, "dx": (dz * gain - lift - x * tilt) / deviation}
    if w is not None:
        out["dweight"], out["dbias"] = products.sum(0), sums.sum(0)
    return out


def _exact_adamw(case, state):
    b1, b2 = _BETAS
    t = float(_STEPS_DONE + 1)
    g = state["grad"].double()
    if case["max_norm"]:
        g = g * min(1.0, case["max_norm"] / (float(g.norm()) + 1e-6))
    moments = state["moments"]
    if case["bits"] == 32:
        m, v = moments["exp_avg"].double(), moments["exp_avg_sq"].double()
    else:
        def value(kind):
            scale = moments[kind + "_scale"].double()
            return (moments[kind].double().reshape(-1, _BLOCK)
                    * scale[:, None]).reshape(-1)

        m, v = value("exp_avg"), value("root_avg_sq") ** 2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = state["param"].double()
    p = p - _LR * _DECAY * p - _LR * (m / (1 - b1 ** t)) / (
        (v / (1 - b2 ** t)) ** 0.5 + _EPS)
    step = state["step"] + 1
    out = {"param": p, "step": step}
    if case["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    bits = _random_bits(state, step).reshape(-1)
    for kind, x, part in (("exp_avg", m, bits & 0xFFFF),
                          ("root_avg_sq", v ** 0.5, bits >> 16)):
        x = x.reshape(-1, _BLOCK)
        scale = x.abs().amax(1).clamp(min=_SCALE_FLOOR) / _E4M3_MAX
        a = (x.abs() / scale[:, None]).reshape(-1)
        # the distance of e4m3 values: 2^-3 of the power of two below, 2^-9 at
        # least; the next 20 bits decide, against 16 random ones and a half
        _, e = torch.frexp(a.clamp(min=2.0 ** -6))
        gap = torch.ldexp(torch.ones_like(a), e - 4)
        a = torch.floor(a / gap + (part * 16 + 8) / 2.0 ** 20) * gap
        a = a.clamp(max=_E4M3_MAX)
        if kind == "root_avg_sq":
            a = torch.where(x.reshape(-1) > 0, a.clamp(min=2.0 ** -9), a)
        out[kind] = a * torch.sign(x.reshape(-1))
        out[kind + "_scale"] = scale
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "group_norm":
            return _exact_norm(case, state)
        if case["op"] == "grad_norm":
            return torch.linalg.vector_norm(state["grad"].double())
        return _exact_adamw(case, state)
