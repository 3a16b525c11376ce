"""AdamW over many tensors and the norm over many tensors
(opendressi_b200.optim) against the formulas in 64 bits, and the 8-bit states
against a plain restatement of their rounding.

Tolerances count roundings of 2^-24 each (U): two products, a sum and the
rounded betas for a moment (and half a denormal step for each product); for
the update about a dozen operations with the
bias corrections; a parameter in type T is rounded once, eps(T) / 2."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BLOCK = 256


def _torch():
    import torch
    return torch


def make(seed, shapes, dtype, scale=1e-2):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for s in shapes:
        p = torch.nn.Parameter(torch.randn(s, generator=g, device="cuda")
                               .to(dtype))
        p.grad = (scale * torch.randn(s, generator=g, device="cuda")).to(dtype)
        out.append(p)
    return out


def formula(p, g, m, v, t, lr, betas, eps, wd, coef=1.0, clamp=None):
    """One step in 64 bits from 32-bit state, and the errors it may have."""
    b1, b2 = betas
    g = g.double() * coef
    g_err = 3 * U * (coef != 1.0)  # the clip factor and its product
    m1 = b1 * m + (1 - b1) * g
    m_err = 4 * U * ((b1 * m).abs() + ((1 - b1) * g).abs() * (1 + g_err / U))
    v1 = b2 * v + (1 - b2) * g * g
    v_err = 5 * U * (b2 * v + (1 - b2) * g * g * (1 + 2 * g_err / U)) \
        + 2.0 ** -148  # two products that may be denormal
    c1, c2 = 1 - b1 ** t, 1 - b2 ** t
    den = (v1 / c2).sqrt() + eps
    step = lr / c1 * m1 / den
    # the moments' errors, then 16 roundings: sqrt, bias corrections, quotient
    step_err = (lr / c1 * m_err / den
                + step.abs() * (v_err / (2 * v1).clamp(min=1e-300) + 16 * U))
    p64 = p.double()
    p1 = p64 * (1 - lr * wd) - step
    p_err = 3 * U * (p64.abs() + p1.abs()) + step_err
    if clamp is not None:
        p1 = p1.clamp(*clamp)
    return p1, p_err, m1, m_err, v1, v_err


def near(got, exp, err):
    torch = _torch()
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * 2 * half
    tol = err * (1 + half) + half * exp.abs() + tiny
    off = (got.double() - exp).abs()
    assert (off <= tol).all(), float((off / tol).max())


SHAPES = [(1,), (7, 5), (256,), (255,), (257,), (0,), (3, 1000), (64, 3, 3, 3),
          (), (100003,), (512, 512)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
def test_steps_in_32_bits(cuda, dtype, max_norm):
    torch = _torch()
    from opendressi_b200 import optim

    dtype = getattr(torch, dtype)
    params = make(1, SHAPES, dtype)
    kw = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    opt = optim.AdamW(params, max_norm=max_norm, **kw)
    for t in range(1, 5):
        g = torch.Generator(device="cuda").manual_seed(100 + t)
        for p in params:
            p.grad = (10.0 ** (t - 3) * torch.randn(
                p.shape, generator=g, device="cuda")).to(dtype)
        coef = 1.0
        if max_norm is not None:
            norm = math.sqrt(sum(float((p.grad.double() ** 2).sum())
                                 for p in params))
            coef = min(1.0, max_norm / (norm + 1e-6))
        before = [(p.detach().clone(), opt.state[p]["exp_avg"].double(),
                   opt.state[p]["exp_avg_sq"].double()) for p in params]
        opt.step()
        if max_norm is not None:
            assert abs(float(opt.last_norm) / norm - 1) <= 2 * U
        for p, (p0, m0, v0) in zip(params, before):
            p1, pe, m1, me, v1, ve = formula(p0, p.grad, m0, v0, t,
                                             coef=coef, **{
                "lr": kw["lr"], "betas": kw["betas"], "eps": kw["eps"],
                "wd": kw["weight_decay"]})
            st = opt.state[p]
            assert int(st["step"]) == t
            near(st["exp_avg"], m1, me)
            near(st["exp_avg_sq"], v1, ve)
            near(p.detach(), p1, pe)


def test_denormal_second_moments(cuda):
    """With eps 0 the root of a denormal number counts."""
    torch = _torch()
    from opendressi_b200 import optim

    p = make(21, [(1000,)], torch.float32)[0]
    p0 = p.detach().clone()
    p.grad = 3e-19 * (1 + torch.rand(1000, device="cuda"))
    opt = optim.AdamW([p], lr=1e-2, betas=(0.9, 0.99), eps=0.0,
                      weight_decay=0.0)
    opt.step()
    z = torch.zeros(1000, device="cuda").double()
    p1, pe, m1, me, v1, ve = formula(p0, p.grad, z, z, 1, 1e-2, (0.9, 0.99),
                                     0.0, 0.0)
    assert float(v1.max()) < 2.0 ** -126
    near(opt.state[p]["exp_avg_sq"], v1, ve)
    near(p.detach(), p1, pe)


def test_clip_over_groups_and_types(cuda):
    """One norm for all groups and element types, and a launch for each."""
    torch = _torch()
    from opendressi_b200 import optim

    a = make(22, [(700,), (3, 9)], torch.float32, scale=1.0)
    b = make(23, [(64, 65)], torch.bfloat16, scale=1.0)
    c = make(24, [(501,)], torch.float16, scale=1.0)
    params = a + b + c
    opt = optim.AdamW([{"params": a + b}, {"params": c, "lr": 1e-2}],
                      lr=1e-3, max_norm=0.25)
    before = [p.detach().clone() for p in params]
    norm = math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in params))
    opt.step()
    assert abs(float(opt.last_norm) / norm - 1) <= 2 * U
    for p, p0 in zip(params, before):
        z = torch.zeros_like(p0).double()
        lr = 1e-2 if p is c[0] else 1e-3
        p1, pe, m1, me, v1, ve = formula(p0, p.grad, z, z, 1, lr,
                                         (0.9, 0.999), 1e-8, 1e-2,
                                         0.25 / (norm + 1e-6))
        near(opt.state[p]["exp_avg"], m1, me)
        near(opt.state[p]["exp_avg_sq"], v1, ve)
        near(p.detach(), p1, pe)


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(cuda, bits):
    """Odd addresses, transposed and channels-last parameters, gradients in
    another order than theirs: what a packed copy of each would do."""
    torch = _torch()
    from opendressi_b200 import optim

    base = torch.randn(5000, device="cuda")
    for off in range(0, 9):
        n = 1500 + off
        p = torch.nn.Parameter(base.clone()[off:off + n])
        q = torch.nn.Parameter(base[off:off + n].clone())
        grad = torch.randn(n + 3, device="cuda")
        p.grad, q.grad = grad[3:], grad[3:].clone()
        a = optim.AdamW([p], state_bits=bits, seed=5)
        b = optim.AdamW([q], state_bits=bits, seed=5)
        for _ in range(3):
            a.step()
            b.step()
        assert torch.equal(p, q)
        for k in a.packed_state():
            assert torch.equal(a.packed_state()[k].float(),
                               b.packed_state()[k].float()), k
    for perm in ((1, 0, 2, 3), (0, 2, 3, 1), (3, 2, 1, 0)):
        t = torch.randn(12, 9, 5, 7, device="cuda")
        p = torch.nn.Parameter(t.clone().permute(perm))
        q = torch.nn.Parameter(t.clone())
        g = torch.randn(12, 9, 5, 7, device="cuda")
        p.grad = g.permute(perm).contiguous()  # not in p's order
        q.grad = g
        a = optim.AdamW([p], state_bits=bits)
        b = optim.AdamW([q], state_bits=bits)
        for _ in range(2):
            a.step()
            b.step()
        assert torch.equal(p.detach(), q.detach().permute(perm))
        assert a.state[p]["exp_avg"].shape == p.shape
        assert torch.equal(a.state[p]["exp_avg"].float(),
                           b.state[q]["exp_avg"].float().permute(perm))


def mix(x):
    """Wang's integer hash."""
    x = np.asarray(x, np.uint64) & np.uint64(0xFFFFFFFF)
    m = np.uint64(0xFFFFFFFF)
    x = (x ^ np.uint64(61)) ^ (x >> np.uint64(16))
    x = (x * np.uint64(9)) & m
    x ^= x >> np.uint64(4)
    x = (x * np.uint64(0x27D4EB2D)) & m
    return x ^ (x >> np.uint64(15))


def codes(x, scale, bits16, root):
    """The e4m3 values of x [n] (float64) with their block's scale, rounded
    by 16 random bits each: plain arithmetic in 64 bits."""
    pad = -len(x) % BLOCK
    a = np.abs(np.pad(x, (0, pad)).reshape(-1, BLOCK) / scale[:, None])
    u = np.pad(bits16, (0, pad)).reshape(-1, BLOCK).astype(np.float64)
    _, e = np.frexp(np.maximum(a, 2.0 ** -6))
    gap = np.ldexp(1.0, e - 4)
    a = np.minimum(np.floor(a / gap + (u * 16 + 8) / 2.0 ** 20) * gap, 448)
    a = a.reshape(-1)[:len(x)]
    if root:
        a = np.where((x > 0) & (a < 2.0 ** -9), 2.0 ** -9, a)
    return np.copysign(a, x)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_8_bit_state_bit_by_bit(cuda, dtype):
    """Codes and scales over steps that start from zeros, with values of many
    magnitudes, zeros and what is not finite, against plain arithmetic with
    the same random bits. For given bits a code grows with its value, so it
    lies between the codes of the value less and plus what 32-bit arithmetic
    may be off by: 4 U of a moment's terms, 6 U of a root's value, 4 U for the
    scale and 8 U for its inverse and the quotient; below 2^-6 the quotient
    keeps 20 bits below its last, another 2^-29."""
    torch = _torch()
    from opendressi_b200 import optim

    dtype = getattr(torch, dtype)
    params = make(4, [(5,), (300,), (256,), (1000, 3), (70001,)], dtype)
    seed = 0x9ABCDEF1
    kw = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    opt = optim.AdamW(params, state_bits=8, seed=seed, **kw)
    b1, b2 = kw["betas"]
    exact = total = 0
    for t in range(1, 5):
        g = torch.Generator(device="cuda").manual_seed(50 + t)
        for p in params:
            mag = torch.randn(p.shape, generator=g, device="cuda") * 4
            x = torch.randn(p.shape, generator=g, device="cuda") * mag.exp()
            x *= torch.rand(p.shape, generator=g, device="cuda") < 0.8
            if t == 3 and p.numel() > 400:
                x.view(-1)[300] = math.inf
                x.view(-1)[301] = math.nan
            p.grad = x.to(dtype)
        before = []
        for p in params:
            s = opt.state[p]
            before.append([
                s[k].double().cpu().numpy().reshape(-1)
                * np.repeat(s[k + "_scale"].double().cpu().numpy(),
                            BLOCK)[:p.numel()]
                for k in ("exp_avg", "root_avg_sq")])
        opt.step()
        for i, (p, (m, r)) in enumerate(zip(params, before)):
            x = p.grad.double().cpu().numpy().reshape(-1)
            with np.errstate(all="ignore"):
                m_err = 4 * U * (np.abs(b1 * m) + np.abs((1 - b1) * x))
                m = b1 * m + (1 - b1) * x
                r = np.sqrt(b2 * r * r + (1 - b2) * x * x)
                r_err = 6 * U * r
            key = mix(mix(np.uint64(seed) ^ mix(t)) + np.uint64(i))
            bits = mix(key + np.arange(p.numel(), dtype=np.uint64))
            s = opt.state[p]
            for kind, val, err, part, root in (
                    ("exp_avg", m, m_err, bits & np.uint64(0xFFFF), False),
                    ("root_avg_sq", r, r_err, bits >> np.uint64(16), True)):
                got = s[kind].double().cpu().numpy().reshape(-1)
                fine = np.isfinite(val)
                assert np.array_equal(np.isnan(got), ~fine), (t, i, kind)
                val, err = np.where(fine, val, 0), np.where(fine, err, 0)
                pad = -len(val) % BLOCK
                top = np.pad(np.abs(val), (0, pad)).reshape(-1, BLOCK).max(1)
                top_err = np.pad(err, (0, pad)).reshape(-1, BLOCK).max(1)
                scale = np.maximum(top, 2.0 ** -100) / 448
                off = np.abs(s[kind + "_scale"].double().cpu().numpy() - scale)
                assert (off <= 4 * U * scale + top_err / 448).all()
                wide = np.repeat(top_err / np.maximum(top, 2.0 ** -100),
                                 BLOCK)[:len(val)]
                each = np.repeat(scale, BLOCK)[:len(val)]
                mag = np.abs(val)
                low = np.maximum(mag * (1 - 12 * U - wide) - err
                                 - each * 2.0 ** -29, 0)
                high = mag * (1 + 12 * U + wide) + err + each * 2.0 ** -29
                if root:  # 0 stays 0, and what is not does not become it
                    low = np.where(mag > 0, np.maximum(low, 1e-300), 0)
                    high = np.where(mag > 0, high, 0)
                lo = codes(low, scale, part, root)
                hi = codes(high, scale, part, root)
                size = np.abs(np.where(fine, got, 0))
                sure = fine & (mag > err)
                assert ((size >= lo) & (size <= hi))[fine].all(), (t, i, kind)
                assert (np.sign(got) * np.sign(val) >= 0)[sure].all()
                exact += int((lo == hi).sum())
                total += len(val)
    assert exact > 0.999 * total  # the bounds say something


def test_8_bit_parameters_follow_the_formula(cuda):
    """The parameters see the moments before they are coded: the 64-bit
    formula from the decoded state."""
    torch = _torch()
    from opendressi_b200 import optim

    params = make(6, [(5000,), (33, 77)], torch.float32)
    opt = optim.AdamW(params, state_bits=8, lr=1e-2, weight_decay=0.05)
    for t in range(1, 4):
        for p in params:
            p.grad = torch.randn_like(p) * 0.1
        olds = []
        for p in params:
            s = opt.state[p]
            val = lambda k: (s[k].double().reshape(-1) * s[  # noqa: E731
                k + "_scale"].double().repeat_interleave(BLOCK)[:p.numel()]
            ).reshape(p.shape)
            olds.append((p.detach().clone(), val("exp_avg"),
                         val("root_avg_sq") ** 2))
        opt.step()
        for p, (p0, m0, v0) in zip(params, olds):
            p1, pe, *_ = formula(p0, p.grad, m0, v0, t, 1e-2, (0.9, 0.999),
                                 1e-8, 0.05)
            # decoding rounds twice more
            near(p.detach(), p1, 1.5 * pe + 1e-2 * 8 * U)


def test_8_bit_rounding_has_the_right_mean(cuda):
    """Over 4096 seeds a code's mean is its value: within 5 deviations of the
    mean of two-valued draws (at most half a gap each), which is 5 / 128 of
    a gap."""
    torch = _torch()
    from opendressi_b200 import optim

    x = torch.logspace(-5, 0, BLOCK, device="cuda")
    total = {k: torch.zeros(BLOCK, dtype=torch.float64, device="cuda")
             for k in ("exp_avg", "root_avg_sq")}
    n = 4096
    p = torch.nn.Parameter(torch.zeros(BLOCK, device="cuda"))
    p.grad = x
    opt = optim.AdamW([p], state_bits=8, betas=(0.5, 0.75))
    s = opt.packed_state()
    for seed in range(n):
        for k in s:
            s[k].zero_()
        opt.seed = seed * 7919
        opt.step()
        for k in total:
            total[k] += s[k].double() * s[k + "_scale"].double()
    for k, exact in (("exp_avg", 0.5 * x.double()),
                     ("root_avg_sq", 0.5 * x.double())):
        a = exact / s[k + "_scale"].double()
        gap = torch.ldexp(torch.ones_like(a),
                          torch.frexp(a.clamp(min=2.0 ** -6))[1] - 4)
        off = (total[k] / n / s[k + "_scale"].double() - a).abs() / gap
        assert float(off.max()) <= 5.0 / 128.0, k


def test_8_bit_average_moves_by_less_than_a_gap(cuda):
    """A second moment whose root moves by 0.0005 of itself a step, where the
    gap between codes is 1/16 to 1/8 of it, still reaches its gradient's
    square (rounding to the nearest would leave it where it began).

    The square v of a root that goes up or down a gap with the right mean
    gains the variance of that: gap^2 f (1 - f), f the share of a gap that the
    step moves. With gap <= r / 8 and gap f <= 0.0005 r that is at most
    0.0005 / 8 v a step. So the mean of v follows v <- v (1 - 0.001) + 1e-5
    from below and v <- v (1 - 0.001 + 0.0000625) + 1e-5 from above. 2% for
    the mean of 16320 draws, each off by no more than about itself."""
    torch = _torch()
    from opendressi_b200 import optim

    n = 64 * BLOCK
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = optim.AdamW([p], state_bits=8, lr=0.0)
    p.grad = torch.full((n,), 0.1, device="cuda")
    p.grad[::BLOCK] = 1.0  # holds the scale of each block
    s = opt.packed_state()
    s["exp_avg"].zero_()
    s["root_avg_sq"].copy_(torch.full((n,), 448.0, device="cuda"))
    s["root_avg_sq_scale"].fill_(1.0 / 448.0)
    for _ in range(3000):  # 0.999^3000 = 0.05 of the start is left
        opt.step()
    v = (s["root_avg_sq"].double().reshape(-1, BLOCK)
         * s["root_avg_sq_scale"].double()[:, None]) ** 2
    mean = float(v[:, 1:].mean())
    low = 0.01 + 0.99 * 0.999 ** 3000
    end = 1e-5 / 0.0009375
    high = end + (1 - end) * 0.9990625 ** 3000
    assert 0.98 * low <= mean <= 1.02 * high


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite_gradients_stay_with_their_values(cuda, bits):
    torch = _torch()
    from opendressi_b200 import optim

    p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
    q = torch.nn.Parameter(torch.ones(1000, device="cuda"))
    grad = torch.randn(1000, device="cuda")
    p.grad, q.grad = grad.clone(), grad.clone()
    bad = torch.tensor([3, 300, 301], device="cuda")
    q.grad[bad] = torch.tensor([math.nan, math.inf, -math.inf],
                               device="cuda")
    # the largest value of each block is a finite one
    p.grad[::100] = 9.0
    q.grad[::100] = 9.0
    bad = bad[q.grad[bad] != 9.0]
    keep = torch.ones(1000, dtype=torch.bool, device="cuda")
    keep[bad] = False
    a = optim.AdamW([p], state_bits=bits)
    b = optim.AdamW([q], state_bits=bits)
    for _ in range(3):
        # p's values at the bad places must not be the largest of a block
        p.grad[bad] = 0.0
        a.step()
        b.step()
        assert torch.equal(p[keep], q[keep])
        assert torch.isnan(q[bad]).all()
        for k in ("exp_avg", "exp_avg_sq" if bits == 32 else "root_avg_sq"):
            assert torch.equal(a.state[p][k].float()[keep],
                               b.state[q][k].float()[keep])
            assert not torch.isfinite(b.state[q][k].float()[bad]).any()


def test_zero_gradients_leave_zero_state(cuda):
    torch = _torch()
    from opendressi_b200 import optim

    for bits in (32, 8):
        p = torch.nn.Parameter(torch.randn(777, device="cuda"))
        p0 = p.detach().clone()
        p.grad = torch.zeros_like(p)
        opt = optim.AdamW([p], state_bits=bits, weight_decay=0.0)
        for _ in range(3):
            opt.step()
        assert torch.equal(p, p0)
        assert not opt.packed_state()["exp_avg"].float().any()


def test_groups_clamps_and_missing_gradients(cuda):
    torch = _torch()
    from opendressi_b200 import optim

    maps = make(8, [(40, 40, 3), (9,)], torch.float32, scale=1.0)
    env = make(9, [(16, 32, 3)], torch.float32, scale=1.0)
    half = make(10, [(300,), (20, 20)], torch.bfloat16, scale=1.0)
    opt = optim.AdamW([
        {"params": maps, "clamp": (0.0, 1.0), "lr": 0.5},
        {"params": env, "clamp": (0.0, math.inf), "weight_decay": 0.0},
        {"params": half + make(11, [(5,)], torch.float32)}], lr=1e-2)
    late = maps[1]
    kept = late.grad
    late.grad = None
    opt.step()
    assert int(opt.state[late]["step"]) == 0
    assert not opt.state[late]["exp_avg"].any()
    late.grad = kept
    opt.step()
    assert int(opt.state[late]["step"]) == 1
    assert int(opt.state[maps[0]]["step"]) == 2
    for p in maps[:1]:
        assert float(p.detach().min()) >= 0.0
        assert float(p.detach().max()) <= 1.0
    assert float(env[0].detach().min()) >= 0.0
    # the late tensor's first step is a whole one: lr * sign (eps aside)
    p1, pe, *_ = formula(make(8, [(40, 40, 3), (9,)], torch.float32)[1]
                         .detach(), kept, torch.zeros(9).cuda().double(),
                         torch.zeros(9).cuda().double(), 1, 0.5,
                         (0.9, 0.999), 1e-8, 1e-2, clamp=(0.0, 1.0))
    near(late.detach(), p1, pe)
    extra = make(12, [(31,)], torch.float32)
    opt.add_param_group({"params": extra})
    opt.step()
    assert int(opt.state[extra[0]]["step"]) == 1
    # nan is not hidden by a clamp
    maps[0].grad[0, 0, 0] = math.nan
    opt.step()
    assert math.isnan(float(maps[0].detach()[0, 0, 0]))


def test_many_tensors_in_several_launches(cuda):
    """More tensors than one launch's arguments hold, some empty."""
    torch = _torch()
    from opendressi_b200 import optim

    lengths = [(37 * i) % 700 for i in range(1500)]
    flat = torch.randn(sum(lengths), device="cuda")
    grad = torch.randn(sum(lengths), device="cuda")
    ps, at = [], 0
    for n in lengths:
        p = torch.nn.Parameter(flat[at:at + n].clone())
        p.grad = grad[at:at + n].clone()
        ps.append(p)
        at += n
    opt = optim.AdamW(ps, max_norm=3.0)
    opt.step()
    opt.step()
    norm = float((grad.double() ** 2).sum().sqrt())
    assert abs(float(opt.last_norm) / norm - 1) <= 2 * U
    z = torch.zeros_like(flat).double()
    coef = 3.0 / (norm + 1e-6)
    p1, e1, m1, _, v1, _ = formula(flat, grad, z, z, 1, 1e-3, (0.9, 0.999),
                                   1e-8, 1e-2, coef)
    p2, e2, *_ = formula(p1, grad, m1, v1, 2, 1e-3, (0.9, 0.999), 1e-8, 1e-2,
                         coef)
    got = torch.cat([p.detach() for p in ps])
    near(got, p2, e1 + 2 * e2)
    assert all(int(s) == 2 for s in opt.packed_state()["step"].tolist())


def test_learning_rates(cuda):
    torch = _torch()
    from opendressi_b200 import optim

    p, q, r = (make(13, [(999,)], torch.float32)[0] for _ in range(3))
    a = optim.AdamW([p], lr=0.125)
    b = optim.AdamW([q], lr=torch.tensor(0.125, device="cuda"))
    c = optim.AdamW([r], lr=torch.tensor(0.125))
    for o in (a, b, c):
        o.step()
    assert torch.equal(p, q) and torch.equal(p, r)
    sched = torch.optim.lr_scheduler.StepLR(a, 1, gamma=0.5)
    a.step()
    sched.step()
    assert a.param_groups[0]["lr"] == 0.0625

    def closure():
        return torch.tensor(3.5)

    assert float(a.step(closure)) == 3.5


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(cuda, bits):
    """A captured step, replayed with new gradients and a new learning rate,
    counts on; an eager optimizer takes the same steps."""
    torch = _torch()
    from opendressi_b200 import optim

    shapes = [(1000,), (33, 7), (5,)]
    pa, pb = (make(14, shapes, torch.float32) for _ in range(2))
    lr = torch.tensor(2.0 ** -7, device="cuda")
    a = optim.AdamW(pa, lr=lr, state_bits=bits, max_norm=1.0, seed=3)
    b = optim.AdamW(pb, lr=2.0 ** -7, state_bits=bits, max_norm=1.0, seed=3)
    # on a side stream first, as a captured step runs
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for k in range(4):
        for x, y in zip(pa, pb):
            g = torch.randn_like(x) * (k + 1)
            x.grad.copy_(g)
            y.grad.copy_(g)
        lr.fill_(1e-2 / (k + 1))
        b.param_groups[0]["lr"] = float(lr)
        graph.replay()
        b.step()
    for x, y in zip(pa, pb):
        assert torch.equal(x, y)
    for k, v in a.packed_state().items():
        assert torch.equal(v.float(), b.packed_state()[k].float()), k
    assert a.packed_state()["step"].tolist() == [5, 5, 5]


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_loaded(cuda, bits, tmp_path):
    torch = _torch()
    from opendressi_b200 import optim

    shapes = [(700,), (3, 5)]
    pa, pb = (make(15, shapes, torch.bfloat16) for _ in range(2))
    a = optim.AdamW(pa, lr=1e-2, state_bits=bits, seed=11, max_norm=2.0)
    a.step()
    a.step()
    torch.save(a.state_dict(), tmp_path / "opt.pt")
    for x, y in zip(pa, pb):
        y.data.copy_(x.data)
    b = optim.AdamW(pb, state_bits=bits)
    b.load_state_dict(torch.load(tmp_path / "opt.pt"))
    assert b.param_groups[0]["lr"] == 1e-2 and b.max_norm == 2.0
    for _ in range(2):
        a.step()
        b.step()
    for x, y in zip(pa, pb):
        assert torch.equal(x, y)
    other = optim.AdamW(make(15, shapes, torch.bfloat16),
                        state_bits=40 - bits)
    with pytest.raises(ValueError):
        other.load_state_dict(a.state_dict())
    with pytest.raises(ValueError):
        b.load_state_dict(optim.AdamW(make(1, [(700,)], torch.bfloat16),
                                      state_bits=bits).state_dict())


def test_refusals(cuda):
    torch = _torch()
    from opendressi_b200 import DressiError, optim

    def leaf(t):
        return torch.nn.Parameter(t, requires_grad=t.is_floating_point())

    dev = "cuda"
    x = torch.randn(64, device=dev)
    for bad in (torch.randn(4), x.double(), torch.randn(4, 1, device=dev)
                .expand(4, 5), torch.arange(4, device=dev),
                torch.randn(8, 8, device=dev)[:, ::2],
                torch.view_as_complex(x.view(32, 2))):
        with pytest.raises(DressiError):
            optim.AdamW([leaf(bad)])
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamW([leaf(x[:40]), leaf(x[30:])])
    with pytest.raises(ValueError):  # the same parameter twice
        p = leaf(x)
        optim.AdamW([{"params": [p]}, {"params": [p]}])
    with pytest.raises(TypeError):
        optim.AdamW([("name", leaf(x))])
    p = leaf(x.clone())
    opt = optim.AdamW([p])
    with pytest.raises(TypeError, match="state_dict"):
        import copy
        copy.deepcopy(opt)
    p.grad = torch.randn(64, device=dev)
    before = p.detach().clone()
    p.grad = torch.sparse_coo_tensor([[1]], [1.0], (64,), device=dev)
    with pytest.raises(DressiError, match="gradient"):
        opt.step()
    p.grad = torch.randn(64, device=dev)
    p.data = p.data.half()
    with pytest.raises(DressiError, match="changed"):
        opt.step()
    p.data = before[:32]
    with pytest.raises(DressiError, match="changed"):
        opt.step()
    opt = optim.AdamW([leaf(x.clone())])
    opt.param_groups[0]["params"][0].grad = torch.ones(64, device=dev)
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError):
        opt.step()
    with pytest.raises(ValueError):
        optim.AdamW([leaf(x)], lr=torch.tensor(1e-3, device=dev,
                                               dtype=torch.float64))
    assert optim.AdamW([{"params": []}]).step() is None


# -------------------------------------------------------------------- norm

@pytest.mark.parametrize("lengths", [
    [1], [0], [5, 0, 3], [2048], [2049, 1, 4095], [1000003],
    [(13 * i) % 900 for i in range(2500)], [3000000, 17, 2000001]])
def test_norm(cuda, lengths):
    torch = _torch()
    from opendressi_b200 import optim

    types = (torch.float32, torch.bfloat16, torch.float16)
    ts = [torch.randn(n + 1, device="cuda").to(types[i % 3])[1:]
          for i, n in enumerate(lengths)]
    exact = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
    got = optim.grad_norm(ts)
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - exact) <= 2 * U * exact
    assert torch.equal(got, optim.grad_norm(ts))


def test_norm_of_large_small_and_not_finite_values(cuda):
    torch = _torch()
    from opendressi_b200 import optim

    for size in (1e30, 1e-30):  # whose squares 32 bits cannot hold
        t = torch.full((1000,), size, device="cuda")
        exact = float(t[0].double()) * math.sqrt(1000)
        assert abs(float(optim.grad_norm(t)) / exact - 1) <= 2 * U
    t = torch.ones(5000, device="cuda")
    t[4321] = math.inf
    assert float(optim.grad_norm([t])) == math.inf
    t[7] = math.nan
    assert math.isnan(float(optim.grad_norm([t])))
    assert float(optim.grad_norm([])) == 0.0
    strided = torch.randn(40, 50, device="cuda")[:, ::3]
    assert abs(float(optim.grad_norm(strided)) /
               float((strided.double() ** 2).sum().sqrt()) - 1) <= 2 * U


def test_norm_refusals(cuda):
    torch = _torch()
    from opendressi_b200 import DressiError, optim

    for bad in (torch.ones(3), torch.ones(3, device="cuda").double(),
                torch.arange(3, device="cuda")):
        with pytest.raises(DressiError):
            optim.grad_norm([bad])
    with pytest.raises(DressiError):
        optim.grad_norm([torch.ones(3, device="cuda")],
                        out=torch.zeros(2, device="cuda"))


# ---------------------------------------------------------------- together

def test_a_decoder_on_rendered_features(cuda):
    """Rasterize, interpolate learned vertex features, a two-layer decoder
    with group_norm, loss, backward, clipped AdamW over features and weights:
    gradients against the same pipeline in 64 bits from the raster on, the
    step against the formula."""
    torch = _torch()
    from opendressi_b200 import optim, scene, torch_api as dr

    sc = scene.silhouette_scene(level=2, n_views=2, res=48, seed=3)
    nv = sc.n_verts
    pos = []
    for m in sc.mvps:  # column-major matrices, Vulkan depth
        h = np.concatenate([sc.target_pos, np.ones((nv, 1))], 1)
        clip = h @ np.asarray(m, np.float64).reshape(4, 4)
        clip[:, 2] = 2.0 * clip[:, 2] - clip[:, 3]
        pos.append(clip)
    pos = torch.tensor(np.stack(pos), dtype=torch.float32, device=cuda)
    tri = torch.tensor(sc.faces.astype(np.int32), device=cuda)
    g = torch.Generator(device="cuda").manual_seed(2)

    def normal(*s):
        return torch.randn(s, generator=g, device="cuda")

    leaves = [normal(nv, 16), normal(16, 24) / 4, 1 + 0.1 * normal(24),
              0.1 * normal(24), normal(24, 3) / 5]
    leaves = [torch.nn.Parameter(t) for t in leaves]
    target = torch.rand((2, 48, 48, 3), generator=g, device="cuda")
    opt = optim.AdamW([{"params": leaves[:1], "clamp": (-3.0, 3.0)},
                       {"params": leaves[1:]}], lr=1e-2, max_norm=0.1)
    ctx = dr.RasterizeContext()
    with torch.no_grad():
        rast, _ = dr.rasterize(ctx, pos, tri, (48, 48))
    assert float((rast[..., 3] > 0).float().mean()) > 0.05

    feat, w1, gamma, beta, w2 = leaves
    image, _ = dr.interpolate(feat, rast, tri)
    hidden = dr.group_norm(image @ w1, 6, gamma, beta, activation="silu")
    loss = ((hidden @ w2 - target) ** 2).mean()
    opt.zero_grad()
    loss.backward()

    d = [t.detach().double().requires_grad_(True) for t in leaves]
    fid = rast[..., 3].long() - 1
    cov = (fid >= 0)[..., None]
    idx = tri.long()[fid.clamp(min=0)]
    u, v = rast[..., 0:1].double(), rast[..., 1:2].double()
    f = d[0]
    im = torch.where(cov, u * f[idx[..., 0]] + v * f[idx[..., 1]]
                     + (1 - u - v) * f[idx[..., 2]], 0.0)
    z = (im @ d[1]).reshape(2, -1, 6, 4)
    z = (z - z.mean((1, 3), keepdim=True)) / (
        z.var((1, 3), keepdim=True, unbiased=False) + 1e-5).sqrt()
    z = z.reshape(2, 48, 48, 24) * d[2] + d[3]
    exact = (((z * torch.sigmoid(z)) @ d[4] - target.double()) ** 2).mean()
    exact.backward()
    # products in 32 bits (tf32 stays off), a mean of 13824 squares
    assert abs(float(loss.detach()) / float(exact.detach()) - 1) < 1e-4
    for p, e in zip(leaves, d):
        # sums over 4608 pixels of 32-bit products, and the interpolation's
        # atomics: 1e-4 of the largest
        assert float((p.grad.double() - e.grad).abs().max()) <= \
            1e-4 * float(e.grad.abs().max())

    norm = math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in leaves))
    before = [p.detach().clone() for p in leaves]
    opt.step()
    assert abs(float(opt.last_norm) / norm - 1) <= 2 * U
    coef = min(1.0, 0.1 / (norm + 1e-6))
    for i, (p, p0) in enumerate(zip(leaves, before)):
        zero = torch.zeros_like(p0).double()
        p1, pe, *_ = formula(p0, p.grad, zero, zero, 1, 1e-2, (0.9, 0.999),
                             1e-8, 1e-2, coef,
                             (-3.0, 3.0) if i == 0 else None)
        near(p.detach(), p1, pe)
