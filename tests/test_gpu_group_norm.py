"""Group normalisation with an activation over channels-last images
(opendressi_b200.torch_api.group_norm, ops.group_norm*) against the formulas
in 64 bits.

Tolerances. An image in type T is rounded once: eps(T) / 2 of the value. What
is computed in 32 bits before that: a value h = (x - mean) rstd carries the
rounding of mean (2^-24 |mean| rstd), a few of its own and those of rstd, each
2^-24 of |h|; per-thread sums add one rounding a step. K covers the number of
such roundings of a term, taken at the size of the term.

The mean itself is an average of threads' means. Each of those is a first value
less the group's, plus a mean of distances from it: 3 roundings of terms of at
most 2 R deviations, where R is the group's largest |h|. So the average, and
every h, is off by 6 R 2^-24 at most from those; 8 R 2^-24 with the sums of up
to 32 distances behind the means, whose roundings have either sign."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
K = 64.0  # roundings of one term, with those of up to 32 summation steps


def _torch():
    import torch
    return torch


def reference(x, weight, bias, groups, eps, act, dy=None):
    """The formulas in 64 bits, and the sizes of the terms that round."""
    torch = _torch()
    shape = x.shape
    n, c = shape[0], shape[-1]
    x64 = x.detach().double().reshape(n, -1, groups, c // groups)
    mean = x64.mean((1, 3), keepdim=True)
    var = ((x64 - mean) ** 2).mean((1, 3), keepdim=True)
    rstd = 1.0 / (var + eps).sqrt()
    h = (x64 - mean) * rstd
    one = torch.ones(c, device=x.device, dtype=torch.float64)
    w = one if weight is None else weight.detach().double()
    b = one * 0 if bias is None else bias.detach().double()
    w, b = w.reshape(1, 1, groups, -1), b.reshape(1, 1, groups, -1)
    z = h * w + b
    if act == "silu":
        s = torch.sigmoid(z)
        y, slope = z * s, s * (1 + z * (1 - s))
    elif act == "relu":
        y, slope = z.clamp(min=0), (z > 0).double()
    else:
        y, slope = z, torch.ones_like(z)
    off = (mean.abs() * rstd).expand_as(h)      # the mean's own rounding
    out = {"y": y.reshape(shape), "mean": mean.reshape(n, groups),
           "rstd": rstd.reshape(n, groups)}
    reach = 8 / K * h.abs().amax((1, 3), keepdim=True)
    off = off + reach
    z_err = K * U * ((h.abs() + off) * w.abs() + b.abs())
    out["y_err"] = (1.2 * z_err + K * U * y.abs() * (1 + z.abs())
                    ).reshape(shape)
    if dy is None:
        return out
    dy64 = dy.double().reshape(h.shape)
    dz = dy64 * slope
    # |act''| <= 0.5 for silu; relu jumps at 0, where the caller looks away
    dz_err = dy64.abs() * (0.5 * z_err * (act == "silu")
                           + K * U * (slope.abs() + 0.1) * (1 + z.abs()))
    h_err = K * U * (h.abs() + off)
    g = dz * w
    ma, mb = g.mean((1, 3), keepdim=True), (g * h).mean((1, 3), keepdim=True)
    ma_err = ((dz_err + K * U * dz.abs()) * w.abs()).mean((1, 3), keepdim=True)
    mb_err = ((dz_err * h.abs() + dz.abs() * h_err
               + K * U * (dz * h).abs()) * w.abs()).mean((1, 3), keepdim=True)
    out["dx"] = (rstd * (g - ma - h * mb)).reshape(shape)
    out["dx_err"] = (rstd * (
        dz_err * w.abs() + ma_err + h.abs() * mb_err + h_err * mb.abs()
        + K * U * (g.abs() + ma.abs() + (h * mb).abs()))).reshape(shape)
    out["dweight"] = (dz * h).sum((0, 1)).reshape(-1)
    out["dweight_err"] = (dz_err * h.abs() + dz.abs() * h_err + K * U
                          * (dz * h).abs()).sum((0, 1)).reshape(-1)
    out["dbias"] = dz.sum((0, 1)).reshape(-1)
    out["dbias_err"] = (dz_err + K * U * dz.abs()).sum((0, 1)).reshape(-1)
    out["kink"] = ((z.abs() <= z_err) if act == "relu"
                   else torch.zeros_like(z, dtype=torch.bool)).reshape(shape)
    return out


def check(got, ref, kind, where=None):
    torch = _torch()
    exp = ref[kind]
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * 2 * half
    tol = ref[kind + "_err"] * (1 + half) + half * exp.abs() + tiny
    bad = (got.double() - exp).abs() > tol
    if where is not None:
        bad &= ~where
    assert got.shape == exp.shape
    assert not bad.any(), (kind, int(bad.sum()), float(
        ((got.double() - exp).abs() / tol).max().detach()))


def make(seed, shape, dtype, affine=True, offset=0.0):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[-1]
    x = torch.randn(shape, generator=g, device="cuda") + offset
    dy = torch.randn(shape, generator=g, device="cuda")
    w = 1 + 0.3 * torch.randn(c, generator=g, device="cuda")
    b = 0.3 * torch.randn(c, generator=g, device="cuda")
    return (x.to(dtype), dy.to(dtype), w if affine else None,
            b if affine else None)


# rows, channels and groups that take every mapping: whole vectors; rows that
# vectors straddle; samples whose size no vector divides; rows wider than a
# thread block, of narrow and of wide groups, odd too; one value a group
SHAPES = [
    ((1, 1, 1, 1), 1), ((2, 1, 1, 8), 8), ((3, 1, 1, 6), 2),
    ((1, 16, 16, 32), 8), ((2, 7, 5, 3), 1), ((2, 7, 5, 3), 3),
    ((3, 61, 47, 40), 10), ((2, 8, 41), 1), ((2, 33, 31, 41), 41),
    ((5, 9), 3), ((1, 300, 301, 64), 32), ((2, 129, 127, 96), 16),
    ((2, 3, 3, 4096), 32), ((1, 5, 3, 4100), 1), ((2, 2, 3, 5002), 2),
    ((1, 4, 2, 9000), 2), ((2, 3, 1030), 515), ((1, 2, 2, 1021), 1021),
    ((1, 3, 1, 8209), 1), ((17, 4, 4, 16), 4), ((400, 2, 2, 8), 2),
    # more samples than blocks; samples of one block an SM and of two
    ((1500, 3, 5, 12), 3), ((9, 40, 50, 24), 6), ((160, 30, 31, 24), 4),
]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape,groups", SHAPES,
                         ids=["x".join(map(str, s)) + f"g{g}"
                              for s, g in SHAPES])
def test_forward_and_backward(cuda, shape, groups, dtype):
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    dtype = getattr(torch, dtype)
    for k, act in enumerate(("silu", "none", "relu")):
        affine = k < 2 or shape[0] % 2 == 1
        x, dy, w, b = make(7 + k, shape, dtype, affine)
        leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
        y = dr.group_norm(x, groups, w, b, activation=act)
        grads = torch.autograd.grad(y, leaves, dy)
        with torch.no_grad():  # the call without a graph gives the same bits
            assert torch.equal(dr.group_norm(x, groups, w, b, activation=act),
                               y)
        ref = reference(x, w, b, groups, 1e-5, act, dy)
        assert y.dtype == dtype and y.is_contiguous()
        check(y, ref, "y")
        if ref["kink"].any():
            continue  # a sum may hold either side of the kink
        check(grads[0], ref, "dx")
        if affine:
            check(grads[1], ref, "dweight")
            check(grads[2], ref, "dbias")


@pytest.mark.parametrize("offset", [0.0, 100.0, 1.0e4])
def test_mean_far_from_zero(cuda, offset):
    """A mean of 1e4 deviations: a sum of squares in 32 bits would have
    nothing left of the variance."""
    torch = _torch()
    from opendressi_b200 import ops

    x, _, w, b = make(3, (2, 64, 65, 24), torch.float32, offset=offset)
    x[0, 0, 0] = 0.0  # a background corner
    y, mean, rstd = ops.group_norm(x, 4, w, b, stats=True)
    ref = reference(x, w, b, 4, 1e-5, "none")
    check(y, ref, "y")
    assert ((mean.double() - ref["mean"]).abs() <=
            4 * U * (ref["mean"].abs() + 1 / ref["rstd"])).all()
    assert ((rstd / ref["rstd"] - 1).abs() <= K * U).all()


def test_gradients_against_differences(cuda):
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    x, dy, w, b = make(5, (2, 5, 3, 12), torch.float32)
    for t in (x, w, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(
        dr.group_norm(x, 3, w, b, activation="silu"), (x, w, b), dy)

    def loss(xx, ww, bb):
        return (reference(xx, ww, bb, 3, 1e-5, "silu")["y"]
                * dy.double()).sum()

    args = [t.detach().double() for t in (x, w, b)]
    for i, g in enumerate(grads):
        d = torch.randn_like(args[i])
        step = 1e-5
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + step * d, args[i] - step * d
        diff = float((loss(*hi) - loss(*lo)) / (2 * step))
        # differences: step^2 of the third derivative, 1e-16 / step of the sum
        assert abs(float((g.double() * d).sum()) - diff) <= 1e-5 * max(
            1.0, float((g.double() * d).abs().sum()))


def test_unaligned_strided_and_expanded(cuda):
    """Inputs at odd addresses, images cut out of wider ones, a gradient that
    is one value for all: the same values as of packed copies."""
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    for dtype in (torch.float32, torch.bfloat16):
        base = torch.randn(2 * 15 * 17 * 16 + 8, device="cuda").to(dtype)
        want = {}
        for off in (0, 1, 2, 3, 4, 7):
            x = base[off:off + 2 * 15 * 17 * 16].view(2, 15, 17, 16)
            ref = reference(x, None, None, 4, 1e-5, "silu")
            check(dr.group_norm(x, 4, activation="silu"), ref, "y")
            want[off] = x
        wide = torch.randn(2, 9, 11, 40, device="cuda").to(dtype)
        cut = wide[..., 3:27]
        assert torch.equal(dr.group_norm(cut, 4), dr.group_norm(
            cut.contiguous(), 4))
        image = torch.randn(2, 24, 9, 11, device="cuda").to(dtype)
        last = image.to(memory_format=torch.channels_last).permute(0, 2, 3, 1)
        assert last.is_contiguous()
        x = last.detach().requires_grad_(True)
        y = dr.group_norm(x, 3, activation="silu")
        one = torch.ones((), device="cuda", dtype=dtype)
        (g1,) = torch.autograd.grad(y, x, one.expand_as(y), retain_graph=True)
        (g2,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(g1, g2)


def test_needed_gradients_only(cuda):
    torch = _torch()
    from opendressi_b200 import ops, torch_api as dr

    x, dy, w, b = make(9, (3, 9, 7, 20), torch.float32)
    xr, wr, br = (t.clone().requires_grad_(True) for t in (x, w, b))
    full = torch.autograd.grad(dr.group_norm(xr, 5, wr, br), (xr, wr, br), dy)
    (gx,) = torch.autograd.grad(dr.group_norm(xr, 5, w, b), (xr,), dy)
    gw, = torch.autograd.grad(dr.group_norm(x, 5, wr, b), (wr,), dy)
    gb, = torch.autograd.grad(dr.group_norm(x, 5, w, br), (br,), dy)
    (gn,) = torch.autograd.grad(dr.group_norm(x, 5, None, br), (br,), dy)
    ref = reference(x, w, b, 5, 1e-5, "none", dy)
    for got, kind in zip((*full, gx, gw, gb), 2 * ("dx", "dweight", "dbias")):
        check(got, ref, kind)
    check(gn, reference(x, None, b, 5, 1e-5, "none", dy), "dbias")
    y, mean, rstd = ops.group_norm(x, 5, w, b, stats=True)
    got = ops.group_norm_grad(dy, x, 5, w, b, mean, rstd,
                              want=(False, True, False))
    assert got[0] is None and got[2] is None
    check(got[1], ref, "dweight")
    # tables in 16 bits are widened, and their gradients come back in 16
    wh = w.half().requires_grad_(True)
    (gh,) = torch.autograd.grad(dr.group_norm(x, 5, wh, b), (wh,), dy)
    assert gh.dtype == torch.float16


def test_more_samples_than_a_grid_counts(cuda):
    """Over 65535 samples: resident, and (table gradients only) in rounds."""
    torch = _torch()
    from opendressi_b200 import ops

    x, dy, w, b = make(17, (70001, 3, 8), torch.float32)
    y, mean, rstd = ops.group_norm(x, 2, w, b, activation="silu", stats=True)
    ref = reference(x, w, b, 2, 1e-5, "silu", dy)
    check(y, ref, "y")
    for want in ((True, True, True), (False, True, True)):
        dx, dw, db = ops.group_norm_grad(dy, x, 2, w, b, mean, rstd,
                                         activation="silu", want=want)
        if want[0]:
            check(dx, ref, "dx")
        check(dw, ref, "dweight")
        check(db, ref, "dbias")


@pytest.mark.parametrize("shape", [(0, 4, 4, 8), (3, 0, 4, 8), (2, 0, 8)])
def test_nothing_to_normalise(cuda, shape):
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    x = torch.empty(shape, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    b = torch.ones(8, device="cuda", requires_grad=True)
    y = dr.group_norm(x, 2, w, b, activation="silu")
    assert y.shape == shape
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert gx.shape == shape and not gw.any() and not gb.any()


def test_not_finite_stays_in_its_group(cuda):
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    for bad in (math.nan, math.inf, -math.inf):
        for act in ("none", "relu", "silu"):
            x, _, w, b = make(11, (2, 6, 5, 12), torch.float32)
            clean = dr.group_norm(x, 3, w, b, activation=act)
            x[1, 3, 2, 5] = bad  # sample 1, group 1
            y = dr.group_norm(x, 3, w, b, activation=act)
            hit = torch.zeros_like(y, dtype=torch.bool)
            hit[1, :, :, 4:8] = True
            assert torch.equal(y[~hit], clean[~hit])
            assert torch.isnan(y[hit]).all()
    # a group of one pixel and one channel that is infinite
    x = torch.full((1, 1, 1, 1), math.inf, device="cuda")
    assert torch.isnan(dr.group_norm(x, 1)).all()
    # two values, the second infinite: met by one thread
    x = torch.tensor([1.0, math.inf], device="cuda").reshape(1, 2, 1)
    assert torch.isnan(dr.group_norm(x, 1)).all()


def test_constant_groups(cuda):
    """Variance 0 and, with eps 0, the deviation's own limit."""
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    x = torch.full((2, 33, 5, 8), 3.7, device="cuda")
    b = torch.arange(8.0, device="cuda")
    assert torch.equal(dr.group_norm(x, 2, None, b), b.expand_as(x))


def test_repeats_bit_for_bit(cuda):
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    x, dy, w, b = make(13, (2, 256, 250, 32), torch.bfloat16)
    for t in (x, w, b):
        t.requires_grad_(True)
    runs = []
    for _ in range(3):
        y = dr.group_norm(x, 8, w, b, activation="silu")
        runs.append([y, *torch.autograd.grad(y, (x, w, b), dy)])
    for r in runs[1:]:
        for a, e in zip(r, runs[0]):
            assert torch.equal(a, e)


@pytest.mark.parametrize("side", [12, 200])
def test_captured_and_on_another_stream(cuda, side):
    """Forward and backward captured together, replayed on new inputs; two
    captured graphs replayed at once; an eager call on a side stream."""
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    sets = []
    for k in range(2):
        x, dy, w, b = make(20 + k, (2, side, side, 24), torch.float32)
        for t in (x, w, b):
            t.requires_grad_(True)
        sets.append((x, dy, w, b))

    def step(s):
        x, dy, w, b = s
        y = dr.group_norm(x, 6, w, b, activation="silu")
        return [y, *torch.autograd.grad(y, (x, w, b), dy)]

    side_stream = torch.cuda.Stream()
    side_stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side_stream):
        eager = [step(s) for s in sets]
    torch.cuda.current_stream().wait_stream(side_stream)
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, e in zip(outs, eager):
        for a, b in zip(o, e):
            assert torch.equal(a, b)
    # new inputs in the captured addresses
    with torch.no_grad():
        sets[0][0].copy_(sets[1][0])
        sets[0][1].copy_(sets[1][1])
        sets[0][2].copy_(sets[1][2])
        sets[0][3].copy_(sets[1][3])
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs[0], eager[1]):
        assert torch.equal(a, b)


def test_traced_by_compile(cuda):
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    x, dy, w, b = make(30, (2, 14, 9, 16), torch.bfloat16)
    for t in (x, w, b):
        t.requires_grad_(True)

    def f(x, w, b):
        return dr.group_norm(x * 2.0, 4, w, b, activation="silu")

    torch.compiler.reset()
    g = torch.compile(f, backend="aot_eager", fullgraph=True)
    y1, y2 = f(x, w, b), g(x, w, b)
    assert torch.equal(y1, y2)
    for a, e in zip(torch.autograd.grad(y2, (x, w, b), dy),
                    torch.autograd.grad(y1, (x, w, b), dy)):
        assert torch.equal(a, e)
    torch.library.opcheck(
        torch.ops.dressi_b200.group_norm,
        (x.detach(), w.detach(), b.detach(), 4, 1e-5, "silu"),
        test_utils=("test_schema", "test_faketensor"))


def test_more_values_than_32_bits_count(cuda):
    """An image of more than 2^32 values: offsets past 32 bits, in the last
    rows of the last sample."""
    torch = _torch()
    from opendressi_b200 import ops

    free, _ = torch.cuda.mem_get_info()
    n, rows, c = 3, (1 << 25) + 3, 48  # 4.83e9 values, 9.7 GB each
    if free < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    x = torch.empty((n, rows, c), dtype=torch.bfloat16, device="cuda")
    ramp = torch.linspace(-1, 1, 64 * c, device="cuda").to(
        torch.bfloat16).view(64, c)
    x[:, :rows - 3].view(n, -1, 64, c)[:] = ramp  # repeats: known statistics
    x[:, rows - 3:] = ramp[:3]
    y, mean, rstd = ops.group_norm(x, 4, stats=True)
    tail = x[:, -5:].double().reshape(n, 5, 4, 12)
    exp = (tail - mean.double()[:, None, :, None]) * \
        rstd.double()[:, None, :, None]
    got = y[:, -5:].double().reshape(n, 5, 4, 12)
    assert ((got - exp).abs() <= 2 ** -8 * exp.abs() + K * U * 4).all()
    m = ramp.double().view(64, 4, 12).mean((0, 2))
    # 3 rows in 2^25 shift the mean by less than 1e-6
    assert ((mean - m).abs() < 1e-5).all()


def test_refusals(cuda):
    torch = _torch()
    from opendressi_b200 import DressiError, ops, torch_api as dr

    x = torch.randn(2, 4, 4, 12, device="cuda")
    ok = torch.ones(12, device="cuda")
    for args, kw in [
            ((x.cpu(), 3), {}), ((x.double(), 3), {}), ((x, 5), {}),
            ((x, 0), {}), ((x, -3), {}), ((x[0, 0, 0], 3), {}),
            ((x, 3, ok[:6]), {}), ((x, 3, ok.cpu()), {}),
            ((x, 3, None, ok[None]), {}),
            ((x, 3), {"activation": "gelu"}), ((x, 3), {"eps": -1.0}),
            ((x, 3), {"eps": math.nan}),
            ((torch.empty(2, 4, 0, device="cuda"), 1), {})]:
        with pytest.raises(DressiError):
            dr.group_norm(*args, **kw)
    y, mean, rstd = ops.group_norm(x, 3, stats=True)
    for dy in (x[:1], x.half(), x.cpu()):
        with pytest.raises(DressiError):
            ops.group_norm_grad(dy, x, 3, None, None, mean, rstd)
    with pytest.raises(DressiError):
        ops.group_norm_grad(x, x, 3, None, None, mean[:1], rstd)
    assert np.isfinite(float(y.sum()))


def test_differentiable_once(cuda):
    """A second derivative is refused, not taken as zero."""
    torch = _torch()
    from opendressi_b200 import torch_api as dr

    x, dy, w, b = make(31, (2, 4, 3, 8), torch.float32)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = dr.group_norm(x, 2, w, b, activation="silu")
    plain = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    grads = torch.autograd.grad(y, (x, w, b), dy, create_graph=True)
    for a, e in zip(grads, plain):
        assert torch.equal(a, e)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(grads[0].sum(), x)
