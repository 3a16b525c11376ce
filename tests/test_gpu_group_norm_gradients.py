"""Every gradient of group_norm over all mappings, relu's too: against the
formulas in 64 bits with the tolerances of test_gpu_group_norm.py.

A value whose z lies within its own rounding error of relu's kink may pass its
gradient or not. Its dz is then off by |dy| at most; the sums and the means of
its group carry that, all other values are held to what they round."""

import math

import pytest

import test_gpu_group_norm as base

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]
SHAPES = pytest.mark.parametrize(
    "shape,groups", base.SHAPES,
    ids=["x".join(map(str, s)) + f"g{g}" for s, g in base.SHAPES])


def reference(x, weight, bias, groups, eps, act, dy):
    """base.reference with what the kink leaves open in its errors."""
    import torch

    ref = base.reference(x, weight, bias, groups, eps, act, dy)
    n, c = x.shape[0], x.shape[-1]
    shape = (n, -1, groups, c // groups)
    h = ((x.detach().double().reshape(shape)
          - ref["mean"].reshape(n, 1, groups, 1))
         * ref["rstd"].reshape(n, 1, groups, 1))
    w = torch.ones((), device=x.device, dtype=torch.float64) \
        if weight is None else weight.detach().double().reshape(
            1, 1, groups, -1)
    open_ = dy.double().abs().reshape(shape) * ref["kink"].reshape(shape)
    gw = open_ * w.abs()
    ref["dx_err"] = ref["dx_err"] + (
        ref["rstd"].reshape(n, 1, groups, 1)
        * (gw + gw.mean((1, 3), keepdim=True) + h.abs()
           * (gw * h.abs()).mean((1, 3), keepdim=True))).reshape(x.shape)
    ref["dweight_err"] = ref["dweight_err"] + (
        open_ * h.abs()).sum((0, 1)).reshape(-1)
    ref["dbias_err"] = ref["dbias_err"] + open_.sum((0, 1)).reshape(-1)
    # z's error is some 1e-5 of its range: few values lie that near to 0 (all
    # do where a group is one value and has no bias: z is 0 then)
    if h.shape[1] * h.shape[3] > 1 or bias is not None:
        assert int(ref["kink"].sum()) <= 1 + 0.01 * x.numel()
    return ref


def check(got, ref, kind):
    """|got - exact| <= its error and half a step of its type; a value that is
    not a number is none of them."""
    import torch

    exp, err = ref[kind], ref[kind + "_err"]
    assert torch.isfinite(exp).all() and torch.isfinite(err).all()
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * 2 * half
    tol = err * (1 + half) + half * exp.abs() + tiny
    off = (got.detach().double() - exp).abs()
    assert got.shape == exp.shape
    assert (off <= tol).all(), (kind, int((~(off <= tol)).sum()),
                                float((off / tol).max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "silu", "none"])
@SHAPES
def test_gradients(cuda, shape, groups, dtype, act):
    import torch

    from opendressi_b200 import torch_api as dr

    for affine in (True, False):
        x, dy, w, b = base.make(41 + affine, shape, getattr(torch, dtype),
                                affine)
        leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
        y = dr.group_norm(x, groups, w, b, activation=act)
        grads = torch.autograd.grad(y, leaves, dy)
        ref = reference(x, w, b, groups, 1e-5, act, dy)
        check(y, ref, "y")
        for got, kind in zip(grads, ("dx", "dweight", "dbias")):
            check(got, ref, kind)


def test_more_samples_than_a_grid_counts(cuda):
    import torch

    from opendressi_b200 import ops

    for act in ("relu", "silu"):
        x, dy, w, b = base.make(42, (70001, 3, 8), torch.bfloat16)
        y, mean, rstd = ops.group_norm(x, 2, w, b, activation=act, stats=True)
        ref = reference(x, w, b, 2, 1e-5, act, dy)
        check(y, ref, "y")
        for want in ((True, True, True), (False, True, True)):
            got = ops.group_norm_grad(dy, x, 2, w, b, mean, rstd,
                                      activation=act, want=want)
            for t, kind in zip(got, ("dx", "dweight", "dbias")):
                if t is not None:
                    check(t, ref, kind)


def test_several_rounds_of_launches(cuda):
    """Samples of 90 MB, more than one round takes together."""
    import torch

    from opendressi_b200 import torch_api as dr

    x, dy, w, b = base.make(44, (3, 700, 801, 40), torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = dr.group_norm(x, 10, w, b, activation="silu")
    grads = torch.autograd.grad(y, leaves, dy)
    for k in range(3):  # sample by sample: the reference is large
        xs = x.detach()[k:k + 1]
        ref = reference(xs, w, b, 10, 1e-5, "silu", dy[k:k + 1])
        check(y[k:k + 1], ref, "y")
        check(grads[0][k:k + 1], ref, "dx")
        sums = ref if k == 0 else {t: sums[t] + ref[t] for t in (
            "dweight", "dbias", "dweight_err", "dbias_err")}
    check(grads[1], sums, "dweight")
    check(grads[2], sums, "dbias")


@pytest.mark.parametrize("far", [1e2, 1e4, 1e6])
@pytest.mark.parametrize("shape,groups,steps", [
    ((1, 64, 64, 32), 8, 4), ((3, 40, 40, 16), 4, 13),
    ((8, 256, 256, 64), 16, 56), ((1, 2048, 2048, 32), 8, 222),
    ((2, 1201, 1013, 3), 1, 139)])
def test_values_far_from_the_others(cuda, shape, groups, steps, far):
    """A bright corner, the first row, the last row: what a thread meets first
    must not cancel its sums. A sum of squares about a centre is at most 4
    times what it is about the mean; its `steps` roundings of 2^-24 (of either
    sign) add up to sqrt(steps) of them, the rest is the 64 of `base`, which
    cover 32."""
    import torch

    from opendressi_b200 import ops

    tol = base.K * base.U * max(1.0, math.sqrt(steps / 32.0))
    for where in ((0, 0), (0,), (-1,), (0, slice(None, None, 7))):
        g = torch.Generator(device="cuda").manual_seed(9)
        x = torch.randn(shape, generator=g, device="cuda")
        x[(slice(None), *where)] += far
        y, mean, rstd = ops.group_norm(x, groups, stats=True)
        n, c = shape[0], shape[-1] // groups
        for k in range(groups):
            d = x[..., k * c:(k + 1) * c].reshape(n, -1).double()
            mu = d.mean(1, keepdim=True)
            dev = (((d - mu) ** 2).mean(1) + 1e-5).sqrt()
            assert ((rstd[:, k].double() * dev - 1).abs() <= tol).all()
            # 8 roundings of the largest distance from it (the proof stands in
            # test_gpu_group_norm.py: a thread's mean is its centre and a mean
            # of distances from there, 3 roundings of at most twice that, and
            # those of the sum) and the mean's own
            reach = (d - mu).abs().amax(1)
            assert ((mean[:, k].double() - mu[:, 0]).abs() <=
                    base.U * (8 * reach + mu[:, 0].abs())).all()


@pytest.mark.parametrize("size", [1e-18, 1.0, 1e15])
def test_no_eps(cuda, size):
    """With eps 0 the deviation alone scales: any size of values gives the
    same."""
    import torch

    from opendressi_b200 import torch_api as dr

    for shape in ((2, 9, 7, 12), (1, 200, 180, 12)):
        x, dy, w, b = base.make(43, shape, torch.float32)
        x = (x * size).requires_grad_(True)
        y = dr.group_norm(x, 3, w, b, eps=0.0, activation="silu")
        (dx,) = torch.autograd.grad(y, (x,), dy)
        ref = reference(x, w, b, 3, 0.0, "silu", dy)
        check(y, ref, "y")
        check(dx, ref, "dx")
    # 0 / 0 as the formula has it, in that group alone
    x = torch.randn((1, 6, 5, 12), device="cuda")
    x[..., 4:8] = 3.0
    y = dr.group_norm(x, 3, eps=0.0)
    assert torch.isnan(y[..., 4:8]).all()
    assert torch.isfinite(y[..., :4]).all() and math.isfinite(
        float(y[..., 8:].sum()))
