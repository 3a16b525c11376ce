"""The learning operators at their far sizes: values that 32 bits do not
count, and rows of a million channels."""

import math

import pytest

import test_gpu_group_norm as base
import test_gpu_group_norm_gradients as grads

pytestmark = pytest.mark.gpu


def room(gb):
    import torch

    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip(f"needs {gb} GB of free device memory")


@pytest.mark.parametrize("bits", [32, 8])
def test_step_of_more_values_than_32_bits_count(cuda, bits):
    """Gradients in the first and the last values alone: a first step moves
    those by lr (eps aside), no other, and the norm is theirs."""
    import torch

    from opendressi_b200 import optim

    room(70)
    n, ends = (1 << 32) + 777, 5000
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    g = torch.randn(2, ends, device="cuda").to(torch.bfloat16)
    g[g.abs() < 0.01] = 1.0
    p.grad[:ends], p.grad[-ends:] = g[0], g[1]
    opt = optim.AdamW([p], lr=2.0 ** -6, eps=0.0, weight_decay=0.0,
                      state_bits=bits, max_norm=1e9)
    opt.step()
    # m / sqrt(v) is sign(g) to some 2^-20: one rounding away from 2^-6
    step = 2.0 ** -6
    for got, grad in ((p.detach()[:ends], g[0]), (p.detach()[-ends:], g[1])):
        assert ((got.double() + step * grad.double().sign()).abs() <=
                2.0 ** -8 * step).all()
    # 0 / 0 as the formula has it where there was never a gradient
    assert torch.isnan(p.detach()[ends:ends + 999]).all()
    norm = math.sqrt(float((g.double() ** 2).sum()))
    assert abs(float(opt.last_norm) / norm - 1) <= 2 * base.U
    m = opt.state[p]["exp_avg"]
    assert bool((m[-ends:].float() != 0).all())
    assert not m[ends:1 << 20].float().any()


def test_gradient_of_more_values_than_32_bits_count(cuda):
    """A periodic image: its sums are known, its last rows are looked at."""
    import torch

    from opendressi_b200 import ops

    room(60)
    rows, c, per, groups = (1 << 25) + 64, 136, 64, 4
    x = torch.empty((1, rows, c), dtype=torch.bfloat16, device="cuda")
    dy = torch.empty_like(x)
    a, b = (torch.randn(per, c, device="cuda").to(torch.bfloat16)
            for _ in range(2))
    x.view(-1, per, c)[:] = a
    dy.view(-1, per, c)[:] = b
    assert x.numel() > 1 << 32
    y, mean, rstd = ops.group_norm(x, groups, stats=True)
    w = torch.ones(c, device="cuda")
    dx, dw, db = ops.group_norm_grad(dy, x, groups, w, 0 * w, mean, rstd)
    ref = grads.reference(a[None], w, 0 * w, groups, 1e-5, "none", b[None])
    assert ((mean.double() - ref["mean"]).abs() <= 1e-6).all()
    # A thread adds 7600 values in 32 bits (a 296th of the rows, 15 lanes of a
    # block). Each addition rounds by U of the running sum at most, which grows
    # to the sum of their sizes: on average half of it, 7600 / 2 U in all. They
    # need not cancel: the terms repeat, and so do their roundings.
    tol = 3800 * base.U
    times = rows // per
    sizes = {}
    for got, kind, other in ((dw, "dweight", ref["y"][0]), (db, "dbias", 1.0)):
        sizes[kind] = (b.double() * other).abs().sum(0)
        assert ((got.double() - times * ref[kind]).abs() <=
                tol * sizes[kind] * times).all()
    # dx takes the means of those sums over a group: off by tol of their terms
    share = {k: v.reshape(groups, -1).mean(1).repeat_interleave(c // groups)
             / per for k, v in sizes.items()}
    more = tol * (rstd.double().repeat_interleave(c // groups, 1)[0]
                  * (share["dbias"] + ref["y"][0].abs() * share["dweight"]))
    for got, kind, wide in ((y, "y", 0.0), (dx, "dx", more)):
        for at in (slice(0, per), slice(rows - per, rows)):
            exp = ref[kind][0]
            off = (got[0, at].double() - exp).abs()
            assert (off <= 2.0 ** -8 * exp.abs() + 4 * ref[kind + "_err"][0]
                    + wide).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape,groups", [
    ((2, 3, 1 << 20), 4), ((2, 3, 1 << 20), 1 << 20), ((1, 2, 1000003), 1),
    ((1, 5, 999990), 333330)])
def test_rows_of_a_million_channels(cuda, shape, groups, dtype):
    import torch

    from opendressi_b200 import torch_api as dr

    x, dy, w, b = base.make(51, shape, getattr(torch, dtype))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = dr.group_norm(x, groups, w, b, activation="silu")
    got = torch.autograd.grad(y, leaves, dy)
    ref = grads.reference(x, w, b, groups, 1e-5, "silu", dy)
    grads.check(y, ref, "y")
    for t, kind in zip(got, ("dx", "dweight", "dbias")):
        grads.check(t, ref, kind)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_copies_gradients_of_another_order(cuda, bits):
    import torch

    from opendressi_b200 import optim

    t = torch.randn(40, 24, device="cuda")
    p, q = (torch.nn.Parameter(t.clone()) for _ in range(2))
    p.grad = torch.zeros(24, 40, device="cuda").t()
    q.grad = torch.zeros(40, 24, device="cuda")
    a, b = (optim.AdamW([v], state_bits=bits, max_norm=1.0) for v in (p, q))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(3):
        g = torch.randn_like(t)
        p.grad.copy_(g)
        q.grad.copy_(g)
        graph.replay()
        b.step()
    assert torch.equal(p, q)
    assert torch.equal(a.last_norm, b.last_norm)
