"""What autograd, forward mode and tracing see of the learning operators."""

import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def leaves(*shapes, dtype=None):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(3)
    return [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda")
                               .to(dtype or torch.float32)) for s in shapes]


# ------------------------------------------------------------------ versions

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_graph_of_the_values_before_a_step_is_refused(cuda, dtype, bits):
    torch = _torch()
    from opendressi_b200 import optim

    p, q = leaves((300,), (7, 5), dtype=getattr(torch, dtype))
    opt = optim.AdamW([p, q], state_bits=bits)
    loss = (p * p).sum() + (q * q).sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_versions_grow_where_a_step_writes(cuda, bits):
    torch = _torch()
    from opendressi_b200 import optim

    a, late, b = leaves((300,), (9,), (33, 4))
    (h,) = leaves((70,), dtype=torch.float16)
    opt = optim.AdamW([{"params": [a, late]}, {"params": [b, h]}],
                      state_bits=bits, max_norm=1.0)
    for p in (a, b, h):
        p.grad = torch.ones_like(p)
    watched = {"last_norm": opt.last_norm}
    for g in range(2):
        for k, t in opt.packed_state(g).items():
            watched[k, g] = t
    watched["a"], watched["b"], watched["h"] = a, b, h
    watched["view"] = opt.state[a]["exp_avg"]
    before = {k: t._version for k, t in watched.items()}
    kept = late._version, a.grad._version
    opt.step()
    for k, t in watched.items():
        assert t._version > before[k], k
    assert (late._version, a.grad._version) == kept


def test_norm_into_a_tensor_that_a_graph_keeps(cuda):
    torch = _torch()
    from opendressi_b200 import DressiError, optim

    (p,) = leaves((300,))
    out = torch.ones((), device="cuda")
    w = torch.ones((), device="cuda", requires_grad=True)
    kept = w * out
    got = optim.grad_norm([p], out=out)
    assert got.data_ptr() == out.data_ptr() and not got.requires_grad
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        kept.backward()
    with pytest.raises(DressiError, match="requires a gradient"):
        optim.grad_norm([p], out=w)


# -------------------------------------------------------------- forward mode

@pytest.mark.parametrize("which", ["x", "weight", "bias"])
@pytest.mark.parametrize("with_grad", [False, True])
def test_forward_mode_is_refused(cuda, which, with_grad):
    """A tangent is not dropped, which would read as a derivative of zero."""
    torch = _torch()
    import torch.autograd.forward_ad as fw

    from opendressi_b200 import torch_api as dr

    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((2, 5, 4, 8), generator=g, device="cuda")
    args = {"x": x, "weight": torch.ones(8, device="cuda"),
            "bias": torch.zeros(8, device="cuda")}
    clean = dr.group_norm(num_groups=2, **args)
    with fw.dual_level():
        primal = args[which].clone().requires_grad_(with_grad)
        dual = fw.make_dual(primal, torch.ones_like(primal))
        with pytest.raises(RuntimeError, match="forward"):
            dr.group_norm(num_groups=2, **{**args, which: dual})
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
            dr.group_norm(num_groups=2, **{**args, which: dual})
        # where tangents are switched off none is expected
        with fw._set_fwd_grad_enabled(False):
            y = dr.group_norm(num_groups=2, **{**args, which: dual})
        assert torch.equal(y, clean)
        # a call without one inside a dual level
        assert torch.equal(dr.group_norm(num_groups=2, **args), clean)

    def f(t):
        return dr.group_norm(num_groups=2, **{**args, which: t})

    with pytest.raises(RuntimeError, match="forward"):
        torch.func.jvp(f, (args[which],), (torch.ones_like(args[which]),))


# ------------------------------------------------------------------- tracing

def inputs(seed):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=g, device="cuda")

    return normal(2, 9, 7, 12) + 1, 1 + normal(12) / 4, normal(12)


def norm(x, w, b):
    from opendressi_b200 import torch_api as dr

    return dr.group_norm(x * 2.0, 3, w, b, activation="silu") + 1.0


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_traced_by_make_fx(cuda, mode):
    torch = _torch()
    from torch.fx.experimental.proxy_tensor import make_fx

    traced = make_fx(norm, tracing_mode=mode)(*inputs(1))
    assert any("dressi_b200.group_norm" in str(n.target)
               for n in traced.graph.nodes)
    new = inputs(2)
    torch.empty(1 << 20, device="cuda").fill_(7.0)  # what memory held before
    assert torch.equal(traced(*new), norm(*new))


def test_traced_by_jit(cuda):
    torch = _torch()
    with torch.no_grad():
        traced = torch.jit.trace(norm, inputs(1))
        assert "dressi_b200::group_norm" in str(traced.graph)
        new = inputs(2)
        assert torch.equal(traced(*new), norm(*new))


def test_functional_transforms(cuda):
    """vmap takes sample after sample; grad is refused."""
    torch = _torch()
    x, w, b = inputs(3)
    xs = torch.stack([x, x + 1.0, -x])
    got = torch.vmap(lambda t: norm(t, w, b))(xs)
    assert torch.equal(got, torch.stack([norm(t, w, b) for t in xs]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: norm(t, w, b).square().sum())(x)


def test_a_dispatch_mode_sees_the_operator(cuda):
    torch = _torch()
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    args = inputs(5)
    with Log():
        y = norm(*args)
    assert any("dressi_b200.group_norm" in s for s in seen)
    assert torch.equal(y, norm(*args))


def test_selective_recomputation(cuda):
    """Checkpointing that keeps some operators' results runs under a dispatch
    mode: what it recomputes is computed."""
    torch = _torch()
    from torch.utils import checkpoint as ck

    def policy(ctx, op, *a, **k):
        return (ck.CheckpointPolicy.MUST_SAVE if "empty" in str(op)
                else ck.CheckpointPolicy.PREFER_RECOMPUTE)

    x, w, b = inputs(6)

    def f(x, w, b):
        return norm(norm(x, w, b), w, b)

    def gradients(call):
        ts = [t.clone().requires_grad_(True) for t in (x, w, b)]
        return torch.autograd.grad(call(*ts).square().sum(), ts)

    got = gradients(lambda *t: ck.checkpoint(
        f, *t, use_reentrant=False,
        context_fn=lambda: ck.create_selective_checkpoint_contexts(policy)))
    for a, e in zip(got, gradients(f)):
        assert torch.equal(a, e)


def test_norm_and_step_refuse_a_trace(cuda):
    """Their result is not a value of the trace, and their writes no part of
    it: better refused than left out."""
    torch = _torch()
    from torch.fx.experimental.proxy_tensor import make_fx

    from opendressi_b200 import DressiError, optim

    (p,) = leaves((300,))
    p.grad = torch.ones_like(p)
    opt = optim.AdamW([p])
    before = p.detach().clone()

    def step(t):
        opt.step()
        return t + 1.0

    for trace in (lambda f: make_fx(f)(p.grad),
                  lambda f: torch.jit.trace(f, (p.grad,))):
        with pytest.raises(DressiError, match="traced"):
            trace(lambda t: optim.grad_norm([t]) + 1.0)
        with pytest.raises(DressiError, match="traced"):
            trace(step)
    assert torch.equal(p, before)
    assert int(opt.state[p]["step"]) == 0
    # other dispatch modes look on
    from torch.utils.flop_counter import FlopCounterMode

    with FlopCounterMode(display=False):
        opt.step()
        n = optim.grad_norm([p.grad])
    assert int(opt.state[p]["step"]) == 1 and float(n) > 17.3


# ---------------------------------------------------------------- relu's kink

@pytest.mark.parametrize("rows", [23, 600])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_relu_gradient_where_its_output_is_not_zero(cuda, dtype, rows):
    """The backward pass takes a value for positive exactly where the forward
    pass did, to the last bit: biases put one value of each channel next to
    zero. dbias is then a sum of powers of two, one for each positive value of
    23 rows (the others have no gradient)."""
    import torch

    from opendressi_b200 import ops

    dtype = getattr(torch, dtype)
    c = 512
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randn((1, rows, c), generator=g, device="cuda") + 2).to(dtype)
    w = 1 + 0.3 * torch.randn(c, generator=g, device="cuda")
    y, mean, rstd = ops.group_norm(x, 16, w, None, stats=True)
    e = x[0].float() - mean.repeat_interleave(c // 16, 1)
    z = e * (rstd.repeat_interleave(c // 16, 1) * w)
    k = torch.arange(c, device="cuda") % 23
    b = -z.gather(0, k[None]).reshape(-1).contiguous()
    y, mean, rstd = ops.group_norm(x, 16, w, b, activation="none", stats=True)
    small = (y[0].float().abs() < 1e-6).sum()
    assert int(small) >= c // 4  # the biases reach the kink
    dy = torch.zeros((1, rows, c), device="cuda")
    dy[0, :23] = 2.0 ** (torch.arange(23, device="cuda") - 11)[:, None]
    for want in ((True, True, True), (False, False, True)):
        _, _, db = ops.group_norm_grad(dy.to(dtype), x, 16, w, b, mean, rstd,
                                       activation="relu", want=want)
        on = (db.double() * 2.0 ** 11).long()
        relu = ops.group_norm(x, 16, w, b, activation="relu")[0, :23]
        # a positive value may round to 0 in the output's type; f32 does not
        bits = (y[0, :23].float() > 0) if dtype == torch.float32 else relu > 0
        said = (on[None] >> torch.arange(23, device="cuda")[:, None]) & 1
        if dtype == torch.float32:
            assert torch.equal(said.bool(), bits)
        else:
            assert not (bits & ~said.bool()).any()
            assert not ((y[0, :23].float() < 0) & said.bool()).any()


def test_lazily_negated_tensors(cuda):
    """Tensors whose sign is a bit of theirs (the imaginary part of a lazily
    conjugated tensor): their values count, not what memory holds."""
    import torch

    from opendressi_b200 import ops, optim, torch_api as dr

    x, w, b = inputs(7)
    dy = torch.randn_like(x)
    nx, nw, nb, ndy = (torch._neg_view(-t) for t in (x, w, b, dy))
    assert nx.is_neg() and nx.is_contiguous() and torch.equal(nx, x)
    y, mean, rstd = ops.group_norm(x, 3, w, b, activation="silu", stats=True)
    for got in (ops.group_norm(nx, 3, nw, nb, activation="silu"),
                dr.group_norm(nx, 3, w, b, activation="silu"),
                dr.group_norm(x, 3, nw, nb, activation="silu")):
        assert torch.equal(got, y)
    want = ops.group_norm_grad(dy, x, 3, w, b, mean, rstd, activation="silu")
    for got in (ops.group_norm_grad(ndy, nx, 3, nw, nb, torch._neg_view(-mean),
                                    torch._neg_view(-rstd),
                                    activation="silu"),):
        for a, e in zip(got, want):
            assert torch.equal(a, e)
    leaf = x.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(dr.group_norm(leaf, 3, w, b,
                                              activation="silu"), leaf, ndy)
    assert torch.equal(gx, want[0])

    p, q = leaves((300,), (300,))
    with torch.no_grad():
        q.copy_(p)
    p.grad = torch.randn_like(p)
    q.grad = torch._neg_view(-p.grad)
    for t in (p, q):
        optim.AdamW([t], max_norm=1.0).step()
    assert torch.equal(p, q)
    from opendressi_b200 import DressiError

    with pytest.raises(DressiError):
        optim.AdamW([torch.nn.Parameter(torch._neg_view(x))])
    opt = optim.AdamW([p])
    p.data = torch._neg_view(p.detach())
    for call in (opt.step, lambda: optim.grad_norm(
            [x], out=torch._neg_view(torch.ones((), device="cuda")))):
        with pytest.raises(DressiError):
            call()
