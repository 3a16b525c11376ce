"""AdamW's options and tensors where a program changes them between steps."""

import math

import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def leaves(*shapes):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(8)
    out = [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda"))
           for s in shapes]
    for p in out:
        p.grad = torch.randn(p.shape, generator=g, device="cuda")
    return out


def tensor_lr(value):
    return _torch().tensor(value, device="cuda")


# ---------------------------------------------------------- loaded options

def test_loading_shares_no_learning_rate(cuda):
    torch = _torch()
    from opendressi_b200 import optim

    a = optim.AdamW(leaves((9,)), lr=tensor_lr(0.125))
    b = optim.AdamW(leaves((9,)), lr=tensor_lr(0.5))
    c = optim.AdamW(leaves((9,)), lr=0.5, clamp=[0.0, 1.0])
    own = b.param_groups[0]["lr"]
    b.load_state_dict(a.state_dict())
    c.load_state_dict(a.state_dict())
    assert b.param_groups[0]["lr"] is own and float(own) == 0.125
    got = c.param_groups[0]["lr"]
    assert got.is_cuda and float(got) == 0.125
    a.param_groups[0]["lr"].fill_(0.25)
    assert float(own) == 0.125 and float(got) == 0.125
    # a number into a tensor, a CPU copy into a tensor, a list is copied
    number = optim.AdamW(leaves((9,)), lr=0.0625, clamp=[0.0, 2.0])
    b.load_state_dict(number.state_dict())
    assert b.param_groups[0]["lr"] is own and float(own) == 0.0625
    assert b.param_groups[0]["clamp"] == [0.0, 2.0]
    assert b.param_groups[0]["clamp"] is not number.param_groups[0]["clamp"]
    state = a.state_dict()
    state["param_groups"][0]["lr"] = torch.tensor(0.75, dtype=torch.float64)
    b.load_state_dict(state)
    assert b.param_groups[0]["lr"] is own and float(own) == 0.75


@pytest.mark.parametrize("bad", [-1.0, math.nan, math.inf])
def test_a_refused_load_changes_nothing(cuda, bad):
    torch = _torch()
    from opendressi_b200 import optim

    a = optim.AdamW(leaves((9,), (4,)), lr=tensor_lr(0.125))
    a.step()
    b = optim.AdamW([{"params": p} for p in leaves((9,), (4,))], lr=0.5)
    one = optim.AdamW([{"params": p} for p in leaves((9,), (4,))], lr=0.25)
    one.step()
    for lr in (bad, torch.tensor(bad)):
        state = one.state_dict()
        state["param_groups"][1]["lr"] = lr
        with pytest.raises(ValueError):
            b.load_state_dict(state)
        assert [g["lr"] for g in b.param_groups] == [0.5, 0.5]
        assert not b.packed_state()["exp_avg"].any()


def test_a_captured_step_reads_a_loaded_learning_rate(cuda):
    torch = _torch()
    from opendressi_b200 import optim

    pa, pb = leaves((700,), (3, 5)), leaves((700,), (3, 5))
    a = optim.AdamW(pa, lr=tensor_lr(2.0 ** -7))
    b = optim.AdamW(pb, lr=2.0 ** -7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    saved = b.state_dict()
    saved["param_groups"][0]["lr"] = 2.0 ** -4
    saved = {**saved, "state": {k: {n: t.clone() for n, t in v.items()}
                                for k, v in saved["state"].items()}}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    a.load_state_dict(saved)
    b.load_state_dict(saved)
    graph.replay()
    b.step()
    a.param_groups[0]["lr"].fill_(2.0 ** -3)
    b.param_groups[0]["lr"] = 2.0 ** -3
    graph.replay()
    b.step()
    for x, y in zip(pa, pb):
        assert torch.equal(x, y)


def test_load_hooks_run(cuda):
    from opendressi_b200 import optim

    a, b = optim.AdamW(leaves((9,)), lr=0.125), optim.AdamW(leaves((9,)))
    seen = []

    def before(opt, state):
        seen.append("before")
        state = dict(state)
        state["param_groups"] = [{**g, "lr": 0.75}
                                 for g in state["param_groups"]]
        return state

    b.register_load_state_dict_pre_hook(before)
    b.register_load_state_dict_post_hook(lambda opt: seen.append(
        opt.param_groups[0]["lr"]))
    b.load_state_dict(a.state_dict())
    assert seen == ["before", 0.75]


# ------------------------------------------------------- changed parameters

def test_a_parameter_of_another_shape_is_refused(cuda):
    """Also one with as many values and the same strides, which are then no
    longer dense: (3, 2) cut out of (3, 3), or one value as six."""
    torch = _torch()
    from opendressi_b200 import DressiError, optim

    wide = torch.randn(3, 3, device="cuda")
    p = torch.nn.Parameter(torch.randn(2, 3, device="cuda"))
    opt = optim.AdamW([p])
    p.data = wide[:, :2]
    p.grad = torch.ones_like(p)
    assert p.stride() == (3, 1) and p.numel() == 6
    before = wide.clone()
    with pytest.raises(DressiError, match="changed"):
        opt.step()
    row = torch.randn(1, 6, device="cuda").as_strided((1, 6), (0, 1))
    q = torch.nn.Parameter(row)
    opt = optim.AdamW([q])
    one = torch.randn(8, device="cuda")
    q.data = one[:1].as_strided((6, 1), (0, 1))
    q.grad = torch.ones(6, 1, device="cuda")
    assert q.numel() == 6
    kept = one.clone()
    with pytest.raises(DressiError, match="changed"):
        opt.step()
    assert torch.equal(wide, before) and torch.equal(one, kept)


def test_a_group_that_fails_to_be_added_leaves_no_trace(cuda, monkeypatch):
    torch = _torch()
    from opendressi_b200 import optim

    p, q, r = leaves((9,), (4,), (5,))
    opt = optim.AdamW([p], lr=0.5)

    def full(*args, **kw):
        raise torch.OutOfMemoryError("no memory for the state")

    with monkeypatch.context() as m:
        m.setattr(optim, "_Pack", full)
        with pytest.raises(torch.OutOfMemoryError):
            opt.add_param_group({"params": [q], "lr": 0.25})
    assert len(opt.param_groups) == 1 and q not in opt.state
    opt.add_param_group({"params": [r], "lr": 0.0, "weight_decay": 0.0})
    opt.add_param_group({"params": [q], "lr": 0.25})
    before = [t.detach().clone() for t in (p, q, r)]
    opt.step()
    assert not torch.equal(p, before[0]) and not torch.equal(q, before[1])
    assert torch.equal(r, before[2])  # its own learning rate


def test_a_host_learning_rate_is_checked_before_any_group_steps(cuda):
    torch = _torch()
    from opendressi_b200 import optim

    p, q = leaves((9,), (4,))
    with pytest.raises(ValueError):
        optim.AdamW([p], lr=torch.tensor(-1.0))
    opt = optim.AdamW([{"params": p}, {"params": q}], lr=torch.tensor(0.5))
    opt.param_groups[1]["lr"] = torch.tensor(math.nan)
    before = p.detach().clone()
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(p, before) and int(opt.state[p]["step"]) == 0


@pytest.mark.parametrize("bits", [8, 32])
def test_loading_into_another_order_of_memory(cuda, bits):
    """Codes go with the scale of 256 neighbours in memory: in another order
    they would stand for other values. 32-bit moments go anywhere."""
    torch = _torch()
    from opendressi_b200 import optim

    t = torch.randn(64, 24, 3, 3, device="cuda")
    t *= torch.logspace(-4, 0, 64, device="cuda")[:, None, None, None]
    p = torch.nn.Parameter(t.clone())
    q = torch.nn.Parameter(t.to(memory_format=torch.channels_last))
    p.grad, q.grad = t.clone(), t.clone()
    a, b = (optim.AdamW([x], state_bits=bits) for x in (p, q))
    a.step()
    if bits == 8:
        with pytest.raises(ValueError, match="order"):
            b.load_state_dict(a.state_dict())
        assert not b.packed_state()["exp_avg"].float().any()
        return
    b.load_state_dict(a.state_dict())
    q.data.copy_(p.data)
    a.step()
    b.step()
    assert torch.equal(p, q)


def test_loading_8_bit_state_of_odd_strides(cuda):
    """Strides of extents of 1 do not count."""
    torch = _torch()
    from opendressi_b200 import optim

    t = torch.randn(1, 5, 1, 700, device="cuda")
    p = torch.nn.Parameter(t.clone())
    q = torch.nn.Parameter(t.clone().as_strided(t.shape, (9, 700, 1, 1)))
    p.grad, q.grad = t.clone(), t.clone()
    a, b = (optim.AdamW([x], state_bits=8, seed=5) for x in (p, q))
    a.step()
    b.load_state_dict(a.state_dict())
    q.data.copy_(p.data)
    a.step()
    b.step()
    assert torch.equal(p, q)
