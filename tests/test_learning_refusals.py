"""The learning operators refuse wrong arguments before any CUDA call (no GPU
needed; the fake addresses are never read)."""

import ctypes as C
import math
from array import array

import pytest

from opendressi_b200 import _native as N

FAKE = C.c_void_p(1 << 20)


def norm_desc(**kw):
    d = dict(struct_size=C.sizeof(N.GroupNormDesc), dtype=N.F32,
             activation=N.ACT_SILU, channels=32, groups=8, eps=1e-5, n=2,
             rows=64)
    d.update(kw)
    return N.GroupNormDesc(**d)


def refused(name, *args, text):
    rc = getattr(N.load(), name)(*args)
    assert rc == N.ERR_INVALID, (name, rc)
    assert text in N.last_error(), N.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(struct_size=3), "struct_size"), (dict(dtype=7), "dtype"),
    (dict(dtype=-1), "dtype"), (dict(activation=3), "activation"),
    (dict(activation=-1), "activation"), (dict(channels=0), "channels"),
    (dict(channels=1 << 25, groups=1), "channels"),
    (dict(groups=0), "divide"), (dict(groups=5), "divide"),
    (dict(groups=64), "divide"), (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"),
    (dict(n=1 << 40), "too many"), (dict(rows=1 << 40), "too many"),
    (dict(n=1 << 20, rows=1 << 30), "too many"),
])
def test_group_norm_descriptor(kw, text):
    d, size = norm_desc(**kw), C.c_size_t()
    refused("dressi_group_norm_workspace", C.byref(d), 0, C.byref(size),
            text=text)
    refused("dressi_group_norm", C.byref(d), FAKE, None, None, FAKE, None,
            None, FAKE, 1 << 40, None, text=text)
    refused("dressi_group_norm_grad", C.byref(d), FAKE, FAKE, None, None,
            FAKE, FAKE, FAKE, None, None, FAKE, 1 << 40, None, text=text)


def test_group_norm_pointers_and_workspace():
    d, size = norm_desc(), C.c_size_t()
    assert N.load().dressi_group_norm_workspace(C.byref(d), 0,
                                                C.byref(size)) == N.OK
    need = size.value
    assert need > 0
    big = 1 << 30
    refused("dressi_group_norm", None, FAKE, None, None, FAKE, None, None,
            FAKE, big, None, text="null pointer")
    refused("dressi_group_norm", C.byref(d), None, None, None, FAKE, None,
            None, FAKE, big, None, text="null pointer")
    refused("dressi_group_norm", C.byref(d), FAKE, None, None, FAKE, FAKE,
            None, FAKE, big, None, text="mean and rstd")
    refused("dressi_group_norm", C.byref(d), C.c_void_p((1 << 20) + 2), None,
            None, FAKE, None, None, FAKE, big, None, text="aligned")
    refused("dressi_group_norm", C.byref(d), FAKE, None, None, FAKE, None,
            None, FAKE, need - 1, None, text="too small")
    refused("dressi_group_norm", C.byref(d), FAKE, None, None, FAKE, None,
            None, C.c_void_p((1 << 20) + 8), big, None, text="16 bytes")
    refused("dressi_group_norm_grad", C.byref(d), FAKE, FAKE, None, None,
            None, FAKE, FAKE, None, None, FAKE, big, None,
            text="null pointer")
    refused("dressi_group_norm_workspace", C.byref(d), 0, None,
            text="null pointer")
    # nothing to do: accepted with null images
    empty = norm_desc(n=0)
    assert N.load().dressi_group_norm(C.byref(empty), None, None, None, None,
                                      None, None, None, 0, None) == N.OK


def test_grad_norm_arguments():
    need = C.c_size_t()
    assert N.load().dressi_grad_norm_workspace(C.byref(need)) == N.OK
    ptr, n, t = array("Q", [1 << 20]), array("Q", [8]), array("i", [N.F32])

    keep = []  # the host arrays of a call outlive it

    def call(ptr=ptr, n=n, t=t, out=FAKE, space=FAKE, size=1 << 20, count=1):
        keep.append((ptr, n, t))
        return (count, ptr and ptr.buffer_info()[0],
                n and n.buffer_info()[0], t and t.buffer_info()[0], out,
                space, size, None)

    name = "dressi_grad_norm"
    refused(name, *call(out=None), text="null pointer")
    refused(name, *call(space=None), text="null pointer")
    refused(name, *call(ptr=None), text="null pointer")
    refused(name, *call(size=need.value - 1), text="workspace")
    refused(name, *call(space=C.c_void_p(4)), text="workspace")
    refused(name, *call(t=array("i", [9])), text="dtype")
    refused(name, *call(ptr=array("Q", [0])), text="null or misaligned")
    refused(name, *call(ptr=array("Q", [2])), text="null or misaligned")
    refused(name, *call(n=array("Q", [1 << 50])), text="too long")


def adamw_desc(keep, **kw):
    one = {k: array("Q", [1 << 20]) for k in
           ("params", "grads", "exp_avg", "exp_avg_sq", "exp_avg_scale",
            "exp_avg_sq_scale", "steps")}
    one["numel"] = array("Q", [8])
    d = dict(struct_size=C.sizeof(N.AdamWDesc), n_tensors=1, dtype=N.F32,
             state_bits=32, index=None, lr=1e-3, beta1=0.9, beta2=0.999,
             eps=1e-8, weight_decay=1e-2, lr_device=None, max_norm=0.0,
             grad_norm=None, clamp_lo=-math.inf, clamp_hi=math.inf, seed=0,
             ticket=1 << 20)
    for k, v in kw.items():
        if isinstance(v, array):
            one[k] = v
        else:
            d[k] = v
    keep.append(one)
    for k, v in one.items():
        d.setdefault(k, v.buffer_info()[0])
    return N.AdamWDesc(**d)


@pytest.mark.parametrize("kw,text", [
    (dict(struct_size=8), "struct_size"), (dict(dtype=3), "dtype"),
    (dict(state_bits=16), "state_bits"), (dict(lr=-1.0), "lr"),
    (dict(lr=math.nan), "lr"), (dict(lr=math.inf), "lr"),
    (dict(beta1=1.0), "betas"), (dict(beta1=-0.1), "betas"),
    (dict(beta2=math.nan), "betas"), (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"), (dict(weight_decay=-1.0), "weight_decay"),
    (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=math.inf), "max_norm"),
    (dict(max_norm=1.0), "grad_norm"),
    (dict(clamp_lo=1.0, clamp_hi=0.0), "clamp"),
    (dict(clamp_lo=math.nan), "clamp"), (dict(ticket=None), "null pointer"),
    (dict(params=None), "null pointer"), (dict(steps=None), "null pointer"),
    (dict(state_bits=8, exp_avg_scale=None), "null pointer"),
    (dict(numel=array("Q", [1 << 45])), "too long"),
    (dict(params=array("Q", [0])), "null tensor"),
    (dict(grads=array("Q", [0])), "null tensor"),
    (dict(exp_avg=array("Q", [0])), "null tensor"),
    (dict(state_bits=8, exp_avg_scale=array("Q", [0])), "null tensor"),
    (dict(steps=array("Q", [0])), "null step"),
    (dict(params=array("Q", [1 << 20 | 2])), "aligned"),
    (dict(exp_avg=array("Q", [1 << 20 | 1])), "aligned"),
    (dict(state_bits=8, exp_avg_sq_scale=array("Q", [1 << 20 | 2])),
     "aligned"),
    (dict(steps=array("Q", [1 << 20 | 2])), "null step"),
])
def test_adamw_descriptor(kw, text):
    keep = []
    d = adamw_desc(keep, **kw)
    refused("dressi_adamw_step", C.byref(d), None, text=text)


def test_adamw_of_nothing():
    keep = []
    d = adamw_desc(keep, n_tensors=0)
    assert N.load().dressi_adamw_step(C.byref(d), None) == N.OK
    refused("dressi_adamw_step", None, None, text="null pointer")


def test_python_refuses_host_tensors():
    import torch
    from opendressi_b200 import DressiError, optim, ops, torch_api

    p = torch.zeros(4, requires_grad=True)
    with pytest.raises(DressiError, match="CUDA"):
        optim.AdamW([p])
    with pytest.raises(DressiError, match="CUDA"):
        ops.grad_norm([p])
    with pytest.raises(DressiError, match="CUDA"):
        torch_api.group_norm(torch.zeros(2, 4, 4, 8), 2)
    for kw in (dict(state_bits=16), dict(max_norm=-1.0), dict(max_norm=0.0),
               dict(lr=-1.0), dict(lr=math.nan), dict(betas=(0.9, 1.0)),
               dict(betas=(0.9,)), dict(eps=-1.0), dict(weight_decay=-1.0),
               dict(clamp=(1.0, 0.0)), dict(clamp=(math.nan, 1.0))):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
