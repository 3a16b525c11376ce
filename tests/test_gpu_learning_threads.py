"""The learning operators called from several host threads at once."""

import ctypes as C
import os
import subprocess
import sys
import threading

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
def test_one_kernel_with_much_and_with_little_shared_memory(cuda, grad):
    """Two threads, two streams, the same kernel over samples that take 200
    KB and 60 KB of a block's shared memory."""
    import torch

    from opendressi_b200 import _native as N

    lib = N.load()
    images = 2 if grad else 1
    jobs = []
    for k, kb in enumerate((190, 56)):
        rows = kb * 1024 // (32 * 4 * images)
        g = torch.Generator(device="cuda").manual_seed(k)
        x = torch.randn((1, rows, 32), generator=g, device="cuda")
        dy = torch.randn((1, rows, 32), generator=g, device="cuda")
        d = N.GroupNormDesc(
            struct_size=C.sizeof(N.GroupNormDesc), dtype=N.F32,
            activation=N.ACT_SILU, channels=32, groups=4, eps=1e-5, n=1,
            rows=rows)
        need = C.c_size_t()
        N.check(lib.dressi_group_norm_workspace(C.byref(d), int(grad),
                                                C.byref(need)))
        outs = [torch.empty_like(x), torch.empty(1, 4, device="cuda"),
                torch.empty(1, 4, device="cuda"),
                torch.empty(32, device="cuda"),
                torch.empty(32, device="cuda")]
        space = torch.empty(need.value, dtype=torch.uint8, device="cuda")
        stream = torch.cuda.Stream()

        def call(d=d, x=x, dy=dy, outs=outs, space=space, stream=stream):
            y, mean, rstd, dw, db = (C.c_void_p(t.data_ptr()) for t in outs)
            at, end = C.c_void_p(space.data_ptr()), space.numel()
            on = C.c_void_p(stream.cuda_stream)
            if grad:
                return lib.dressi_group_norm_grad(
                    C.byref(d), dy.data_ptr(), x.data_ptr(), None, None, mean,
                    rstd, y, dw, db, at, end, on)
            return lib.dressi_group_norm(C.byref(d), x.data_ptr(), None, None,
                                         y, mean, rstd, at, end, on)

        if grad:
            h = x.double().reshape(rows, 4, 8)
            outs[1].copy_(h.mean((0, 2)))
            outs[2].copy_((h.var((0, 2), unbiased=False) + 1e-5).rsqrt())
        jobs.append((call, outs, stream))
    torch.cuda.synchronize()
    alone = []
    for call, outs, stream in jobs:
        assert call() == N.OK, N.last_error()
        stream.synchronize()
        alone.append([t.clone() for t in outs])
    failed = []

    def work(call):
        for _ in range(4000):
            if call() != N.OK:
                failed.append(N.last_error())
                return

    threads = [threading.Thread(target=work, args=(j[0],)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for (_, outs, _), want in zip(jobs, alone):
        for a, e in zip(outs, want):
            assert torch.equal(a, e)


def test_shared_memory_next_to_what_needs_no_leave(cuda):
    """The first call of a process, with just under and just over 48 KB of a
    block's shared memory (9 and 10 steps of 4 KB, 8 KB of sums and 8 bytes
    for each of up to 512 groups)."""
    code = """
import torch
from opendressi_b200 import torch_api as dr
for c, rows in ((256, 36), (508, 18), (512, 18), (512, 20)):
    x = torch.randn(1, rows, c, device="cuda")
    y = dr.group_norm(x, c)
    d = x.double()
    mean, dev = d.mean(1), (d.var(1, unbiased=False) + 1e-5).sqrt()
    e = (d - mean) / dev
    # 64 roundings of a term: of the value, of its group's mean and of an
    # eighth of the group's largest value (as in test_gpu_group_norm.py)
    tol = 64 * 2.0 ** -24 * (e.abs() + (mean / dev).abs()
                             + e.abs().amax(1) / 8)
    assert ((y - e).abs() <= tol).all(), (c, rows)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], cwd=root, check=True,
                   timeout=280)
