"""q4k_linear_lora in a process whose workspace is as small as the case makes it.

What a call finds in the workspace depends on every call before it, so these
cases need a fresh process: the parent test (test_gpu_adapter_workspace.py) runs
``python adapter_child.py CASE``.  Exit status 0 means every check passed.
"""
import ctypes
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import mtlqwen_amd as q4k  # noqa: E402
from mtlqwen_amd import operators as ops  # noqa: E402
from mtlqwen_amd._lib import EHIP  # noqa: E402
from q4k_ref import TYPE_Q4_K, TYPE_Q6_K, make_weight, make_x  # noqa: E402

dev = torch.device("cuda:0")
rng = np.random.default_rng(9600)


class Call:
    """A linear_lora call over one stack of two adapters."""

    def __init__(self, t, counts, n, k, r, post, dtype=torch.float32):
        m = sum(counts)
        self.name = f"type {t} {m}x{k}->{n} rank {r} post {post} {dtype}"
        print(self.name, flush=True)
        self.W = q4k.Weight(make_weight(rng, n, k, t), n, k, ggml_type=t)
        self.x = torch.from_numpy(make_x(rng, m, k, 0.25)).to(dev).to(dtype)
        self.aux = torch.from_numpy(make_x(rng, m, n, 0.5)).to(dev).to(dtype)
        self.a = torch.from_numpy((rng.standard_normal((2, r, k)) / np.sqrt(k)).astype(np.float16)).to(dev)
        self.b = torch.from_numpy((rng.standard_normal((2, n, r)) / np.sqrt(r)).astype(np.float16)).to(dev)
        self.ids = torch.ones(len(counts), dtype=torch.int32, device=dev)
        self.m, self.counts, self.post = m, counts, post

    def __call__(self, y, aux=None):
        q4k.linear_lora(self.x, self.W, self.a, self.b, self.ids, self.m, y, auxiliary=aux if self.post else None, gated=self.post == 2,
                        query_counts=self.counts)


def refused(call):
    """In a capture that needs more workspace, in place over the auxiliary: the
    error, and a graph that holds nothing of the call."""
    y, count = call.aux.clone(), torch.zeros(1, device=dev)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        count.add_(1)
        try:
            call(y, y)
            code = 0
        except q4k.Q4KError as e:
            code = e.code
    assert code == q4k.ECAPTURE, (call.name, code)
    for i in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert count.item() == i + 1 and torch.equal(y, call.aux), call.name


def eager(call):
    """The call out of place, and in place over the auxiliary."""
    y, z = torch.empty_like(call.aux), call.aux.clone()
    call(y, call.aux)
    call(z, z)
    torch.cuda.synchronize()
    assert torch.isfinite(y).all() and (call.post == 0 or torch.equal(y, z)), call.name
    return y


case = sys.argv[1]
if case == "refused":
    # No workspace at all: adapters of a single launch, which need none, beside
    # projections that do (split-K, staged, persistent, packed).
    ones = [1] * 8
    for post in (1, 2):
        for t, n, k in ((TYPE_Q4_K, 4096, 12288), (TYPE_Q4_K, 512, 1024), (TYPE_Q4_K, 65536, 2048), (TYPE_Q6_K, 512, 1024), (TYPE_Q6_K, 1024, 8192)):
            refused(Call(t, ones, n, k, 8, post))
    # Adapters that fit what a small call reserved, beside a projection that stages more.
    small = Call(TYPE_Q4_K, [3], 512, 1024, 8, 1)
    eager(small)
    for t in (TYPE_Q4_K, TYPE_Q6_K):
        for post in (1, 2):
            large = Call(t, [8000, 192], 256, 8192, 16, post)
            refused(large)
            if (t, post) == (TYPE_Q6_K, 2):
                eager(large)
elif case == "captured":
    # Any first call reserves what gated calls of few rows need.
    q4k.linear(torch.zeros((3, 1024), device=dev), q4k.Weight(make_weight(rng, 512, 1024, TYPE_Q4_K), 512, 1024), 3, torch.empty((3, 512), device=dev))
    for t, counts, n, k, r, dtype in ((TYPE_Q4_K, [1] * 8, 12288, 4096, 8, torch.float32), (TYPE_Q4_K, [5] * 8, 32768, 512, 64, torch.float32),
                                      (TYPE_Q6_K, [60, 3], 1024, 1024, 16, torch.float16)):
        call = Call(t, counts, n, k, r, 2, dtype)
        y = call.aux.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            call(y, y)
        want = eager(call)
        for _ in range(3):
            y.copy_(call.aux)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), call.name
            eager(call)
elif case == "growth":
    # Rising row counts: the sums' buffer at least doubles, from 8.4 MB to 16.8
    # at 528 rows and 33.5 at 1040.  Two more allocations are the row scales of the
    # projection's staging (1024 rows reserved; rows in steps of 128): 1152 and 1280.
    def allocations():
        c = ctypes.c_uint64()
        assert q4k.lib.q4k_workspace_allocations(ctypes.byref(c)) == 0
        return c.value

    call = Call(TYPE_Q4_K, [1200], 4096, 256, 8, 2)
    every = call.x, call.aux
    call.x, call.aux, call.m, call.counts = every[0][:8], every[1][:8], 8, [8]
    eager(call)
    before = allocations()
    for m in range(528, 1201, 16):  # from 8.7 to 19.7 MB of sums
        call.x, call.aux, call.m, call.counts = every[0][:m], every[1][:m], m, [m]
        y = eager(call)
        base, delta = torch.empty_like(y), torch.empty_like(y)
        q4k.linear(call.x, call.W, m, base, query_counts=[m])
        q4k.lora(call.x, call.a, call.b, call.ids, m, delta)
        want = torch.nn.functional.silu(call.aux) * (base + delta)
        assert ((y - want).norm(dim=1) <= 1e-5 * want.norm(dim=1)).all(), m
    assert allocations() - before <= 4, allocations() - before
elif case == "errors":
    # A call that the runtime refuses reports that once: the next calls, the
    # library's and torch's, run.  The first asks for 2.2 TB of sums, before
    # anything is launched; its addresses are only compared.
    call = Call(TYPE_Q4_K, [3], 32768, 256, 8, 2)
    want = eager(call)
    m, address = 1 << 24, 1 << 40
    ad = ops._ADAPTERS(address, 2 * address, 3 * address, 0, 0, 1, 8)
    rc = q4k.lib.q4k_linear_lora(None, call.W.handle, ad, 4 * address, 8 * address, 8 * address, m, ops._COUNTS[1](m), 1, 2, 0)
    assert rc == q4k.ENOMEM, rc
    assert torch.equal(eager(call), want)
    # A device that is not there.
    x, y = torch.randn((2, 4, 64), device=dev), torch.empty((2, 4, 64), device=dev)
    f, p = torch.ones(32, device=dev, dtype=torch.float64), torch.zeros(2, device=dev, dtype=torch.int32)
    heads = ops._HEADS(x.data_ptr(), y.data_ptr(), 0, 256, 64, 256, 64, 4)
    rc = q4k.lib.q4k_rope(None, torch.cuda.device_count(), heads, ops._ROTATION(f.data_ptr(), p.data_ptr(), 64, 0, 1.0), 2, 64, 0)
    assert rc == EHIP, rc
    q4k.rope(x, f, p, y)
    assert torch.equal(x + 0, y) and torch.cuda.current_device() == 0
else:
    raise SystemExit(f"no case {case}")
print("ok", flush=True)
