"""The operators around the projections as programs use them beyond plain
calls: on streams other than the current one and two at a time, storage whose
offsets pass 32 bits, the smallest calls, captures in a process that has no
workspace yet, and graphs that share it."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
HERE = os.path.dirname(os.path.abspath(__file__))


def _i32(gpu, *v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _lora_inputs(gpu, rng, m, k, n, r, slots, dtype):
    a = torch.from_numpy((rng.standard_normal((slots, r, k)) / np.sqrt(k)).astype(np.float16)).to(gpu)
    b = torch.from_numpy((rng.standard_normal((slots, n, r)) / np.sqrt(r)).astype(np.float16)).to(gpu)
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(gpu).to(dtype)
    return x, a, b


def test_streams(q4k, gpu):
    """Each operator on a side stream behind work that makes its inputs there,
    given as argument and as the current stream, beside another on a second
    stream: the results of the plain call."""
    rng = np.random.default_rng(1)
    m, k, n, r = 40, 1024, 512, 24
    x, a, b = _lora_inputs(gpu, rng, m, k, n, r, 2, F32)
    ids, f = _i32(gpu, 1), torch.from_numpy(10000.0 ** (-np.arange(0, 128, 2) / 128)).to(gpu)
    q = torch.randn((64, 8, 128), device=gpu)
    kk = torch.randn((64, 2, 128), device=gpu)
    w = torch.ones(128, device=gpu)
    pos = torch.arange(64, dtype=torch.int32, device=gpu)
    logits = torch.randn((4, 30000), device=gpu)
    tokens, lengths = torch.randint(0, 30000, (4, 100), device=gpu, dtype=torch.int32), _i32(gpu, 100, 50, 0, 7)
    rep = torch.full((4,), 1.3, device=gpu)

    def calls(scale, stream):
        y, qo, ko, out, ro = torch.empty((m, n), device=gpu), torch.empty_like(q), torch.empty_like(kk), torch.empty_like(logits), torch.empty_like(q)
        q4k.lora(x * scale, a, b, ids, m, y, stream=stream)
        q4k.qk_norm_rope(q * scale, kk * scale, w, w, f, pos, qo, ko, stream=stream)
        q4k.rope(q * scale, f, pos, ro, stream=stream)
        q4k.process_logits(logits * scale, out, tokens=tokens, lengths=lengths, repetition=rep, stream=stream)
        return y, qo, ko, out, ro

    want = [t.clone() for t in calls(2.0, None)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        big = torch.randn((4096, 4096), device=gpu)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            scale = (big @ big).sum() * 0 + 2.0  # the inputs wait for it
            got = calls(scale, None)
            given = calls(scale, s1)
        with torch.cuda.stream(s2):  # no workspace: may run beside the first stream's
            other = torch.empty_like(q)
            q4k.rope(q * 2.0, f, pos, other)
        torch.cuda.synchronize()
        for g, h, v in zip(got, given, want):
            assert torch.equal(g, v) and torch.equal(h, v)
        assert torch.equal(other, want[4])


def test_rope_offsets_past_32_bits(q4k, gpu):
    step = (1 << 30) + 128
    store = torch.empty(2 * step + 128, device=gpu, dtype=F16)
    x = store.as_strided((3, 1, 128), (step, 128, 1))
    rng = np.random.default_rng(2)
    host = torch.from_numpy(rng.standard_normal((3, 1, 128)).astype(np.float32)).half()
    x.copy_(host)
    f, p = torch.from_numpy(10000.0 ** (-np.arange(0, 128, 2) / 128)), _i32(gpu, 5, 6, 7)
    q4k.rope(x, f.to(gpu), p, x)
    torch.cuda.synchronize()
    want, size = ref.rotate(host.float().numpy(), f.numpy(), [5, 6, 7], False, 1.0)
    ref.assert_close(x.cpu().float().numpy(), want, ref.rotate_bound(size, 1.0), True)


def test_logits_text_past_32_bits(q4k, gpu):
    tokens = torch.zeros((3, 1 << 30), device=gpu, dtype=torch.int32)
    tokens[2, :3] = _i32(gpu, 7, 9, 7)
    x = torch.ones((1, 64), device=gpu)
    out = torch.empty_like(x)
    q4k.process_logits(x, out, tokens=tokens, slots=_i32(gpu, 2), lengths=_i32(gpu, 3), frequency=torch.full((1,), 0.25, device=gpu))
    got = out.cpu()[0]
    assert got[7] == 0.5 and got[9] == 0.75 and got[0] == 1.0


def test_adapters_past_32_bits(q4k, gpu):
    slots, n, r, k = 18, 248320, 512, 256
    a, b = torch.zeros((slots, r, k), device=gpu, dtype=F16), torch.zeros((slots, n, r), device=gpu, dtype=F16)
    assert b.numel() > 1 << 31
    a[17, 511, 255], b[17, n - 1, 511], b[17, 0, 511] = 2.0, 3.0, -1.0
    x = torch.ones((1, k), device=gpu)
    y = torch.empty((1, n), device=gpu)
    q4k.lora(x, a, b, _i32(gpu, 17), 1, y)
    torch.cuda.synchronize()
    assert y[0, n - 1] == 6.0 and y[0, 0] == -2.0 and bool((y[0, 1:n - 1] == 0).all())


@pytest.mark.parametrize("dtype", [F32, F16])
def test_smallest_calls(q4k, gpu, dtype):
    x = torch.tensor([[[3.0]]], device=gpu, dtype=dtype)
    y = torch.empty_like(x)
    none = torch.zeros(0, device=gpu, dtype=torch.float64)
    one = torch.ones(1, device=gpu)
    q4k.qk_norm_rope(x, x, one, 2 * one, none, _i32(gpu, 4), y, torch.empty_like(x), eps=0.0)
    assert y.item() == 1.0
    a, b = torch.ones((1, 1, 256), device=gpu, dtype=F16), torch.ones((1, 16, 1), device=gpu, dtype=F16)
    v = torch.ones((1, 256), device=gpu, dtype=dtype)
    out = torch.empty((1, 16), device=gpu, dtype=dtype)
    q4k.lora(v, a, b, _i32(gpu, 0), 1, out)
    assert bool((out == 256).all())
    q4k.lora(v.repeat(3, 1), a, b, _i32(gpu, 0), 3, torch.empty((3, 16), device=gpu, dtype=dtype))
    z = torch.tensor([[1.0]], device=gpu, dtype=dtype)
    q4k.process_logits(z, z, tokens=_i32(gpu, 0).view(1, 1), lengths=_i32(gpu, 1), presence=one)
    assert z.item() == 0.0


def test_extreme_values_of_adapters(q4k, gpu):
    """Rows of the largest and smallest magnitudes, alone and mixed with others
    2^17 and more below them, keep the bound relative to their sums; an
    infinity stays one."""
    rng = np.random.default_rng(5)
    m, k, n, r = 33, 512, 64, 16
    x, a, b = _lora_inputs(gpu, rng, m, k, n, r, 1, F32)
    x[0] *= 1e34
    x[1] *= 1e-36
    x[2] *= torch.where(torch.rand(k, device=gpu) < 0.5, 1.0, 2.0 ** -18)
    x[3] = 0
    x[4, 1:] = 0
    x[5] *= 2.0 ** torch.randint(-60, 60, (k,), device=gpu)
    y = torch.empty((m, n), device=gpu)
    q4k.lora(x, a, b, _i32(gpu, 0), m, y)
    torch.cuda.synchronize()
    want, bound = ref.lora(x.cpu().numpy(), a.cpu().numpy(), b.cpu().numpy(), [0], [m], None, None, None)
    # Products of x below the smallest normal fp32 value round to subnormals.
    ref.assert_close(y.cpu().numpy(), want, bound + 1e-42, False)
    assert bool((y[3] == 0).all())
    a.abs_()
    b.abs_()
    x.abs_()
    x[7, 3] = float("inf")
    q4k.lora(x, a, b, _i32(gpu, 0), m, y)
    torch.cuda.synchronize()
    assert bool((y[7] == float("inf")).all()) and bool(torch.isfinite(y[8:]).all())


def test_graphs_that_share_the_workspace(q4k, gpu):
    """Two captured adapter calls of different shapes and an eager projection's
    worth of others, replayed in turn on one stream."""
    rng = np.random.default_rng(6)
    sets = []
    for m, k, n, r in [(40, 1024, 512, 32), (100, 2048, 256, 64)]:
        x, a, b = _lora_inputs(gpu, rng, m, k, n, r, 2, F32)
        y, want = torch.empty((m, n), device=gpu), torch.empty((m, n), device=gpu)
        args = (x, a, b, _i32(gpu, 1, 0), m)
        kw = {"query_counts": [m - 7, 7]}
        q4k.lora(*args, want, **kw)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            q4k.lora(*args, y, **kw)
        sets.append((g, y, want, args, kw))
    for _ in range(3):
        for g, y, want, args, kw in sets:
            y.zero_()
        for g, y, want, args, kw in sets:
            g.replay()
        for g, y, want, args, kw in sets:
            q4k.lora(*args, torch.empty_like(y), **kw)
        torch.cuda.synchronize()
        for g, y, want, args, kw in sets:
            assert torch.equal(y, want)


CHILD = """
import sys
sys.path[:0] = [{here!r}, {root!r}]
import torch
import mtlqwen_amd as q4k
dev = torch.device("cuda:0")
def capture(fn):
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        fn()
    return g
ids = torch.zeros(1, dtype=torch.int32, device=dev)
def lora(m, r):
    a, b = torch.ones((1, r, 512), device=dev, dtype=torch.half), torch.ones((1, 64, r), device=dev, dtype=torch.half)
    x, y = torch.ones((m, 512), device=dev), torch.zeros((m, 64), device=dev)
    return lambda: q4k.lora(x, a, b, ids, m, y), y
# A single row of few ranks needs no workspace.
fn, y = lora(1, 16)
g = capture(fn)
for _ in range(3):
    y.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert bool((y == 512 * 16).all())
fn, y = lora(40, 32)
try:
    capture(fn)
    raise SystemExit("captured without a workspace")
except q4k.Q4KError as e:
    assert e.code == q4k.ECAPTURE, e.message
torch.cuda.synchronize()
lora(3, 8)[0]()  # any call of several rows reserves what usual batches need
torch.cuda.synchronize()
g = capture(fn)
for _ in range(3):
    y.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert bool((y == 512 * 32).all())
print("ok", flush=True)
"""


def test_capture_without_a_workspace(gpu):
    code = CHILD.format(here=HERE, root=os.path.dirname(HERE))
    r = subprocess.run([sys.executable, "-u", "-c", code], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), f"{r.returncode}:\n{r.stdout[-800:]}\n{r.stderr[-1500:]}"
