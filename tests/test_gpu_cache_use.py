"""The paged cache as a server uses it: prompts and steps with beams that fork
and end, pages that move, all against attention over each sequence's own
keys in 64 bits; streams, captured and replayed steps, graphs that share the
workspace, a process without one, storage whose offsets pass 32 bits, calls that
take several launches or are refused."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import cache_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
HERE = os.path.dirname(os.path.abspath(__file__))


def _i32(gpu, *v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _dense(q, keys, values, kw, f16):
    """attention() of the rows behind a sequence's own keys and values [tokens, heads, dim]: one page holds them."""
    n, page = len(keys), 1 << max(4, (len(keys) - 1).bit_length())
    kc = np.zeros((1, keys.shape[1], page, keys.shape[2]))
    vc = kc.copy()
    kc[0, :, :n], vc[0, :, :n] = keys.transpose(1, 0, 2), values.transpose(1, 0, 2)
    return ref.attention(q, kc, vc, [[0]], [n - len(q)], [len(q)], f16=f16, **kw)


@pytest.mark.parametrize("dtype,kw", [(F16, {}), (F32, {"softcap": 20.0, "window": 70})])
def test_beams_together(q4k, gpu, dtype, kw):
    """Two layers in one pool: prompts in chunks, then steps in which beams take
    over others' states, end and start anew, with the pages moved in between."""
    rng = np.random.default_rng(8)
    slots, layers, kv, heads, dim, page, pages, width = 6, 2, 2, 6, 64, 16, 90, 12
    pool = torch.full((pages, layers, 2, kv, page, dim), float("nan"), device=gpu, dtype=F16)  # what nobody wrote reaches nobody
    tables, lengths = torch.full((slots, width), -1, device=gpu, dtype=torch.int32), torch.zeros(slots, device=gpu, dtype=torch.int32)
    texts = [[(np.zeros((0, kv, dim)), np.zeros((0, kv, dim))) for _ in range(layers)] for _ in range(slots)]  # keys, values of every layer

    def assign(parents, counts):
        nonlocal tables, lengths, texts
        new_tables, new_lengths, missing = torch.empty_like(tables), torch.empty_like(lengths), _i32(gpu, 7)
        q4k.cache_assign(pool, tables, lengths, None if parents is None else _i32(gpu, *parents), new_tables, new_lengths,
                         counts=_i32(gpu, *counts), missing=missing)
        assert missing.item() == 0
        tables, lengths = new_tables, new_lengths
        if parents is not None:
            empty = (np.zeros((0, kv, dim)), np.zeros((0, kv, dim)))
            texts = [[texts[p][i] if p >= 0 else empty for i in range(layers)] for p in parents]

    def step(counts):
        nonlocal lengths
        rows = sum(counts)
        for i in range(layers):
            q, k, v = (torch.from_numpy(rng.standard_normal((rows, h, dim)).astype(np.float32)).to(dtype).to(gpu) for h in (heads, kv, kv))
            out = torch.empty_like(q)
            kc, vc = pool[:, i, 0], pool[:, i, 1]
            q4k.cache_write(k, v, kc, vc, tables, lengths, query_counts=counts)
            q4k.attention(q, kc, vc, tables, lengths, out, query_counts=counts, **kw)
            torch.cuda.synchronize()
            got, start = out.cpu().double().numpy(), 0
            for s, n in enumerate(counts):
                keys, values = (np.concatenate([t, x[start:start + n].half().cpu().double().numpy()]) for t, x in zip(texts[s][i], (k, v)))
                texts[s][i] = (keys, values)
                if n:
                    want, bound = _dense(q[start:start + n].cpu().double().numpy(), keys, values, kw, dtype == F16)
                    off = np.abs(got[start:start + n] - want)
                    assert (off <= bound).all(), (counts, s, i, float(np.nanmax(off / bound)))
                start += n
        lengths = lengths + _i32(gpu, *counts)

    def compact():
        nonlocal tables
        new, used = torch.empty_like(tables), _i32(gpu, -1)
        q4k.cache_compact(pool, tables, lengths, new, used=used)
        tables = new
        assert used.item() <= pages and int(tables.max()) < used.item()
        pool[used.item():] = float("nan")  # what is behind them is nobody's

    prompts = [33, 0, 70, 1, 16, 5]
    assign(None, prompts)
    step([20, 0, 64, 1, 16, 5])
    step([13, 0, 6, 0, 0, 0])
    for turn, parents in enumerate([[0, 0, 2, 2, 4, 5], [1, 0, 3, 3, 3, -1], [0, 1, 2, 4, 4, 0], None, [5, 4, 3, 2, 1, 0], [2, 2, 2, 2, 2, 2]]):
        counts = [1, 2, 1, 5, 1, 3] if turn % 2 else [1] * 6
        assign(parents, counts)
        step(counts)
        if turn in (1, 4):
            compact()


def _calls(gpu, rng, dtype=F16, counts=(1, 3, 1), contexts=(300, 77, 900), heads=8, kv=2, dim=128, page=32):
    need = [-(-c // page) for c in contexts]
    order = rng.permutation(sum(need) + 2)
    tables, at = np.full((len(counts), max(need) + 1), -1, np.int32), 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    cache = torch.from_numpy(rng.standard_normal((sum(need) + 2, 2, kv, page, dim)).astype(np.float16)).to(gpu)
    x = [torch.from_numpy(rng.standard_normal((sum(counts), h, dim)).astype(np.float32)).to(dtype).to(gpu) for h in (heads, kv, kv)]
    return {"cache": cache, "tables": torch.from_numpy(tables).to(gpu), "first": _i32(gpu, *[c - n for c, n in zip(contexts, counts)]), "counts": list(counts),
            "q": x[0], "k": x[1], "v": x[2]}


def _step(q4k, s, out, stream=None):
    kc, vc = s["cache"][:, 0], s["cache"][:, 1]
    q4k.cache_write(s["k"], s["v"], kc, vc, s["tables"], s["first"], query_counts=s["counts"], stream=stream)
    return q4k.attention(s["q"], kc, vc, s["tables"], s["first"], out, query_counts=s["counts"], stream=stream)


def test_streams(q4k, gpu):
    """On a side stream behind work that makes the inputs there, given as argument and as the current stream."""
    rng = np.random.default_rng(1)
    for s in (_calls(gpu, rng), _calls(gpu, rng, counts=(90, 1, 70))):
        want = _step(q4k, s, torch.empty_like(s["q"])).clone()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        for _ in range(3):
            big = torch.randn((4096, 4096), device=gpu)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                late = dict(s, q=s["q"] * ((big @ big).sum() * 0 + 1.0).to(s["q"].dtype))
                first = _step(q4k, late, torch.empty_like(want))
                second = _step(q4k, late, torch.empty_like(want), stream=side)
            torch.cuda.synchronize()
            assert torch.equal(first, want) and torch.equal(second, want)


@pytest.mark.parametrize("counts,contexts", [((1, 1, 1), (300, 77, 900)), ((60, 5, 64), (300, 77, 900))])
def test_captured_steps_follow_the_device(q4k, gpu, counts, contexts):
    """A captured step of writes, attention and tables follows positions, tables
    and lengths from replay to replay with the eager call's bits, beside eager
    work and another graph that shares the workspace."""
    rng = np.random.default_rng(2)
    s, other = _calls(gpu, rng, counts=counts, contexts=contexts), _calls(gpu, rng, counts=(40, 2, 1), heads=4, dim=256)
    pool, lengths = s["cache"], s["first"].clone()
    new, new_lengths, moved = torch.empty_like(s["tables"]), torch.empty_like(lengths), torch.empty_like(s["tables"])
    parents = _i32(gpu, 0, 0, 2)

    def work(out):
        _step(q4k, s, out)
        q4k.cache_assign(pool, s["tables"], lengths, parents, new, new_lengths)
        q4k.cache_compact(pool.clone(), s["tables"], lengths, moved)
        return out

    out, out2 = torch.empty_like(s["q"]), torch.empty_like(other["q"])
    work(out)
    want2 = _step(q4k, other, out2).clone()
    torch.cuda.synchronize()
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        work(out)
    with torch.cuda.graph(g2, stream=torch.cuda.Stream()):
        _step(q4k, other, out2)
    for turn in range(4):
        s["first"].copy_(torch.tensor([max(0, c - n - 40 * turn) for c, n in zip(contexts, counts)], dtype=torch.int32))
        lengths.copy_(s["first"])
        s["tables"].copy_(s["tables"][[1, 0, 2]] if turn == 2 else s["tables"])
        want = work(torch.empty_like(out)).clone()
        tables, moves, held = new.clone(), moved.clone(), new_lengths.clone()
        out.zero_(), out2.zero_(), new.zero_(), moved.zero_(), new_lengths.zero_()
        torch.cuda.synchronize()
        g.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want2)
        assert torch.equal(new, tables) and torch.equal(moved, moves) and torch.equal(new_lengths, held)


CHILD = """
import sys
sys.path[:0] = [{here!r}, {root!r}]
import numpy as np, torch
import mtlqwen_amd as q4k
import test_gpu_cache_use as t
gpu = torch.device("cuda:0")
rng = np.random.default_rng(3)
few, many = t._calls(gpu, rng), t._calls(gpu, rng, counts=(100, 30, 60), dim=256)
def capture(s, out):
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    code = 0
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        out.add_(1)
        try:
            t._step(q4k, s, out)
        except q4k.Q4KError as e:
            code = e.code
    return g, code
out = torch.zeros_like(few["q"])
print("few rows captured first", flush=True)
g, code = capture(few, out)
assert code == q4k.ECAPTURE, code
g.replay(); torch.cuda.synchronize()
assert bool((out == 1).all())
x, y = torch.zeros((8, 4096), device=gpu), torch.empty((8, 256), device=gpu)
W = q4k.Weight(np.zeros(256 * 16 * 144, np.uint8), 256, 4096)
print("a projection, then few rows", flush=True)
q4k.linear(x, W, 8, y, query_counts=[1] * 8)
g, code = capture(few, out)
assert code == 0
for _ in range(3):
    out.zero_(); g.replay(); torch.cuda.synchronize()
    want = t._step(q4k, few, torch.empty_like(out))
    assert torch.equal(out, want)
print("many rows: refused, then eager, then captured", flush=True)
out = torch.zeros_like(many["q"])
g, code = capture(many, out)
assert code == q4k.ECAPTURE, code
want = t._step(q4k, many, torch.empty_like(out)).clone()
g, code = capture(many, out)
assert code == 0
for _ in range(3):
    out.zero_(); g.replay(); torch.cuda.synchronize()
    assert torch.equal(out, want)
print("ok")
"""


def test_process_without_a_workspace(gpu):
    """A capture before any call is refused and holds nothing of it; behind any
    projection few rows need no more, many rows one call of theirs."""
    env = {k: v for k, v in os.environ.items() if not k.startswith(("Q4K_", "Q6K_"))}
    code = CHILD.format(here=HERE, root=os.path.dirname(HERE))
    r = subprocess.run([sys.executable, "-u", "-c", code], env=env, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), f"{r.returncode}:\n{r.stdout[-1500:]}\n{r.stderr[-2000:]}"


def _check(q4k, gpu, q, kc, vc, tables, first, counts, out):
    q4k.attention(q, kc, vc, tables, first, out, query_counts=counts)
    torch.cuda.synchronize()
    want, bound = ref.attention(q.cpu().float().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), tables.tolist(), first.tolist(), counts, f16=q.dtype == F16)
    off = np.abs(out.cpu().double().numpy() - want)
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("counts", [[2], [40]])
def test_offsets_past_32_bits(q4k, gpu, counts):
    """Pages, heads and rows more than 2^31 elements apart; tokens 2^26 apart."""
    rng = np.random.default_rng(4)
    heads, kv, dim, page, pages, far = 4, 2, 64, 16, 3, (1 << 30) + 64
    x = torch.from_numpy(rng.standard_normal((counts[0], kv, dim)).astype(np.float32)).to(gpu)
    q = torch.from_numpy(rng.standard_normal((counts[0], heads, dim)).astype(np.float32)).to(gpu)
    tables, first = _i32(gpu, 2, 0, 1).view(1, 3), _i32(gpu, 48 - counts[0])
    for strides in [(far, 1024, 64), (2048, far, 64), (1024, 64, 1 << 26)]:
        size = sum((n - 1) * s for n, s in zip((pages, kv, page), strides)) + dim
        kc, vc = (torch.empty(size, device=gpu, dtype=F16).as_strided((pages, kv, page, dim), (*strides, 1)) for _ in range(2))
        for c in (kc, vc):
            c.copy_(torch.from_numpy(rng.standard_normal(c.shape).astype(np.float16)))
        q4k.cache_write(x, -x, kc, vc, tables, first)
        last = tables[0, 2].item()
        assert torch.equal(kc[last, :, 15], x[-1].half()) and torch.equal(vc[last, :, 15], -x[-1].half())
        _check(q4k, gpu, q, kc, vc, tables, first, counts, torch.empty_like(q))
        del kc, vc, c
    rows = torch.empty((counts[0] - 1) * ((1 << 31) // counts[0] + 256) + heads * dim, device=gpu)
    wide = rows.as_strided((counts[0], heads, dim), ((1 << 31) // counts[0] + 256, dim, 1))
    cache = torch.from_numpy(rng.standard_normal((pages, 2, kv, page, dim)).astype(np.float16)).to(gpu)
    wide.copy_(q)
    out = torch.empty_like(q)
    _check(q4k, gpu, wide, cache[:, 0], cache[:, 1], tables, first, counts, out)
    _check(q4k, gpu, q, cache[:, 0], cache[:, 1], tables, first, counts, wide)
    assert torch.equal(wide, out)


def test_heads_of_several_launches(q4k, gpu):
    """Tables of 2^30 tokens: the line of work of 130 heads takes three launches; and one of a single head that no launch holds is refused."""
    rng = np.random.default_rng(5)
    heads, dim, page = 130, 8, 1024
    cache = torch.from_numpy(rng.standard_normal((2, 2, heads, page, dim)).astype(np.float16)).to(gpu)
    tables = torch.full((1, 1 << 20), -1, device=gpu, dtype=torch.int32)
    tables[0, :2] = _i32(gpu, 1, 0)
    for n in (1, 100):
        q = torch.from_numpy(rng.standard_normal((n, heads, dim)).astype(np.float32)).to(gpu)
        out = torch.empty_like(q)
        q4k.attention(q, cache[:, 0], cache[:, 1], tables, _i32(gpu, 1100), out)
        torch.cuda.synchronize()
        c = cache.cpu().numpy()
        want, bound = ref.attention(q.cpu().numpy(), c[:, 0], c[:, 1], [[1, 0]], [1100], [n])
        assert (np.abs(out.cpu().double().numpy() - want) <= bound).all()
    q = torch.zeros((1, 1, dim), device=gpu, dtype=F16).expand(1 << 20, 1, dim)
    with pytest.raises(q4k.Q4KError) as e:
        q4k.attention(q, cache[:, 0, :1], cache[:, 1, :1], tables, _i32(gpu, 0), torch.empty(q.shape, device=gpu, dtype=F16))
    assert e.value.code == -3


def test_same_place_twice(q4k, gpu):
    """Two rows with one place: one of them stays there, whole values of it."""
    cache = torch.zeros((2, 2, 1, 16, 64), device=gpu, dtype=F16)
    x = torch.stack([torch.full((1, 64), float(i + 1)) for i in range(4)]).to(gpu)
    q4k.cache_write(x, x, cache[:, 0], cache[:, 1], _i32(gpu, 1).view(1, 1), _i32(gpu, 2, 2, 3), query_counts=[1, 2, 1], slots=_i32(gpu, 0, 0, 0))
    torch.cuda.synchronize()
    assert set(cache[1, 0, 0, 2].tolist()) <= {1.0, 2.0} and set(cache[1, 0, 0, 3].tolist()) <= {3.0, 4.0}
    assert (cache[0] == 0).all() and (cache[1, :, :, :2] == 0).all() and (cache[1, :, :, 4:] == 0).all()


def test_runs_are_alike(q4k, gpu):
    """The same call gives the same bits: parts join in one order whoever comes last."""
    rng = np.random.default_rng(6)
    for s in (_calls(gpu, rng, contexts=(9000, 40, 5000)), _calls(gpu, rng, counts=(200, 3, 90), contexts=(3000, 40, 900)), _calls(gpu, rng, dtype=F32, contexts=(9000, 40, 5000))):
        want = _step(q4k, s, torch.empty_like(s["q"])).clone()
        for _ in range(20):
            assert torch.equal(_step(q4k, s, torch.empty_like(want)), want)
