"""Attention of few rows where every wave of a workgroup has several key tiles one
behind the other, so that its buffers are refilled under the products: all
paddings of a head, one row to many, with the caches emptied before the call, against
64-bit numpy (cache_ref) for some heads of some sequences."""
import numpy as np
import pytest
import torch

import cache_ref as ref
from test_gpu_attention import _close, _i32, _tables

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
CONTEXTS = [4096, 5003, 4500, 6001, 4097, 5555, 4800, 7777]


def _run(q4k, gpu, n, heads, kv, dim, page, dtype, window=0, bad=False, probe=((0, 0), (3, 1), (7, -1)), contexts=CONTEXTS):
    rng = np.random.default_rng(dim + page + 97 * n + heads)
    # Places of the line of work: tiles of 32 keys and a unit's beginning and end, as 16 of them.  Four waves share a workgroup's.
    tiles = sum((min(c, window + 32 + n) if window else c) // 32 + 16 for c in contexts) * kv
    assert tiles > 2 * 4 * torch.cuda.get_device_properties(gpu).multi_processor_count, "a wave has one tile only"
    tables, pages = _tables(rng, contexts, page)
    g = torch.Generator(device=gpu)
    g.manual_seed(dim + 7 * n)
    cache = torch.randn((pages, 2, kv, page, dim), generator=g, device=gpu).to(F16)
    rows, first = n * len(contexts), [c - n for c in contexts]
    if bad:  # what no row of a sequence sees: tokens before every window, places behind the last token
        for t, c, f in zip(tables, contexts, first):
            for at in range(0, f + 1 - window, 61):
                cache[t[at // page], :, :, at % page] = float("nan")
            if c % page:
                cache[t[c // page], :, :, c % page:] = float("inf")
    q = torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32)).to(dtype)
    out = torch.full((rows, heads, dim), 7.0, device=gpu, dtype=dtype)
    there, at = _i32(gpu, tables), _i32(gpu, first)
    queries = q.to(gpu)
    torch.empty(1 << 30, device=gpu, dtype=torch.uint8).fill_(1)  # keys and values leave the caches
    q4k.attention(queries, cache[:, 0], cache[:, 1], there, at, out, query_counts=[n] * len(contexts), window=window)
    torch.cuda.synchronize()
    for s, h in probe:
        s, h = s % len(contexts), h % heads
        mine = [p for p in tables[s] if p >= 0]
        c = cache[torch.tensor(mine, device=gpu), :, h * kv // heads].cpu().numpy()[:, :, None]
        want, bound = ref.attention(q[s * n:(s + 1) * n, h:h + 1].float().numpy(), c[:, 0], c[:, 1], [list(range(len(mine)))], [first[s]], [n],
                                    window=window, f16=dtype == F16)
        _close(out[s * n:(s + 1) * n, h:h + 1], want, bound, f"sequence {s} head {h}: {n} rows, {heads}/{kv} heads of {dim}, pages of {page}, {dtype}")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [8, 24, 32, 40, 64, 72, 80, 104, 128, 136, 144, 152, 160, 168, 192, 200, 208, 216, 224, 232, 256])
def test_refilled_tiles(q4k, gpu, dim, dtype):
    _run(q4k, gpu, 1, 4, 4, dim, 16, dtype)
    _run(q4k, gpu, 5, 8, 4, dim, 32, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv,dim", [(24, 4, 32), (36, 4, 64), (24, 4, 80), (36, 4, 128)])
def test_refilled_tiles_of_more_rows(q4k, gpu, heads, kv, dim, dtype):
    """Two and three tiles of 16 rows of a cache head."""
    _run(q4k, gpu, 5, heads, kv, dim, 32, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [32, 64, 80, 160, 224, 256])
def test_refilled_tiles_behind_a_window(q4k, gpu, dim, dtype):
    _run(q4k, gpu, 1, 8, 8, dim, 16, dtype, window=1500, bad=True)
    _run(q4k, gpu, 4, 8, 8, dim, 64, dtype, window=1999, bad=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [32, 160, 224])
def test_keys_past_the_memory_side_cache(q4k, gpu, dim, dtype):
    """400 MB and more of keys and values a call: transfers that take long."""
    contexts = [16384 * 6 * 32 // dim - 32 * i - 5 for i in range(8)]
    _run(q4k, gpu, 1, 4, 4, dim, 128, dtype, probe=((0, 0), (5, 3)), contexts=contexts)
