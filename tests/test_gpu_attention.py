"""Attention over a paged cache on the GPU against 64-bit numpy (cache_ref),
within bounds that count the roundings: head sizes, groups, page sizes, one
row to many, one key to many, ragged batches, caps, windows, biases, strides,
tables in any order, pages that are not there, rows that see nothing, and
infinities and NaN where a row does not look."""
import numpy as np
import pytest
import torch

import cache_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def _i32(gpu, v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _cache(rng, gpu, pages, heads, page, dim):
    return torch.from_numpy(rng.standard_normal((pages, 2, heads, page, dim)).astype(np.float16)).to(gpu)


def _tables(rng, contexts, page, spare=2):
    need = [-(-c // page) for c in contexts]
    order = rng.permutation(sum(need) + spare)
    width, at, tables = max(need) + 1, 0, []
    for n in need:
        tables.append([int(p) for p in order[at:at + n]] + [-1] * (width - n))
        at += n
    return tables, sum(need) + spare


def _close(got, want, bound, what):
    got = got.cpu().double().numpy()
    off = np.abs(got - want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    bad = off > bound
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(off / bound):.2f} times the bound at {np.unravel_index(np.nanargmax(off / bound), off.shape)}"


def _check(q4k, gpu, counts, contexts, heads, kv, dim, page, dtype, seed=0, softcap=0.0, window=0, slopes=False, scale=None, size=1.0):
    rng = np.random.default_rng(seed + 7919 * heads + 104729 * dim + 31 * page + sum(contexts))
    tables, pages = _tables(rng, contexts, page)
    cache = _cache(rng, gpu, pages, kv, page, dim)
    rows = sum(counts)
    q = torch.from_numpy((size * rng.standard_normal((rows + 1, heads, dim))).astype(np.float32)).to(dtype)
    first = [c - n for c, n in zip(contexts, counts)]
    sl = torch.from_numpy(rng.uniform(0.0, 0.5, heads).astype(np.float32)) if slopes else None
    out = torch.full((rows + 1, heads, dim), 7.0, device=gpu, dtype=dtype)
    got = q4k.attention(q.to(gpu), cache[:, 0], cache[:, 1], _i32(gpu, tables), _i32(gpu, first), out, query_counts=counts, scale=scale,
                        softcap=softcap, window=window, slopes=None if sl is None else sl.to(gpu))
    torch.cuda.synchronize()
    assert got is out and (out[rows].cpu() == 7.0).all()
    c = cache.cpu().numpy()
    want, bound = ref.attention(q[:rows].float().numpy(), c[:, 0], c[:, 1], tables, first, counts, scale=scale, softcap=softcap, window=window,
                                slopes=None if sl is None else sl.numpy().astype(np.float64), f16=dtype == F16)
    _close(out[:rows], want, bound, f"{counts} of {contexts}, {heads}/{kv} heads of {dim}, pages of {page}, {dtype}")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [8, 16, 40, 64, 72, 80, 96, 112, 128, 136, 160, 192, 200, 256])
def test_head_sizes(q4k, gpu, dim, dtype):
    _check(q4k, gpu, [1], [77], 4, 2, dim, 16, dtype)
    _check(q4k, gpu, [1, 3], [200, 3], 4, 1, dim, 32, dtype)
    _check(q4k, gpu, [70], [130], 2, 1, dim, 64, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_page_sizes(q4k, gpu, page, dtype):
    _check(q4k, gpu, [1, 1], [1, 2 * page + 3], 4, 2, 128, page, dtype)
    _check(q4k, gpu, [5, 2, 1], [page, page + 1, 3 * page - 1], 8, 2, 64, page, dtype)
    _check(q4k, gpu, [40, 17], [page + 40, 555], 4, 2, 128, page, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 2), (3, 1), (7, 1), (8, 1), (16, 1), (24, 3), (16, 4), (20, 1), (33, 1), (50, 2), (130, 1)])
def test_groups(q4k, gpu, heads, kv, dtype):
    _check(q4k, gpu, [1], [300], heads, kv, 64, 32, dtype)
    _check(q4k, gpu, [2, 5], [31, 100], heads, kv, 128, 32, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 2049])
def test_lengths(q4k, gpu, n, dtype):
    _check(q4k, gpu, [1], [n], 4, 2, 128, 32, dtype)
    _check(q4k, gpu, [1], [n], 8, 1, 256, 64, dtype)
    if n >= 31:
        _check(q4k, gpu, [min(n, 300)], [n], 2, 2, 64, 64, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("kw", [{}, {"softcap": 30.0}, {"softcap": 2.0, "size": 3.0}, {"window": 1}, {"window": 37}, {"window": 64}, {"window": 5000},
                                {"slopes": True}, {"scale": 0.3, "size": 2.0}, {"softcap": 20.0, "window": 100, "slopes": True}])
def test_options(q4k, gpu, kw, dtype):
    _check(q4k, gpu, [1, 1, 1], [5, 400, 1029], 8, 2, 128, 64, dtype, **kw)
    _check(q4k, gpu, [4, 0, 5], [4, 100, 333], 8, 2, 256, 16, dtype, **kw)
    _check(q4k, gpu, [100, 3, 61], [300, 333, 61], 4, 2, 64, 32, dtype, **kw)
    _check(q4k, gpu, [150], [520], 4, 1, 128, 128, dtype, **kw)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_ragged_prompts(q4k, gpu, dtype):
    """Rows of one to many sequences, contexts of none to long, more heads than a tile."""
    counts = [51, 37, 1, 1, 90, 5, 1, 64]
    _check(q4k, gpu, counts, [51, 500, 1, 800, 333, 1005, 64, 64], 8, 2, 128, 64, dtype)
    _check(q4k, gpu, [1] * 64, list(range(1, 65)), 4, 2, 64, 16, dtype)
    _check(q4k, gpu, [3] * 20, [17 * i + 3 for i in range(20)], 8, 1, 80, 16, dtype)
    _check(q4k, gpu, [300, 1], [300, 301], 5, 1, 256, 32, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_long_contexts(q4k, gpu, dtype):
    _check(q4k, gpu, [1, 1], [20000, 8191], 4, 1, 128, 64, dtype)
    _check(q4k, gpu, [5], [12345], 4, 2, 64, 128, dtype, softcap=50.0)
    _check(q4k, gpu, [33], [6000], 2, 1, 128, 128, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_large_scores(q4k, gpu, dtype):
    """Weights that fall on one key, and scores whose spread passes what fp16 holds."""
    _check(q4k, gpu, [1, 2], [600, 700], 4, 2, 128, 64, dtype, size=30.0)
    _check(q4k, gpu, [80], [300], 4, 2, 128, 64, dtype, size=30.0)


def _strided(q4k, gpu, dtype, counts, contexts):
    """q and out in rows of a joined projection, k and v token by token, slots that reorder the tables."""
    rng = np.random.default_rng(5)
    heads, kv, dim, page = 6, 3, 64, 32
    tables, pages = _tables(rng, contexts, page)
    store = torch.from_numpy(rng.standard_normal((pages, page, 2, kv, dim)).astype(np.float16)).to(gpu)
    kc, vc = store[:, :, 0].transpose(1, 2), store[:, :, 1].transpose(1, 2)
    rows = sum(counts)
    joined = torch.from_numpy(rng.standard_normal((rows, 2 * heads * dim + 40)).astype(np.float32)).to(dtype).to(gpu)
    q = joined[:, 8:8 + 2 * heads * dim].view(rows, heads, 2 * dim)[:, :, :dim]
    store_out = torch.full((heads, rows, dim + 3), 3.0, device=gpu, dtype=dtype)
    out = store_out.transpose(0, 1)[:, :, 1:dim + 1]
    slots = list(range(len(counts)))[::-1]
    first = [contexts[s] - n for s, n in zip(slots, counts)]
    q4k.attention(q, kc, vc, _i32(gpu, tables), _i32(gpu, first), out, query_counts=counts, slots=_i32(gpu, slots))
    torch.cuda.synchronize()
    want, bound = ref.attention(q.cpu().float().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), tables, first, counts, slots=slots, f16=dtype == F16)
    _close(out, want, bound, "strided")
    assert (store_out[..., 0] == 3.0).all() and (store_out[..., dim + 1:] == 3.0).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides_and_slots(q4k, gpu, dtype):
    _strided(q4k, gpu, dtype, [1, 2, 1], [70, 33, 200])
    _strided(q4k, gpu, dtype, [40, 1, 100], [170, 133, 200])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("counts", [[2, 3, 1, 1], [40, 65, 1, 1]])
def test_pages_that_are_not_there(q4k, gpu, dtype, counts):
    """Numbers below and past the cache's are no pages, at the front, within and
    behind; positions before the table and behind it; slots outside it."""
    rng = np.random.default_rng(11)
    page, dim, kv, heads = 16, 64, 1, 4
    cache = _cache(rng, gpu, 9, kv, page, dim)
    tables = [[-1, 3, 9, 2, -7, 1 << 30, 8, 0, -1, -1], [4, 5, -1, -1, -1, -1, -1, -1, -1, -1], [7] * 10, [-1] * 10]
    q = torch.from_numpy(rng.standard_normal((sum(counts), heads, dim)).astype(np.float32)).to(dtype)
    c = cache.cpu().numpy()
    for first, slots in [([100, 10, 5, 30], [0, 1, 2, 3]), ([-1, 158, 160, 3], [0, 2, 2, 1]), ([-100, 1 << 29, -2, 0], [1, 2, 0, -1]),
                         ([0, 20, 31, 1], [1 << 30, 1, 4, 0])]:
        out = torch.full(q.shape, 5.0, device=gpu, dtype=dtype)
        q4k.attention(q.to(gpu), cache[:, 0], cache[:, 1], _i32(gpu, tables), _i32(gpu, first), out, query_counts=counts, slots=_i32(gpu, slots))
        torch.cuda.synchronize()
        want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts, slots=slots, f16=dtype == F16)
        _close(out, want, bound, f"{first} {slots}")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), 65504.0])
@pytest.mark.parametrize("counts,contexts,window", [([1, 2], [70, 45], 0), ([5], [300], 20), ([90], [200], 0), ([70, 66], [200, 90], 33), ([150], [150], 0)])
def test_what_a_row_does_not_see(q4k, gpu, dtype, bad, counts, contexts, window):
    """Keys and values of later tokens, of tokens before the window, of places
    behind the sequence and of pages of nobody do not reach a row; what it
    sees does: a NaN among its values makes it NaN."""
    rng = np.random.default_rng(3)
    heads, kv, dim, page = 4, 2, 128, 32
    tables, pages = _tables(rng, contexts, page)
    cache = _cache(rng, gpu, pages, kv, page, dim)
    rows, first = sum(counts), [c - n for c, n in zip(contexts, counts)]
    q = torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32)).to(dtype)
    used = {p for t in tables for p in t}
    for p in range(pages):
        if p not in used:
            cache[p] = bad
    for t, n in zip(tables, contexts):
        if n % page:
            cache[t[n // page], :, :, n % page:] = bad
    # One token of the last sequence that some of its rows see: before the window's end, or a later row's own.
    token = contexts[-1] - max(1, counts[-1] // 2) if counts[-1] > 1 else contexts[-1] - 30
    cache[tables[-1][token // page], 1, :, token % page, 5] = bad
    if window:  # tokens before every row's window
        for at in range(0, max(0, first[-1] + 1 - window), 7):
            cache[tables[-1][at // page], :, :, at % page] = bad
    out = torch.empty(q.shape, device=gpu, dtype=dtype)
    q4k.attention(q.to(gpu), cache[:, 0], cache[:, 1], _i32(gpu, tables), _i32(gpu, first), out, query_counts=counts, window=window)
    torch.cuda.synchronize()
    c = cache.cpu().numpy()
    want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts, window=window, f16=dtype == F16)
    fine = np.isfinite(want)
    if np.isfinite(bad):
        fine[:] = True
    got = out.cpu().double().numpy()
    assert np.isfinite(got[fine]).all() and not np.isfinite(got[~fine]).any()
    _close(out.cpu().masked_fill(torch.from_numpy(~fine), 0.0), np.where(fine, want, 0.0), np.where(fine, bound, 1.0), f"{bad}")


@pytest.mark.parametrize("dtype", [F16, F32])
def test_infinite_and_nan_queries(q4k, gpu, dtype):
    """A query with a NaN makes its own head's row NaN and nothing else."""
    rng = np.random.default_rng(4)
    for counts, contexts in [([2], [90]), ([70], [200])]:
        tables, pages = _tables(rng, contexts, 32)
        cache = _cache(rng, gpu, pages, 2, 32, 128)
        q = torch.from_numpy(rng.standard_normal((counts[0], 4, 128)).astype(np.float32)).to(dtype)
        q[1, 2, 3] = float("nan")
        out = torch.empty(q.shape, device=gpu, dtype=dtype)
        first = [contexts[0] - counts[0]]
        q4k.attention(q.to(gpu), cache[:, 0], cache[:, 1], _i32(gpu, tables), _i32(gpu, first), out)
        torch.cuda.synchronize()
        c = cache.cpu().numpy()
        want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts, f16=dtype == F16)
        assert np.isnan(out[1, 2].cpu().numpy()).all()
        want[1, 2] = np.nan
        _close(out, want, np.where(np.isnan(bound), 1.0, bound), "NaN query")


def test_no_rows(q4k, gpu):
    cache = torch.zeros((2, 2, 1, 16, 64), device=gpu, dtype=F16)
    q = torch.empty((0, 2, 64), device=gpu)
    out = torch.empty_like(q)
    q4k.attention(q, cache[:, 0], cache[:, 1], _i32(gpu, [[0]]), _i32(gpu, [0]), out)
    q4k.attention(q, cache[:, 0], cache[:, 1], _i32(gpu, [[0], [1]]), _i32(gpu, [0, 0]), out, query_counts=[0, 0])
    # A cache without pages, tables without room: every row sees nothing.
    q = torch.randn((3, 2, 64), device=gpu)
    out = torch.ones_like(q)
    q4k.attention(q, cache[:0, 0], cache[:0, 1], _i32(gpu, [[0]]), _i32(gpu, [0]), out)
    assert (out == 0).all()
    out.fill_(1.0)
    q4k.attention(q, cache[:, 0], cache[:, 1], torch.empty((1, 0), device=gpu, dtype=torch.int32), _i32(gpu, [0]), out)
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("counts", [[1, 3], [40, 17]])
def test_smallest_scores(q4k, gpu, counts, dtype):
    """Scores that underflow: a plain mean of the values that a row sees."""
    _check(q4k, gpu, counts, [77, 130], 4, 2, 128, 16, dtype, scale=1e-38)
    _check(q4k, gpu, counts, [77, 130], 4, 2, 128, 16, dtype, scale=1e-30, size=1e-7 if dtype == F16 else 1e-35)
    _check(q4k, gpu, counts, [77, 130], 4, 2, 128, 16, dtype, softcap=2.0 ** -64, window=30)


@pytest.mark.parametrize("counts", [[1, 3], [40, 17]])
def test_largest_cap(q4k, gpu, counts):
    """A cap of 2^64 leaves scores as they are: their cubes over 3 * 2^128 are
    nothing.  The cap's function is good to 2^-21 of its value, so scores up to x
    are off by 2^-21 x more, and outputs by twice that of the largest value."""
    rng = np.random.default_rng(5)
    tables, pages = _tables(rng, [77, 130], 16)
    cache = _cache(rng, gpu, pages, 2, 16, 64)
    q = torch.from_numpy(rng.standard_normal((sum(counts), 4, 64)).astype(np.float32))
    first = [77 - counts[0], 130 - counts[1]]
    out = q4k.attention(q.to(gpu), cache[:, 0], cache[:, 1], _i32(gpu, tables), _i32(gpu, first), torch.empty_like(q, device=gpu), query_counts=counts,
                        softcap=2.0 ** 64)
    c = cache.cpu().numpy()
    want, bound = ref.attention(q.numpy(), c[:, 0], c[:, 1], tables, first, counts)
    x = 0.125 * np.sqrt((q.numpy() ** 2).sum(-1).max() * (c[:, 0].astype(np.float64) ** 2).sum(-1).max())  # no score is above
    _close(out, want, bound + 2 * 2.0 ** -21 * x * np.abs(c[:, 1]).max(), "cap of 2^64")
