"""Writes into a paged cache, slots that take over others' states, and
compaction on the GPU, against plain Python (cache_ref): every table, every
length and every byte of the pool."""
import numpy as np
import pytest
import torch

import cache_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def _i32(gpu, v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,dim,page", [(1, 8, 16), (4, 256, 128), (3, 80, 32), (8, 128, 64), (2, 136, 1024)])
def test_write(q4k, gpu, heads, dim, page, dtype):
    rng = np.random.default_rng(heads * dim + page)
    pages, width = 11, 5
    tables = [[int(p) for p in rng.permutation(pages)[:width]] for _ in range(4)]
    tables[1] = [p for p in range(pages) if p not in tables[0]][:width]
    tables[2], tables[3] = [-1, 3, pages, -5, 1 << 30], [-1] * width
    for counts, first, slots in [([1, 1], [0, page], None), ([page + 3, 2], [page - 1, 5 * page - 1], [1, 0]), ([3, 0, 4, 5], [7, 0, page - 2, -3], [0, 1, 2, 3]),
                                 ([2, 2], [-1, 4 * page + 1], [1, -1]), ([1], [2 ** 31 - 1], None), ([2], [1], [9])]:
        rows = sum(counts)
        joined = torch.from_numpy(rng.standard_normal((rows + 2, 3 * heads * dim + 5)).astype(np.float32) * 3).to(dtype).to(gpu)
        k = joined[:, 1:1 + heads * dim].view(rows + 2, heads, dim)
        v = joined[:, 2 * heads * dim + 3:3 * heads * dim + 3].view(rows + 2, heads, dim)
        for order in range(2):  # heads outside tokens, and inside
            if order:
                store = torch.full((pages, page, 2, heads, dim), 2.0, device=gpu, dtype=F16)
                kc, vc = store[:, :, 0].transpose(1, 2), store[:, :, 1].transpose(1, 2)
            else:
                store = torch.full((pages, 2, heads, page, dim), 2.0, device=gpu, dtype=F16)
                kc, vc = store[:, 0], store[:, 1]
            want_k, want_v = kc.cpu().clone(), vc.cpu().clone()
            got = q4k.cache_write(k, v, kc, vc, _i32(gpu, tables), _i32(gpu, first), query_counts=counts, slots=None if slots is None else _i32(gpu, slots))
            torch.cuda.synchronize()
            assert got[0] is kc and got[1] is vc
            r = 0
            for s, n in enumerate(counts):
                slot = s if slots is None else slots[s]
                for t in range(n):
                    p = first[s] + t
                    if 0 <= p < width * page and 0 <= slot < 4 and 0 <= tables[slot][p // page] < pages:
                        want_k[tables[slot][p // page], :, p % page] = k[r].half().cpu()
                        want_v[tables[slot][p // page], :, p % page] = v[r].half().cpu()
                    r += 1
            assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v), (counts, first, slots, order)


def test_write_extreme_values(q4k, gpu):
    """Values past fp16's become infinite, NaN stays, the smallest round to nearest."""
    x = torch.tensor([65504.0, 65519.0, 65520.0, -1e30, float("inf"), float("nan"), 3e-8, 2e-8], device=gpu).view(1, 1, 8)
    cache = torch.zeros((1, 2, 1, 16, 8), device=gpu, dtype=F16)
    q4k.cache_write(x, -x, cache[:, 0], cache[:, 1], _i32(gpu, [[0]]), _i32(gpu, [3]))
    assert torch.equal(cache[0, 0, 0, 3].nan_to_num(7.0), x[0, 0].half().nan_to_num(7.0))
    assert torch.equal(cache[0, 1, 0, 3].nan_to_num(7.0), (-x[0, 0]).half().nan_to_num(7.0))
    assert (cache[0, :, :, :3] == 0).all() and (cache[0, :, :, 4:] == 0).all()


def _pool(rng, gpu, pages, blocks, page, token):
    return torch.from_numpy(rng.integers(0, 255, (pages, blocks, page, token), dtype=np.uint8)).to(gpu)


def _assign(q4k, gpu, pool, page, tables, lengths, parents, counts):
    slots, width = len(tables), len(tables[0])
    pages = pool.shape[0]
    want_pool = pool.cpu().clone()
    new, length, missing = torch.full((slots, width), 99, device=gpu, dtype=torch.int32), torch.full((slots,), 99, device=gpu, dtype=torch.int32), _i32(gpu, [55])
    q4k.cache_assign(pool, _i32(gpu, tables), _i32(gpu, lengths), None if parents is None else _i32(gpu, parents), new, length,
                     counts=None if counts is None else _i32(gpu, counts), missing=missing)
    torch.cuda.synchronize()
    want, want_length, want_missing, copies = ref.assign(pages, page, tables, lengths, parents if parents is not None else list(range(slots)), counts or [0] * slots)
    assert new.tolist() == want
    assert length.tolist() == want_length and missing.tolist() == [want_missing]
    for a, b, n in copies:
        want_pool[b, :, :n] = want_pool[a, :, :n]
    assert torch.equal(pool.cpu(), want_pool)
    return want, want_length


@pytest.mark.parametrize("page,blocks,token", [(16, 1, 16), (32, 4, 64), (128, 2, 512), (1, 3, 16), (1024, 1, 48)])
def test_assign(q4k, gpu, page, blocks, token):
    rng = np.random.default_rng(page + blocks)
    pages, slots, width = 40, 6, 7
    pool = _pool(rng, gpu, pages, blocks, page, token)
    order = [int(p) for p in rng.permutation(pages)]
    tables, lengths = [], [0, 1, page, 3 * page + page // 2, 2 * page + 1, 4 * page]
    for n in lengths:
        k = -(-n // page)
        tables.append([order.pop() for _ in range(k)] + [-1] * (width - k))
    for parents, counts in [(None, None), (None, [1] * slots), ([0, 1, 2, 3, 4, 5], [1, page, page + 1, 0, 5, 3 * page]), ([3] * slots, [1] * slots),
                            ([3, 3, 4, 4, -1, 6], [2, 2, 1, page, 9, 1]), ([5, 4, 3, 2, 1, 0], [0] * slots), ([-1] * slots, None),
                            ([4, 3, 4, 3, 4, 3], [7 * page, -5, 1, 1, 2, 2 ** 31 - 1])]:
        _assign(q4k, gpu, pool.clone(), page, tables, lengths, parents, counts)


def test_assign_shared_tables(q4k, gpu):
    """Slots that share full and last pages already, a page that is one slot's last
    and another's full one, numbers that are no pages, lengths outside the table."""
    rng = np.random.default_rng(2)
    pool = _pool(rng, gpu, 12, 2, 16, 32)
    tables = [[0, 1, 2, -1], [0, 1, 2, -1], [0, 1, 5, -1], [0, 7, -1, 3], [12, -4, 6, 6]]
    for lengths in ([40, 40, 48, 33, 64], [33, 48, 40, 17, 60], [-3, 1000, 20, 64, 5], [47, 46, 45, 1, 33]):
        for parents in (None, [1, 0, 2, 2, 4], [4, 4, 3, 3, 0]):
            for counts in (None, [1, 2, 30, 0, 4]):
                _assign(q4k, gpu, pool.clone(), 16, tables, lengths, parents, counts)


def test_assign_pool_runs_out(q4k, gpu):
    rng = np.random.default_rng(3)
    pool = _pool(rng, gpu, 5, 1, 16, 16)
    tables = [[0, 1, -1, -1, -1], [2, -1, -1, -1, -1], [-1] * 5]
    for counts in ([16, 16, 16], [0, 0, 100], [100, 0, 0], [30, 20, 0]):
        for parents in ([0, 1, 2], [0, 0, 0], [0, 1, 1]):
            _assign(q4k, gpu, pool.clone(), 16, tables, [20, 16, 0], parents, counts)


@pytest.mark.parametrize("seed", range(6))
def test_assign_many(q4k, gpu, seed):
    rng = np.random.default_rng(seed)
    slots, page, pages, width = [64, 1024, 200, 33, 1, 500][seed], [16, 16, 64, 32, 16, 16][seed], [700, 20000, 3000, 262144, 64, 1500][seed], [9, 16, 12, 2000, 64, 40][seed]
    pool = _pool(rng, gpu, pages, 1, page, 16)
    order = [int(p) for p in rng.permutation(pages)]
    tables, lengths = [], []
    for _ in range(slots):
        n = min(int(rng.integers(0, width * page + 1)), len(order) * page // 2)
        k = -(-n // page)
        tables.append([order.pop() for _ in range(k)] + [-1] * (width - k))
        lengths.append(n)
    parents = [int(p) for p in rng.integers(-1, slots, slots)]
    counts = [int(c) for c in rng.integers(0, 3 * page, slots)]
    now, length = _assign(q4k, gpu, pool, page, tables, lengths, parents, counts)
    # And on from there, the tokens written: beams in a new order again.
    length = [min(n + c, width * page) for n, c in zip(length, counts)]
    _assign(q4k, gpu, pool, page, now, length, [int(p) for p in rng.integers(-1, slots, slots)], [1] * slots)


@pytest.mark.parametrize("page,blocks,token", [(16, 1, 16), (32, 4, 64), (128, 8, 512), (1, 1, 16), (16, 3, 2064)])
def test_compact(q4k, gpu, page, blocks, token):
    rng = np.random.default_rng(page + token)
    for pages, slots, width in [(1, 1, 1), (40, 5, 6), (33, 8, 4), (500, 64, 7), (64, 3, 30)]:
        pool = _pool(rng, gpu, pages, blocks, page, token)
        for kind in range(4):
            order = [int(p) for p in rng.permutation(pages)]
            tables, lengths = [], []
            for _ in range(slots):
                n = min(int(rng.integers(0, width * page + 1)), len(order) * page // 2)
                k = -(-n // page)
                tables.append([order.pop() for _ in range(k)] + [int(p) for p in rng.integers(-2, pages + 2, width - k)])
                lengths.append(n)
            if kind == 1:
                tables = [list(tables[0]) for _ in tables]  # all share their pages
            if kind == 2:
                tables = [[-1 if e % 2 else p for e, p in enumerate(t)] for t in tables]
            if kind == 3:
                lengths = [-5 if s % 2 else 10 * width * page for s in range(slots)]
            got_pool, want_pool = pool.clone(), pool.cpu().clone()
            new, used = torch.full((slots, width), 99, device=gpu, dtype=torch.int32), _i32(gpu, [77])
            q4k.cache_compact(got_pool, _i32(gpu, tables), _i32(gpu, lengths), new, used=used)
            torch.cuda.synchronize()
            want, n, moves = ref.compact(pages, page, tables, lengths)
            assert new.tolist() == want and used.tolist() == [n]
            for a, b in moves:
                want_pool[b] = want_pool[a]
            assert torch.equal(got_pool.cpu(), want_pool)


def test_nothing_to_do(q4k, gpu):
    pool = torch.zeros((4, 1, 16, 16), device=gpu, dtype=torch.uint8)
    none, empty = torch.empty((0, 3), device=gpu, dtype=torch.int32), torch.empty(0, device=gpu, dtype=torch.int32)
    n = _i32(gpu, [9])
    q4k.cache_assign(pool, none, empty, empty, none.clone(), empty.clone(), missing=n)
    assert n.tolist() == [0]
    n.fill_(9)
    q4k.cache_compact(pool, none, empty, none.clone(), used=n)
    assert n.tolist() == [0]
    flat = torch.empty((2, 0), device=gpu, dtype=torch.int32)
    length = _i32(gpu, [7, 7])
    q4k.cache_assign(pool, flat, _i32(gpu, [3, 4]), _i32(gpu, [1, 0]), flat.clone(), length, counts=_i32(gpu, [1, 17]), missing=n)
    assert length.tolist() == [0, 0] and n.tolist() == [3]


def test_assign_missing_at_most(q4k, gpu):
    """More pages asked for than 32 bits count: 40 slots of 2^27 each."""
    pool = torch.zeros((3, 1, 16, 16), device=gpu, dtype=torch.uint8)
    for n, want in ((40, 2 ** 31 - 1), (15, 15 * 2 ** 27 - 3)):
        tables, lengths = _i32(gpu, [[-1]] * n), _i32(gpu, [0] * n)
        new, length, missing = torch.empty_like(tables), torch.empty_like(lengths), _i32(gpu, [55])
        q4k.cache_assign(pool, tables, lengths, None, new, length, counts=_i32(gpu, [2 ** 31 - 1] * n), missing=missing)
        assert missing.item() == want and new.flatten().tolist() == [0, 1, 2] + [-1] * (n - 3)


def test_assign_many_blocks(q4k, gpu):
    """A page of 2^24 blocks: more than a launch has workgroups for, one each."""
    blocks = 1 << 24
    pool = torch.zeros((2, blocks, 2, 16), device=gpu, dtype=torch.uint8)
    pool[0] = torch.arange(blocks, device=gpu).view(blocks, 1, 1).remainder(251).to(torch.uint8)
    new, length = _i32(gpu, [[9], [9]]), _i32(gpu, [9, 9])
    q4k.cache_assign(pool, _i32(gpu, [[0], [-1]]), _i32(gpu, [1, 0]), _i32(gpu, [0, 0]), new, length)
    assert new.tolist() == [[0], [1]] and length.tolist() == [1, 1]
    assert torch.equal(pool[0, :, 0], pool[1, :, 0]) and (pool[1, :, 1] == 0).all()
