"""Copies that cache_assign makes of pages that are written on: a single slot whose
table lists a page twice, few and many slots that fork among many that do not, pages of one block to
many, against plain Python (cache_ref): tables, lengths and every byte of the pool."""
import numpy as np
import pytest

from test_gpu_cache import _assign, _pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [1, 2, 3])
@pytest.mark.parametrize("parents", [None, [0, 0, 0]])
def test_a_page_listed_twice(q4k, gpu, slots, parents):
    """A slot's last page that is one of its own full ones too is copied, in whatever number of slots."""
    rng = np.random.default_rng(slots)
    pool = _pool(rng, gpu, 9, 3, 16, 32)
    tables, lengths = [[3, 3, -1, -1], [4, 5, 4, -1], [7, -1, -1, -1]][:slots], [20, 40, 0][:slots]
    for counts in (None, [0, 1, 5][:slots], [14, 30, 1][:slots]):
        _assign(q4k, gpu, pool.clone(), 16, tables, lengths, None if parents is None else parents[:slots], counts)


@pytest.mark.parametrize("slots,page,blocks,token", [(5, 16, 1, 16), (64, 32, 7, 32), (257, 16, 2, 16), (300, 64, 3, 512), (1024, 2, 1, 48)])
@pytest.mark.parametrize("forks", [0, 1, 2, 1000])
def test_forks_among_many_slots(q4k, gpu, slots, page, blocks, token, forks):
    """No slot, the last one, two and nearly all that start from others' pages; blocks of less and more than a workgroup copies at once."""
    rng = np.random.default_rng(slots + forks)
    lengths = [int(n) for n in rng.integers(0, 3 * page, slots)]
    tables, used = [], 0
    for n in lengths:
        k = -(-n // page)
        tables.append(list(range(used, used + k)) + [-1] * (4 - k))
        used += k
    pages = used + 2 * slots + 3
    order = [int(p) for p in rng.permutation(pages)]
    tables = [[order[p] if p >= 0 else -1 for p in t] for t in tables]
    parents = list(range(slots))
    if forks == 1000:
        parents = [int(p) for p in rng.integers(-1, slots, slots)]
    else:
        for s in range(slots - forks, slots):
            parents[s] = int(rng.integers(0, slots - forks))
            lengths[parents[s]] = lengths[parents[s]] // page * page + page // 2 if lengths[parents[s]] else 0
    _assign(q4k, gpu, _pool(rng, gpu, pages, blocks, page, token), page, tables, lengths, parents, [int(n) for n in rng.integers(0, page, slots)])
