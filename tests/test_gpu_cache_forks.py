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
