"""Adapters in the forms that only some sizes take, against 64-bit numpy: the
one-launch kernel with two rows, with a long K in several rounds and with ranks
of three, storage off alignment in every form, values past the ranks in use of
large stacks, four row tiles to a workgroup at the ranks whose B stays in
registers, and workgroups of several column steps."""
import numpy as np
import pytest
import torch

from test_gpu_lora import _check, _stacks

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("k", [256, 4096])
@pytest.mark.parametrize("r", [1, 5, 8])
@pytest.mark.parametrize("counts,ids", [([2], [1]), ([2, 1, 2], [2, 0, 1]), ([1, 0, 2, 2], [0, 1, -1, 2])])
def test_one_launch_of_two_rows(q4k, gpu, counts, ids, r, k, dtype):
    _check(q4k, gpu, counts, ids, k, 1040, r, dtype)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("r", [3, 8])
@pytest.mark.parametrize("k", [3840, 4352, 8192, 11776, 12288])
def test_one_launch_of_a_long_k(q4k, gpu, k, r, dtype):
    _check(q4k, gpu, [1, 1], [1, 0], k, 528, r, dtype)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("r", [9, 16, 17, 23, 24])
def test_one_launch_of_many_ranks(q4k, gpu, r, dtype):
    _check(q4k, gpu, [1] * 4, [2, 0, 1, 2], 4096, 4096, r, dtype, ranks=[r, 5, r - 1])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("counts,r", [([1, 1], 6), ([1, 1], 16), ([1, 1], 24), ([2, 1], 8), ([1, 40], 33), ([30, 3], 64), ([5, 18], 70), ([20, 1], 300)])
def test_shifted_storage_of_every_form(q4k, gpu, counts, r, dtype):
    """Every tensor one element off alignment: the bits of aligned ones."""
    rng = np.random.default_rng(r)
    m, k, n = sum(counts), 512, 272
    a, b = (torch.from_numpy(v).to(gpu) for v in _stacks(rng, 2, r, k, n))
    x, h = (torch.from_numpy(rng.standard_normal((m, w)).astype(np.float32)).to(gpu).to(dtype) for w in (k, n))
    ids = torch.tensor([1, 0], dtype=torch.int32, device=gpu)
    shift = lambda t: torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    y, ys = torch.empty_like(h), shift(torch.zeros_like(h))
    q4k.lora(x, a, b, ids, m, y, auxiliary=h, query_counts=counts)
    q4k.lora(shift(x), shift(a), shift(b), shift(ids), m, ys, auxiliary=shift(h), query_counts=counts)
    torch.cuda.synchronize()
    assert torch.equal(y, ys)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("r,ranks", [(24, [9, 24, 1]), (32, [32, 17, 3]), (64, [20, 64, 33]), (64, [0, 1, 63]), (300, [1, 70, 300]), (300, [257, 64, 16]),
                                     (512, [511, 255, 512])])
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 5, 70]])
def test_ranks_in_use_of_large_stacks(q4k, gpu, counts, r, ranks, dtype):
    """NaN in a and infinities in b past every adapter's rank."""
    _check(q4k, gpu, counts, [2, 0, 1], 768, 80, r, dtype, ranks=ranks)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("r", [8, 16, 24, 32, 48, 64])
def test_four_row_tiles(q4k, gpu, r, dtype):
    _check(q4k, gpu, [700, 868], [1, 0], 512, 12288, r, dtype, slots=2)


@pytest.mark.parametrize("r,dtype", [(16, F16), (32, F16), (64, F16), (64, F32), (72, F16)])
def test_several_column_steps(q4k, gpu, r, dtype):
    """Two steps of 256 columns to a workgroup, the last one of 16."""
    _check(q4k, gpu, [2000, 112], [1, 0], 256, 16400, r, dtype, slots=2)
