"""Adapters with outputs on both sides of the size from which they are written
past the caches (64 MB of aux and y): with aux, then in place, which moves half
as much, on either side of it or both past it, with few and many K-slices."""
import pytest
import torch

from test_gpu_lora import _check

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


@pytest.mark.parametrize("r", [16, 32, 64, 100])
@pytest.mark.parametrize("k,counts,dtype", [(1024, [1000, 24], F32), (1024, [1300, 108], F16), (512, [1000, 24], F32), (1024, [1311, 64], F32)])
def test_outputs_past_the_caches(q4k, gpu, k, counts, dtype, r):
    _check(q4k, gpu, counts, [1, 0], k, 12288, r, dtype, slots=2)
