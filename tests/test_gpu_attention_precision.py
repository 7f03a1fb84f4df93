"""Attention of few fp16 rows: the output's own rounding to fp16 and what fp32 rows
may be off by (cache_ref's bound for weights of 22 bits), no more."""
import pytest
import torch

import cache_ref as ref
from operators_ref import half_step
from test_gpu_attention import _close
from test_gpu_attention_values import _attend, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (12, 1, 64), (9, 1, 80), (4, 1, 128), (8, 1, 128), (4, 2, 192), (4, 2, 256)])
@pytest.mark.parametrize("counts,contexts", [([1], [1]), ([1, 1], [60, 5000]), ([3, 4], [300, 1500])])
def test_few_rows(q4k, gpu, counts, contexts, heads, kv, dim):
    if max(counts) * heads // kv > (48 if dim <= 128 else 16):
        counts = [1] * len(counts)
    tables, cache, q, first = _case(gpu, counts, contexts, heads, kv, dim, 32, torch.float16)
    out = _attend(q4k, gpu, q, cache, tables, first, counts)
    c = cache.cpu().numpy()
    want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts)
    _close(out, want, bound + half_step(want, True), f"{counts} of {contexts}, {heads}/{kv} heads of {dim}")
