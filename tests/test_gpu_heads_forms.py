"""Rotary positions and head norms of many rows, where a lane takes two rows at
a time: with the norm, in both layouts, whole and in part, out of place, in place
in the rows of a joined projection, and head-major, against 64-bit numpy."""
import numpy as np
import pytest
import torch

import operators_ref as ref
from test_gpu_heads import _check_rope, _freq, _host, _x

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
SHAPES = [(2047, 32, 8, 128, 128, False), (2047, 32, 8, 128, 128, True), (1801, 16, 4, 256, 64, False), (1801, 16, 4, 256, 64, True),
          (4099, 9, 3, 64, 32, True), (4099, 7, 2, 64, 64, False)]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,hq,hk,dim,rot,inter", SHAPES)
def test_norms_of_many_rows(q4k, gpu, rows, hq, hk, dim, rot, inter, dtype):
    rng = np.random.default_rng(rows + hq)
    joined = _x(rng, rows, (hq + 2 * hk) * dim, dtype=dtype).to(gpu)
    wq, wk = (torch.from_numpy(rng.uniform(0.5, 1.5, dim).astype(np.float32)) for _ in range(2))
    f, p = _freq(rot), torch.arange(50000, 50000 + rows, dtype=torch.int32)

    def views(t):
        return t[:, :hq * dim].unflatten(1, (hq, dim)), t[:, hq * dim:(hq + hk) * dim].unflatten(1, (hk, dim))

    def call(q, k, qo, ko):
        q4k.qk_norm_rope(q, k, wq.to(gpu), wk.to(gpu), f.to(gpu), p.to(gpu), qo, ko, interleaved=inter, scale=1.25, eps=1e-5)
        torch.cuda.synchronize()

    q, k = views(joined)
    qo, ko = torch.full((rows + 1, hq, dim), 7.0, device=gpu, dtype=dtype), torch.full((rows + 1, hk, dim), 7.0, device=gpu, dtype=dtype)
    call(q, k, qo[:rows], ko[:rows])
    for x, w, o, name in ((q, wq, qo, "q"), (k, wk, ko, "k")):
        n = ref.head_norm(_host(x), w.numpy(), np.float32(1e-5))
        want, size = ref.rotate(n, f.numpy(), p.numpy(), inter, np.float32(1.25))
        ref.assert_close(_host(o[:rows]), want, ref.norm_bound(size, want, 1.25), dtype == F16, name)
        assert bool((o[rows] == 7.0).all())
    inplace = joined.clone()
    call(*views(inplace), *views(inplace))
    for got, want in zip(views(inplace), (qo, ko)):
        assert torch.equal(got, want[:rows])
    assert torch.equal(inplace[:, (hq + hk) * dim:], joined[:, (hq + hk) * dim:])
    major = [torch.empty((h, rows, dim), device=gpu, dtype=dtype).transpose(0, 1) for h in (hq, hk)]
    call(q, k, *major)
    assert torch.equal(major[0], qo[:rows]) and torch.equal(major[1], ko[:rows])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,heads,dim,rot,inter", [(2047, 40, 128, 128, True), (4099, 9, 128, 64, True), (1801, 20, 256, 64, False)])
def test_rope_of_many_rows(q4k, gpu, rows, heads, dim, rot, inter, dtype):
    _check_rope(q4k, gpu, rows, heads, dim, rot, inter, dtype, np.arange(rows) + 100000, scale=1.2)
    rng = np.random.default_rng(rows)
    x, f, p = _x(rng, rows, heads, dim, dtype=dtype).to(gpu), _freq(rot).to(gpu), torch.arange(rows, dtype=torch.int32, device=gpu)
    y = torch.empty_like(x)
    q4k.rope(x, f, p, y, interleaved=inter)
    q4k.rope(x, f, p, x, interleaved=inter)
    torch.cuda.synchronize()
    assert torch.equal(x, y)
