"""Rotary positions and head norms on the GPU against 64-bit numpy
(operators_ref), within bounds that count the roundings: head sizes and rotated
parts that take each vector width, both layouts, both types, strided and
head-major storage, in place, far positions, one row to many, norms of zero
rows, infinities and NaN."""
import numpy as np
import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def _x(rng, *shape, dtype):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype)


def _freq(rot, base=10000.0):
    return torch.from_numpy(base ** (-np.arange(0, rot, 2, dtype=np.float64) / max(rot, 1)))


def _host(t):
    return t.cpu().float().numpy()


def _check_rope(q4k, gpu, rows, heads, dim, rot, inter, dtype, positions, scale=1.0, far=False, seed=0):
    rng = np.random.default_rng(seed + rows * 131 + heads * 17 + dim * 3 + rot)
    x, f = _x(rng, rows, heads, dim, dtype=dtype), _freq(rot)
    p = torch.tensor(positions, dtype=torch.int32)
    y = torch.full((rows + 1, heads, dim), float("nan"), device=gpu, dtype=dtype)
    got = q4k.rope(x.to(gpu), f.to(gpu), p.to(gpu), y[:rows], interleaved=inter, scale=scale)
    torch.cuda.synchronize()
    want, size = ref.rotate(_host(x), f.numpy(), p.numpy(), inter, np.float32(scale))
    ref.assert_close(_host(got), want, ref.rotate_bound(size, scale, far), dtype == F16, f"{rows}x{heads}x{dim} rot {rot}")
    # Behind the pairs a copy, behind the rows nothing.
    assert torch.equal(got.cpu()[..., rot:], x[..., rot:])
    assert torch.isnan(y[rows]).all()


SIZES = [(128, 128), (256, 64), (64, 64), (80, 80), (96, 48), (112, 28), (80, 20), (128, 2), (2, 2), (65, 64), (7, 6), (66, 66), (192, 128),
         (320, 320), (576, 64), (1024, 1024), (1024, 510), (1023, 1022)]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dim,rot", SIZES)
def test_rope_sizes(q4k, gpu, dim, rot, inter, dtype):
    rng = np.random.default_rng(dim + rot)
    for rows, heads in [(1, 1), (3, 5), (9, 4)]:
        _check_rope(q4k, gpu, rows, heads, dim, rot, inter, dtype, rng.integers(0, 70000, rows))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,heads,dim,rot", [(8, 32, 128, 128), (821, 16, 256, 64), (2047, 40, 128, 128), (4099, 9, 128, 64), (5000, 1, 64, 64)])
def test_rope_many_rows(q4k, gpu, rows, heads, dim, rot, dtype):
    _check_rope(q4k, gpu, rows, heads, dim, rot, False, dtype, np.arange(rows) + 100000, scale=1.2)


def test_heads_of_millions_of_rows(q4k, gpu):
    """More rows than one launch takes: around its end, and at both ends, the
    bits of calls on those rows alone."""
    rows, f = (1 << 23) + 70, _freq(2).to(gpu)
    x = torch.randn((rows, 2, 2), device=gpu).half()
    p = torch.arange(rows, dtype=torch.int32, device=gpu)
    w = torch.tensor([0.5, 2.0], device=gpu)
    y, q, k = torch.empty_like(x), torch.empty_like(x)[:, :1], torch.empty_like(x)[:, :1]
    q4k.rope(x, f, p, y)
    q4k.qk_norm_rope(x[:, :1], x[:, 1:], w, w, f, p, q, k)
    for part in (slice(0, 100), slice((1 << 23) - 50, (1 << 23) + 50), slice(rows - 30, rows)):
        want, wq, wk = torch.empty_like(x[part]), torch.empty_like(q[part]), torch.empty_like(k[part])
        q4k.rope(x[part], f, p[part], want)
        q4k.qk_norm_rope(x[part, :1], x[part, 1:], w, w, f, p[part], wq, wk)
        torch.cuda.synchronize()
        assert torch.equal(y[part], want) and torch.equal(q[part], wq) and torch.equal(k[part], wk)


def test_rope_far_and_negative_positions(q4k, gpu):
    _check_rope(q4k, gpu, 7, 3, 128, 128, False, F32, [2**31 - 1, -(2**31), 2**30 + 7, -1, 0, 1 << 24, 12345678], far=True)
    # Up to 2^20 the near bound holds.
    _check_rope(q4k, gpu, 4, 3, 128, 128, True, F32, [(1 << 20) - 1, 999999, -(1 << 20), 777777])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("norm", [False, True])
def test_heads_in_place_and_strided(q4k, gpu, dtype, norm):
    """q and k inside the rows of a joined projection, in place (values and
    what lies between heads stay), then head-major outputs and shifted storage:
    every form gives the bits of the contiguous one."""
    rows, hq, hk, dim, rot = 13, 6, 2, 128, 64
    rng = np.random.default_rng(5)
    joined = _x(rng, rows, (2 * hq + 2 * hk) * dim, dtype=dtype).to(gpu)
    f, p = _freq(rot).to(gpu), torch.arange(7, 7 + rows, dtype=torch.int32, device=gpu)
    wq, wk = (torch.from_numpy(rng.uniform(0.5, 1.5, dim).astype(np.float32)).to(gpu) for _ in range(2))

    def views(t):
        q = t[:, :2 * hq * dim].unflatten(1, (hq, 2 * dim))[:, :, :dim]  # a gate of dim values behind every query head
        k = t[:, 2 * hq * dim:(2 * hq + hk) * dim].unflatten(1, (hk, dim))
        return q, k

    def call(q, k, qo, ko):
        if norm:
            q4k.qk_norm_rope(q, k, wq, wk, f, p, qo, ko)
        else:
            q4k.rope(q, f, p, qo)
            q4k.rope(k, f, p, ko)
        torch.cuda.synchronize()

    q, k = views(joined)
    qo, ko = torch.empty((rows, hq, dim), device=gpu, dtype=dtype), torch.empty((rows, hk, dim), device=gpu, dtype=dtype)
    call(q, k, qo, ko)
    inplace = joined.clone()
    qi, ki = views(inplace)
    call(qi, ki, qi, ki)
    assert torch.equal(qi, qo) and torch.equal(ki, ko)
    keep = torch.ones_like(joined, dtype=torch.bool)
    for v in views(keep):
        v.fill_(False)
    assert torch.equal(inplace[keep], joined[keep])
    # Head-major outputs ([heads, rows, dim] storage), one element off alignment.
    store = torch.full((hq * (rows + 3) * dim + 1,), 7.0, device=gpu, dtype=dtype)
    q_hm = store[1:].view(hq, rows + 3, dim).transpose(0, 1)[:rows]
    k_hm = torch.empty((hk, rows, dim), device=gpu, dtype=dtype).transpose(0, 1)
    call(q, k, q_hm, k_hm)
    assert torch.equal(q_hm, qo) and torch.equal(k_hm, ko)
    assert bool((store[1:].view(hq, rows + 3, dim)[:, rows:] == 7.0).all()) and store[0] == 7.0
    # A row broadcast over all rows (stride 0).
    one = q[:1].expand(rows, hq, dim)
    each, copied = torch.empty_like(qo), torch.empty_like(qo)
    call(one, k, each, ko)
    call(one.contiguous(), k, copied, ko)
    assert torch.equal(each, copied)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows", [1, 9])
def test_qk_heads_in_turn(q4k, gpu, rows, dtype):
    """q, k and v heads in turn in the rows of one projection, in place and
    into one buffer of the same form: the bits of separate tensors, v as it was."""
    rng = np.random.default_rng(31)
    qkv = _x(rng, rows, 6, 3, 64, dtype=dtype).to(gpu)
    f, p = _freq(64).to(gpu), torch.arange(5, 5 + rows, dtype=torch.int32, device=gpu)
    wq, wk = (torch.from_numpy(rng.uniform(0.5, 1.5, 64).astype(np.float32)).to(gpu) for _ in range(2))
    q, k = qkv[:, :, 0].contiguous(), qkv[:, :, 1].contiguous()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    q4k.qk_norm_rope(q, k, wq, wk, f, p, qo, ko)
    other = torch.full_like(qkv, 7.0)
    q4k.qk_norm_rope(qkv[:, :, 0], qkv[:, :, 1], wq, wk, f, p, other[:, :, 0], other[:, :, 1])
    got = qkv.clone()
    q4k.qk_norm_rope(got[:, :, 0], got[:, :, 1], wq, wk, f, p, got[:, :, 0], got[:, :, 1])
    torch.cuda.synchronize()
    for t, v in ((got, qkv[:, :, 2]), (other, torch.full_like(q, 7.0))):
        assert torch.equal(t[:, :, 0], qo) and torch.equal(t[:, :, 1], ko) and torch.equal(t[:, :, 2], v)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("dim,rot,inter", [(128, 128, False), (256, 64, False), (64, 64, True), (80, 20, False), (96, 96, True), (112, 28, True),
                                          (65, 64, False), (128, 0, False), (1024, 1024, False), (7, 6, True), (576, 64, False), (1, 0, False)])
def test_qk_norm_rope(q4k, gpu, dim, rot, inter, dtype):
    for rows, hq, hk, scale in [(1, 1, 1, 1.0), (5, 7, 2, 1.3), (70, 32, 8, 1.0)]:
        rng = np.random.default_rng(dim * 7 + rot + rows)
        q, k = _x(rng, rows, hq, dim, dtype=dtype) * 3, _x(rng, rows, hk, dim, dtype=dtype)
        q[0, 0] = 0  # a zero head stays zero
        wq, wk = (torch.from_numpy(rng.standard_normal(dim).astype(np.float32)) for _ in range(2))
        f, p = _freq(rot), torch.from_numpy(rng.integers(0, 100000, rows).astype(np.int32))
        qo, ko = torch.full_like(q, float("nan")).to(gpu), torch.full_like(k, float("nan")).to(gpu)
        q4k.qk_norm_rope(q.to(gpu), k.to(gpu), wq.to(gpu), wk.to(gpu), f.to(gpu), p.to(gpu), qo, ko, interleaved=inter, scale=scale, eps=1e-5)
        torch.cuda.synchronize()
        for x, w, o, name in ((q, wq, qo, "q"), (k, wk, ko, "k")):
            n = ref.head_norm(_host(x), w.numpy(), np.float32(1e-5))
            want, size = ref.rotate(n, f.numpy(), p.numpy(), inter, np.float32(scale))
            ref.assert_close(_host(o), want, ref.norm_bound(size, want, scale), dtype == F16, f"{name} {rows}x{dim} rot {rot}")
        assert bool((qo[0, 0] == 0).all())


def test_qk_norm_keeps_bad_values_to_their_head(q4k, gpu):
    """NaN and infinity make their own head NaN (the formula's inf / inf) and
    no other."""
    rows, hq, hk, dim = 4, 5, 2, 128
    rng = np.random.default_rng(11)
    q, k = _x(rng, rows, hq, dim, dtype=F32).to(gpu), _x(rng, rows, hk, dim, dtype=F32).to(gpu)
    w, f, p = torch.ones(dim, device=gpu), _freq(dim).to(gpu), torch.arange(rows, dtype=torch.int32, device=gpu)
    clean = [torch.empty_like(q), torch.empty_like(k)]
    q4k.qk_norm_rope(q, k, w, w, f, p, *clean)
    q[1, 2, 5], q[3, 0, 127], k[2, 1, 0] = float("nan"), float("inf"), float("-inf")
    got = [torch.empty_like(q), torch.empty_like(k)]
    q4k.qk_norm_rope(q, k, w, w, f, p, *got)
    torch.cuda.synchronize()
    bad = [torch.zeros(rows, hq, dtype=torch.bool), torch.zeros(rows, hk, dtype=torch.bool)]
    bad[0][1, 2] = bad[0][3, 0] = bad[1][2, 1] = True
    for g, c, b in zip(got, clean, bad):
        g, c = g.cpu(), c.cpu()
        assert torch.equal(g[~b], c[~b])
        assert torch.isnan(g[b]).any(dim=-1).all()


def test_heads_follow_positions_in_a_graph(q4k, gpu):
    """A captured call reads positions and inputs anew at every replay, and
    allocates nothing."""
    rows, hq, hk, dim = 8, 32, 8, 128
    rng = np.random.default_rng(12)
    q, k = _x(rng, rows, hq, dim, dtype=F16).to(gpu), _x(rng, rows, hk, dim, dtype=F16).to(gpu)
    w, f, p = torch.ones(dim, device=gpu), _freq(dim).to(gpu), torch.zeros(rows, dtype=torch.int32, device=gpu)
    qo, ko, qr, kr = (torch.empty_like(t) for t in (q, k, q, k))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        q4k.qk_norm_rope(q, k, w, w, f, p, qo, ko)
    for step in range(4):
        p.copy_(torch.from_numpy(rng.integers(0, 50000, rows).astype(np.int32)))
        q.mul_(1.25)
        g.replay()
        q4k.qk_norm_rope(q, k, w, w, f, p, qr, kr)
        torch.cuda.synchronize()
        assert torch.equal(qo, qr) and torch.equal(ko, kr)


def test_heads_python_refusals(q4k, gpu):
    x = torch.zeros((2, 4, 128), device=gpu)
    f, p = _freq(128).to(gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    for bad in [lambda: q4k.rope(x, f.float(), p, x), lambda: q4k.rope(x, f, p.long(), x), lambda: q4k.rope(x, f, p[:1], x),
                lambda: q4k.rope(x, f, p, x.half()), lambda: q4k.rope(x, f, p, x[:1]), lambda: q4k.rope(x[0], f, p, x[0]),
                lambda: q4k.rope(x.transpose(1, 2), f, p, x.transpose(1, 2)), lambda: q4k.rope(x, f.cpu(), p, x),
                lambda: q4k.qk_norm_rope(x, x[:1], f, f, f, p, x, x[:1]), lambda: q4k.qk_norm_rope(x, x, p, p, f, p, x, x)]:
        with pytest.raises((TypeError, ValueError)):
            bad()
    with pytest.raises(q4k.Q4KError):
        q4k.rope(x[:, :, :64], f, p, x[:, :, :64])  # rot_dim 128 of 64
    with pytest.raises(q4k.Q4KError):
        q4k.rope(x, f, p, x[:1].expand(2, 4, 128))  # both rows into one
    assert q4k.rope(x[:0], f, p, x[:0]).shape[0] == 0
