"""attention, cache_write, cache_assign and cache_compact without a GPU: every
refusal comes before any HIP call."""
import struct

import pytest
import torch

from mtlqwen_amd import operators as ops

EINVAL, ESHAPE, EALIAS = -1, -3, -4
# Addresses that are only compared, never read: the calls below are refused.
Q, O, K, V, T, S, P = 0x10000000, 0x20000000, 0x30000000, 0x40000000, 0x50000000, 0x50100000, 0x50200000


def heads(i=Q, o=O, strides=(512, 64, 512, 64), n=8):
    return ops._HEADS(i, o, 0, *strides, n)


def cache(k=K, v=V, strides=(4096, 2048, 64), t=T, s=0, pages=10, size=32, n=2, dim=64, rows=8, width=4):
    return ops._CACHE(k, v, *strides, t, s, pages, size, n, dim, rows, width)


def params(scale=0.1, cap=0.0, slopes=0, window=0):
    return ops._ATTENTION(scale, cap, slopes, window)


def counts(*v):
    return ops._COUNTS[len(v)](*v)


SEQUENCES = [
    ({"rows": 1 << 25}, ESHAPE),
    ({"counts": counts(1, 2), "nq": 2, "rows": 4}, EINVAL),
    ({"counts": None, "nq": 2}, EINVAL),
    ({"counts": counts(1), "nq": 0}, EINVAL),
    ({"counts": b"\0" * 4 * 65, "nq": 65}, EINVAL),
    ({"dtype": 2}, EINVAL),
    ({"p": 0}, EINVAL),
]
CACHES = [
    (cache(size=8), ESHAPE), (cache(size=48), ESHAPE), (cache(size=2048), ESHAPE),
    (cache(dim=0), ESHAPE), (cache(dim=60), ESHAPE), (cache(dim=264), ESHAPE),
    (cache(n=0), ESHAPE), (cache(n=65536), ESHAPE),
    (cache(strides=(4096, 2048, 60)), ESHAPE), (cache(strides=(-4096, 2048, 64)), ESHAPE), (cache(strides=(1 << 41, 2048, 64)), ESHAPE),
    (cache(pages=1 << 31), ESHAPE), (cache(rows=1 << 31), ESHAPE), (cache(width=(1 << 25) + 1), ESHAPE),
    (cache(k=0), EINVAL), (cache(v=0), EINVAL), (cache(k=K + 8), EINVAL), (cache(v=V + 2), EINVAL), (cache(t=0), EINVAL),
    (cache(rows=0), ESHAPE),
]


def run_attention(q4k, h=heads(), c=cache(), pr=params(), p=P, counts=None, nq=0, rows=8, dtype=0):
    return q4k.lib.q4k_attention(None, 0, h, c, pr, p, counts, nq, rows, dtype)


def run_write(q4k, k=heads(o=0, n=2), c=cache(), v=heads(i=O, o=0, n=2), p=P, counts=None, nq=0, rows=8, dtype=0):
    return q4k.lib.q4k_cache_write(None, 0, c, k, v, p, counts, nq, rows, dtype)


@pytest.mark.parametrize("kw,code", SEQUENCES)
def test_sequences(q4k, kw, code):
    assert run_attention(q4k, **kw) == code and q4k.lib.q4k_last_error()
    assert run_write(q4k, **kw) == code


@pytest.mark.parametrize("c,code", CACHES)
def test_caches(q4k, c, code):
    assert run_attention(q4k, c=c) == code and q4k.lib.q4k_last_error()
    assert run_write(q4k, c=c) == code


@pytest.mark.parametrize("kw,code", [
    ({"h": heads(n=7)}, ESHAPE), ({"h": heads(n=0)}, ESHAPE), ({"h": heads(i=0)}, EINVAL), ({"h": heads(o=0)}, EINVAL),
    ({"h": heads(strides=(512, 64, 511, 64))}, ESHAPE), ({"h": heads(strides=(512, 64, -512, 64))}, ESHAPE),
    ({"h": heads(o=Q)}, EALIAS), ({"h": heads(o=Q + 256)}, EALIAS),
    ({"h": heads(o=K)}, EALIAS), ({"h": heads(o=V - 4)}, EALIAS), ({"h": heads(o=T + 4 * 8 * 4 - 4)}, EALIAS), ({"h": heads(o=P)}, EALIAS),
    ({"h": heads(o=S), "c": cache(s=S)}, EALIAS), ({"h": heads(o=S), "pr": params(slopes=S + 28)}, EALIAS),
    ({"pr": params(scale=float("inf"))}, EINVAL), ({"pr": params(scale=float("nan"))}, EINVAL), ({"pr": params(cap=-1.0)}, EINVAL),
    ({"pr": params(cap=float("nan"))}, EINVAL), ({"pr": params(window=1 << 31)}, EINVAL),
    ({"pr": params(cap=2.0 ** -65)}, EINVAL), ({"pr": params(cap=2.0 ** 65)}, EINVAL), ({"rows": (1 << 24) - 1, "h": heads(n=66)}, ESHAPE),
    ({"c": cache(rows=2), "counts": counts(1, 2, 5), "nq": 3}, ESHAPE),
])
def test_attention_refusals(q4k, kw, code):
    assert run_attention(q4k, **kw) == code and q4k.lib.q4k_last_error()


@pytest.mark.parametrize("kw,code", [
    ({"c": cache(v=K)}, ESHAPE), ({"c": cache(v=K + 64)}, ESHAPE), ({"c": cache(strides=(4096, 1024, 64))}, ESHAPE), ({"c": cache(strides=(0, 2048, 64))}, ESHAPE),
    ({"c": cache(strides=(4096, 2048, 32))}, ESHAPE), ({"c": cache(v=K + 2 * 4096)}, ESHAPE), ({"c": cache(strides=(4096, 32, 128), v=K + 128)}, ESHAPE),
    ({"k": heads(i=0, n=2)}, EINVAL), ({"v": heads(i=0, n=2)}, EINVAL), ({"k": heads(strides=(-1, 64, 0, 0))}, ESHAPE),
    ({"k": heads(i=K + 4096)}, EALIAS), ({"v": heads(i=V)}, EALIAS), ({"c": cache(t=K)}, EALIAS), ({"p": V + 100}, EALIAS), ({"c": cache(s=K)}, EALIAS),
    ({"rows": 1 << 24, "c": cache(n=16, dim=64, strides=(64 * 16 * 32, 64 * 32, 64))}, ESHAPE),
])
def test_write_refusals(q4k, kw, code):
    assert run_write(q4k, **kw) == code and q4k.lib.q4k_last_error()


def pool(d=K, pages=16, blocks=2, size=16, token=64):
    return ops._POOL(d, pages, blocks, size, token)


def run_tables(q4k, what, p=pool(), t=T, n=S, slots=4, width=8, parents=P, counts=0, new=Q, lengths=Q + 4096, out=Q + 8192):
    if what == "assign":
        return q4k.lib.q4k_cache_assign(None, 0, p, t, n, slots, width, parents, counts, new, lengths, out)
    return q4k.lib.q4k_cache_compact(None, 0, p, t, n, slots, width, new, out)


@pytest.mark.parametrize("what", ["assign", "compact"])
@pytest.mark.parametrize("kw,code", [
    ({"p": pool(pages=0)}, ESHAPE), ({"p": pool(pages=262145)}, ESHAPE), ({"p": pool(size=0)}, ESHAPE), ({"p": pool(size=24)}, ESHAPE),
    ({"p": pool(size=1 << 21)}, ESHAPE), ({"p": pool(blocks=0)}, ESHAPE), ({"p": pool(token=0)}, ESHAPE), ({"p": pool(token=40)}, ESHAPE),
    ({"p": pool(size=1 << 16, token=1 << 15)}, ESHAPE), ({"p": pool(blocks=1 << 20, size=1 << 10, token=1 << 10)}, ESHAPE),
    ({"p": pool(d=0)}, EINVAL), ({"p": pool(d=K + 8)}, EINVAL), ({"t": 0}, EINVAL), ({"n": 0}, EINVAL), ({"new": 0}, EINVAL),
    ({"slots": 1025}, ESHAPE), ({"width": (1 << 26) + 1}, ESHAPE),
    ({"new": T}, EALIAS), ({"new": T + 124}, EALIAS), ({"new": S - 4}, EALIAS), ({"new": K + 64}, EALIAS), ({"out": T + 8}, EALIAS), ({"out": Q}, EALIAS),
    ({"t": K + 32}, EALIAS), ({"n": K + 16 * 2 * 16 * 64 - 4}, EALIAS),
])
def test_table_refusals(q4k, what, kw, code):
    assert run_tables(q4k, what, **kw) == code and q4k.lib.q4k_last_error()


@pytest.mark.parametrize("kw,code", [
    ({"lengths": 0}, EINVAL), ({"lengths": S}, EALIAS), ({"lengths": Q + 100}, EALIAS), ({"parents": Q}, EALIAS), ({"counts": K}, EALIAS), ({"lengths": P + 12}, EALIAS),
])
def test_assign_refusals(q4k, kw, code):
    assert run_tables(q4k, "assign", **kw) == code and q4k.lib.q4k_last_error()


def test_null_arguments(q4k):
    lib = q4k.lib
    assert lib.q4k_attention(None, 0, None, cache(), params(), P, None, 0, 8, 0) == EINVAL
    assert lib.q4k_attention(None, 0, heads(), None, params(), P, None, 0, 8, 0) == EINVAL
    assert lib.q4k_attention(None, 0, heads(), cache(), None, P, None, 0, 8, 0) == EINVAL
    assert lib.q4k_cache_write(None, 0, None, heads(), heads(), P, None, 0, 8, 0) == EINVAL
    assert lib.q4k_cache_assign(None, 0, None, T, S, 4, 8, P, 0, Q, Q + 4096, 0) == EINVAL
    assert lib.q4k_cache_compact(None, 0, None, T, S, 4, 8, Q, 0) == EINVAL


def test_nothing_is_refused_with_nothing_to_do(q4k):
    """No rows, no slots, no pages to write to: done before any HIP call."""
    assert run_attention(q4k, rows=0) == 0
    assert run_write(q4k, rows=0) == 0 and run_write(q4k, c=cache(pages=0)) == 0 and run_write(q4k, c=cache(width=0)) == 0
    assert run_tables(q4k, "assign", slots=0, out=0) == 0 and run_tables(q4k, "compact", slots=0, out=0) == 0


def test_python_checks(q4k):
    """The Python faces refuse what is no GPU tensor, or does not fit, before the library sees it."""
    x, c, i = torch.zeros(2, 4, 64), torch.zeros(3, 2, 16, 64, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.attention(x, c, c, i, i[0], x)
    with pytest.raises(TypeError):
        ops.attention(x.double(), c, c, i, i[0], x)
    with pytest.raises(ValueError):
        ops.cache_write(x, x, c, c, i, i[0])
    with pytest.raises(ValueError):
        ops.cache_assign(c, i, i[0], i[0], i, i[0])
    with pytest.raises(ValueError):
        ops.cache_compact(c, i, i[0], i)
    with pytest.raises(ValueError):
        ops._sequences([3, 2], 4)
    assert ops._sequences([3], 4) == (counts(3), 1, 3) and ops._sequences(None, 4)[2] == 4
    with pytest.raises(ValueError):
        ops._cache_shape(c, c[:, :1])
    with pytest.raises(ValueError):
        ops._cache_shape(c[0], c[0])
    of = ops._cache_shape(c, c)
    with pytest.raises(TypeError):
        ops._cache(c.float(), c.float(), of, i, None, i[0], 1, -1)
    with pytest.raises(ValueError):
        t = c.transpose(2, 3).contiguous().transpose(2, 3)
        ops._cache(c, t, of, i, None, i[0], 1, -1)
    with pytest.raises(TypeError):
        ops._cache(c, c, of, i.long(), None, i[0], 1, -1)
    with pytest.raises(ValueError):
        ops._cache(c, c, of, i, None, i[0, :0], 1, -1)
    with pytest.raises(ValueError):
        ops._cache(c, c, of, i[0], None, i[0], 1, -1)
    with pytest.raises(ValueError):
        ops._rows_of(x.transpose(1, 2), 64, "k")
    with pytest.raises(struct.error):
        ops._sequences([3, -1], 4)
