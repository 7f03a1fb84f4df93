"""Attention over scores and values that are not finite and that a row does see:
what the formula gives, in tiles that all rows of a unit see and in others, in one
stretch of the keys or several."""
import numpy as np
import pytest
import torch

import cache_ref as ref
from test_gpu_attention import _cache, _close, _i32, _tables

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def _case(gpu, counts, contexts, heads, kv, dim, page, dtype):
    rng = np.random.default_rng(sum(contexts) + dim)
    tables, pages = _tables(rng, contexts, page)
    cache = _cache(rng, gpu, pages, kv, page, dim)
    q = torch.from_numpy(rng.standard_normal((sum(counts), heads, dim)).astype(np.float32)).to(dtype)
    return tables, cache, q, [c - n for c, n in zip(contexts, counts)]


def _attend(q4k, gpu, q, cache, tables, first, counts, window=0):
    out = torch.full(q.shape, 9.0, device=gpu, dtype=q.dtype)
    q4k.attention(q.to(gpu), cache[:, 0], cache[:, 1], _i32(gpu, tables), _i32(gpu, first), out, query_counts=counts, window=window)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [64, 80, 128, 200, 256])
@pytest.mark.parametrize("counts,contexts,window", [([1], [40], 0), ([1, 2], [1, 3000], 0), ([5], [90], 7), ([70], [200], 0), ([3, 90], [50, 4000], 333)])
def test_scores_of_minus_infinity_alone(q4k, gpu, counts, contexts, window, dim, dtype):
    """An infinite element of a query whose products are all -inf: 0 / 0, not a row that sees nothing."""
    tables, cache, q, first = _case(gpu, counts, contexts, 4, 2, dim, 16, dtype)
    cache[:, 0, :, :, 5] = -cache[:, 0, :, :, 5].abs() - 0.5
    r, h = sum(counts) - 1, 2
    q[r, h, 5] = float("inf")
    out = _attend(q4k, gpu, q, cache, tables, first, counts, window)
    c = cache.cpu().numpy()
    want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts, window=window, f16=dtype == F16)
    assert np.isnan(want[r, h]).all()
    _close(out, want, bound, "one row of -inf")


@pytest.mark.parametrize("dim", [64, 80, 128, 200, 256])
@pytest.mark.parametrize("counts,contexts", [([1, 2], [40, 6000]), ([4, 5], [30, 8000]), ([70], [200]), ([100, 90], [6000, 500])])
def test_scores_of_minus_infinity_among_others(q4k, gpu, counts, contexts, dim):
    """Keys with an infinite element leave nothing in rows that see others, in whichever part of the keys they are,
    and make those that see no other NaN.  fp16 rows: fp32 ones, of two parts, become NaN.  For the bounds those keys have a score of
    -4000 / sqrt(dim), whose weight is below 2^-300."""
    page, window = 16, 0
    for window in (0, 3):
        tables, cache, q, first = _case(gpu, counts, contexts, 4, 2, dim, page, F16)
        q[:, :, 5] = 4.0
        cache[:, 0, :, :, 5] = 0.0
        plain = cache.clone()
        # The first half of the last sequence's tokens before its rows, and its rows' own but the last three.
        n, t = contexts[-1], tables[-1]
        bad = [at for at in range(n - 3) if at >= first[-1] or at < first[-1] // 2]
        for at in bad:
            cache[t[at // page], 0, :, at % page, 5] = float("-inf")
            plain[t[at // page], 0, :, at % page, 5] = -1000.0
        out = _attend(q4k, gpu, q, cache, tables, first, counts, window)
        c = plain.cpu().numpy()
        want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts, window=window, f16=True)
        for i in range(counts[-1]):
            p, r = first[-1] + i, sum(counts[:-1]) + i
            if all(at in set(bad) for at in range(max(0, p + 1 - window) if window else 0, p + 1)):
                want[r] = np.nan
        _close(out, want, bound, f"window {window}")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [8, 64, 72, 80, 96, 112, 128, 160, 192, 200, 256])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("counts,contexts,window", [([1, 3], [77, 500], 60), ([5], [900], 65), ([70], [130], 0), ([150], [900], 500)])
def test_values_that_no_row_sees(q4k, gpu, counts, contexts, window, bad, dim, dtype):
    """Keys and values before every row's window and behind the last token, then
    values of one token that some rows see, at every place of a tile."""
    tables, cache, q, first = _case(gpu, counts, contexts, 2, 1, dim, 32, dtype)
    for t, n, p in zip(tables, contexts, first):
        for at in list(range(0, max(0, p + 1 - window) if window else 0)) + list(range(n, -(-n // 32) * 32)):
            cache[t[at // 32], :, :, at % 32] = bad
    out = _attend(q4k, gpu, q, cache, tables, first, counts, window)
    c = cache.cpu().numpy()
    want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts, window=window, f16=dtype == F16)
    assert np.isfinite(want).all()
    _close(out, want, bound, f"{bad} that no row sees")
    # A token that the first row of the last sequence does not see yet, or does not see any more.
    at = contexts[-1] - 1 if counts[-1] > 1 and not window else max(0, first[-1] + 1 - window)
    cache[tables[-1][at // 32], 1, :, at % 32] = bad
    out = _attend(q4k, gpu, q, cache, tables, first, counts, window)
    c = cache.cpu().numpy()
    with np.errstate(invalid="ignore"):
        want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts, window=window, f16=dtype == F16)
    fine = np.isfinite(want)
    got = out.cpu().double().numpy()
    assert np.isfinite(got[fine]).all() and not np.isfinite(got[~fine]).any() and fine.any() and not fine.all()
    _close(torch.from_numpy(np.where(fine, got, 0.0)), np.where(fine, want, 0.0), np.where(fine, bound, 1.0), f"{bad} that some rows see")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [64, 80, 128, 200, 256])
@pytest.mark.parametrize("size", [1.0, 20.0])
@pytest.mark.parametrize("counts,contexts,window", [([1, 1], [150, 5000], 0), ([5], [700], 0), ([70], [500], 0), ([90, 3], [4000, 3000], 0),
                                                    ([150], [900], 500), ([2, 4], [900, 4000], 1500)])
def test_values_of_infinity(q4k, gpu, counts, contexts, window, size, dim, dtype):
    """Values of infinity, -infinity, both and NaN that rows see, among keys of weights of any size (those of 2^-200 too, whose
    share no fp32 holds), in tiles that all rows see: weights are positive, so the sum is what it is in the reals."""
    tables, cache, q, first = _case(gpu, counts, contexts, 4, 2, dim, 32, dtype)
    q *= size
    for t, n in zip(tables, contexts):
        for at in range(n):
            if at % 41 == 7:
                cache[t[at // 32], 1, :, at % 32, 3] = float("inf")
            if at % 611 == 40:
                cache[t[at // 32], 1, :, at % 32, 8] = float("-inf")
            if at % 300 == 50:
                cache[t[at // 32], 1, :, at % 32, 15] = float("-inf") if at % 600 == 50 else float("inf")
            if at == 111:
                cache[t[at // 32], 1, :, at % 32, dim - 1] = float("nan")
    out = _attend(q4k, gpu, q, cache, tables, first, counts, window)
    c = cache.cpu().numpy()
    with np.errstate(invalid="ignore"):
        want, bound = ref.attention(q.float().numpy(), c[:, 0], c[:, 1], tables, first, counts, window=window, f16=dtype == F16)
    got = out.cpu().double().numpy()
    assert np.isinf(want).any() and np.isnan(want).any()
    for what in (np.isposinf, np.isneginf, np.isnan):
        off = np.argwhere(what(got) != what(want))
        assert not len(off), f"{what.__name__}: {len(off)} places, row, head and element {off[0]}"
    fine = np.isfinite(want)
    _close(torch.from_numpy(np.where(fine, got, 0.0)), np.where(fine, want, 0.0), np.where(fine, bound, 1.0), "finite ones")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 24, 2.0 ** 26, 1.3 * 2.0 ** 27, 1.7 * 2.0 ** 27, 2.0 ** 29, 2.0 ** 33])
@pytest.mark.parametrize("counts,contexts", [([1, 2], [70, 3000]), ([5], [900]), ([70], [300]), ([90, 40], [3000, 500])])
@pytest.mark.parametrize("dim,softcap,slopes", [(64, 0.0, False), (128, 0.0, True), (256, 0.0, False), (80, 2.0 ** 40, False)])
def test_scores_of_any_size(q4k, gpu, counts, contexts, size, dim, softcap, slopes, dtype):
    """One key whose score is above all others', by a hundredth of `size` and more, where scores of that size have steps of
    2^-23 of it: its values, but for the roundings of one weight and the output (2^-11 each in fp16).  Once with all scores above zero, once
    below, once with that key's at zero and the others' far below."""
    rng = np.random.default_rng(dim)
    for sign in (1.0, -1.0, 0.0):
        tables, cache, q, first = _case(gpu, counts, contexts, 4, 2, dim, 32, dtype)
        cache[:, 0] = 0.0
        # Scores are size * k[0] (fp16 k): q[0] k[0] / sqrt(dim).
        a = float(np.sqrt(size * np.sqrt(dim)))
        small = min(a, 30000.0)
        q.zero_()
        q[:, :, 0] = a * a / small if dtype is F32 else min(a * a / small, 60000.0)
        q[:, :, 1] = 0.5
        best = [min(f, n - 3) for f, n in zip(first, contexts)]
        for t, n, b in zip(tables, contexts, best):
            for at in range(n):
                x = 1.0 if at == b else float(rng.uniform(0.25, 0.99))
                x = small * (x if sign > 0 else x - 1.25 if sign < 0 else 0.0 if at == b else -x)
                cache[t[at // 32], 0, :, at % 32, 0] = x
        sl = torch.full((4,), 0.25, device=gpu) if slopes else None
        out = torch.full(q.shape, 9.0, device=gpu, dtype=dtype)
        q4k.attention(q.to(gpu), cache[:, 0], cache[:, 1], _i32(gpu, tables), _i32(gpu, first), out, query_counts=counts, softcap=softcap, slopes=sl)
        torch.cuda.synchronize()
        v, got, r = cache[:, 1].double().cpu().numpy(), out.double().cpu().numpy(), 0
        for s, (t, n, b) in enumerate(zip(tables, counts, best)):
            want = v[t[b // 32], :, b % 32]  # [kv, dim]
            want = np.repeat(want, 2, axis=0)[None]
            off = np.abs(got[r:r + n] - want)
            bad = ~(off <= 2.0 ** -10 * np.abs(want) + 2.0 ** -24)
            assert not bad.any(), f"{sign} sequence {s}: {bad.sum()} of {bad.size}, {np.isnan(off).sum()} NaN"
            r += n


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("dim", [64, 80, 160, 256])
@pytest.mark.parametrize("n,window", [(1, 0), (3, 3000), (40, 0), (60, 2500)])
def test_rare_sums_of_long_contexts(q4k, gpu, n, window, dim, dtype):
    """Infinite values, then scores too large for the tiles' way with weights, in eight sequences whose waves have several tiles each,
    some of whose pages are not there: two heads of two sequences against 64 bits, every output for NaN."""
    rng = np.random.default_rng(dim + n)
    kv, heads, page = 4, 8, 16
    contexts = [4000 + 311 * i for i in range(8)]
    counts, first = [n] * 8, [c - n for c in contexts]
    tables, pages = _tables(rng, contexts, page)
    for t, c in zip(tables, contexts):
        for e in range(5, c // page - 20, 17):
            t[e] = -1
    cache = _cache(rng, gpu, pages, kv, page, dim)
    q = torch.from_numpy(rng.standard_normal((8 * n, heads, dim)).astype(np.float32)).to(dtype)
    probes = ((1, 0), (6, 7))

    def compare(out, far):
        for s, h in probes:
            mine = [p for p in tables[s] if p >= 0]
            c = cache[torch.tensor(mine, device=gpu), :, h // 2].cpu().numpy()[:, :, None]
            table = [mine.index(p) if p >= 0 else -1 for p in tables[s]]
            rows = slice(s * n, (s + 1) * n)
            with np.errstate(invalid="ignore"):
                want, bound = ref.attention(q[rows, h:h + 1].float().numpy(), c[:, 0], c[:, 1], [table], [first[s]], [n], window=window, f16=dtype == F16)
            got = out[rows, h:h + 1].cpu().double().numpy()
            if far:  # one key alone has a weight, one of 22 or 11 bits
                bound = 2.0 ** -10 * np.abs(want) + 2.0 ** -24
            for what in (np.isposinf, np.isneginf, np.isnan):
                assert np.array_equal(what(got), what(want)), (what.__name__, s, h)
            fine = np.isfinite(want)
            _close(torch.from_numpy(np.where(fine, got, 0.0)), np.where(fine, want, 0.0), np.where(fine, bound, 1.0), f"sequence {s} head {h}")

    for t, c in zip(tables, contexts):
        for at in range(c % 50, c, 97):
            if t[at // page] >= 0:
                cache[t[at // page], 1, :, at % page, 3] = float("inf")
                cache[t[at // page], 1, :, at % page, dim - 1] = float("inf") if at % 2 else float("-inf")
    compare(_attend(q4k, gpu, q, cache, tables, first, counts, window), False)
    # One key's score 2^30 / sqrt(dim), which passes 2^26 / log2(e), all others' at most 0.9 of it.
    cache = _cache(rng, gpu, pages, kv, page, dim)
    cache[:, 0] = 0.0
    cache[:, 0, :, :, 0] = torch.from_numpy(rng.uniform(-0.9, 0.9, (pages, 1, page))).to(gpu).to(F16) * 2.0 ** 15
    q.zero_()
    q[:, :, 0] = 2.0 ** 15
    for t, f in zip(tables, first):
        at = f - n if t[(f - n) // page] >= 0 else f - n - page
        assert t[at // page] >= 0
        cache[t[at // page], 0, :, at % page, 0] = 2.0 ** 15
    compare(_attend(q4k, gpu, q, cache, tables, first, counts, window), True)
