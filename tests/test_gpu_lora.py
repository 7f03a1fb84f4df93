"""Low-rank adapters on the GPU against 64-bit numpy (operators_ref), within
bounds that count the roundings: ragged batches of one row to prompts, ranks of
one to the largest, several per stack, sequences without an adapter, both types,
with and without an auxiliary, in place, values past an adapter's rank that
must not be read, and q4k_linear_lora against the projection of the summed
weights."""
import numpy as np
import pytest
import torch

import operators_ref as ref
from q4k_ref import TYPE_Q4_K, TYPE_Q6_K, make_q4k, make_weight, make_x, row_rel_err

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def _stacks(rng, slots, r, k, n):
    a = (rng.standard_normal((slots, r, k)) / np.sqrt(k)).astype(np.float16)
    b = (rng.standard_normal((slots, n, r)) / np.sqrt(r)).astype(np.float16)
    return a, b


def _check(q4k, gpu, counts, ids, k, n, r, dtype, slots=3, ranks=None, scales=True, aux=True, seed=0):
    m = sum(counts)
    rng = np.random.default_rng(seed + m + 7 * r + k // 256 + n)
    a, b = _stacks(rng, slots, r, k, n)
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(dtype)
    h = torch.from_numpy(rng.standard_normal((m, n)).astype(np.float32)).to(dtype) if aux else None
    sc = rng.uniform(-2, 2, slots).astype(np.float32) if scales else None
    if ranks is not None:  # what lies past an adapter's rank is never used
        for i, v in enumerate(ranks):
            a[i, max(0, v):], b[i, :, max(0, v):] = np.nan, np.inf
    t = lambda v: None if v is None else torch.from_numpy(np.ascontiguousarray(v)).to(gpu)  # noqa: E731
    kw = {"query_counts": counts, "ranks": t(None if ranks is None else np.array(ranks, np.int32)), "scales": t(sc)}
    args = (x.to(gpu), t(a), t(b), t(np.array(ids, np.int32)), m)
    y = torch.full((m + 1, n), 7.0, device=gpu, dtype=dtype)
    q4k.lora(*args, y, auxiliary=None if h is None else h.to(gpu), **kw)
    torch.cuda.synchronize()
    want, bound = ref.lora(x.float().numpy(), a, b, ids, counts, ranks, sc, None if h is None else h.float().numpy())
    got = y[:m].cpu().float().numpy()
    what = f"{counts} k={k} n={n} r={r} {dtype}"
    ref.assert_close(got, want, bound, dtype == F16, what)
    # On the whole the roundings do not line up: a chain of k / 8 of them drifts
    # by its root, 23 * 2^-24 = 1.4e-6 of a sum; and half a step of fp16.
    off = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert off <= 5e-6 + (2.0 ** -11 if dtype == F16 else 0.0), what
    assert bool((y[m] == 7.0).all()), what
    if h is not None:
        start = 0
        for q, rows in enumerate(counts):  # no adapter: a copy
            if not 0 <= ids[q] < slots:
                assert torch.equal(y[start:start + rows].cpu(), h[start:start + rows]), what
            start += rows
        inplace = h.to(gpu)
        q4k.lora(*args, inplace, auxiliary=inplace, **kw)
        torch.cuda.synchronize()
        assert torch.equal(inplace, y[:m]), what


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("counts,ids", [
    ([1], [0]), ([1] * 8, [2, 0, 1, 1, -1, 3, 0, 2]), ([5, 1, 4], [1, -7, 2**31 - 1]), ([0, 3, 0, 17, 0], [0, 1, 2, 2, 1]), ([16, 16], [0, 1]),
    ([33, 1, 100, 5], [2, 2, 0, 1]), ([15], [-1]), ([512, 37, 1, 1, 200, 5, 1, 64], [0, 1, 2, 0, 1, -1, 2, 0]),
])
def test_lora_batches(q4k, gpu, counts, ids, dtype):
    _check(q4k, gpu, counts, ids, 512, 144, 16, dtype)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("r", [1, 2, 3, 5, 8, 15, 16, 17, 24, 31, 32, 33, 48, 64, 65, 100, 128, 240, 256, 300, 512])
def test_lora_ranks(q4k, gpu, r, dtype):
    _check(q4k, gpu, [3, 70, 2], [1, 0, 2], 768, 80, r, dtype, aux=r % 2 == 0, scales=r % 3 == 0)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("r", [128, 224, 225, 256, 257])
def test_lora_large_ranks_of_many_rows(q4k, gpu, r, dtype):
    """Enough rows and columns for the largest row tiles, at the ranks where
    their shared memory decides."""
    _check(q4k, gpu, [700, 868], [1, 0], 256, 12288, r, dtype, slots=2)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("ranks", [[1, 4, 20], [0, 20, 7], [20, 19, 18], [-5, 21, 3], [16, 1, 2**31 - 1]])
def test_lora_mixed_ranks(q4k, gpu, ranks, dtype):
    """Ranks of 0 (and below) are no adapter, above the stack's all of it."""
    _check(q4k, gpu, [2, 40, 5, 1], [0, 1, 2, 0], 256, 48, 20, dtype, ranks=[min(v, 1 << 30) for v in ranks], aux=False)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("k,n,counts", [(4096, 12288, [1] * 8), (12288, 4096, [5] * 8), (4096, 6144, [9, 1, 130, 60]), (4096, 1024, [300, 212]),
                                        (256, 16, [1, 1]), (4096, 248320, [1, 2])])
def test_lora_projections(q4k, gpu, k, n, counts, dtype):
    _check(q4k, gpu, counts, [(2 * i) % 3 for i in range(len(counts))], k, n, 16, dtype)


def test_lora_shifted_storage(q4k, gpu):
    """Every tensor one element off alignment: the bits of aligned ones."""
    rng = np.random.default_rng(1)
    for dtype in (F32, F16):
        for r in (6, 16):
            m, k, n = 21, 512, 96
            a, b = (torch.from_numpy(v).to(gpu) for v in _stacks(rng, 2, r, k, n))
            x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(gpu).to(dtype)
            h = torch.from_numpy(rng.standard_normal((m, n)).astype(np.float32)).to(gpu).to(dtype)
            ids = torch.tensor([1, 0], dtype=torch.int32, device=gpu)
            shift = lambda t: torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
            y = torch.empty_like(h)
            ys = shift(torch.zeros_like(h))
            q4k.lora(x, a, b, ids, m, y, auxiliary=h, query_counts=[4, 17])
            q4k.lora(shift(x), shift(a), shift(b), shift(ids), m, ys, auxiliary=shift(h), query_counts=[4, 17])
            torch.cuda.synchronize()
            assert torch.equal(y, ys)


def test_lora_bad_values_stay_in_their_rows(q4k, gpu):
    rng = np.random.default_rng(2)
    m, k, n, r = 20, 512, 64, 12
    a, b = (torch.from_numpy(v).to(gpu) for v in _stacks(rng, 2, r, k, n))
    ids = torch.tensor([1, 0], dtype=torch.int32, device=gpu)
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(gpu)
    clean, got = torch.empty((m, n), device=gpu), torch.empty((m, n), device=gpu)
    q4k.lora(x, a, b, ids, m, clean, query_counts=[6, 14])
    x[3, 7], x[10, 500] = float("nan"), 1e38
    q4k.lora(x, a, b, ids, m, got, query_counts=[6, 14])
    torch.cuda.synchronize()
    assert torch.isnan(got[3]).all() and bool((got[10].abs() > 1e30).any())
    rest = [i for i in range(m) if i not in (3, 10)]
    assert torch.equal(got[rest], clean[rest])


def test_lora_follows_its_batch_in_a_graph(q4k, gpu):
    """Adapter ids, ranks and scales are read at every replay; replays with
    eager calls of other shapes between them give the eager call's bits."""
    rng = np.random.default_rng(3)
    m, k, n, r, slots = 8, 4096, 1024, 16, 4
    a, b = (torch.from_numpy(v).to(gpu) for v in _stacks(rng, slots, r, k, n))
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(gpu).half()
    ids = torch.zeros(m, dtype=torch.int32, device=gpu)
    ranks = torch.full((slots,), r, dtype=torch.int32, device=gpu)
    scales = torch.ones(slots, device=gpu)
    y, want = torch.empty((m, n), device=gpu, dtype=F16), torch.empty((m, n), device=gpu, dtype=F16)
    kw = {"query_counts": [1] * m, "ranks": ranks, "scales": scales}
    q4k.lora(x, a, b, ids, m, want, **kw)  # the workspace exists before the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        q4k.lora(x, a, b, ids, m, y, **kw)
    for step in range(4):
        ids.copy_(torch.from_numpy(rng.integers(-1, slots, m).astype(np.int32)))
        ranks.copy_(torch.from_numpy(rng.integers(0, r + 1, slots).astype(np.int32)))
        scales.mul_(1.5)
        g.replay()
        q4k.lora(x, a, b, ids, m, want, **kw)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        big = torch.empty((400, n), device=gpu, dtype=F16)
        q4k.lora(x.repeat(50, 1), a, b, ids[:1], 400, big)


@pytest.mark.parametrize("t,dtype,m,counts", [(TYPE_Q4_K, F32, 8, [1] * 8), (TYPE_Q4_K, F16, 40, [5] * 8), (TYPE_Q6_K, F32, 19, [19]),
                                              (TYPE_Q4_K, F32, 200, [150, 50]), (TYPE_Q6_K, F16, 100, [99, 1])])
@pytest.mark.parametrize("post", [0, 1, 2])
def test_linear_lora(q4k, oracle, gpu, t, dtype, m, counts, post):
    """Against the oracle's projection plus the adapters' part in 64 bits: the
    projection's bar of 1e-3 per row, plus two roundings to fp16 of at most
    half a step (2^-11) each where the type is fp16."""
    k, n, r = 1024, 512, 8
    rng = np.random.default_rng(40 + m + post)
    wb = make_weight(rng, n, k, t)
    W = q4k.Weight(wb, n, k, ggml_type=t)
    a, b = _stacks(rng, 3, r, k, n)
    ids = [(i + 1) % 3 if i % 3 != 1 else -1 for i in range(len(counts))]
    x = make_x(rng, m, k, 0.25)
    aux = make_x(rng, m, n, 0.5)
    xt, at = torch.from_numpy(x).to(gpu).to(dtype), torch.from_numpy(aux).to(gpu).to(dtype)
    xh, ah = xt.cpu().float().numpy(), at.cpu().float().numpy()
    plain = oracle.linear(xh, wb, n, k, ggml_type=t)
    sc = np.array([0.5, 2.0, -1.0], np.float32)
    delta, _ = ref.lora(xh, a, b, ids, counts, None, sc, None)
    acc = np.asarray(plain, np.float64) + delta
    want = acc if post == 0 else acc + ah if post == 1 else ah / (1 + np.exp(-ah.astype(np.float64))) * acc
    args = (xt, W, torch.from_numpy(a).to(gpu), torch.from_numpy(b).to(gpu), torch.tensor(ids, dtype=torch.int32, device=gpu), m)
    kw = {"query_counts": counts, "scales": torch.from_numpy(sc).to(gpu), "gated": post == 2}
    y = torch.empty((m, n), device=gpu, dtype=dtype)
    q4k.linear_lora(*args, y, auxiliary=at if post else None, **kw)
    torch.cuda.synchronize()
    err = row_rel_err(y.cpu().float().numpy(), want)
    assert err <= 1e-3 + (2 * 2.0 ** -11 if dtype == F16 else 0.0)
    if post:  # in place over the auxiliary
        z = at.clone()
        q4k.linear_lora(*args, z, auxiliary=z, **kw)
        torch.cuda.synchronize()
        assert torch.equal(z, y)
    # No sequence has an adapter: the projection itself.
    none = torch.full((len(counts),), -1, dtype=torch.int32, device=gpu)
    q4k.linear_lora(xt, W, args[2], args[3], none, m, y, auxiliary=at if post == 1 else None, query_counts=counts)
    base = torch.empty_like(y)
    q4k.linear(xt, W, m, base, auxiliary=at if post == 1 else None, query_counts=counts)
    torch.cuda.synchronize()
    assert torch.equal(y, base)


def test_lora_python_refusals(q4k, gpu):
    x, y = torch.zeros((4, 512), device=gpu), torch.zeros((4, 64), device=gpu)
    a, b = torch.zeros((2, 8, 512), device=gpu, dtype=F16), torch.zeros((2, 64, 8), device=gpu, dtype=F16)
    ids = torch.zeros(1, dtype=torch.int32, device=gpu)
    for bad in [lambda: q4k.lora(x, a.float(), b, ids, 4, y), lambda: q4k.lora(x, a, b[:1], ids, 4, y), lambda: q4k.lora(x, a, b, ids.long(), 4, y),
                lambda: q4k.lora(x, a, b, ids, 5, y), lambda: q4k.lora(x, a, b, ids, 4, y.half()), lambda: q4k.lora(x, a, b, ids, 4, y[:, ::2]),
                lambda: q4k.lora(x, a, b, ids, 4, y, query_counts=[2, 2]), lambda: q4k.lora(x, a, b, ids, 4, y, ranks=ids),
                lambda: q4k.lora(x, a, b, ids, 4, y, scales=ids), lambda: q4k.lora(x, a[0], b[0], ids, 4, y),
                lambda: q4k.lora(x, a, b, ids, 4, y, auxiliary=y[:3])]:
        with pytest.raises((TypeError, ValueError)):
            bad()
    with pytest.raises(q4k.Q4KError):
        q4k.lora(x, a, b, ids, 4, x[:, :64].contiguous(), query_counts=[3])


def test_pass_around_the_projections(q4k, oracle, gpu):
    """One attention input and one set of logits as an engine runs them: the
    joined projection with adapters, norms and rotation of its heads in place,
    the LM-head rows' norm, the head's projection, penalties and a mask; each
    step against 64 bits from the step before it, and the whole captured and
    replayed."""
    rng = np.random.default_rng(60)
    k, hq, hk, dim, vocab, r = 1024, 6, 2, 64, 4096, 8
    n = (hq + 2 * hk) * dim
    counts, samples = [5, 1, 3], [2, 1, 1]
    m, rows = sum(counts), sum(samples)
    wb, hb = make_q4k(rng, n, k), make_q4k(rng, vocab, k)
    W, H = q4k.Weight(wb, n, k), q4k.Weight(hb, vocab, k)
    a, b = _stacks(rng, 2, r, k, n)
    x = make_x(rng, m, k, 0.5)
    t = lambda v, d=None: torch.from_numpy(np.ascontiguousarray(v)).to(gpu)  # noqa: E731
    xt, at, bt = t(x), t(a), t(b)
    ids, pos = t(np.array([1, -1, 0], np.int32)), t(np.array([40, 41, 42, 43, 44, 900, 7, 8, 9], np.int32))
    wq, wk, wn = (t(rng.uniform(0.5, 1.5, s).astype(np.float32)) for s in (dim, dim, k))
    f, scale = q4k.rope_frequencies(dim, scaling="yarn", factor=4.0, original_context=2048)
    tokens = t(rng.integers(0, vocab, (3, 64)).astype(np.int32))
    slots, lengths, prompts = (t(np.array(v, np.int32)) for v in ([0, 0, 1, 2], [44, 45, 64, 10], [40, 40, 5, 10]))
    rep, freq, pres = (t(np.array(v, np.float32)) for v in ([1.1] * 4, [0.2] * 4, [0.1] * 4))
    mask, mrow = t(rng.integers(-2**31, 2**31, (1, vocab // 32)).astype(np.int32)), t(np.array([-1, 0, 0, -1], np.int32))
    qkv, normed = torch.empty((m, n), device=gpu), torch.empty((rows, k), device=gpu)
    logits = torch.empty((rows, vocab), device=gpu)
    raw_qkv, raw_logits = torch.empty_like(qkv), torch.empty_like(logits)

    def step():
        q4k.linear_lora(xt, W, at, bt, ids, m, qkv, query_counts=counts)
        raw_qkv.copy_(qkv)
        q = qkv[:, :hq * dim].view(m, hq, dim)
        kk = qkv[:, hq * dim:(hq + hk) * dim].view(m, hk, dim)
        q4k.qk_norm_rope(q, kk, wq, wk, f, pos, q, kk, scale=scale)
        q4k.rms_norm_gather(xt, wn, normed, counts, samples)
        q4k.linear(normed, H, rows, logits, query_counts=samples)
        raw_logits.copy_(logits)
        q4k.process_logits(logits, logits, tokens=tokens, slots=slots, lengths=lengths, prompts=prompts, repetition=rep, frequency=freq,
                           presence=pres, mask=mask, mask_rows=mrow)

    step()
    torch.cuda.synchronize()
    delta, _ = ref.lora(x, a, b, [1, -1, 0], counts, None, None, None)
    assert row_rel_err(raw_qkv.cpu().numpy(), oracle.linear(x, wb, n, k) + delta) <= 1e-3
    raw = raw_qkv.cpu().numpy()
    for lo, heads, w in ((0, hq, wq), (hq * dim, hk, wk)):
        part = raw[:, lo:lo + heads * dim].reshape(m, heads, dim)
        want, size = ref.rotate(ref.head_norm(part, w.cpu().numpy(), np.float32(1e-6)), f.cpu().numpy(), pos.cpu().numpy(), False, np.float32(scale))
        ref.assert_close(qkv[:, lo:lo + heads * dim].reshape(m, heads, dim).cpu().numpy(), want, ref.norm_bound(size, want, scale), False)
    assert torch.equal(qkv[:, (hq + hk) * dim:], raw_qkv[:, (hq + hk) * dim:])  # values untouched
    bits = ((mask.cpu().numpy().view(np.uint32)[0][np.arange(vocab) // 32] >> (np.arange(vocab) % 32).astype(np.uint32)) & 1).astype(bool)
    every = np.ones(vocab, bool)
    text = tokens.cpu().numpy()
    want, bound = ref.logits(raw_logits.cpu().numpy(), texts=[text[0, :44], text[0, :45], text[1, :64], text[2, :10]], prompts=[40, 40, 5, 10],
                             repetition=rep.cpu().numpy(), frequency=freq.cpu().numpy(), presence=pres.cpu().numpy(),
                             allowed=np.stack([every, bits, bits, every]))
    ref.assert_close(logits.cpu().numpy(), want, bound, False)
    eager = (qkv.clone(), logits.clone())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        step()
    for _ in range(3):
        qkv.zero_()
        logits.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(qkv, eager[0]) and torch.equal(logits, eager[1])


@pytest.mark.parametrize("slots", [1, 63, 64, 65, 200])
def test_lora_many_slots(q4k, gpu, slots):
    """Stacks on both sides of the 64 slots whose ranks one wave reads at once,
    the last slot in use, in every form (one launch, two)."""
    rng = np.random.default_rng(slots)
    for counts, r in (([1, 1], 8), ([1, 20], 24)):
        ranks = [int(v) for v in rng.integers(1, r + 1, slots)]
        _check(q4k, gpu, counts, [slots - 1, slots // 2], 256, 48, r, F32, slots=slots, ranks=ranks)
