"""The largest sizes that the operators document, one at a time, against 64-bit
numpy."""
import numpy as np
import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
MOST = 1 << 24


def _half(rng, *shape):
    return (rng.standard_normal(shape) / np.sqrt(shape[-1])).astype(np.float16)


def test_adapters_of_a_long_k(q4k, gpu):
    rng = np.random.default_rng(1)
    x, a, b = rng.standard_normal((3, MOST), np.float32), _half(rng, 1, 4, MOST), _half(rng, 1, 16, 4)
    y = torch.empty((3, 16), device=gpu)
    q4k.lora(torch.from_numpy(x).to(gpu), torch.from_numpy(a).to(gpu), torch.from_numpy(b).to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu), 3, y)
    want, bound = ref.lora(x, a, b, [0], [3], None, None, None)
    ref.assert_close(y.cpu().numpy(), want, bound, False)
    assert np.linalg.norm(y.cpu().numpy() - want) <= 1e-4 * np.linalg.norm(want)  # a chain of k / 64 rounds by its root: 512 * 2^-24 = 3e-5


def test_adapters_of_many_columns(q4k, gpu):
    rng = np.random.default_rng(2)
    x, a, b = rng.standard_normal((3, 256)).astype(np.float32), _half(rng, 1, 4, 256), _half(rng, 1, MOST, 4)
    y = torch.empty((3, MOST), device=gpu, dtype=F16)
    xt = torch.from_numpy(x).to(gpu).half()
    for rows in (1, 3):  # one launch, two
        q4k.lora(xt, torch.from_numpy(a).to(gpu), torch.from_numpy(b).to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu), rows, y)
        want, bound = ref.lora(xt[:rows].cpu().float().numpy(), a, b, [0], [rows], None, None, None)
        ref.assert_close(y[:rows].cpu().float().numpy(), want, bound, True)


def test_adapters_of_many_rows(q4k, gpu):
    rng = np.random.default_rng(3)
    a, b = _half(rng, 2, 4, 256), _half(rng, 2, 16, 4)
    g = torch.Generator(device=gpu)
    g.manual_seed(3)
    x = torch.randn((MOST, 256), device=gpu, generator=g, dtype=F16)
    y = torch.empty((MOST, 16), device=gpu, dtype=F16)
    counts = [MOST - 100, 0, 100]
    q4k.lora(x, torch.from_numpy(a).to(gpu), torch.from_numpy(b).to(gpu), torch.tensor([0, 0, 1], dtype=torch.int32, device=gpu), MOST, y,
             query_counts=counts)
    torch.cuda.synchronize()
    for lo, hi, i in ((0, 200, 0), (MOST // 2 - 100, MOST // 2 + 100, 0), (MOST - 250, MOST - 100, 0), (MOST - 100, MOST, 1)):
        want, bound = ref.lora(x[lo:hi].cpu().float().numpy(), a, b, [i], [hi - lo], None, None, None)
        ref.assert_close(y[lo:hi].cpu().float().numpy(), want, bound, True, f"rows {lo}")


@pytest.mark.parametrize("counts", [[1, 1], [1, 30]])
def test_adapters_of_many_slots(q4k, gpu, counts):
    rng = np.random.default_rng(4)
    slots = 65536
    a, b = _half(rng, slots, 2, 256), _half(rng, slots, 16, 2)
    x = rng.standard_normal((sum(counts), 256)).astype(np.float32)
    ranks, scales = rng.integers(1, 3, slots).astype(np.int32), rng.uniform(0.5, 2, slots).astype(np.float32)
    t = lambda v: torch.from_numpy(v).to(gpu)  # noqa: E731
    y = torch.empty((sum(counts), 16), device=gpu)
    ids = [65535, 40000]
    q4k.lora(t(x), t(a), t(b), t(np.array(ids, np.int32)), sum(counts), y, query_counts=counts, ranks=t(ranks), scales=t(scales))
    want, bound = ref.lora(x, a, b, ids, counts, ranks, scales, None)
    ref.assert_close(y.cpu().numpy(), want, bound, False)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,dim,rot", [(65535, 2, 2), (65535, 64, 16), (65535, 1024, 1024)])
def test_many_heads(q4k, gpu, heads, dim, rot, norm):
    rng = np.random.default_rng(heads + dim)
    x = torch.from_numpy(rng.standard_normal((2, heads, dim), np.float32)).half()
    f, p = torch.from_numpy(10000.0 ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)), torch.tensor([9, 70000], dtype=torch.int32)
    w = torch.from_numpy(rng.uniform(0.5, 1.5, dim).astype(np.float32))
    y = torch.empty_like(x).to(gpu)
    if norm:
        k, ko = x[:, :, :dim].flip(1).contiguous().to(gpu), torch.empty_like(y)
        q4k.qk_norm_rope(x.to(gpu), k, w.to(gpu), w.to(gpu), f.to(gpu), p.to(gpu), y, ko)
        torch.cuda.synchronize()
        assert torch.equal(ko.flip(1), y)
    else:
        q4k.rope(x.to(gpu), f.to(gpu), p.to(gpu), y)
    part = slice(0, heads, 97)
    for s in (part, slice(heads - 50, heads)):
        v = x[:, s].float().numpy()
        v = ref.head_norm(v, w.numpy(), np.float32(1e-6)) if norm else v
        want, size = ref.rotate(v, f.numpy(), p.numpy(), False, 1.0)
        ref.assert_close(y[:, s].cpu().float().numpy(), want, ref.norm_bound(size, want, 1.0) if norm else ref.rotate_bound(size, 1.0), True)


@pytest.mark.parametrize("rows,vocab", [(2, MOST), (65535, 1), (65535, 33), (65535, 5000)])
def test_most_logits(q4k, gpu, rows, vocab):
    """Texts of one token, of both halves of the rows: l / 2 - 0.25 - 0.5 of that
    token where positive, l * 2 - 0.75 else (exact: powers of two of fp16 values)."""
    g = torch.Generator(device=gpu)
    g.manual_seed(5)
    x = torch.randn((rows, vocab), device=gpu, generator=g).half().float()
    tokens = torch.tensor([[vocab - 1], [vocab // 2]], device=gpu, dtype=torch.int32)
    slots = (torch.arange(rows, device=gpu) % 2).to(torch.int32)
    full = lambda v, d=F32: torch.full((rows,), v, device=gpu, dtype=d)  # noqa: E731
    out = torch.empty_like(x)
    q4k.process_logits(x, out, tokens=tokens, slots=slots, lengths=full(1, torch.int32), repetition=full(2.0), frequency=full(0.25), presence=full(0.5))
    at = tokens[slots.long(), 0].long().unsqueeze(1)
    l = x.gather(1, at)
    want = x.scatter(1, at, torch.where(l > 0, l / 2, l * 2) - 0.25 - 0.5)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
