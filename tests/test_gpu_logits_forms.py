"""process_logits in the forms that only some sizes take, against 64-bit numpy:
the large ranges with odd vocabularies, wide rows off alignment and in place,
those that long texts choose, and rows of more biases than share a word with
the count of a large token buffer."""
import numpy as np
import pytest
import torch

import operators_ref as ref
from test_gpu_logits import _args, _batch, _reference

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
STEPS = ("text", "bias", "mask")


def _check(q4k, gpu, b, dtype, what):
    want, bound = _reference(b, STEPS)
    x, args = b["x"].to(gpu), _args(b, STEPS, gpu)
    rows, vocab = x.shape
    out = torch.empty_like(x)
    q4k.process_logits(x, out, **args)
    torch.cuda.synchronize()
    ref.assert_close(out.cpu().float().numpy(), want, bound, dtype == F16, what)
    inplace = x.clone()
    q4k.process_logits(inplace, inplace, **args)
    # Rows of wider buffers, one element off alignment, nothing written between them.
    wide_in = torch.full((rows * (vocab + 6) + 1,), 3.0, device=gpu, dtype=dtype)
    wide_out = torch.full((rows * (vocab + 9) + 1,), 7.0, device=gpu, dtype=dtype)
    vi, vo = wide_in[1:].view(rows, vocab + 6)[:, :vocab], wide_out[1:].view(rows, vocab + 9)[:, :vocab]
    vi.copy_(x)
    q4k.process_logits(vi, vo, **args)
    torch.cuda.synchronize()
    assert torch.equal(inplace, out) and torch.equal(vo, out), what
    assert bool((wide_out[1:].view(rows, vocab + 9)[:, vocab:] == 7.0).all()) and wide_out[0] == 7.0, what
    q4k.process_logits(vi, vi, **args)
    torch.cuda.synchronize()
    assert torch.equal(vi, out), what
    assert bool((wide_in[1:].view(rows, vocab + 6)[:, vocab:] == 3.0).all()) and wide_in[0] == 3.0, what


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,vocab,capacity", [(17, 248319, 900), (85, 50257, 120), (9, 248321, 32769), (44, 50261, 33001)])
def test_large_ranges(q4k, gpu, rows, vocab, capacity, dtype):
    """16384 tokens to a workgroup: by the logits, and by the texts' capacity."""
    rng = np.random.default_rng(rows)
    b = _batch(rng, rows, vocab, capacity, rows, 60, 3, dtype)
    b["lengths"][0] = capacity
    _check(q4k, gpu, b, dtype, f"{rows}x{vocab}")


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,vocab", [(5, 4999), (17, 248320)])
def test_biases_beside_the_counts_of_a_large_buffer(q4k, gpu, rows, vocab, dtype):
    """A buffer of 2^22 tokens leaves 8 bits of a word to the biases: rows of up
    to 255 share it with the count, others take a round of their own."""
    rng = np.random.default_rng(vocab)
    b = _batch(rng, rows, vocab, 16, 2, 900, 3, dtype)
    tokens = np.zeros((2, 1 << 22), np.int32)
    tokens[:, :600] = rng.integers(0, 700, (2, 600))
    b["tokens"], b["slots"] = tokens, rng.integers(0, 2, rows).astype(np.int32)
    b["lengths"] = rng.integers(300, 601, rows).astype(np.int32)
    b["prompts"] = rng.integers(0, 300, rows).astype(np.int32)
    per = rng.integers(256, 901, rows)
    per[:4] = 255, 256, 0, 900
    b["bias_offsets"] = np.concatenate([[0], np.cumsum(per)]).astype(np.int32)
    b["bias_tokens"] = rng.integers(-2, 900, int(per.sum())).astype(np.int32)  # repeated ones, on tokens of the texts
    b["bias_values"] = (5 * rng.standard_normal(int(per.sum()))).astype(np.float32)
    _check(q4k, gpu, b, dtype, f"{rows}x{vocab}")
