"""process_logits on the GPU against 64-bit numpy (operators_ref): each step
alone and together, both types, vocabularies of one token to the model's, odd
strides, texts of no token to long ones, repeated and foreign tokens, biases
given twice, masks that forbid everything, infinities and NaN, in place, and
captured."""
import numpy as np
import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16
NEG = float("-inf")


def _bits(mask):
    return ((mask[:, np.arange(mask.shape[1] * 32) // 32].view(np.uint32) >> (np.arange(mask.shape[1] * 32) % 32).astype(np.uint32)) & 1).astype(bool)


def _batch(rng, rows, vocab, capacity, nslots, nbias, nmasks, dtype):
    """Host values of every argument; texts hold foreign tokens too."""
    b = {"x": torch.from_numpy((4 * rng.standard_normal((rows, vocab))).astype(np.float32)).to(dtype)}
    tokens = (vocab * rng.random((nslots, capacity)) ** 3).astype(np.int32)
    if capacity > 4:
        tokens[:, 3], tokens[:, 4] = -1, vocab
    b["tokens"] = tokens
    b["slots"] = rng.integers(0, nslots, rows).astype(np.int32)
    b["lengths"] = rng.integers(0, capacity + 1, rows).astype(np.int32)
    b["prompts"] = (b["lengths"] * rng.random(rows)).astype(np.int32)
    b["repetition"] = rng.uniform(0.8, 1.5, rows).astype(np.float32)
    b["frequency"] = rng.uniform(-0.2, 0.6, rows).astype(np.float32)
    b["presence"] = rng.uniform(0, 1, rows).astype(np.float32)
    per = rng.integers(0, nbias + 1, rows)
    b["bias_offsets"] = np.concatenate([[0], np.cumsum(per)]).astype(np.int32)
    total = max(1, int(per.sum()))
    b["bias_tokens"] = rng.integers(-2, vocab + 2, total).astype(np.int32)
    b["bias_values"] = (5 * rng.standard_normal(total)).astype(np.float32)
    b["mask"] = rng.integers(-2**31, 2**31, (nmasks, (vocab + 31) // 32)).astype(np.int32)
    b["mask_rows"] = rng.integers(-1, nmasks, rows).astype(np.int32)
    return b


def _reference(b, steps):
    rows, vocab = b["x"].shape
    kw = {}
    if "text" in steps:
        kw["texts"] = [b["tokens"][b["slots"][r], :b["lengths"][r]] for r in range(rows)]
        kw.update(prompts=b["prompts"], repetition=b["repetition"], frequency=b["frequency"], presence=b["presence"])
    if "bias" in steps:
        o = b["bias_offsets"]
        kw["biases"] = [list(zip(b["bias_tokens"][o[r]:o[r + 1]], b["bias_values"][o[r]:o[r + 1]])) for r in range(rows)]
    if "mask" in steps:
        bits = _bits(b["mask"])[:, :vocab]
        kw["allowed"] = np.stack([bits[m] if m >= 0 else np.ones(vocab, bool) for m in b["mask_rows"]])
    return ref.logits(b["x"].float().numpy(), **kw)


TEXT = ("tokens", "slots", "lengths", "prompts", "repetition", "frequency", "presence")
NAMES = {"text": TEXT, "bias": ("bias_offsets", "bias_tokens", "bias_values"), "mask": ("mask", "mask_rows")}


def _args(b, steps, gpu):
    return {n: torch.from_numpy(b[n]).to(gpu) for s in steps for n in NAMES[s]}


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("steps", [(), ("text",), ("bias",), ("mask",), ("text", "bias", "mask")])
@pytest.mark.parametrize("rows,vocab,capacity", [(1, 1, 1), (3, 31, 5), (2, 1000, 7), (5, 4097, 300), (7, 32001, 4100), (64, 8200, 130)])
def test_process_logits(q4k, gpu, rows, vocab, capacity, steps, dtype):
    rng = np.random.default_rng(rows + vocab + capacity + len(steps))
    b = _batch(rng, rows, vocab, capacity, rows + 2, 40, 3, dtype)
    want, bound = _reference(b, steps)
    x = b["x"].to(gpu)
    out = torch.full_like(x, float("nan"))
    q4k.process_logits(x, out, **_args(b, steps, gpu))
    torch.cuda.synchronize()
    ref.assert_close(out.cpu().float().numpy(), want, bound, dtype == F16, f"{rows}x{vocab} {steps}")
    same = (want == b["x"].float().numpy()) & (bound == 0)
    assert np.array_equal(out.cpu().float().numpy()[same], b["x"].float().numpy()[same])
    inplace = x.clone()
    q4k.process_logits(inplace, inplace, **_args(b, steps, gpu))
    torch.cuda.synchronize()
    assert torch.equal(inplace, out)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,capacity", [(2, 65536), (48, 3000)])
def test_full_vocabulary(q4k, gpu, rows, capacity, dtype):
    """The model's vocabulary; the kernel of few rows and that of many."""
    rng = np.random.default_rng(rows)
    b = _batch(rng, rows, 248320, capacity, rows, 300, 2, dtype)
    b["lengths"][0] = capacity
    steps = ("text", "bias", "mask")
    want, bound = _reference(b, steps)
    x = b["x"].to(gpu)
    out = torch.empty_like(x)
    q4k.process_logits(x, out, **_args(b, steps, gpu))
    torch.cuda.synchronize()
    ref.assert_close(out.cpu().float().numpy(), want, bound, dtype == F16, f"{rows} rows")


@pytest.mark.parametrize("dtype", [F32, F16])
def test_strides_and_storage(q4k, gpu, dtype):
    """Rows of a wider buffer, one element off alignment: the bits of the
    contiguous call, and nothing written between the rows."""
    rng = np.random.default_rng(3)
    b = _batch(rng, 5, 1003, 50, 6, 9, 3, dtype)
    steps = ("text", "bias", "mask")
    x, args = b["x"].to(gpu), _args(b, steps, gpu)
    out = torch.empty_like(x)
    q4k.process_logits(x, out, **args)
    wide_in = torch.full((5 * 1100 + 1,), 3.0, device=gpu, dtype=dtype)
    wide_out = torch.full((5 * 1021 + 1,), 7.0, device=gpu, dtype=dtype)
    vi, vo = wide_in[1:].view(5, 1100)[:, :1003], wide_out[1:].view(5, 1021)[:, :1003]
    vi.copy_(x)
    q4k.process_logits(vi, vo, **args)
    torch.cuda.synchronize()
    assert torch.equal(vo, out)
    assert bool((wide_out[1:].view(5, 1021)[:, 1003:] == 7.0).all()) and wide_out[0] == 7.0
    # One row's logits for all rows (stride 0).
    q4k.process_logits(x[:1].expand(5, 1003), out, **args)
    again = torch.empty_like(x)
    q4k.process_logits(x[:1].expand(5, 1003).contiguous(), again, **args)
    torch.cuda.synchronize()
    assert torch.equal(out, again)


def test_special_values(q4k, gpu):
    """Masked places are -inf whatever they held; infinities take penalties by
    IEEE rules; NaN stays where it is allowed."""
    x = torch.tensor([[float("nan"), float("inf"), NEG, 1.0, -1.0, 0.0, 2.0, float("nan")]], device=gpu)
    tokens = torch.tensor([[1, 2, 3, 4, 5, 3, 3, 0]], dtype=torch.int32, device=gpu)
    out = torch.empty_like(x)
    mask = torch.tensor([[0b01111111]], dtype=torch.int32, device=gpu)
    one = torch.ones(1, device=gpu)
    n = torch.tensor([7], dtype=torch.int32, device=gpu)
    q4k.process_logits(x, out, tokens=tokens, lengths=n, prompts=torch.tensor([2], dtype=torch.int32, device=gpu), repetition=2 * one,
                       frequency=0.5 * one, presence=0.25 * one, mask=mask)
    got = out.cpu().numpy()[0]
    assert np.isnan(got[0]) and got[1] == np.inf and got[2] == NEG and got[7] == NEG
    # token 3: 1 / 2 - 3 * 0.5 - 0.25; 4: -1 * 2 - 0.5 - 0.25; 5: 0 - 0.5 - 0.25; 6 untouched
    assert list(got[3:7]) == [-1.25, -2.75, -0.75, 2.0]
    # Everything forbidden; a mask row out of range forbids nothing.
    q4k.process_logits(x, out, mask=torch.zeros((1, 1), dtype=torch.int32, device=gpu))
    assert bool((out == NEG).all())
    q4k.process_logits(x, out, mask=torch.zeros((1, 1), dtype=torch.int32, device=gpu), mask_rows=torch.tensor([1], dtype=torch.int32, device=gpu))
    assert torch.equal(out[:, 1:7], x[:, 1:7])
    # The largest fp16 value pushed past the range.
    h = torch.full((1, 8), 65504.0, device=gpu, dtype=F16)
    ho = torch.empty_like(h)
    q4k.process_logits(h, ho, bias_offsets=torch.tensor([0, 1], dtype=torch.int32, device=gpu), bias_tokens=n, bias_values=1000 * one)
    assert ho[0, 7] == float("inf") and bool((ho[0, :7] == 65504.0).all())


def test_out_of_range_descriptions(q4k, gpu):
    """Slots, lengths, offsets and prompts outside their buffers are clamped
    or ignored, never followed."""
    rng = np.random.default_rng(9)
    vocab, cap = 500, 20
    x = torch.from_numpy(rng.standard_normal((6, vocab)).astype(np.float32)).to(gpu)
    tokens = torch.from_numpy(rng.integers(0, vocab, (3, cap)).astype(np.int32)).to(gpu)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    rep = torch.full((6,), 2.0, device=gpu)
    pres = torch.full((6,), 0.5, device=gpu)
    out, want = torch.empty_like(x), torch.empty_like(x)
    q4k.process_logits(x, out, tokens=tokens, slots=i32(-1, 3, 2**31 - 1, 0, 1, 2), lengths=i32(5, 5, 5, -7, 2**31 - 1, 20),
                       prompts=i32(0, 0, 0, 0, -5, 2**31 - 1), repetition=rep, presence=pres)
    q4k.process_logits(x, want, tokens=tokens, slots=i32(0, 0, 0, 0, 1, 2), lengths=i32(0, 0, 0, 0, 20, 20), prompts=i32(0, 0, 0, 0, 0, 20),
                       repetition=rep, presence=pres)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(out[:4], x[:4]) and not torch.equal(out[4], x[4])
    q4k.process_logits(x, out, bias_offsets=i32(-3, 1, 0, 2**31 - 1, 5, -1, 7), bias_tokens=i32(7, 7, 8), bias_values=torch.ones(3, device=gpu))
    q4k.process_logits(x, want, bias_offsets=i32(0, 1, 1, 4, 4, 4, 4)[:7], bias_tokens=i32(7, 7, 7, 8), bias_values=torch.ones(4, device=gpu))
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], x[1]) and torch.equal(out[2], want[2]) and torch.equal(out[3], x[3])
    # The last row runs from the clamped start to the clamped end: all three entries.
    assert out[5, 7] == x[5, 7] + 1 and out[5, 8] == x[5, 8] + 1


def test_last_bias_of_a_token_counts(q4k, gpu):
    x = torch.zeros((1, 100), device=gpu)
    out = torch.empty_like(x)
    rng = np.random.default_rng(4)
    t = rng.integers(0, 100, 5000).astype(np.int32)
    v = rng.standard_normal(5000).astype(np.float32)
    for _ in range(3):
        q4k.process_logits(x, out, bias_offsets=torch.tensor([0, 5000], dtype=torch.int32, device=gpu), bias_tokens=torch.from_numpy(t).to(gpu),
                           bias_values=torch.from_numpy(v).to(gpu))
        got = out.cpu().numpy()[0]
        assert all(got[token] == value for token, value in dict(zip(t, v)).items())


def test_empty_groups(q4k, gpu):
    x = torch.randn((2, 50), device=gpu)
    out = torch.empty_like(x)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    zeros = torch.zeros(3, dtype=torch.int32, device=gpu)
    q4k.process_logits(x, out, tokens=none.view(2, 0), lengths=zeros, repetition=torch.ones(2, device=gpu), bias_offsets=zeros, bias_tokens=none,
                       bias_values=none.float(), mask=none.view(0, 2), mask_rows=zeros)
    torch.cuda.synchronize()
    assert torch.equal(out, x)
    assert q4k.process_logits(x[:0], out[:0]).shape[0] == 0
    for bad in [lambda: q4k.process_logits(x, out[:1]), lambda: q4k.process_logits(x, out.half()), lambda: q4k.process_logits(x.t(), out.t()),
                lambda: q4k.process_logits(x, out, tokens=none), lambda: q4k.process_logits(x, out, tokens=zeros.view(1, 3), lengths=zeros[:1]),
                lambda: q4k.process_logits(x, out, mask=zeros.view(1, 3).long())]:
        with pytest.raises((TypeError, ValueError)):
            bad()
    with pytest.raises(q4k.Q4KError):
        q4k.process_logits(x, out, repetition=torch.ones(2, device=gpu))


def test_masks_and_texts_too_few(q4k, gpu):
    """Descriptions with nothing in them are refused where rows would need
    them, never taken for a step left out; no rows need none."""
    x = torch.randn((2, 50), device=gpu)
    out = torch.empty_like(x)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    rows = torch.zeros(2, dtype=torch.int32, device=gpu)
    for bad in [{"mask": none.view(0, 2)}, {"mask": none.view(2, 0)}, {"mask": none.view(2, 0), "mask_rows": rows},
                {"mask": rows.view(2, 1)}, {"mask": rows.view(1, 2)}, {"tokens": none.view(0, 5), "lengths": rows},
                {"tokens": rows.view(1, 2), "lengths": rows}]:
        with pytest.raises(ValueError):
            q4k.process_logits(x, out, **bad)
    got = q4k.process_logits(x[:0], out[:0], tokens=rows.view(1, 2), lengths=none, repetition=none.float(), mask=rows.view(1, 2), mask_rows=none)
    assert got.shape == (0, 50)


def test_captured_call_follows_its_descriptions(q4k, gpu):
    rng = np.random.default_rng(8)
    b = _batch(rng, 4, 5000, 200, 5, 10, 3, F32)
    steps = ("text", "bias", "mask")
    x, args = b["x"].to(gpu), _args(b, steps, gpu)
    out, want = torch.empty_like(x), torch.empty_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        q4k.process_logits(x, out, **args)
    for step in range(4):
        args["lengths"].copy_(torch.from_numpy(rng.integers(0, 201, 4).astype(np.int32)))
        args["mask_rows"].copy_(torch.from_numpy(rng.integers(-1, 3, 4).astype(np.int32)))
        args["tokens"].add_(1)
        g.replay()
        q4k.process_logits(x, want, **args)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
