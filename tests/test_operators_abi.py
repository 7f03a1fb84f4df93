"""rope, qk_norm_rope, lora, linear_lora and process_logits without a GPU:
every refusal comes before any HIP call, and the rotary frequencies (host
arithmetic) match their formulas."""
import ctypes
import math

import numpy as np
import pytest
import torch

from mtlqwen_amd import operators as ops

EINVAL, ESHAPE, EALIAS = -1, -3, -4
# Addresses that are only compared, never read: the calls below are refused.
X, Y, W, F, P = 0x10000000, 0x20000000, 0x30000000, 0x30100000, 0x30200000


def heads(i=X, o=Y, w=W, strides=(4096, 128, 4096, 128), n=32):
    return ops._HEADS(i, o, w, *strides, n)


def rotation(f=F, p=P, rot=128, layout=0, scale=1.0):
    return ops._ROTATION(f, p, rot, layout, scale)


def rope(q4k, h, r, rows=8, dim=128, dtype=0):
    return q4k.lib.q4k_rope(None, 0, h, r, rows, dim, dtype)


def qk(q4k, a, b, r, rows=8, dim=128, eps=1e-6, dtype=0):
    return q4k.lib.q4k_qk_norm_rope(None, 0, a, b, r, rows, dim, eps, dtype)


@pytest.mark.parametrize("h,r,kw,code", [
    (heads(), rotation(), {"dtype": 2}, EINVAL),
    (heads(), rotation(), {"dim": 0}, ESHAPE),
    (heads(), rotation(), {"dim": 1025}, ESHAPE),
    (heads(), rotation(rot=127), {}, ESHAPE),
    (heads(), rotation(rot=130), {}, ESHAPE),
    (heads(), rotation(rot=0), {}, ESHAPE),
    (heads(), rotation(layout=2), {}, EINVAL),
    (heads(), rotation(f=0), {}, EINVAL),
    (heads(), rotation(p=0), {}, EINVAL),
    (heads(i=0), rotation(), {}, EINVAL),
    (heads(o=0), rotation(), {}, EINVAL),
    (heads(n=0), rotation(), {}, ESHAPE),
    (heads(n=65536), rotation(), {}, ESHAPE),
    (heads(strides=(-1, 128, 4096, 128)), rotation(), {}, ESHAPE),
    (heads(strides=(4096, 128, 4095, 128)), rotation(), {}, ESHAPE),  # rows of the output share elements
    (heads(strides=(4096, 128, 4096, 127)), rotation(), {}, ESHAPE),  # heads do
    (heads(strides=(4096, 128, 0, 128)), rotation(), {}, ESHAPE),
    (heads(strides=(4096, 128, 128, 1023)), rotation(), {}, ESHAPE),  # rows inside heads, heads too close
    (heads(o=X + 4), rotation(), {}, EALIAS),
    (heads(o=X, strides=(4096, 128, 8192, 128)), rotation(), {}, EALIAS),
    (heads(), rotation(p=Y + 100), {}, EALIAS),
    (heads(), rotation(f=Y + 8 * 4096 * 4 - 8), {}, EALIAS),
])
def test_rope_refusals(q4k, h, r, kw, code):
    assert rope(q4k, h, r, **kw) == code
    assert q4k.lib.q4k_last_error()


def test_rope_takes_no_rows(q4k):
    assert rope(q4k, heads(i=0, o=0), rotation(f=0, p=0), rows=0) == 0


def test_rope_null_structures(q4k):
    assert rope(q4k, None, rotation()) == EINVAL
    assert rope(q4k, heads(), None) == EINVAL
    assert qk(q4k, heads(), None, rotation()) == EINVAL


# q and k in rows of a joined projection of 6144: 32 + 8 heads of 128.
JOINED = (6144, 128, 6144, 128)
K0 = X + 4096 * 4


@pytest.mark.parametrize("a,b,kw,code", [
    (heads(w=0), heads(i=K0, o=Y + 0x1000000, n=8), {}, EINVAL),
    (heads(), heads(i=K0, o=Y + 0x1000000, w=0, n=8), {}, EINVAL),
    (heads(strides=JOINED), heads(i=K0, o=Y + 0x1000000, n=8), {"eps": -1.0}, EINVAL),
    (heads(strides=JOINED), heads(i=K0, o=Y + 0x1000000, n=8), {"eps": float("nan")}, EINVAL),
    (heads(strides=JOINED), heads(i=K0, o=Y + 4, strides=JOINED, n=8), {}, EALIAS),  # outputs overlap
    (heads(o=X, strides=JOINED), heads(i=X + 4095 * 4, o=Y, strides=JOINED, n=8), {}, EALIAS),  # q in place over k's input
    (heads(o=X, strides=JOINED), heads(i=K0, o=X + 4, strides=JOINED, n=8), {}, EALIAS),
    (heads(o=W - 8, strides=JOINED), heads(i=K0, o=Y, strides=JOINED, n=8), {}, EALIAS),  # over the weights
])
def test_qk_refusals(q4k, a, b, kw, code):
    assert qk(q4k, a, b, rotation(), **kw) == code


# q, k and v heads in turn: [rows, 4 heads, q k v, 128].
TURNS = (1536, 384, 1536, 384)
T1 = 128 * 4


@pytest.mark.parametrize("a,b", [
    (heads(o=X, strides=TURNS, n=4), heads(i=X + T1, o=X + T1 + 4, strides=TURNS, n=4)),  # k moves by one element
    (heads(o=X, strides=TURNS, n=4), heads(i=X + T1, o=X + T1 - 4, strides=TURNS, n=4)),  # into q
    (heads(o=X, strides=TURNS, n=4), heads(i=X + T1, o=X + T1, strides=(1600, 384, 1600, 384), n=4)),  # rows out of turn
    (heads(o=X, strides=TURNS, n=4), heads(i=X + T1, o=X + T1, strides=(1536, 256, 1536, 256), n=4)),  # heads out of turn
])
def test_qk_in_turn_refusals(q4k, a, b):
    assert qk(q4k, a, b, rotation()) == EALIAS


def test_frequencies():
    rot, base, factor, ctx = 64, 10000.0, 8.0, 4096
    i = np.arange(rot // 2)
    plain = base ** (-2.0 * i / rot)

    def check(got, want, scale):
        assert np.allclose(got[0].numpy(), want, rtol=1e-14, atol=0) and abs(got[1] - scale) <= 2 ** -23 * scale

    check(ops.rope_frequencies(rot, base, device="cpu"), plain, 1.0)
    check(ops.rope_frequencies(rot, base, "linear", factor, device="cpu"), plain / factor, 1.0)
    check(ops.rope_frequencies(rot, base, "ntk", factor, device="cpu"), (base * factor ** (rot / (rot - 2))) ** (-2.0 * i / rot), 1.0)
    kept = np.clip((ctx * plain / (2 * math.pi) - 1) / 31, 0, 1)
    assert kept.min() == 0 and kept.max() == 1
    check(ops.rope_frequencies(rot, base, "yarn", factor, ctx, device="cpu"), (1 - kept) * plain / factor + kept * plain,
          0.1 * math.log(factor) + 1)
    check(ops.rope_frequencies(2, device="cpu"), np.ones(1), 1.0)


@pytest.mark.parametrize("args", [(0,), (63,), (1026,), (64, 0.0), (64, float("inf")), (64, 1e4, "linear", 0.0), (64, 1e4, "yarn", 2.0, 0),
                                  (64, 1e4, "yarn", 2.0, 4096, 32.0, 1.0), (2, 1e4, "ntk", 2.0)])
def test_frequency_refusals(q4k, args):
    with pytest.raises(q4k.Q4KError):
        ops.rope_frequencies(*args, device="cpu")


def test_frequency_scaling_name():
    with pytest.raises(ValueError):
        ops.rope_frequencies(64, scaling="other", device="cpu")


def adapters(a=F, b=P, ids=W, ranks=0, scales=0, slots=4, rank=16):
    return ops._ADAPTERS(a, b, ids, ranks, scales, slots, rank)


def lora(q4k, ad, x=X, y=Y, aux=None, m=8, k=4096, n=1024, counts=(8,), nq=None, dtype=0):
    arr = None if counts is None else ops._COUNTS[len(counts)](*counts)
    nq = (0 if counts is None else len(counts)) if nq is None else nq
    return q4k.lib.q4k_lora(None, 0, ad, x, y, aux, m, k, n, arr, nq, dtype)


@pytest.mark.parametrize("ad,kw,code", [
    (None, {}, EINVAL),
    (adapters(), {"dtype": 2}, EINVAL),
    (adapters(), {"k": 4000}, ESHAPE),
    (adapters(), {"k": 0}, ESHAPE),
    (adapters(), {"n": 1000}, ESHAPE),
    (adapters(), {"m": 0, "counts": (0,)}, ESHAPE),
    (adapters(), {"m": (1 << 24) + 1, "counts": ((1 << 24) + 1,)}, ESHAPE),
    (adapters(rank=0), {}, ESHAPE),
    (adapters(rank=513), {}, ESHAPE),
    (adapters(slots=0), {}, ESHAPE),
    (adapters(slots=65537), {}, ESHAPE),
    (adapters(a=0), {}, EINVAL),
    (adapters(b=0), {}, EINVAL),
    (adapters(ids=0), {}, EINVAL),
    (adapters(), {"x": None}, EINVAL),
    (adapters(), {"y": None}, EINVAL),
    (adapters(), {"counts": (3, 4)}, EINVAL),
    (adapters(), {"counts": (1,) * 8 + (0,)}, EINVAL),
    (adapters(), {"counts": None, "nq": 1}, EINVAL),
    (adapters(), {"y": X + 4}, EALIAS),
    (adapters(), {"aux": Y + 4}, EALIAS),
    (adapters(a=Y + 64), {}, EALIAS),
    (adapters(b=Y + 64), {}, EALIAS),
    (adapters(ids=Y), {}, EALIAS),
    (adapters(ranks=Y), {}, EALIAS),
    (adapters(scales=Y + 8 * 1024 * 4 - 4), {}, EALIAS),
])
def test_lora_refusals(q4k, ad, kw, code):
    assert lora(q4k, ad, **kw) == code


def test_linear_lora_null_weight(q4k):
    assert q4k.lib.q4k_linear_lora(None, None, adapters(), X, Y, None, 8, None, 0, 0, 0) == EINVAL


def params(tokens=0, slots=0, lengths=0, prompts=0, rep=0, freq=0, pres=0, bo=0, bt=0, bv=0, mask=0, mrows=0, nslots=0, capacity=0, nbias=0,
           nmasks=0, words=0):
    return ops._LOGITS(tokens, slots, lengths, prompts, rep, freq, pres, bo, bt, bv, mask, mrows, nslots, capacity, nbias, nmasks, words)


def logits(q4k, p, i=X, o=Y, rows=4, vocab=1000, si=1000, so=1000, dtype=0):
    return q4k.lib.q4k_process_logits(None, 0, i, o, rows, vocab, si, so, p, dtype)


@pytest.mark.parametrize("p,kw,code", [
    (None, {}, EINVAL),
    (params(), {"dtype": 2}, EINVAL),
    (params(), {"vocab": 0}, ESHAPE),
    (params(), {"vocab": (1 << 24) + 1}, ESHAPE),
    (params(), {"rows": 65536}, ESHAPE),
    (params(), {"so": 999}, ESHAPE),
    (params(), {"si": -1}, ESHAPE),
    (params(tokens=W, nslots=4, capacity=16), {}, EINVAL),  # no lengths
    (params(rep=W), {}, EINVAL),  # no text
    (params(lengths=W), {}, EINVAL),
    (params(tokens=W, lengths=F, nslots=3, capacity=16), {}, ESHAPE),  # row 3 has no text
    (params(tokens=W, lengths=F, nslots=4, capacity=(1 << 30) + 1), {}, ESHAPE),
    (params(bo=W), {}, EINVAL),
    (params(bo=W, bt=F), {}, EINVAL),
    (params(bt=F, bv=P), {}, EINVAL),
    (params(mrows=W), {}, EINVAL),
    (params(mask=W, nmasks=4, words=31), {}, ESHAPE),
    (params(mask=W, nmasks=3, words=32), {}, ESHAPE),  # row 3 has no mask
    (params(), {"i": None}, EINVAL),
    (params(), {"o": None}, EINVAL),
    (params(), {"o": X + 4}, EALIAS),
    (params(), {"o": X, "so": 1001}, EALIAS),
    (params(tokens=Y, lengths=F, nslots=4, capacity=16), {}, EALIAS),
    (params(tokens=W, lengths=Y + 3 * 4000, nslots=4, capacity=16), {}, EALIAS),
    (params(mask=Y - 4, nmasks=4, words=32), {}, EALIAS),
    (params(bo=W, bt=F, bv=Y, nbias=1), {}, EALIAS),
])
def test_logits_refusals(q4k, p, kw, code):
    assert logits(q4k, p, **kw) == code


def test_logits_takes_no_rows(q4k):
    assert logits(q4k, params(), i=None, o=None, rows=0) == 0


def test_structures_have_the_header_sizes(tmp_path):
    """The packed structures are those that a C compiler lays out."""
    import os
    import subprocess

    from q4k_ref import ROOT
    src = '#include <stdio.h>\n#include "q4k.h"\nint main(void){printf("%zu %zu %zu %zu", sizeof(q4k_heads), sizeof(q4k_rotation), ' \
          'sizeof(q4k_adapters), sizeof(q4k_logits_params));return 0;}\n'
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), "-x", "c", "-", "-o", exe], input=src, text=True, check=True)
    sizes = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [len(heads()), len(rotation()), len(adapters()), len(params())]


def test_python_checks_refuse_host_tensors(q4k):
    x = torch.zeros(2, 4, 128)
    f = torch.zeros(64, dtype=torch.float64)
    p = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        q4k.rope(x, f, p, x)
    with pytest.raises(TypeError):
        q4k.rope(x.to(torch.bfloat16), f, p, x)
    with pytest.raises(ValueError):
        q4k.process_logits(torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(ValueError):
        q4k.lora(torch.zeros(2, 256), torch.zeros(1, 4, 256, dtype=torch.half), torch.zeros(1, 16, 4, dtype=torch.half), p, 2, torch.zeros(2, 16))
    assert ctypes.sizeof(ctypes.c_void_p) == 8
