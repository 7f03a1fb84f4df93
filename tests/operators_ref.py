"""Plain 64-bit implementations of rope, qk_norm_rope, lora and
process_logits (numpy, on the host), with the bounds that their fp32
arithmetic keeps.  Each bound counts roundings of u = 2^-24 (half a step of
fp32, relative); an fp16 result adds half a step of its own, 2^-11 of the value
(2^-25 below the normal range)."""
import numpy as np

U = 2.0 ** -24


def half_step(y, f16):
    return np.maximum(np.abs(y) * 2.0 ** -11, 2.0 ** -25) if f16 else 0.0


def rotate(x, inv_freq, positions, interleaved, scale):
    """(y, |a| + |b| of each element's pair) of x [rows, heads, dim]."""
    x = np.asarray(x, np.float64)
    h = len(inv_freq)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)
    c, n = (scale * np.cos(angle))[:, None, :], (scale * np.sin(angle))[:, None, :]
    first, second = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    y, size = x.copy(), np.zeros_like(x)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * n, b * c + a * n
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    return y, size


def rotate_bound(size, scale, far=False):
    """Cosine and sine: the reduced angle rounded to fp32 (2^-26 turns =
    9.4e-8 rad), two steps of the function (1.2e-7), the scale (6e-8); then a
    product and a fused product, two roundings (1.2e-7): 4e-7 of |a| + |b|.
    Positions up to 2^31: the product of position and turns carries three
    roundings of 2^-53 at 3.4e8 turns (7e-7 rad), the reference's one of 2^-53
    at 2^31 rad (2.4e-7): 1e-6 more."""
    return size * scale * (4e-7 + (1e-6 if far else 0.0))


def head_norm(x, weight, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * np.asarray(weight, np.float64)


def norm_bound(size, y, scale):
    """The sum of squares of up to 1024 values: at most 24 roundings on a
    value's way, half of that on its root; division, root, two products: 16
    roundings, 1e-6, on top of the rotation's."""
    return size * scale * (4e-7 + 1.1e-6) + np.abs(y) * 1.1e-6


def lora(x, a, b, ids, counts, ranks, scales, aux, slices_of_k=1):
    """(y, bound before the result's rounding)."""
    x, k, n = np.asarray(x, np.float64), a.shape[2], b.shape[1]
    m = x.shape[0]
    y = np.zeros((m, n)) if aux is None else np.asarray(aux, np.float64).copy()
    # aux + sum: one rounding of each.
    bound = np.zeros((m, n)) if aux is None else np.abs(y) * 2 * U
    start = 0
    for q, rows in enumerate(counts):
        here, i = slice(start, start + rows), int(ids[q])
        start += rows
        if not 0 <= i < a.shape[0]:
            continue
        r = a.shape[1] if ranks is None else int(np.clip(ranks[i], 0, a.shape[1]))
        s = 1.0 if scales is None else float(scales[i])
        A, B = a[i, :r].astype(np.float64), b[i, :, :r].astype(np.float64)
        u = x[here] @ A.T
        y[here] += s * (u @ B.T)
        # A wave sums at most k / 8 products in turn, then waves and slices; the
        # second product sums r.
        long = (np.abs(x[here]) @ np.abs(A).T) @ np.abs(B).T
        bound[here] += abs(s) * (k / 8 + 32) * U * long + abs(s) * (r + 6) * U * (np.abs(u) @ np.abs(B).T) + 2 * U * np.abs(y[here])
    return y, bound


def logits(x, texts=None, prompts=None, repetition=None, frequency=None, presence=None, biases=None, allowed=None):
    """(y, bound before the result's rounding) of x [rows, vocab]; texts[r] and
    biases[r] = [(token, value), ...] of row r, allowed [rows, vocab] or None."""
    y = np.asarray(x, np.float64).copy()
    bound = np.zeros_like(y)
    with np.errstate(invalid="ignore", over="ignore"):
        for r in range(y.shape[0]):
            if texts is not None:
                text = np.asarray(texts[r], np.int64)
                prompt = 0 if prompts is None else max(0, int(prompts[r]))
                seen = np.zeros(y.shape[1], bool)
                count = np.zeros(y.shape[1])
                for i, t in enumerate(text):
                    if 0 <= t < y.shape[1]:
                        seen[t] = True
                        count[t] += i >= prompt
                if repetition is not None:
                    p = float(repetition[r])
                    y[r] = np.where(seen, np.where(y[r] > 0, y[r] / p, y[r] * p), y[r])
                    bound[r] += np.where(seen, np.abs(y[r]) * U, 0.0)
                f = 0.0 if frequency is None else float(frequency[r])
                p = 0.0 if presence is None else float(presence[r])
                less = count > 0
                y[r] = np.where(less, y[r] - f * count - p, y[r])
                bound[r] += np.where(less, 3 * U * (np.abs(y[r]) + np.abs(f * count) + abs(p)), 0.0)
            if biases is not None:
                for token, value in dict((int(t), float(v)) for t, v in biases[r] if 0 <= t < y.shape[1]).items():
                    y[r, token] += value
                    bound[r, token] += U * (np.abs(y[r, token]) + abs(value))
        if allowed is not None:
            y = np.where(allowed, y, -np.inf)
    return y, np.where(np.isfinite(bound), bound, 0.0)


def assert_close(got, want, bound, f16, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    if f16:
        want_inf = np.abs(want) >= 65520.0  # rounds to infinity in fp16
        assert np.array_equal(np.isinf(got) & ~np.isnan(want), want_inf), what
        want = np.where(want_inf, np.copysign(np.inf, want), want)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), what
    d = np.abs(got[fine] - want[fine])
    allow = (bound + half_step(want, f16))[fine] if np.ndim(bound) else bound + half_step(want[fine], f16)
    worst = float(np.max(d - allow)) if d.size else 0.0
    assert worst <= 0.0, f"{what}: off by {float(d.max())}, {worst} past its bound"
