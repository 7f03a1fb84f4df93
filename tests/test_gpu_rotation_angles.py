"""The rotation's cosines and sines themselves: pairs (1, 0) turn into them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("first", [0, 1000, 130000])
def test_cosines_and_sines(q4k, gpu, first, inter):
    """Relative to each value, near zero too: the function within 2 units (4 *
    2^-24), the correction's fused product (2^-24).  Beside that the angle in 64
    bits: 131072 * 1 rad carries half a step of 2^-52 * 2^17 rad here (1.5e-11), in
    the kernel three roundings of 2^-53 * 20861 turns (7e-12 turns, 4.4e-11 rad);
    the part that 32 bits of the fraction leave, at most 9.4e-8 rad, is good to
    2^-23 of itself (1.2e-14)."""
    rows, dim = 1000, 128
    x = torch.zeros((rows, 1, dim), device=gpu)
    at, to = (slice(0, dim, 2), slice(1, dim, 2)) if inter else (slice(0, dim // 2), slice(dim // 2, dim))
    x[..., at] = 1.0
    f = 10000.0 ** (-np.arange(0, dim, 2) / dim)
    p = np.arange(first, first + rows)
    y = torch.empty_like(x)
    q4k.rope(x, torch.from_numpy(f).to(gpu), torch.from_numpy(p.astype(np.int32)).to(gpu), y, interleaved=inter)
    got, angle = y.cpu().double().numpy()[:, 0], p[:, None] * f
    for part, want in ((at, np.cos(angle)), (to, np.sin(angle))):
        off = np.abs(got[:, part] - want)
        assert (off <= 5 * 2.0 ** -24 * np.abs(want) + 6e-11).all(), float((off - 5 * 2.0 ** -24 * np.abs(want)).max())
