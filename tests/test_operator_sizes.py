"""Sizes past the C ABI's 32 bits are refused, never cut to them."""
import pytest
import torch

from mtlqwen_amd import operators as ops


@pytest.mark.parametrize("rot,context", [((1 << 32) + 64, 4096), (64 - (1 << 32), 4096), (-64, 4096), (64, (1 << 32) + 4096), (64, 4096 - (1 << 32)),
                                         (64, -4096)])
def test_frequencies(rot, context):
    with pytest.raises(ValueError):
        ops.rope_frequencies(rot, 1e4, "yarn", 2.0, context, device="cpu")


@pytest.mark.gpu
def test_rows_and_columns(q4k, gpu):
    """Tensors of 2^32 elements and a few (34 GB at a time, not written): their
    sizes, cut to 32 bits, would be valid."""
    many = (1 << 32) + 8
    empty = lambda *shape, dtype=torch.float16: torch.empty(shape, device=gpu, dtype=dtype)  # noqa: E731
    f, w, id0 = torch.ones(1, device=gpu, dtype=torch.float64), torch.ones(2, device=gpu), torch.zeros(1, device=gpu, dtype=torch.int32)
    x, p = empty(many, 1, 2), empty(many, dtype=torch.int32)
    with pytest.raises(ValueError):
        q4k.rope(x, f, p, x)
    with pytest.raises(ValueError):
        q4k.qk_norm_rope(x, x, w, w, f, p, x, x)
    del x, p
    torch.cuda.empty_cache()
    logits = empty(1, many)
    with pytest.raises(ValueError):
        q4k.process_logits(logits, logits)
    del logits
    torch.cuda.empty_cache()
    a = empty(1, 1, (1 << 32) + 256)
    with pytest.raises(ValueError):
        q4k.lora(a.view(1, -1), a, empty(1, 16, 1), id0, 1, empty(1, 16))
    del a
    torch.cuda.empty_cache()
