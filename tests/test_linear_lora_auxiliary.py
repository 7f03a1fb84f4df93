"""linear_lora takes no up weight as auxiliary, which linear does (the fused
gate/up pair)."""
import pytest
import torch

import mtlqwen_amd as q4k


def test_a_weight_is_refused():
    w = q4k.Weight.__new__(q4k.Weight)
    w._h, w.n, w.k, w.type, w.device = None, 16, 256, q4k.GGML_TYPE_Q4_K, 0
    a, b = torch.zeros((1, 4, 256), dtype=torch.half), torch.zeros((1, 16, 4), dtype=torch.half)
    with pytest.raises(TypeError, match="auxiliary"):
        q4k.linear_lora(torch.zeros(2, 256), w, a, b, torch.zeros(1, dtype=torch.int32), 2, torch.zeros(2, 16), auxiliary=w, gated=True)
