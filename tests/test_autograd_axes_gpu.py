"""Gradient of rotary_embedding_axes: what it keeps of the forward pass (GPU)."""
import numpy as np
import pytest
import torch

import dsa_triton_ascend_b200 as dsa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [list, np.array])
def test_gradient_keeps_its_sections(kind):
    """The backward pass turns by the sections that the forward pass had, though the caller's change since."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(5, 2, 32, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    d = torch.randn(5, 2, 32, generator=g, device="cuda", dtype=torch.bfloat16)
    table = dsa.rotary_table(64, 32)
    at = torch.randint(0, 64, (3, 5), generator=g, device="cuda", dtype=torch.int32)
    sections = kind([4, 6, 6])
    out = dsa.RotaryEmbeddingAxesFunction.apply(x, table, at, sections)
    sections[0], sections[1] = 6, 4
    out.backward(d)
    assert torch.equal(x.grad, dsa.rotary_embedding_axes(d, table, at, (4, 6, 6), inverse=True))
