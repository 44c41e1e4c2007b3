"""AdamW: its states' types, gradients and norms that are not finite, captures
replayed, and tensors that have moved."""
import pytest
import torch

import graphzero_b200 as gz
from test_adamw_gpu import gradients, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("default", [torch.bfloat16, torch.float16, torch.float64])
def test_states_do_not_follow_the_default_type(cuda, bits, default):
    """States, scales and norm are 32-bit floats (or the 8-bit ones) whatever type torch gives new tensors."""
    shapes = [(300, 3), (17,)]
    a, b, gs = make(shapes), make(shapes), gradients(shapes, 1)
    want = gz.AdamW(a, state_bits=bits, max_norm=0.01)
    torch.set_default_dtype(default)
    try:
        got = gz.AdamW(b, state_bits=bits, max_norm=0.01)
        for k in ("m", "v", "m_scale", "v_scale"):
            t, u = getattr(got, k), getattr(want, k)
            assert (t is None and u is None) or (t.dtype == u.dtype and t.shape == u.shape)
        norm = got.step(gs)
    finally:
        torch.set_default_dtype(torch.float32)
    assert norm.dtype == torch.float32 and torch.equal(norm, want.step(gs))
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(want.m.float(), got.m.float())
