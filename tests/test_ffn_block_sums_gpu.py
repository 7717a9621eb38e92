"""Sums over pixels in the gradients of gated_ffn and block_norm.

Equal terms: every rounding of a long chain of f32 sums then goes the same way."""
import pytest
import torch

from superresolution_amd import _lib, ops
from tests import ffn_block_ref as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16


@pytest.mark.parametrize("dt,h", [(F16, 1 << 15), (F32, 1 << 12)])
def test_hidden_bias_sums_of_equal_terms(dt, h):
    """2^25 (2^22) pixels, all 1.1, identities for weights, b_up = 1: every term of d_b_gate is 1.1, of d_b_up 1.1 * 1.1.  A tile's sum of 128
    pixels passes five levels of a tree and three sums of waves, the terms and the tiles' joint sum are rounded three times at most."""
    c, w = 16, 1024
    x = ops.Planes.wrap(torch.full((1, c // ops.cpb(dt), h, w, ops.cpb(dt)), 1.1, dtype=R.TORCH_DT[dt], device="cuda"))
    one = torch.eye(c, dtype=R.TORCH_DT[dt], device="cuda")
    got = ops.gated_ffn_backward(x, x, one, torch.zeros_like(one), one, b_gate=torch.zeros(c, device="cuda"), b_up=torch.ones(c, device="cuda"),
                                 act=_lib.ACT_NONE)
    term = float(x.buf.flatten()[0].double())
    for k, want in (("d_b_gate", term * h * w), ("d_b_up", term * term * h * w)):
        assert float((got[k].double() / want - 1).abs().max()) <= 11 * R.U, k
