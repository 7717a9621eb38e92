"""Infinities in gated_ffn's inputs and weights give what the formula gives: tiles that the hidden units, channels or pixels do not fill add
nothing (0 * infinity would be NaN).  All inputs are positive, so that no sum holds infinities of both signs."""
import pytest
import torch

from superresolution_amd import _lib, ops
from tests import ffn_block_ref as R
from tests.test_gated_ffn_gpu import NAMES, back, gradients, make, planes, rows, weights

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16
# c and hidden: tiles of 32 hidden units and four planes filled and not, in every form of the forward and backward pass
SIZES = [(F16, 48, 48), (BF16, 16, 80), (BF16, 64, 64), (F16, 208, 112), (BF16, 272, 48), (F32, 24, 40), (F32, 8, 8), (F32, 112, 72), (F32, 136, 56)]


def positive(s):
    return {k: v.abs() if isinstance(v, torch.Tensor) else v for k, v in s.items()}


def as_it_is(v, s, dt):
    """A plane tensor of the values by plain copies (the library's conversion to f16 stores an infinity as 65504)."""
    n, m, c = v.shape
    cpb = ops.cpb(dt)
    return ops.Planes.wrap(v.to(R.TORCH_DT[dt]).reshape(n, s["h"], s["w"], c // cpb, cpb).permute(0, 3, 1, 2, 4).contiguous().cuda())


def run_backward(s, dt):
    return ops.gated_ffn_backward(as_it_is(s["x"], s, dt), planes(s["d_out"], s, dt), **weights(s, dt), act=_lib.ACT_RELU, res_scale=0.5)


def alike(got, ref, dt, what):
    """Infinities and finite values in the same places, NaN nowhere.  (f16 stores hold +-65504 instead, also of the hidden values, which small
    factors bring back into the range: there only NaN is looked for.)"""
    got, ref = got.double(), ref.double()
    assert not bool(torch.isnan(ref).any()) and not bool(torch.isnan(got).any()), f"{what}: NaN"
    if dt != F16 or what.startswith("d_b"):
        assert torch.equal(got == float("inf"), ref == float("inf")), f"{what}: infinite elsewhere than by the formula"


@pytest.mark.parametrize("dt,c,hidden", SIZES)
def test_an_infinite_input(dt, c, hidden):
    s = positive(make(c + hidden, 1, 7, 11, c, hidden, dt))
    s["x"][0, 40, c // 2] = float("inf")
    ref = R.gated_ffn(rows(s["x"]), *(s[k] for k in NAMES), _lib.ACT_RELU, rows(s["res"]), 0.5)
    got = ops.gated_ffn(as_it_is(s["x"], s, dt), **weights(s, dt), act=_lib.ACT_RELU, res=planes(s["res"], s, dt), res_scale=0.5)
    have = back(got)
    assert bool((ref[40] == float("inf")).all())
    alike(have, ref, dt, "out")
    ref, got = gradients(s, _lib.ACT_RELU, 0.5), run_backward(s, dt)
    for k, v in ref.items():
        alike(back(got[k]) if k == "dx" else got[k].cpu(), v, dt, k)


@pytest.mark.parametrize("dt,c,hidden", SIZES)
def test_an_infinite_weight(dt, c, hidden):
    """77 pixels fill no workgroup: the lanes without one take no part in the sums over pixels."""
    s = positive(make(c + hidden, 1, 7, 11, c, hidden, dt))
    s["w_up"][hidden // 2, c // 2] = float("inf")
    got, ref = run_backward(s, dt), gradients(s, _lib.ACT_RELU, 0.5)
    assert bool((ref["d_b_gate"][hidden // 2] == float("inf")).all())
    for k, v in ref.items():
        alike(back(got[k]) if k == "dx" else got[k].cpu(), v, dt, k)
