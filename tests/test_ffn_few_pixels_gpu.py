"""gated_ffn on few pixels and without a residual in the half types: up to one workgroup's pixels (128, from 208 channels on 256) the hidden values' rounding is carried along, so that outputs
are off by little more than their own rounding.

Bound: FfnBounds' for f32 hidden values (ffn_block_ref), their two halves' relative error of half_step^2 (f16 below the smallest
normal number: 2^-25 absolutely), twice as many additions, and one rounding of the output.  One rounding of the hidden values alone moves
outputs by about 0.6 half steps on top (512 errors of up to a half step, with random signs), over this bound for many."""
import pytest
import torch

from superresolution_amd import _lib, ops
from tests import ffn_block_ref as R
from tests.test_gated_ffn_gpu import F16, BF16, NAMES, back, bounds, make, planes, rows, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [_lib.ACT_SILU, _lib.ACT_GELU, _lib.ACT_NONE])
@pytest.mark.parametrize("dt,n,h,w,c,hidden", [(F16, 1, 1, 1, 256, 512), (BF16, 1, 1, 1, 16, 64), (BF16, 2, 5, 11, 64, 128), (F16, 1, 9, 14, 32, 96), (F16, 1, 3, 5, 48, 32), (BF16, 3, 1, 1, 192, 112),
                                               (F16, 1, 12, 20, 240, 80)])
def test_the_hidden_values_rounding_does_not_show(dt, n, h, w, c, hidden, act):
    s = make(c + hidden + act, n, h, w, c, hidden, dt, res=False)
    got = back(ops.gated_ffn(planes(s["x"], s, dt), **weights(s, dt), act=act))
    ref = R.gated_ffn(rows(s["x"]), *(s[k] for k in NAMES), act, None, 1.0)
    b = bounds(s, dt, act, 1.0)
    wd = s["w_down"].abs()
    hid = b.eh_f32 + 2 * R.half_step(dt) ** 2 * b.hid.abs() + R.half_step(dt) * torch.finfo(R.TORCH_DT[dt]).tiny
    e = hid @ wd.t() + (2 * hidden + 4) * R.U * (b.hid.abs() @ wd.t() + s["b_down"].abs())
    R.assert_within(got, ref, e + R.rounding(dt, ref.abs() + e), "out")


def test_saturated_hidden_values_stay_so():
    """Hidden values of 2^20 count as 65504 and infinite ones too, nothing is left over for the second half (64 hidden units: two parts)."""
    c, hidden = 16, 64
    x = ops.Planes(1, c, 2, 2, F16)
    x.buf.fill_(0.0)
    x.buf[..., 0] = 1024.0
    gate = torch.zeros(hidden, c, dtype=torch.float16, device="cuda")
    gate[0, 0] = gate[40, 0] = 1.0
    gate[41, 0] = float("inf")
    down = torch.zeros(c, hidden, dtype=torch.float16, device="cuda")
    down[0, 0] = down[1, 40] = 0.5
    down[2, 41] = 0.25
    up = torch.ones_like(gate)
    out = ops.gated_ffn(x, gate, up, down, act=_lib.ACT_NONE).buf[0, 0, 0, 0].cpu()
    assert out[:4].tolist() == [32752.0, 32752.0, 16376.0, 0.0]
