"""The GELU of gated_ffn and its slope, one value at a time, relative to their own size.

With identities for w_gate and w_down, no w_up and b_up = 1 the block's output is gelu(x) itself (every sum has one term that is not
zero) and, for d_out = 1, dx is the slope.

Bounds, U = 2^-24.  f32: with x = |a|, the reciprocal and exp2 err by 2 U each, 1 + k x by U, the fitted polynomials by less than U with
their evaluation's 3 U, the products and the last sum by U each; Q moves by at most 1.7 times a relative error of t, so 1.7 * 3 + 2 + 4 + 4 = 16 U
of |gelu(a)| (for a > 0 of a smaller part of it).  The slope is a sum of Phi and a phi, each with that error.  Half types: log2 Q is a
polynomial fitted to 1.2e-5 of Q for |a| <= 4 and 4.5e-4 beyond; its evaluation errs by about 3 roundings of its terms, whose magnitudes sum
to 26 at 4 and 300 at 9.5, so by 26 * 3 U = 5e-6 and 300 * 3 U = 5e-5: 2^-15 and 2^-11 in all; then one rounding to the type."""
import math

import pytest
import torch

from superresolution_amd import _lib, ops
from tests import ffn_block_ref as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16
DEEPEST = {F32: 12.0, F16: 9.5, BF16: 9.5}


def arguments(dt, count):
    """Arguments of both signs from 1e-6 (half types: 1e-4) to 4 and on to -DEEPEST and 30, as doubles the type holds."""
    size = torch.logspace(-6 if dt == F32 else -4, math.log10(4.0), count // 4, dtype=torch.float64)
    rest = count - 2 * size.numel() - 2
    a = torch.cat([size, -size, torch.linspace(-DEEPEST[dt], 30.0, rest, dtype=torch.float64), torch.tensor([0.0, -0.0], dtype=torch.float64)])
    return R.rounded(a, dt)


def block(dt, c):
    one = torch.eye(c, dtype=R.TORCH_DT[dt], device="cuda")
    return dict(w_gate=one, w_up=torch.zeros_like(one), w_down=one, b_up=torch.ones(c, device="cuda"), act=_lib.ACT_GELU)


def relative(dt, a):
    if dt == F32:
        return torch.full_like(a, 16 * R.U)
    return torch.where(a.abs() <= 4.0, 2.0 ** -15, 2.0 ** -11)


def planes(v, dt, c):  # [pixels * c] values -> one image of one row
    return ops.Planes.from_nchw(v.reshape(1, -1, 1, c).permute(0, 3, 2, 1).float().contiguous(), dt)


def values(p):
    return p.to_nchw().cpu().double().permute(0, 3, 2, 1).reshape(-1)


def phi(a):
    return 0.5 * torch.special.erfc(-a * math.sqrt(0.5)), torch.exp(-0.5 * a * a) / math.sqrt(2.0 * math.pi)


# 16 channels: the form with hidden values in registers; 400 (f32: 136): the tile form
@pytest.mark.parametrize("dt,c", [(F32, 16), (F32, 136), (F16, 16), (F16, 400), (BF16, 16), (BF16, 400)])
def test_value_and_slope(dt, c):
    a = arguments(dt, 200 * c)
    x = planes(a, dt, c)
    big, small = phi(a)
    gelu = a * big
    bound = relative(dt, a) * gelu.abs()
    R.assert_within(values(ops.gated_ffn(x, **block(dt, c))), gelu, bound + R.rounding(dt, gelu.abs() + bound), "gelu")
    ones = ops.Planes.wrap(torch.ones_like(x.buf))
    got = ops.gated_ffn_backward(x, ones, **block(dt, c))
    bound = relative(dt, a) * (big + a.abs() * small)
    R.assert_within(values(got["dx"]), big + a * small, bound + R.rounding(dt, (big + a * small).abs() + bound), "slope")


@pytest.mark.parametrize("dt,c", [(F32, 16), (F32, 136), (F16, 16), (BF16, 208)])
def test_hidden_values_of_the_backward_pass(dt, c):
    """One pixel and d_out = 1: every row of w_down's gradient is the hidden values, gelu(x)."""
    a = arguments(dt, 200 * c).reshape(-1, c)
    for row in a[:: max(1, a.shape[0] // 8)]:
        x = planes(row, dt, c)
        got = ops.gated_ffn_backward(x, ops.Planes.wrap(torch.ones_like(x.buf)), **block(dt, c))["d_w_down"].cpu().double()
        gelu = row * phi(row)[0]
        bound = relative(dt, row) * gelu.abs()
        R.assert_within(got, gelu.expand(c, c), (bound + R.rounding(dt, gelu.abs() + bound)).expand(c, c), "hidden")


@pytest.mark.parametrize("scale", [1.0, 0.1, 0.01, 0.001])
def test_f32_of_small_arguments(scale):
    """Gates of one size: outputs and slopes in f32 relative to their 2-norm.  Each errs by 16 U of itself at most (the slope of its two
    terms, 1.3 times itself here), so the norm does too."""
    gen = torch.Generator().manual_seed(5)
    a = R.rounded(R.rnd(gen, 4096 * 16, scale=scale), F32)
    x = planes(a, F32, 16)
    big, small = phi(a)
    got = ops.gated_ffn_backward(x, ops.Planes.wrap(torch.ones_like(x.buf)), **block(F32, 16))
    for have, want in ((ops.gated_ffn(x, **block(F32, 16)), a * big), (got["dx"], big + a * small)):
        assert float((values(have) - want).norm() / want.norm()) <= 1.3 * 16 * R.U


@pytest.mark.parametrize("dt,c", [(F32, 16), (F32, 136), (F16, 16), (BF16, 400)])
def test_limits(dt, c):
    """At +infinity the value is infinite (f16: 65504) and the slope 1, at -infinity both are 0, and NaN stays NaN.  The half types take |a|
    beyond 11 as 11, so their values there end at -11 Phi(-11) = -11 * 1.91e-28 = -2.1e-27 (a zero in f16).  Arguments come in as b_gate; rows of w_down's gradient are the hidden values, b_gate's gradient the slopes (one pixel, x = 0, every column of w_down holds one 1)."""
    special = torch.tensor([float("inf"), -float("inf"), float("nan"), 1e30, -1e30, 60.0, -60.0, 0.0])
    x = ops.Planes(1, c, 1, 1, dt)
    x.buf.fill_(0.0)
    args = dict(block(dt, c), b_gate=special.repeat(c // 8).cuda())
    got = ops.gated_ffn_backward(x, ops.Planes.wrap(torch.ones_like(x.buf)), **args)
    top = 65504.0 if dt == F16 else float("inf")
    want = torch.tensor([top, 0.0, float("nan"), min(top, 1e30), 0.0, 60.0, 0.0, 0.0]).to(R.TORCH_DT[dt]).repeat(c // 8)
    slope = torch.tensor([1.0, 0.0, float("nan"), 1.0, 0.0, 1.0, 0.0, 0.5]).repeat(c // 8)
    for row in got["d_w_down"].cpu():
        row, none = row.double().nan_to_num(nan=-1.0), want == 0
        assert torch.equal(row[~none], want.double().nan_to_num(nan=-1.0)[~none]) and float(row[none].abs().max()) <= (2.2e-27 if dt == BF16 else 0.0)
    have = got["d_b_gate"].cpu()
    assert torch.equal(have.isnan(), slope.isnan()) and float((have - slope).nan_to_num(nan=0.0).abs().max()) <= 2.0 ** -20
