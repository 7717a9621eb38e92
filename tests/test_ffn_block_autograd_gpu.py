"""The feed-forward block inside an autograd.Function of the caller's own, as the integration guide shows it, and under no_grad with
parameters."""
import pytest
import torch

from superresolution_amd import _lib, ops
from tests.test_gated_ffn_gpu import F16, make, planes, weights

pytestmark = pytest.mark.gpu


class Ffn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, *w):
        ctx.save_for_backward(x, *w)
        return ops.gated_ffn(ops.Planes.wrap(x), *w).buf

    @staticmethod
    def backward(ctx, dy):
        x, *w = ctx.saved_tensors
        g = ops.gated_ffn_backward(ops.Planes.wrap(x), ops.Planes.wrap(dy.contiguous()), *w)
        return g["dx"].buf, g["d_w_gate"], g["d_w_up"], g["d_w_down"]


def test_inside_an_autograd_function():
    s = make(21, 2, 9, 11, 48, 80, F16, bias=False, res=False)
    x, dy = planes(s["x"], s, F16), planes(s["d_out"], s, F16)
    w = [weights(s, F16)[k] for k in ("w_gate", "w_up", "w_down")]
    want = ops.gated_ffn_backward(x, dy, *w)
    leaves = [t.clone().requires_grad_() for t in (x.buf, *w)]
    with pytest.raises(_lib.SrmiError, match="requires a gradient"):
        ops.gated_ffn(ops.Planes.wrap(leaves[0]), *leaves[1:])
    out = Ffn.apply(*leaves)
    assert torch.equal(out, ops.gated_ffn(x, *w).buf)
    out.backward(dy.buf)
    for leaf, grad in zip(leaves, (want["dx"].buf, want["d_w_gate"], want["d_w_up"], want["d_w_down"])):
        assert torch.equal(leaf.grad, grad)
    with torch.no_grad():
        assert torch.equal(ops.gated_ffn(ops.Planes.wrap(leaves[0]), *leaves[1:]).buf, out)
