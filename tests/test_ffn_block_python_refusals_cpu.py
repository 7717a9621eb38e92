"""What the Python surface of block_norm and gated_ffn refuses by itself, beyond shapes and types (tests/test_ffn_block_refusals_cpu.py)."""
import pytest
import torch

from superresolution_amd import _lib, ops

F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16


def test_a_type_for_out_that_y_contradicts():
    """out has the type of y; another one asked for is an error, not a tensor of y's type without a word."""
    x, y = ops.Planes(1, 32, 4, 4, F32, device="cpu"), ops.Planes(1, 32, 4, 4, F16, device="cpu")
    one = torch.ones(32)
    for wrong in (F32, BF16):
        with pytest.raises(_lib.SrmiError, match="type of y"):
            ops.block_norm(x, y, pre=(one, None), out_dtype=wrong)
    with pytest.raises(_lib.SrmiError, match="on a GPU"):
        ops.block_norm(x, y, pre=(one, None), out_dtype=F16)


def calls():
    x, one = ops.Planes(1, 32, 4, 4, F16, device="cpu"), torch.ones(32)
    y, res = (ops.Planes(1, 32, 4, 4, F16, device="cpu") for _ in range(2))
    w = {k: torch.zeros(48, 32, dtype=torch.float16) for k in ("w_gate", "w_up")}
    w["w_down"], w["b_gate"] = torch.zeros(32, 48, dtype=torch.float16), torch.zeros(48)
    gate, weight = torch.ones(1, 32), torch.ones(32)
    norm = dict(post=(weight, None), pre=(one, None), gate=gate)
    return [(ops.block_norm, (x, y), norm, [x.buf, y.buf, gate, weight]), (ops.block_norm_backward, (x, y), dict(norm, d_sum=res), [x.buf, y.buf, res.buf, gate, weight]),
            (ops.gated_ffn, (x,), dict(w, res=res), [x.buf, res.buf, w["w_up"], w["b_gate"]]), (ops.gated_ffn_backward, (x, y), w, [x.buf, y.buf, w["w_down"], w["b_gate"]])]


@pytest.mark.parametrize("i", range(4))
def test_a_tensor_that_requires_a_gradient(i):
    """Without a word the outputs would be detached and the gradient lost.  Under no_grad, as in an autograd.Function, the call goes on (here
    to the refusal of tensors that are not on a GPU)."""
    call, args, kw, tensors = calls()[i]
    for t in tensors:
        t.requires_grad_()
        with pytest.raises(_lib.SrmiError, match="requires a gradient"):
            call(*args, **kw)
        with torch.no_grad(), pytest.raises(_lib.SrmiError, match="on a GPU"):
            call(*args, **kw)
        t.requires_grad_(False)
    with pytest.raises(_lib.SrmiError, match="on a GPU"):
        call(*args, **kw)
