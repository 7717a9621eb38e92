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
