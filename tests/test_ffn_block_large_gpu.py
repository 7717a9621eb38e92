"""block_norm and gated_ffn on tensors whose offsets pass 32 bits, and instances whose first call of all is captured.

Every pixel is computed by itself, so a tensor that repeats 60 rows of pixels 100 times has outputs that repeat bit for bit. The
first pixels are held to the 64-bit form (gated_ffn) or to a call on 60 rows alone (block_norm)."""
import pytest
import torch

from superresolution_amd import _lib, ops
from tests import ffn_block_ref as R
from tests.test_gated_ffn_gpu import NAMES, make, rows, weights, wide

pytestmark = pytest.mark.gpu
ROWS, TIMES, WIDTH, C = 60, 100, 6000, 64  # 36 million pixels x 128 bytes: 4.6 GB a tensor


def repeated(seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tile = (torch.randn((1, C // 16, ROWS, WIDTH, 16), generator=gen, device="cuda") * scale).to(torch.float16)
    return ops.Planes.wrap(tile.repeat(1, 1, TIMES, 1, 1))


def assert_repeats(p, what):
    t = p.buf.view(C // 16, TIMES, ROWS, WIDTH, 16)
    for i in range(1, TIMES):
        assert torch.equal(t[:, i], t[:, 0]), f"{what}: repetition {i}"


def first_pixels(p, count):
    """[count][c] doubles of the first pixels."""
    return p.buf[0, :, 0, :count].double().permute(1, 0, 2).reshape(count, C)


def test_gated_ffn_beyond_32_bit_offsets():
    s = make(31, 1, 1, 1, C, 16, _lib.F16)
    args, g = weights(s, _lib.F16), wide(s, _lib.F16)
    x = repeated(1)
    out = ops.gated_ffn(x, **args, act=_lib.ACT_SILU, res=x, res_scale=0.3)
    assert_repeats(out, "out")
    some = first_pixels(x, 500)
    ref = R.gated_ffn(some, *(g[k] for k in NAMES), _lib.ACT_SILU, some, 0.3)
    b = R.FfnBounds(some, *(g[k] for k in NAMES), _lib.ACT_SILU, 0.3, _lib.F16)
    R.assert_within(first_pixels(out, 500), ref, b.forward(ref, some), "out")
    del out
    dy = repeated(2, 0.1)
    got = ops.gated_ffn_backward(x, dy, **args, act=_lib.ACT_SILU, res_scale=0.3)
    assert_repeats(got["dx"], "dx")
    leaf = some.clone().requires_grad_()
    R.gated_ffn(leaf, *(g[k] for k in NAMES), _lib.ACT_SILU, None, 0.3).backward(first_pixels(dy, 500))
    grads = {"d_" + k: torch.zeros_like(g[k]) for k in NAMES}
    R.assert_within(first_pixels(got["dx"], 500), leaf.grad, b.backward(first_pixels(dy, 500), leaf.grad, grads)["dx"], "dx")
    assert all(bool(torch.isfinite(got["d_" + k]).all()) for k in NAMES)


def test_block_norm_beyond_32_bit_offsets():
    x, y = repeated(3), repeated(4)
    vec = lambda i: torch.linspace(0.5, 1.0 + i, C, device="cuda")  # noqa: E731
    post, pre, gate = (vec(0), vec(1)), (vec(2), vec(3)), vec(0.1)
    total, out = ops.block_norm(x, y, post=post, pre=pre, gate=gate, res_scale=0.5)
    assert_repeats(total, "sum")
    assert_repeats(out, "out")
    d_sum, d_out = repeated(5, 0.1), repeated(6, 0.1)
    got = ops.block_norm_backward(x, y, d_sum=d_sum, d_out=d_out, post=post, pre=pre, gate=gate, res_scale=0.5)
    assert_repeats(got["dx"], "dx")
    assert_repeats(got["dy"], "dy")
    # the same pixels by themselves
    few = [ops.Planes.wrap(p.buf[:, :, :ROWS].contiguous()) for p in (x, y, d_sum, d_out)]
    small, small_out = ops.block_norm(few[0], few[1], post=post, pre=pre, gate=gate, res_scale=0.5)
    assert torch.equal(small.buf, total.buf[:, :, :ROWS]) and torch.equal(small_out.buf, out.buf[:, :, :ROWS])
    part = ops.block_norm_backward(few[0], few[1], d_sum=few[2], d_out=few[3], post=post, pre=pre, gate=gate, res_scale=0.5)
    assert torch.equal(part["dx"].buf, got["dx"].buf[:, :, :ROWS]) and torch.equal(part["dy"].buf, got["dy"].buf[:, :, :ROWS])


@pytest.mark.parametrize("dt,c,hidden", [(_lib.F32, 88, 56), (_lib.BF16, 240, 144), (_lib.F32, 176, 40)])
def test_the_first_call_of_an_instance_may_be_captured(dt, c, hidden):
    """Nothing else uses these types, channels and this activation: whatever a first call sets up has to be allowed in a capture."""
    s = make(c, 1, 9, 11, c, hidden, dt)
    x, dy = (ops.Planes.from_nchw(R.to_nchw(s[k], 9, 11).float(), dt) for k in ("x", "d_out"))
    args = weights(s, dt)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.gated_ffn(x, **args, act=_lib.ACT_LRELU, res_scale=0.3)
        got = ops.gated_ffn_backward(x, dy, **args, act=_lib.ACT_LRELU, res_scale=0.3)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.buf, ops.gated_ffn(x, **args, act=_lib.ACT_LRELU, res_scale=0.3).buf)
        for k, v in ops.gated_ffn_backward(x, dy, **args, act=_lib.ACT_LRELU, res_scale=0.3).items():
            assert torch.equal(v.buf, got[k].buf) if k == "dx" else torch.equal(v, got[k]), k
    ref = R.gated_ffn(rows(s["x"]), *(s[k] for k in NAMES), _lib.ACT_LRELU, None, 0.3)
    b = R.FfnBounds(rows(s["x"]), *(s[k] for k in NAMES), _lib.ACT_LRELU, 0.3, dt)
    R.assert_within(rows(R.from_nchw(out.to_nchw().cpu())), ref, b.forward(ref), "out")
