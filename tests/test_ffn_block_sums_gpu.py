"""Sums over pixels in the gradients of gated_ffn and block_norm.

Exact ones: inputs of +-1 and small powers of two, of which every product and every partial sum is held exactly in f32 and the types used, so
that results have to be EQUAL to those in 64 bits, in whatever order they are summed.  The gradient of the output is +-1 in one channel of every
pixel, so one pixel left out, taken twice or taken from elsewhere moves a sum by a whole step.

Equal terms: every rounding of a long chain of f32 sums then goes the same way."""
import ctypes as C

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


# ---- exact sums: gated_ffn -----------------------------------------------------------------------------------------------
def signs(gen, *shape):
    return torch.empty(shape, dtype=torch.float16, device="cuda").bernoulli_(0.5, generator=gen).mul_(2).sub_(1)


def one_channel(gen, m, c):
    """[m][c]: +-1 in one channel of every row, the channels in turn."""
    d = torch.zeros((m, c), dtype=torch.float16, device="cuda")
    at = torch.arange(m, device="cuda")
    d[at, (at * 7 + at // c) % c] = signs(gen, m)
    return d


def selections(gen, hidden, c):
    """[hidden][c]: +-1 in one channel of every row."""
    w = torch.zeros((hidden, c), dtype=torch.float64, device="cuda")
    w[torch.arange(hidden, device="cuda"), torch.randint(0, c, (hidden,), generator=gen, device="cuda")] = signs(gen, hidden).double()
    return w


def as_planes(v, dt, n, h, w):
    """[n * h * w][c] -> plane tensor."""
    cpb = ops.cpb(dt)
    return ops.Planes.wrap(v.to(R.TORCH_DT[dt]).reshape(n, h, w, -1, cpb).permute(0, 3, 1, 2, 4).contiguous())


def as_rows(p):
    n, k, h, w, cpb = p.buf.shape
    return p.buf.permute(0, 2, 3, 1, 4).reshape(n * h * w, k * cpb)


def ffn_reference(x, dy, wg, wu, wd, scale):
    """Without activation: out, dx and the sums over these rows, in 64 bits."""
    x, dy = x.double(), dy.double()
    g, u, dh = x @ wg.t(), x @ wu.t(), scale * (dy @ wd)
    dg, du = dh * u, dh * g
    return (scale * ((g * u) @ wd.t()), dg @ wg + du @ wu,
            {"d_w_gate": dg.t() @ x, "d_w_up": du.t() @ x, "d_w_down": scale * (dy.t() @ (g * u)), "d_b_gate": dg.sum(0), "d_b_up": du.sum(0), "d_b_down": scale * dy.sum(0)})


def ffn_exact(dt, n, h, w, c, hidden, chunk=1 << 20):
    gen = torch.Generator(device="cuda").manual_seed(c * hidden)
    m = n * h * w
    wg, wu, wd = selections(gen, hidden, c), selections(gen, hidden, c), selections(gen, hidden, c).t().contiguous()
    x, dy = as_planes(signs(gen, m, c), dt, n, h, w), as_planes(one_channel(gen, m, c), dt, n, h, w)
    args = {k: v.to(R.TORCH_DT[dt]) for k, v in (("w_gate", wg), ("w_up", wu), ("w_down", wd))}
    args.update(b_gate=torch.zeros(hidden, device="cuda"), b_up=torch.zeros(hidden, device="cuda"), b_down=torch.zeros(c, device="cuda"))
    out = ops.gated_ffn(x, **args, act=_lib.ACT_NONE, res_scale=0.5)
    got = ops.gated_ffn_backward(x, dy, **args, act=_lib.ACT_NONE, res_scale=0.5)
    sums = {}
    # images, rows of pixels: whole ones per part
    per = max(1, chunk // w)
    for i in range(n):
        for r in range(0, h, per):
            part = [as_rows(ops.Planes.wrap(p.buf[i:i + 1, :, r:r + per].contiguous())) for p in (x, dy, out, got["dx"])]
            o, dx, s = ffn_reference(part[0], part[1], wg, wu, wd, 0.5)
            assert torch.equal(part[2].double(), o), f"out, image {i}, rows from {r}"
            assert torch.equal(part[3].double(), dx), f"dx, image {i}, rows from {r}"
            sums = {k: v + sums.get(k, 0.0) for k, v in s.items()}
    for k, v in sums.items():
        assert torch.equal(got[k], v.to(got[k].dtype)), f"{k}: {int((got[k].double() != v.to(got[k].dtype).double()).sum())} of {v.numel()} differ"


# every number of planes that has a form of its own, several splits and steps of the pixels, ragged last ones, images that end inside a step
@pytest.mark.parametrize("dt,n,h,w,c,hidden", [(F16, 3, 97, 103, 64, 256), (BF16, 7, 61, 37, 176, 464), (F16, 1, 187, 190, 256, 272), (BF16, 2, 130, 131, 192, 96),
                                               (F32, 2, 101, 97, 64, 64), (F16, 1, 1, 40003, 16, 48), (F16, 2, 150, 150, 32, 112), (BF16, 1, 200, 301, 128, 320),
                                               (F32, 1, 90, 91, 8, 40), (F32, 3, 61, 67, 120, 136), (F16, 1, 120, 121, 320, 144), (F32, 1, 111, 113, 160, 200),
                                               (F16, 5000, 1, 3, 48, 80), (BF16, 1, 9, 100, 512, 1040), (F16, 1, 300, 401, 96, 64)])
def test_exact_ffn(dt, n, h, w, c, hidden):
    ffn_exact(dt, n, h, w, c, hidden)


@pytest.mark.parametrize("dt,c,hidden,h,w", [(F32, 8, 16384, 150, 160), (F16, 272, 16384, 260, 271), (F32, 8, 16384, 261, 270)])
def test_exact_ffn_in_several_runs_of_pixels(dt, c, hidden, h, w):
    ffn_exact(dt, 1, h, w, c, hidden, chunk=4000)


def test_exact_ffn_beyond_32_bit_offsets():
    """36 million pixels of 64 channels in f16: 4.6 GB a tensor."""
    ffn_exact(F16, 1, 6000, 6000, 64, 16)


# ---- exact sums: block_norm ------------------------------------------------------------------------------------------------
def norm_inputs(dt, xt, n, h, w, c, gate, kind):
    """y and the sum have normalised values t = +-1 (half of a pixel's channels each): y = t, post = (1, 0.5), x = 2 t - k (t + 0.5)
    with k = res_scale * gate = 0.5 or 1, so that the sum is 2 t."""
    gen = torch.Generator(device="cuda").manual_seed(n * h + c)
    m = n * h * w
    half = signs(gen, m, c // 2)
    t = torch.cat([half, -half], 1).float()
    k = torch.empty((n, c) if gate == "image" else (c,), device="cuda").bernoulli_(0.5, generator=gen).mul_(0.5).add_(0.5)
    rows = k.repeat_interleave(h * w, 0) if gate == "image" else k
    x = 2 * t - rows * (t + 0.5)
    d_out, d_sum = one_channel(gen, m, c).float(), one_channel(gen, m, c).flip(1).float()
    vec = lambda v: torch.full((c,), v, device="cuda")  # noqa: E731
    args = dict(post=(vec(1.0), vec(0.5)), pre=(vec(2.0), vec(0.0)), gate=k * 2.0, res_scale=0.5, eps=0.0, kind=kind)
    tensors = {"x": as_planes(x, xt, n, h, w), "y": as_planes(t, dt, n, h, w), "d_sum": as_planes(d_sum, xt, n, h, w), "d_out": as_planes(d_out, dt, n, h, w)}
    return tensors, args, (t, rows, d_sum, d_out)


def norm_reference(t, k, d_sum, d_out, kind, images):
    """(dx, dy, sums) in 64 bits; images: rows of an image (a gate of its own each) or None."""
    t, k, d_sum, d_out = (v.double() for v in (t, k, d_sum, d_out))

    def through(d, r):  # the gradient of normalised values t = hat
        d = d - t * (d * t).mean(1, keepdim=True)
        return r * (d - d.mean(1, keepdim=True) if kind == _lib.NORM_LAYER else d)

    ds = d_sum + through(2.0 * d_out, 0.5)
    dv = k * ds
    gate = 0.5 * ds * (t + 0.5)
    gate = gate.sum(0) if images is None else gate.reshape(-1, images, t.shape[1]).sum(1)
    return ds, through(dv, 1.0), {"d_post_weight": (dv * t).sum(0), "d_post_bias": dv.sum(0), "d_pre_weight": (d_out * t).sum(0), "d_pre_bias": d_out.sum(0), "d_gate": gate}


NORM_SIZES = [(F16, F16, 3, 61, 67, 64, "image"), (BF16, F32, 3, 61, 67, 16, "image"), (F16, F32, 2, 150, 151, 256, "shared"), (F32, F32, 1, 200, 201, 64, "shared"),
              (BF16, BF16, 1100, 1, 3, 16, "image"), (F32, F32, 900, 2, 2, 32, "image"), (F16, F16, 1, 300, 301, 128, "image"), (BF16, BF16, 2, 40, 41, 1024, "shared"),
              (F32, F32, 2, 83, 89, 8, "image"), (F16, F32, 5, 30, 31, 512, "image")]


@pytest.mark.parametrize("kind", [_lib.NORM_LAYER, _lib.NORM_RMS])
@pytest.mark.parametrize("dt,xt,n,h,w,c,gate", NORM_SIZES)
def test_exact_norm(dt, xt, n, h, w, c, gate, kind):
    s, args, parts = norm_inputs(dt, xt, n, h, w, c, gate, kind)
    total, out = ops.block_norm(s["x"], s["y"], **args)
    assert torch.equal(as_rows(total).double(), 2.0 * parts[0].double()) and torch.equal(as_rows(out).double(), 2.0 * parts[0].double())
    got = ops.block_norm_backward(**s, **args)
    dx, dy, sums = norm_reference(*parts, kind, h * w if gate == "image" else None)
    assert torch.equal(as_rows(got["dx"]), dx.to(R.TORCH_DT[xt])) and torch.equal(as_rows(got["dy"]), dy.to(R.TORCH_DT[dt]))
    for k, v in sums.items():
        assert torch.equal(got[k].double(), v), f"{k}: {int((got[k].double() != v).sum())} of {v.numel()} differ"


def test_exact_norm_beyond_32_bit_offsets():
    """36 million pixels of 64 channels in f16, 4.6 GB a tensor: the sums over all of them."""
    s, args, parts = norm_inputs(F16, F16, 1, 600, 6000, 64, "shared", _lib.NORM_LAYER)
    _, _, sums = norm_reference(*parts, _lib.NORM_LAYER, None)
    del parts
    got = ops.block_norm_backward(**{k: ops.Planes.wrap(p.buf.repeat(1, 1, 10, 1, 1)) for k, p in s.items()}, **args)
    for k, v in sums.items():
        assert torch.equal(got[k].double(), 10.0 * v), k


# ---- in place --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("alias", [("d_sum", "y"), ("d_sum", "d_out"), ("d_sum", None), (None, "y"), (None, "d_out")], ids=str)
@pytest.mark.parametrize("dt,xt,n,h,w,c,gate", [(F16, F16, 3, 61, 67, 64, "image"), (BF16, F32, 2, 83, 89, 176, "shared"), (F32, F32, 1, 47, 51, 8, "image"),
                                                (F16, F32, 1, 40, 41, 1024, "shared"), (F16, F16, 900, 1, 3, 48, "image")])
def test_norm_backward_in_place(dt, xt, n, h, w, c, gate, alias):
    """dx written over d_sum, dy over y or d_out: several workgroups, a ragged last step; the bits of a call with places of their own."""
    s, args, _ = norm_inputs(dt, xt, n, h, w, c, gate, _lib.NORM_LAYER)
    want = ops.block_norm_backward(**s, **args)
    d = _lib.BlockNormGradDesc()
    d.n, d.h, d.w, d.c, d.kind, d.gate_per_image, d.eps, d.res_scale = n, h, w, c, _lib.NORM_LAYER, gate == "image", 0.0, 0.5
    dx, dy = (s[alias[0]] if alias[0] else s["x"].new()), (s[alias[1]] if alias[1] else s["y"].new())
    for k, p in dict(s, dx=dx, dy=dy).items():
        setattr(d, k, p.view())
    vectors = dict(post_weight=args["post"][0], post_bias=args["post"][1], pre_weight=args["pre"][0], pre_bias=args["pre"][1], gate=args["gate"])
    grads = {"d_" + k: torch.empty_like(v) for k, v in vectors.items()}
    for k, v in {**vectors, **grads}.items():
        setattr(d, k, v.data_ptr())
    need = _lib.lib().srmi_block_norm_backward_workspace(C.byref(d))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib().srmi_block_norm_backward(C.byref(d), ws.data_ptr(), need, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(dx.buf, want["dx"].buf) and torch.equal(dy.buf, want["dy"].buf)
    for k, v in grads.items():
        assert torch.equal(v, want[k]), k


@pytest.mark.parametrize("dt", [F32, F16])
def test_norm_without_a_body_returns_its_input(dt):
    x = ops.Planes(2, 32, 5, 7, dt)
    x.buf.fill_(1.0)
    total, _ = ops.block_norm(x, pre=(torch.ones(32, device="cuda"), None))
    assert total.buf.data_ptr() == x.buf.data_ptr()
