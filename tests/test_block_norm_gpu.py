"""block_norm and block_norm_backward against 64-bit plain forms.

Bounds.  A lane adds at most 32 values and joins at most 6 times, so a mean over the channels errs by at most 40 * 2^-24 of the
mean magnitude; a centred value then by 64 * 2^-24 * max|v|, its normalised form by r * 64 * 2^-24 * max|v| + 64 * 2^-24 * |hat|
with r = 1 / std.  With A = r * max|v| (how far the values lie from zero in units of their spread) a norm's output errs
by at most 2^-17 * (A + 1) * max|weight| per norm, a second norm behind the first scales the first one's error by its own
r * res_scale * gate (counted in A of the sum), and every store adds half a step of the stored value.  Sums over m pixels add (m +
64) * 2^-24 of the sum of magnitudes."""
import ctypes as C

import pytest
import torch

from superresolution_amd import _lib, ops
from tests import ffn_block_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-5

F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16
TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]  # (block, trunk)


def make(seed, n, h, w, c, dt, xt, *, post=True, pre=True, gate="image", bias=True, y=True, offset=1.0):
    gen = torch.Generator().manual_seed(seed)
    s = {"n": n, "h": h, "w": w, "c": c}
    m = h * w
    s["x"] = R.rounded(R.rnd(gen, n, m, c, scale=1.5) + offset * R.rnd(gen, c), xt)
    s["y"] = R.rounded(R.rnd(gen, n, m, c) + offset * R.rnd(gen, c), dt) if y else None
    vec = lambda mean, scale: (mean + R.rnd(gen, c, scale=scale)).float().double()  # noqa: E731
    s["post"] = (vec(1.0, 0.2), vec(0.0, 0.2) if bias else None) if post and y else None
    s["pre"] = (vec(1.0, 0.2), vec(0.0, 0.2) if bias else None) if pre else None
    shape = {"image": (n, c), "shared": (c,), None: None}[gate if y else None]
    s["gate"] = None if shape is None else torch.sigmoid(R.rnd(gen, *shape)).float().double()
    s["d_sum"] = R.rounded(R.rnd(gen, n, m, c, scale=0.1), xt)
    s["d_out"] = R.rounded(R.rnd(gen, n, m, c, scale=0.1), dt) if pre else None
    return s


def planes(v, s, dt):
    return None if v is None else ops.Planes.from_nchw(R.to_nchw(v, s["h"], s["w"]).float(), dt)


def dev(v):
    return None if v is None else v.float().cuda()


def pair(p):
    return None if p is None else (dev(p[0]), dev(p[1]))


def back(p):
    return R.from_nchw(p.to_nchw().cpu())


def spread(v, kind):
    """r * max|v| of the rows (how much a relative error of a value is enlarged by its norm)."""
    z = v - v.mean(-1, keepdim=True) if kind == _lib.NORM_LAYER else v
    r = 1.0 / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS)
    return r * v.abs().amax(-1, keepdim=True), r


def forward(s, dt, xt, kind, res_scale):
    return ops.block_norm(planes(s["x"], s, xt), planes(s["y"], s, dt), post=pair(s["post"]), pre=pair(s["pre"]), gate=dev(s["gate"]),
                          res_scale=res_scale, eps=EPS, kind=kind, out_dtype=dt)


def check_forward(s, dt, xt, kind, res_scale, got=None):
    total, out = forward(s, dt, xt, kind, res_scale) if got is None else got
    t_ref, o_ref = R.block_norm(s["x"], s["y"], s["post"], s["pre"], s["gate"], res_scale, EPS, kind)
    e_sum = 4 * R.U * s["x"].abs()
    if s["y"] is not None:
        w = s["post"][0].abs().max() if s["post"] else 1.0
        a = spread(s["y"], kind)[0] + 1 if s["post"] else s["y"].abs()
        e_sum = e_sum + 2.0 ** -17 * abs(res_scale) * (a * w + (s["post"][1].abs().max() if s["post"] and s["post"][1] is not None else 0.0))
        R.assert_within(back(total), t_ref, e_sum + R.rounding(xt, t_ref.abs() + e_sum), "sum")
    else:
        assert total.buf.data_ptr()
    if s["pre"] is not None:
        a, r = spread(t_ref, kind)
        hat = ((o_ref - (s["pre"][1] if s["pre"][1] is not None else 0.0)) / s["pre"][0]).abs().amax(-1, keepdim=True)
        e = (2.0 ** -17 * (a + 1) + 4 * r * e_sum.amax(-1, keepdim=True) * (1 + hat)) * s["pre"][0].abs().max() + 4 * R.U * o_ref.abs()
        R.assert_within(back(out), o_ref, e + R.rounding(dt, o_ref.abs() + e), "out")
    else:
        assert out is None


@pytest.mark.parametrize("dt,xt", TYPES)
@pytest.mark.parametrize("kind", [_lib.NORM_LAYER, _lib.NORM_RMS])
@pytest.mark.parametrize("n,h,w,c", [(1, 1, 1, 16), (2, 3, 5, 16), (1, 33, 17, 48), (3, 7, 9, 64), (2, 11, 13, 176), (1, 19, 7, 256), (5, 1, 1, 80),
                                     (2, 5, 3, 512), (1, 2, 3, 1024)])
def test_forward(dt, xt, kind, n, h, w, c):
    check_forward(make(c + n, n, h, w, c, dt, xt), dt, xt, kind, 0.3)


@pytest.mark.parametrize("c", [8, 24, 40, 88, 120, 264, 1016])
def test_forward_f32_planes_of_eight_channels(c):
    check_forward(make(c, 2, 5, 7, c, F32, F32), F32, F32, _lib.NORM_LAYER, 1.0)


@pytest.mark.parametrize("what", [dict(post=False), dict(pre=False), dict(gate="shared"), dict(gate=None), dict(bias=False), dict(y=False),
                                  dict(post=False, gate=None, bias=False), dict(post=False, pre=False)], ids=str)
@pytest.mark.parametrize("dt,xt", [(F16, F32), (BF16, BF16)])
def test_forward_parts(what, dt, xt):
    check_forward(make(7, 3, 9, 11, 96, dt, xt, **what), dt, xt, _lib.NORM_LAYER, -0.5)


def test_forward_far_from_zero():
    """Channels whose common mean is a thousand times their spread: the two-pass variance keeps them."""
    s = make(5, 1, 9, 9, 64, F32, F32)
    s["x"] = (s["x"] + 1000.0).float().double()
    check_forward(s, F32, F32, _lib.NORM_LAYER, 0.3)


def test_forward_in_place_and_strided_views():
    """Views of 32 channels inside tensors of 96, sum written over x and out over y; the other channels stay as they were."""
    s = make(3, 2, 6, 7, 32, F16, F16)
    wide_x, wide_y = (ops.Planes(2, 96, 6, 7, F16, zero=True) for _ in range(2))
    wide_x.buf.fill_(3.0)
    wide_y.buf.fill_(5.0)
    wide_x.buf[:, 2:4] = planes(s["x"], s, F16).buf
    wide_y.buf[:, 2:4] = planes(s["y"], s, F16).buf
    d = _lib.BlockNormDesc()
    post, pre, gate = pair(s["post"]), pair(s["pre"]), dev(s["gate"])
    d.n, d.h, d.w, d.c, d.kind, d.gate_per_image, d.eps, d.res_scale = 2, 6, 7, 32, _lib.NORM_LAYER, 1, EPS, 0.3
    d.x = d.sum = wide_x.view(32)
    d.y = d.out = wide_y.view(32)
    d.post_weight, d.post_bias, d.pre_weight, d.pre_bias, d.gate = (t.data_ptr() for t in (*post, *pre, gate))
    _lib.check(_lib.lib().srmi_block_norm(C.byref(d), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    got = [ops.Planes.wrap(b.buf[:, 2:4].contiguous()) for b in (wide_x, wide_y)]
    check_forward(s, F16, F16, _lib.NORM_LAYER, 0.3, got)
    for b, v in ((wide_x, 3.0), (wide_y, 5.0)):
        assert bool((b.buf[:, :2] == v).all()) and bool((b.buf[:, 4:] == v).all())


def test_forward_vectors_need_no_alignment():
    s = make(4, 2, 5, 5, 64, BF16, BF16)
    def off(v):  # a float's alignment only
        t = torch.empty(v.numel() + 1, dtype=torch.float32, device="cuda")[1:].view(v.shape)
        t.copy_(v)
        return t
    got = ops.block_norm(planes(s["x"], s, BF16), planes(s["y"], s, BF16), post=tuple(map(off, s["post"])), pre=tuple(map(off, s["pre"])),
                         gate=off(s["gate"]), res_scale=0.3, eps=EPS)
    check_forward(s, BF16, BF16, _lib.NORM_LAYER, 0.3, got)


def test_forward_nan_and_infinity_stay_in_their_pixel():
    s = make(6, 1, 8, 8, 64, F16, F16)
    x, y = planes(s["x"], s, F16), planes(s["y"], s, F16)
    clean = ops.block_norm(x, y, post=pair(s["post"]), pre=pair(s["pre"]), gate=dev(s["gate"]), eps=EPS)[1].to_nchw()
    y.buf[0, 1, 3, 4, 5] = float("nan")
    x.buf[0, 0, 6, 2, 0] = float("inf")
    out = ops.block_norm(x, y, post=pair(s["post"]), pre=pair(s["pre"]), gate=dev(s["gate"]), eps=EPS)[1].to_nchw()
    assert bool(torch.isnan(out[0, :, 3, 4]).all()) and bool(torch.isnan(out[0, :, 6, 2]).all())
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, :, 3, 4] = keep[0, :, 6, 2] = False
    assert torch.equal(out[keep], clean[keep])


def gradients(s, kind, res_scale):
    leaf = {"x": s["x"], "y": s["y"], "gate": s["gate"]}
    for side in ("post", "pre"):
        leaf[side + "_weight"], leaf[side + "_bias"] = s[side] if s[side] is not None else (None, None)
    leaf = {k: None if v is None else v.clone().requires_grad_() for k, v in leaf.items()}
    parts = {side: None if s[side] is None else (leaf[side + "_weight"], leaf[side + "_bias"]) for side in ("post", "pre")}
    total, out = R.block_norm(leaf["x"], leaf["y"], parts["post"], parts["pre"], leaf["gate"], res_scale, EPS, kind)
    loss = (total * s["d_sum"]).sum()
    if out is not None:
        loss = loss + (out * s["d_out"]).sum()
    loss.backward()
    return {("d" if k in "xy" else "d_") + k: None if v is None else v.grad for k, v in leaf.items()}


def backward(s, dt, xt, kind, res_scale):
    return ops.block_norm_backward(planes(s["x"], s, xt), planes(s["y"], s, dt), d_sum=planes(s["d_sum"], s, xt), d_out=planes(s["d_out"], s, dt),
                                   post=pair(s["post"]), pre=pair(s["pre"]), gate=dev(s["gate"]), res_scale=res_scale, eps=EPS, kind=kind)


def check_backward(s, dt, xt, kind, res_scale):
    got, ref = backward(s, dt, xt, kind, res_scale), gradients(s, kind, res_scale)
    rows = s["x"].shape[0] * s["x"].shape[1]
    total, _ = R.block_norm(s["x"], s["y"], s["post"], s["pre"], s["gate"], res_scale, EPS, kind)
    # ds: d_sum plus the norm's gradient, r * (D - <D hat> hat - <D>): each of its terms is at most r * max|D| * (1 + max|hat|^2)
    top = s["d_sum"].abs().max()
    e_ds = 4 * R.U * top
    if s["pre"] is not None:
        a, r = spread(total, kind)
        hat = ((total - total.mean(-1, keepdim=True) if kind == _lib.NORM_LAYER else total) * r).abs().amax()
        size = float((r * (s["d_out"] * s["pre"][0]).abs().amax(-1, keepdim=True)).max() * (1 + hat * hat))
        e_ds = e_ds + 2.0 ** -16 * (float(a.max()) + 1) * size
        top = top + size
    R.assert_within(back(got["dx"]), ref["dx"], e_ds + R.rounding(xt, ref["dx"].abs() + e_ds), "dx")
    g = s["gate"].abs().max() if s["gate"] is not None else 1.0
    if s["y"] is not None:
        e_dv, dv_top = abs(res_scale) * g * e_ds * 1.01 + 4 * R.U * abs(res_scale) * g * top, abs(res_scale) * g * top
        ay, ry, yhat_top = 1.0, 1.0, s["y"].abs().max()
        e_dy = e_dv
        if s["post"] is not None:
            a, r = spread(s["y"], kind)
            ay, ry, w = float(a.max()), float(r.max()), s["post"][0].abs().max()
            yhat_top = ((s["y"] - s["y"].mean(-1, keepdim=True) if kind == _lib.NORM_LAYER else s["y"]) * r).abs().max()
            e_dy = ry * w * (1 + yhat_top ** 2) * (4 * e_dv + 2.0 ** -16 * (ay + 1) * dv_top)
        R.assert_within(back(got["dy"]), ref["dy"], e_dy + R.rounding(dt, ref["dy"].abs() + e_dy), "dy")
        v_top = yhat_top if s["post"] is None else yhat_top * s["post"][0].abs().max() + (s["post"][1].abs().max() if s["post"][1] is not None else 0.0)
        sums = rows * ((rows + 64) * R.U)
        if s["gate"] is not None:
            per = rows if s["gate"].dim() == 1 else s["x"].shape[1]
            R.assert_within(got["d_gate"].cpu(), ref["d_gate"], abs(res_scale) * per * (e_ds * v_top + top * 2.0 ** -17 * (ay + 1) * v_top + (per + 64) * R.U * top * v_top), "d_gate")
        if s["post"] is not None:
            R.assert_within(got["d_post_weight"].cpu(), ref["d_post_weight"], rows * (e_dv * yhat_top + dv_top * 2.0 ** -17 * (ay + 1)) + sums * dv_top * yhat_top, "d_post_weight")
            if s["post"][1] is not None:
                R.assert_within(got["d_post_bias"].cpu(), ref["d_post_bias"], rows * e_dv + sums * dv_top, "d_post_bias")
    if s["pre"] is not None:
        d_abs = s["d_out"].abs()
        R.assert_within(got["d_pre_weight"].cpu(), ref["d_pre_weight"], d_abs.sum((0, 1)) * (2.0 ** -16 * (float(a_of(total, kind)) + 1) + (rows + 64) * R.U * hat), "d_pre_weight")
        if s["pre"][1] is not None:
            R.assert_within(got["d_pre_bias"].cpu(), ref["d_pre_bias"], (rows + 64) * R.U * d_abs.sum((0, 1)), "d_pre_bias")
    for k, v in ref.items():
        assert (v is None) == (got[k] is None), k


def a_of(v, kind):
    return spread(v, kind)[0].max()


@pytest.mark.parametrize("dt,xt", TYPES)
@pytest.mark.parametrize("kind", [_lib.NORM_LAYER, _lib.NORM_RMS])
@pytest.mark.parametrize("n,h,w,c", [(1, 1, 1, 16), (2, 3, 5, 16), (1, 33, 17, 48), (3, 7, 9, 64), (2, 11, 13, 176), (1, 19, 7, 256), (5, 1, 1, 80),
                                     (2, 5, 3, 512), (1, 2, 3, 1024)])
def test_backward(dt, xt, kind, n, h, w, c):
    check_backward(make(c + n, n, h, w, c, dt, xt), dt, xt, kind, 0.3)


@pytest.mark.parametrize("c", [8, 24, 40, 88, 120, 264, 1016])
def test_backward_f32_planes_of_eight_channels(c):
    check_backward(make(c, 2, 5, 7, c, F32, F32), F32, F32, _lib.NORM_LAYER, 1.0)


@pytest.mark.parametrize("what", [dict(post=False), dict(pre=False), dict(gate="shared"), dict(gate=None), dict(bias=False), dict(y=False),
                                  dict(post=False, gate=None, bias=False), dict(post=False, pre=False)], ids=str)
@pytest.mark.parametrize("dt,xt", [(F16, F32), (BF16, BF16)])
def test_backward_parts(what, dt, xt):
    check_backward(make(7, 3, 9, 11, 96, dt, xt, **what), dt, xt, _lib.NORM_LAYER, -0.5)


@pytest.mark.parametrize("n,h,w,gate", [(1100, 1, 3, "image"), (1100, 1, 3, "shared"), (3, 61, 67, "image"), (1, 80, 90, "shared")])
def test_backward_many_images_and_many_pixels(n, h, w, gate):
    """More images than workgroups (several per workgroup), and images split over workgroups."""
    check_backward(make(n, n, h, w, 16, F32, F32, gate=gate), F32, F32, _lib.NORM_LAYER, 0.3)


def test_backward_gives_equal_bits_twice():
    s = make(9, 2, 40, 50, 64, BF16, BF16)
    a, b = (backward(s, BF16, BF16, _lib.NORM_LAYER, 0.3) for _ in range(2))
    for k, v in a.items():
        assert torch.equal(v.buf, b[k].buf) if isinstance(v, ops.Planes) else torch.equal(v, b[k])


def test_backward_without_the_sums_gradient():
    s = make(10, 2, 6, 7, 64, F32, F32)
    s["d_sum"] = torch.zeros_like(s["d_sum"])
    want = backward(s, F32, F32, _lib.NORM_LAYER, 0.3)
    got = ops.block_norm_backward(planes(s["x"], s, F32), planes(s["y"], s, F32), d_out=planes(s["d_out"], s, F32), post=pair(s["post"]),
                                  pre=pair(s["pre"]), gate=dev(s["gate"]), res_scale=0.3, eps=EPS)
    for k, v in want.items():
        assert torch.equal(v.buf, got[k].buf) if isinstance(v, ops.Planes) else torch.equal(v, got[k])


def test_backward_against_differences():
    """The f32 gradients along random directions against central differences of the 64-bit forward form.  With step t the
    difference errs by t^2 / 6 of the third derivative (below 1e-6 of the value at t = 1e-3 here) and by 2^-52 / t."""
    s = make(11, 2, 4, 5, 64, F32, F32)
    got = backward(s, F32, F32, _lib.NORM_LAYER, 0.3)
    grad = {"x": back(got["dx"]), "y": back(got["dy"]), "gate": got["d_gate"].cpu().double(), "post": [got["d_post_weight"].cpu().double(), got["d_post_bias"].cpu().double()],
            "pre": [got["d_pre_weight"].cpu().double(), got["d_pre_bias"].cpu().double()]}
    gen = torch.Generator().manual_seed(1)

    def loss(v):
        total, out = R.block_norm(v["x"], v["y"], v["post"], v["pre"], v["gate"], 0.3, EPS, _lib.NORM_LAYER)
        return (total * s["d_sum"]).sum() + (out * s["d_out"]).sum()

    for key in ("x", "y", "gate", "post", "pre"):
        base = s[key]
        dirs = [R.rnd(gen, *b.shape) for b in (base if isinstance(base, tuple) else (base,))]
        moved = lambda t: tuple(b + t * d for b, d in zip(base, dirs)) if isinstance(base, tuple) else base + t * dirs[0]  # noqa: E731
        t = 1e-3
        want = float((loss(dict(s, **{key: moved(t)})) - loss(dict(s, **{key: moved(-t)}))) / (2 * t))
        g = grad[key] if isinstance(grad[key], list) else [grad[key]]
        have = float(sum((a * b).sum() for a, b in zip(g, dirs)))
        size = float(sum((a * b).abs().sum() for a, b in zip(g, dirs)))
        assert abs(have - want) <= 1e-5 * size, (key, have, want, size)


def test_on_another_stream_and_captured():
    """The calls run on the current stream and can be captured; replays on new inputs equal eager calls."""
    s = make(12, 2, 9, 10, 64, F16, F32)
    x, y, ds, do = planes(s["x"], s, F32), planes(s["y"], s, F16), planes(s["d_sum"], s, F32), planes(s["d_out"], s, F16)
    kw = dict(post=pair(s["post"]), pre=pair(s["pre"]), gate=dev(s["gate"]), res_scale=0.3, eps=EPS)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.block_norm(x, y, **kw)
        ops.block_norm_backward(x, y, d_sum=ds, d_out=do, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total, out = ops.block_norm(x, y, **kw)
        grads = ops.block_norm_backward(x, y, d_sum=ds, d_out=do, **kw)
    for i in range(4):
        x.buf.mul_(1.25)
        y.buf.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        t2, o2 = ops.block_norm(x, y, **kw)
        g2 = ops.block_norm_backward(x, y, d_sum=ds, d_out=do, **kw)
        assert torch.equal(total.buf, t2.buf) and torch.equal(out.buf, o2.buf)
        for k, v in grads.items():
            assert torch.equal(v.buf, g2[k].buf) if isinstance(v, ops.Planes) else torch.equal(v, g2[k]), k
