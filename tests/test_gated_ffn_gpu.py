"""gated_ffn and gated_ffn_backward against 64-bit plain forms; the elementwise bounds are derived in ffn_block_ref.FfnBounds."""
import ctypes as C

import pytest
import torch

from superresolution_amd import _lib, ops
from tests import ffn_block_ref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16
ACTS = [_lib.ACT_NONE, _lib.ACT_RELU, _lib.ACT_LRELU, _lib.ACT_SILU, _lib.ACT_GELU]
NAMES = ("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")


def make(seed, n, h, w, c, hidden, dt, bias=True, res=True):
    gen = torch.Generator().manual_seed(seed)
    s = {"n": n, "h": h, "w": w, "c": c, "hidden": hidden}
    m = h * w
    s["x"] = R.rounded(R.rnd(gen, n, m, c) + R.rnd(gen, c, scale=0.3), dt)
    s["w_gate"], s["w_up"] = (R.rounded(R.rnd(gen, hidden, c, scale=c ** -0.5), dt) for _ in range(2))
    s["w_down"] = R.rounded(R.rnd(gen, c, hidden, scale=hidden ** -0.5), dt)
    for k, size in (("b_gate", hidden), ("b_up", hidden), ("b_down", c)):
        s[k] = R.rnd(gen, size, scale=0.2).float().double() if bias else None
    s["res"] = R.rounded(R.rnd(gen, n, m, c), dt) if res else None
    s["d_out"] = R.rounded(R.rnd(gen, n, m, c, scale=0.1), dt)
    return s


def planes(v, s, dt):
    return None if v is None else ops.Planes.from_nchw(R.to_nchw(v, s["h"], s["w"]).float(), dt)


def weights(s, dt):
    args = {k: s[k].to(R.TORCH_DT[dt]).cuda() for k in NAMES[:3]}
    args.update({k: None if s[k] is None else s[k].float().cuda() for k in NAMES[3:]})
    return args


def rows(v):
    return v.reshape(-1, v.shape[-1])


def back(p):
    return rows(R.from_nchw(p.to_nchw().cpu()))


def bounds(s, dt, act, res_scale):
    return R.FfnBounds(rows(s["x"]), *(s[k] for k in NAMES), act, res_scale, dt)


def check_forward(s, dt, act, res_scale, got=None):
    if got is None:
        got = ops.gated_ffn(planes(s["x"], s, dt), **weights(s, dt), act=act, res=planes(s["res"], s, dt), res_scale=res_scale)
    res = None if s["res"] is None else rows(s["res"])
    ref = R.gated_ffn(rows(s["x"]), *(s[k] for k in NAMES), act, res, res_scale)
    R.assert_within(back(got), ref, bounds(s, dt, act, res_scale).forward(ref, res), "out")


def run_backward(s, dt, act, res_scale):
    return ops.gated_ffn_backward(planes(s["x"], s, dt), planes(s["d_out"], s, dt), **weights(s, dt), act=act, res_scale=res_scale)


def gradients(s, act, res_scale):
    leaf = {k: None if s[k] is None else s[k].clone().requires_grad_() for k in NAMES}
    x = rows(s["x"]).clone().requires_grad_()
    y = R.gated_ffn(x, *(leaf[k] for k in NAMES), act, None, res_scale)
    y.backward(rows(s["d_out"]))
    return dict({"d_" + k: None if v is None else v.grad for k, v in leaf.items()}, dx=x.grad)


def check_backward(s, dt, act, res_scale):
    got, ref = run_backward(s, dt, act, res_scale), gradients(s, act, res_scale)
    limit = bounds(s, dt, act, res_scale).backward(rows(s["d_out"]), ref["dx"], ref)
    for k, v in ref.items():
        if v is None:
            assert got[k] is None
            continue
        have = back(got[k]) if k == "dx" else got[k].cpu()
        assert k == "dx" or got[k].dtype == (R.TORCH_DT[dt] if k.startswith("d_w") else torch.float32)
        R.assert_within(have, v, limit[k], k)


# one pixel to several tiles, channels and hidden units that fill no tile, both sides of every size rule
SIZES = [(1, 1, 1, 16, 16), (1, 1, 1, 64, 128), (3, 1, 1, 48, 80), (1, 9, 31, 32, 48), (2, 17, 13, 64, 96), (1, 33, 29, 80, 176), (2, 5, 7, 144, 208),
         (1, 16, 16, 256, 512), (1, 7, 37, 272, 144), (2, 1, 3, 400, 1040), (1, 5, 60, 128, 32), (1, 40, 30, 16, 16), (4, 1, 2, 256, 1024)]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("n,h,w,c,hidden", SIZES)
def test_forward(dt, n, h, w, c, hidden):
    check_forward(make(c + hidden, n, h, w, c, hidden, dt), dt, _lib.ACT_SILU, 0.3)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,res", [(True, False), (False, True)])
def test_forward_activations(dt, act, bias, res):
    check_forward(make(act, 2, 9, 11, 48, 112, dt, bias, res), dt, act, -0.7)


@pytest.mark.parametrize("c,hidden", [(8, 8), (24, 40), (56, 120), (264, 24), (200, 328)])
def test_f32_planes_of_eight_channels(c, hidden):
    s = make(c, 2, 7, 9, c, hidden, F32)
    check_forward(s, F32, _lib.ACT_GELU, 1.0)
    check_backward(s, F32, _lib.ACT_GELU, 1.0)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("n,h,w,c,hidden", SIZES)
def test_backward(dt, n, h, w, c, hidden):
    check_backward(make(c + hidden, n, h, w, c, hidden, dt), dt, _lib.ACT_SILU, 0.3)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [True, False])
def test_backward_activations(dt, act, bias):
    check_backward(make(act, 2, 9, 11, 48, 112, dt, bias), dt, act, -0.7)


@pytest.mark.parametrize("given", [("b_gate",), ("b_up",), ("b_down",), ("b_gate", "b_down")])
def test_each_bias_alone(given):
    s = make(5, 1, 11, 13, 32, 64, F16)
    for k in NAMES[3:]:
        if k not in given:
            s[k] = None
    check_forward(s, F16, _lib.ACT_SILU, 1.0)
    check_backward(s, F16, _lib.ACT_SILU, 1.0)


def test_backward_gives_equal_bits_twice():
    s = make(6, 2, 33, 41, 64, 160, BF16)
    a, b = (run_backward(s, BF16, _lib.ACT_GELU, 0.3) for _ in range(2))
    for k, v in a.items():
        assert torch.equal(v.buf, b[k].buf) if k == "dx" else torch.equal(v, b[k])


def test_strided_views_and_residual_in_place():
    """x, res and out inside wider tensors, out written over res; the other channels stay as they were."""
    s = make(7, 2, 11, 13, 48, 80, F16)
    wide_x, wide_r = (ops.Planes(2, 112, 11, 13, F16) for _ in range(2))
    wide_x.buf.fill_(float("nan"))
    wide_r.buf.fill_(5.0)
    wide_x.buf[:, 3:6] = planes(s["x"], s, F16).buf
    wide_r.buf[:, 1:4] = planes(s["res"], s, F16).buf
    args = weights(s, F16)
    d = _lib.GatedFfnDesc()
    d.dtype, d.n, d.h, d.w, d.c, d.hidden, d.act, d.res_scale = F16, 2, 11, 13, 48, 80, _lib.ACT_SILU, 0.3
    d.x, d.res, d.out = wide_x.view(48), wide_r.view(16), wide_r.view(16)
    for k, v in args.items():
        setattr(d, k, v.data_ptr())
    need = _lib.lib().srmi_gated_ffn_workspace(C.byref(d))
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib().srmi_gated_ffn(C.byref(d), ws.data_ptr(), need, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    check_forward(s, F16, _lib.ACT_SILU, 0.3, ops.Planes.wrap(wide_r.buf[:, 1:4].contiguous()))
    assert bool((wide_r.buf[:, :1] == 5).all()) and bool((wide_r.buf[:, 4:] == 5).all())


def test_nan_stays_in_its_pixel():
    s = make(8, 1, 12, 12, 64, 128, F16)
    x = planes(s["x"], s, F16)
    args = weights(s, F16)
    clean = ops.gated_ffn(x, **args).to_nchw()
    x.buf[0, 2, 5, 7, 3] = float("nan")
    out = ops.gated_ffn(x, **args).to_nchw()
    assert bool(torch.isnan(out[0, :, 5, 7]).all())
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, :, 5, 7] = False
    assert torch.equal(out[keep], clean[keep])


def test_f16_values_beyond_the_range_saturate():
    """x = 2^10 on one channel of weight 1: hidden values of 2^20 are stored as 65504, as every f16 store of the library."""
    s = make(9, 1, 4, 4, 16, 16, F16, bias=False, res=False)
    x = torch.zeros(1, 16, 16, dtype=torch.float64)
    x[..., 0] = 1024.0
    eye = torch.eye(16, dtype=torch.float64)
    s.update(x=x, w_gate=eye, w_up=eye, w_down=eye)
    out = ops.gated_ffn(planes(s["x"], s, F16), **weights(s, F16), act=_lib.ACT_NONE).to_nchw().cpu()
    want = torch.zeros(1, 16, 4, 4)
    want[:, 0] = 65504.0
    assert torch.equal(out, want)


def test_backward_against_differences():
    """f32 gradients along random directions against central differences of the 64-bit forward form (step 1e-3: its error is
    below 1e-6 of the magnitudes summed)."""
    s = make(10, 1, 4, 5, 32, 48, F32, res=False)
    for act in (_lib.ACT_SILU, _lib.ACT_GELU):
        got = run_backward(s, F32, act, 0.3)
        gen = torch.Generator().manual_seed(1)

        def loss(v):
            return (R.gated_ffn(rows(v["x"]), *(v[k] for k in NAMES), act, None, 0.3) * rows(s["d_out"])).sum()

        for key in ("x",) + NAMES:
            direction = R.rnd(gen, *s[key].shape)
            t = 1e-3
            want = float((loss(dict(s, **{key: s[key] + t * direction})) - loss(dict(s, **{key: s[key] - t * direction}))) / (2 * t))
            g = back(got["dx"]).reshape(direction.shape) if key == "x" else got["d_" + key].cpu().double()
            assert abs(float((g * direction).sum()) - want) <= 1e-5 * float((g * direction).abs().sum()), key


def test_on_another_stream_and_captured():
    s = make(11, 2, 19, 21, 64, 96, F16)
    x, dy, res = planes(s["x"], s, F16), planes(s["d_out"], s, F16), planes(s["res"], s, F16)
    args = weights(s, F16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.gated_ffn(x, **args, res=res)
        ops.gated_ffn_backward(x, dy, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.gated_ffn(x, **args, res=res)
        grads = ops.gated_ffn_backward(x, dy, **args)
    for _ in range(4):
        x.buf.mul_(1.25)
        args["w_up"].mul_(0.875)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.buf, ops.gated_ffn(x, **args, res=res).buf)
        for k, v in ops.gated_ffn_backward(x, dy, **args).items():
            assert torch.equal(v.buf, grads[k].buf) if k == "dx" else torch.equal(v, grads[k]), k


def test_a_block_as_it_is_used():
    """norm -> feed-forward -> norm, gate, residual -> norm, forward and backward through both operators, against autograd
    on the 64-bit form.  f32, so that only accumulation order differs: 1e-5 of the largest value of each result (sums of fewer than 600
    terms, three norms of spread below 8)."""
    s = make(12, 2, 6, 7, 48, 96, F32, res=False)
    gen = torch.Generator().manual_seed(3)
    c, n = 48, 2
    vec = lambda m: (m + R.rnd(gen, c, scale=0.1)).float().double()  # noqa: E731
    first, post, pre, gate = (vec(1.0), vec(0.0)), (vec(1.0), None), (vec(1.0), vec(0.0)), torch.sigmoid(R.rnd(gen, n, c)).float().double()
    leaf = {k: v.clone().requires_grad_() for k, v in dict(x=s["x"], first_w=first[0], first_b=first[1], post_w=post[0], pre_w=pre[0], pre_b=pre[1], gate=gate).items()}
    leaf.update({k: s[k].clone().requires_grad_() for k in NAMES})
    _, a = R.block_norm(leaf["x"], None, None, (leaf["first_w"], leaf["first_b"]), None, 1.0, 1e-5, 0)
    f = R.gated_ffn(rows(a), *(leaf[k] for k in NAMES), _lib.ACT_SILU, None, 1.0).reshape(a.shape)
    total, out = R.block_norm(leaf["x"], f, (leaf["post_w"], None), (leaf["pre_w"], leaf["pre_b"]), leaf["gate"], 0.5, 1e-5, 0)
    d_total, d_out = R.rnd(gen, *total.shape).float().double(), R.rnd(gen, *out.shape).float().double()
    torch.autograd.backward([total, out], [d_total, d_out])

    cu = lambda v: None if v is None else v.float().cuda()  # noqa: E731
    x = planes(s["x"], s, F32)
    args = weights(s, F32)
    k_first, k_post, k_pre, k_gate = tuple(map(cu, first)), (cu(post[0]), None), tuple(map(cu, pre)), cu(gate)
    _, ka = ops.block_norm(x, pre=k_first)
    kf = ops.gated_ffn(ka, **args)
    k_total, k_out = ops.block_norm(x, kf, post=k_post, pre=k_pre, gate=k_gate, res_scale=0.5)
    g2 = ops.block_norm_backward(x, kf, d_sum=planes(d_total, s, F32), d_out=planes(d_out, s, F32), post=k_post, pre=k_pre, gate=k_gate, res_scale=0.5)
    gf = ops.gated_ffn_backward(ka, g2["dy"], **args)
    g1 = ops.block_norm_backward(x, d_sum=g2["dx"], d_out=gf["dx"], pre=k_first)

    def close(got, ref, what):
        assert float((got.double().cpu() - ref).abs().max()) <= 1e-5 * float(ref.abs().max()), what

    close(R.from_nchw(k_total.to_nchw()).cpu(), total.detach(), "sum")
    close(R.from_nchw(k_out.to_nchw()).cpu(), out.detach(), "out")
    close(R.from_nchw(g1["dx"].to_nchw()).cpu(), leaf["x"].grad, "dx")
    for k in NAMES:
        close(gf["d_" + k], leaf[k].grad, k)
    for got, k in ((g1["d_pre_weight"], "first_w"), (g1["d_pre_bias"], "first_b"), (g2["d_post_weight"], "post_w"), (g2["d_pre_weight"], "pre_w"),
                   (g2["d_pre_bias"], "pre_b"), (g2["d_gate"], "gate")):
        close(got, leaf[k].grad, k)


def test_between_convolutions():
    """The operators take and give the tensors of the library's other operators: conv3x3 -> block_norm -> gated_ffn -> conv3x3 in
    f32 against the same in 64 bits.  The convolutions sum 9 * 32 terms; 1e-4 of the largest value is over 16 times what
    f32 accumulation through the five operators can err by (sum of 2 * 288 + 32 + 96 terms at 2^-24 each, two norm-like rescalings)."""
    import torch.nn.functional as F
    gen = torch.Generator().manual_seed(4)
    x = R.rnd(gen, 1, 32, 13, 17).float()
    w1, w2 = (R.rnd(gen, 32, 32, 3, 3, scale=0.06).float() for _ in range(2))
    s = make(13, 1, 13, 17, 32, 64, F32)
    t = F.conv2d(x.double(), w1.double(), padding=1)
    rows_t = R.from_nchw(t)
    one = torch.ones(32, dtype=torch.float64)
    _, a = R.block_norm(rows_t, None, None, (one, None), None, 1.0, 1e-5, _lib.NORM_RMS)
    f = R.gated_ffn(rows(a), *(s[k] for k in NAMES), _lib.ACT_SILU, rows(rows_t), 0.2).reshape(a.shape)
    want = F.conv2d(R.to_nchw(f, 13, 17), w2.double(), padding=1)
    kt = ops.conv3x3(ops.Planes.from_nchw(x, F32), ops.PackedConv(w1.numpy(), None, F32))
    _, ka = ops.block_norm(kt, pre=(one.float().cuda(), None), kind=_lib.NORM_RMS)
    kf = ops.gated_ffn(ka, **weights(s, F32), res=kt, res_scale=0.2)
    got = ops.conv3x3(kf, ops.PackedConv(w2.numpy(), None, F32)).to_nchw().cpu().double()
    assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max())


def wide(s, dt):
    """The case's tensors as doubles on the GPU."""
    return {k: v.to("cuda") if isinstance(v, torch.Tensor) else v for k, v in s.items()}


def test_backward_in_several_runs_of_pixels():
    """More pixels than the hidden tensors of one run hold (4 GiB): hidden 16384 in f32 takes 21760 pixels per run."""
    s = make(14, 1, 150, 160, 8, 16384, F32)
    got = run_backward(s, F32, _lib.ACT_SILU, 0.3)
    g = wide(s, F32)
    ref = gradients(g, _lib.ACT_SILU, 0.3)
    limit = R.FfnBounds(rows(g["x"]), *(g[k] for k in NAMES), _lib.ACT_SILU, 0.3, F32).backward(rows(g["d_out"]), ref["dx"], ref)
    for k, v in ref.items():
        have = rows(R.from_nchw(got[k].to_nchw())) if k == "dx" else got[k]
        R.assert_within(have, v, limit[k], k)


def test_forward_in_several_runs_of_pixels():
    """The same for the form with two launches (more than 16 planes of channels): 65536 pixels per run."""
    s = make(15, 1, 260, 270, 136, 16384, F32, bias=False, res=False)
    got = ops.gated_ffn(planes(s["x"], s, F32), **weights(s, F32), act=_lib.ACT_RELU)
    g = wide(s, F32)
    x = rows(g["x"])
    have = rows(R.from_nchw(got.to_nchw()))
    for part in (slice(0, 2000), slice(64500, 66500), slice(x.shape[0] - 2000, x.shape[0])):  # both ends and the runs' border
        b = R.FfnBounds(x[part], *(g[k] for k in NAMES), _lib.ACT_RELU, 1.0, F32)
        ref = R.gated_ffn(x[part], *(g[k] for k in NAMES), _lib.ACT_RELU, None, 1.0)
        R.assert_within(have[part], ref, b.forward(ref), "out")


@pytest.mark.parametrize("dt,c,hidden,pixels", [(F16, 64, 128, 40000), (F16, 16, 512, 33000), (BF16, 128, 96, 36001), (F32, 32, 64, 33333), (F16, 256, 64, 70001)])
def test_forward_with_pixels_for_every_cu(dt, c, hidden, pixels):
    """More workgroups than CUs, ragged last ones."""
    s = make(c, 1, 1, pixels, c, hidden, dt)
    check_forward(s, dt, _lib.ACT_SILU, 0.3)


@pytest.mark.parametrize("dt,c,hidden,n,h,w", [(F16, 64, 256, 3, 97, 103), (BF16, 192, 96, 2, 130, 131), (F32, 64, 64, 2, 101, 97), (F16, 256, 272, 1, 187, 190)])
def test_backward_of_many_pixels(dt, c, hidden, n, h, w):
    """Several steps and splits of the weight gradients, ragged last ones, images that end inside a step."""
    check_backward(make(c + hidden, n, h, w, c, hidden, dt), dt, _lib.ACT_GELU, 0.3)


@pytest.mark.parametrize("dt,c,hidden,pixels", [(F16, 512, 256, 32769), (BF16, 384, 256, 32761), (F16, 640, 160, 13401), (BF16, 272, 416, 13330),
                                                (F32, 256, 256, 33003), (F32, 136, 72, 70), (F16, 1040, 64, 3), (BF16, 1024, 2064, 1), (F32, 144, 1304, 37),
                                                (F16, 528, 1040, 515)])
def test_wide_channels_with_every_size_of_tile(dt, c, hidden, pixels):
    """More than 16 planes of channels: tiles of 8, 6, 4, 2 and 1 blocks of rows, the last pixels in a workgroup with idle waves, and
    reductions in parts (odd steps, both products of dx inside one part)."""
    s = make(c + hidden, 1, 1, pixels, c, hidden, dt)
    out = ops.gated_ffn(planes(s["x"], s, dt), **weights(s, dt), act=_lib.ACT_SILU, res=planes(s["res"], s, dt), res_scale=0.3)
    got = run_backward(s, dt, _lib.ACT_SILU, 0.3)
    g = wide(s, dt)
    limit = R.FfnBounds(rows(g["x"]), *(g[k] for k in NAMES), _lib.ACT_SILU, 0.3, dt)
    ref = R.gated_ffn(rows(g["x"]), *(g[k] for k in NAMES), _lib.ACT_SILU, rows(g["res"]), 0.3)
    R.assert_within(rows(R.from_nchw(out.to_nchw())), ref, limit.forward(ref, rows(g["res"])), "out")
    ref = gradients(g, _lib.ACT_SILU, 0.3)
    bound = limit.backward(rows(g["d_out"]), ref["dx"], ref)
    for k, v in ref.items():
        R.assert_within(rows(R.from_nchw(got[k].to_nchw())) if k == "dx" else got[k], v, bound[k], k)


def test_backward_of_many_single_pixel_images():
    """Every step of 32 pixels then crosses 32 images, inside a wider tensor."""
    s = make(16, 500, 1, 1, 32, 48, F16)
    check_backward(s, F16, _lib.ACT_SILU, 1.0)
    check_forward(s, F16, _lib.ACT_SILU, 1.0)


def test_two_calls_at_once_on_two_streams():
    """Each call has its own workspace; equal inputs give equal bits whatever runs beside."""
    s = make(17, 2, 40, 41, 64, 160, F16)
    x, dy = planes(s["x"], s, F16), planes(s["d_out"], s, F16)
    args = weights(s, F16)
    want_f, want_b = ops.gated_ffn(x, **args), ops.gated_ffn_backward(x, dy, **args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                got.append((ops.gated_ffn(x, **args), ops.gated_ffn_backward(x, dy, **args)))
    torch.cuda.synchronize()
    for f, b in got:
        assert torch.equal(f.buf, want_f.buf)
        for k, v in b.items():
            assert torch.equal(v.buf, want_b[k].buf) if k == "dx" else torch.equal(v, want_b[k]), k
