"""64-bit plain forms of the feed-forward block's operators (block_norm, gated_ffn), their gradients through autograd, and
the error bounds the tests hold the kernels to.  Tensors here are [n][h * w][c] doubles on the CPU."""
import math

import torch

from superresolution_amd import _lib

TORCH_DT = {_lib.F32: torch.float32, _lib.F16: torch.float16, _lib.BF16: torch.bfloat16}
U = 2.0 ** -24  # half a step of f32


def half_step(dt):
    """Largest relative error of one rounding to the type."""
    return torch.finfo(TORCH_DT[dt]).eps / 2


def rounding(dt, v):
    """Largest error of one rounding of a value of magnitude up to v: half a step of the value, and below the smallest normal
    number (2^-14 in f16) half of the fixed step there, which is half_step * 2^-14 = 2^-25."""
    return half_step(dt) * (v + torch.finfo(TORCH_DT[dt]).tiny)


def rnd(gen, *shape, scale=1.0):
    return torch.randn(shape, generator=gen, dtype=torch.float64) * scale


def rounded(v, dt):
    """The values a tensor of the type holds, as doubles."""
    return v.to(TORCH_DT[dt]).double()


def to_nchw(v, h, w):
    n, _, c = v.shape
    return v.reshape(n, h, w, c).permute(0, 3, 1, 2).contiguous()


def from_nchw(v):
    n, c = v.shape[:2]
    return v.double().permute(0, 2, 3, 1).reshape(n, -1, c)


# ---- block_norm ------------------------------------------------------------------------------------------------------
def norm(v, weight, bias, kind, eps):
    if kind == _lib.NORM_LAYER:
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * weight
    return v if bias is None else v + bias


def block_norm(x, y, post, pre, gate, res_scale, eps, kind):
    total = x
    if y is not None:
        v = y if post is None else norm(y, post[0], post[1], kind, eps)
        if gate is not None:
            v = v * (gate if gate.dim() == 1 else gate[:, None, :])
        total = x + res_scale * v
    return total, None if pre is None else norm(total, pre[0], pre[1], kind, eps)


# ---- gated_ffn -------------------------------------------------------------------------------------------------------
def act(a, which):
    if which == _lib.ACT_SILU:
        return a * torch.sigmoid(a)
    if which == _lib.ACT_GELU:
        return a * 0.5 * torch.special.erfc(-a * math.sqrt(0.5))
    if which == _lib.ACT_RELU:
        return torch.where(a > 0, a, torch.zeros_like(a))
    if which == _lib.ACT_LRELU:
        return torch.where(a > 0, a, 0.2 * a)
    return a


def gated_ffn(x, wg, wu, wd, bg, bu, bd, which, res, res_scale):
    g, u = x @ wg.t(), x @ wu.t()
    g, u = (g if bg is None else g + bg), (u if bu is None else u + bu)
    y = (act(g, which) * u) @ wd.t()
    y = res_scale * (y if bd is None else y + bd)
    return y if res is None else res + y


class FfnBounds:
    """Elementwise error bounds of gated_ffn and its gradients on rows x [m][c]: f32 accumulation of k terms errs by at most
    k * 2^-24 times the sum of their magnitudes, the activations (through exp2 and a reciprocal of 1 ulp each, and an erfc of
    absolute error 1.5e-7) and their slopes by 2^-20 of (1 + |a|), and one rounding to the type by half a step of the rounded value."""

    def __init__(self, x, wg, wu, wd, bg, bu, bd, which, res_scale, dt):
        m, c = x.shape
        hidden = wg.shape[0]
        self.round, self.s = lambda v: rounding(dt, v), abs(res_scale)
        zero = torch.zeros((), dtype=torch.float64)
        bg, bu, bd = (zero if b is None else b for b in (bg, bu, bd))
        g, u = x @ wg.t() + bg, x @ wu.t() + bu
        eg = (c + 4) * U * (x.abs() @ wg.abs().t() + bg.abs())
        eu = (c + 4) * U * (x.abs() @ wu.abs().t() + bu.abs())
        a = act(g, which)
        soft = which in (_lib.ACT_SILU, _lib.ACT_GELU)
        ea = 1.2 * eg + (2.0 ** -20 * (1 + g.abs()) if soft else 0.0)
        hid = a * u
        eh = ea * (u.abs() + eu) + a.abs() * eu + 4 * U * hid.abs()
        self.hid, self.eh_f32 = hid, eh
        eh = eh + self.round(hid.abs() + eh)
        self.eh = eh
        ywd = hid.abs() @ wd.abs().t()
        self.y = self.s * (eh @ wd.abs().t() + (hidden + 4) * U * (ywd + bd.abs()))
        self.g, self.u, self.a, self.eg, self.eu, self.ea = g, u, a, eg, eu, ea
        self.x, self.wg, self.wu, self.wd = x, wg, wu, wd
        self.soft, self.which = soft, which
        self.m, self.c, self.hidden = m, c, hidden

    def forward(self, ref, res=None):
        extra = 4 * U * (ref.abs() + (res.abs() if res is not None else 0.0))
        return self.y + extra + self.round(ref.abs() + self.y + extra)

    def backward(self, dy, dx_ref, grads):
        s = self.s
        dh = s * (dy @ self.wd)
        e_dh = (self.c + 4) * U * s * (dy.abs() @ self.wd.abs())
        slope_max = 1.2
        # the slope moves by at most 1.2 times the error of its argument, or jumps where a kink lies inside that error
        e_slope = (1.2 * self.eg + 2.0 ** -20 * (1 + self.g.abs())) if self.soft else (self.g.abs() <= self.eg).double()
        if self.which == _lib.ACT_NONE:
            e_slope = torch.zeros_like(self.g)
        e_dg = e_dh * self.u.abs() * slope_max + dh.abs() * (self.eu * slope_max + self.u.abs() * e_slope) + 2 * e_dh * self.eu
        e_dg = e_dg + 8 * U * dh.abs() * self.u.abs() * slope_max
        e_du = e_dh * (self.a.abs() + self.ea) + dh.abs() * self.ea + 4 * U * (dh * self.a).abs()
        dg_abs, du_abs = dh.abs() * self.u.abs() * slope_max, (dh * self.a).abs()
        rg, ru = e_dg + self.round(dg_abs + e_dg), e_du + self.round(du_abs + e_du)  # after the rounding
        m, x = self.m, self.x.abs()
        bounds = {
            "dx": rg @ self.wg.abs() + ru @ self.wu.abs() + (2 * self.hidden + 8) * U * (dg_abs @ self.wg.abs() + du_abs @ self.wu.abs()),
            "d_w_gate": rg.t() @ x + (m + 64) * U * (dg_abs.t() @ x),
            "d_w_up": ru.t() @ x + (m + 64) * U * (du_abs.t() @ x),
            "d_w_down": s * (dy.abs().t() @ self.eh + (m + 64) * U * (dy.abs().t() @ self.hid.abs())),
            "d_b_gate": e_dg.sum(0) + (m + 64) * U * dg_abs.sum(0),
            "d_b_up": e_du.sum(0) + (m + 64) * U * du_abs.sum(0),
            "d_b_down": (m + 64) * U * s * dy.abs().sum(0),
        }
        refs = dict(grads, dx=dx_ref)
        for k in ("dx", "d_w_gate", "d_w_up", "d_w_down"):
            bounds[k] = bounds[k] + self.round(refs[k].abs() + bounds[k])
        return bounds


def assert_within(got, ref, bound, what=""):
    """|got - ref| <= bound in every element; NaN and infinities where ref has them."""
    got, ref = got.double(), ref.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN elsewhere than in the reference"
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), f"{what}: infinities differ"
    over = ((got - ref).abs() / (bound + 1e-30))[fine]
    if over.numel():
        worst = float(over.max())
        assert worst <= 1.0, f"{what}: error is {worst:.3g} of its bound"
