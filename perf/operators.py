"""Measured cases of the feed-forward block's operators: the norms around a residual block with its gate and residual scale,
and the gated feed-forward block, each forward and backward.

Activations are plane tensors, [n][c / cpb][h][w][cpb] with 32 bytes of channels per pixel and plane (16 halves or 8 floats),
as every operator of `superresolution_amd.ops` takes them.  With v the block's body y, normalised if the block has a norm
behind it (post), a pixel's channels c go through

    sum = x + res_scale * gate[n][c] * v                     out = norm(sum) * pre_weight + pre_bias
    ffn = res + res_scale * (W_down (act(W_gate x + b_gate) * (W_up x + b_up)) + b_down)

`own` False computes them with elementary torch operations in 32 bits, True with the library's operators.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


# ---- the cases ------------------------------------------------------------------------------------------------------
def _norm(name, op, n, h, w, c, dtype, trunk, kind="layer", post=True, pre=True, gate="image", bias=True):
    return dict(name=name, op=op, n=n, h=h, w=w, c=c, dtype=dtype, trunk=trunk, kind=kind, post=post, pre=pre, gate=gate, bias=bias)


def _ffn(name, op, n, h, w, c, hidden, dtype, act="silu", bias=True, res=True):
    return dict(name=name, op=op, n=n, h=h, w=w, c=c, hidden=hidden, dtype=dtype, act=act, bias=bias, res=res)


def listed():
    return [
        # one pooled vector per image, as the squeeze / excite pair of channel attention sees them: a launch's latency
        _norm("norm_pooled", "norm_fwd", 32, 1, 1, 64, "f16", "f16"),
        # the 510 x 339 video frame at 64 features, residual trunk in single precision
        _norm("norm_frame_trunk_f32", "norm_fwd", 1, 339, 510, 64, "f16", "f32"),
        # a batch of 256 x 256 frames at 256 features: pure memory traffic
        _norm("norm_batch_rms", "norm_fwd", 8, 256, 256, 256, "bf16", "bf16", kind="rms", gate="shared", bias=False),
        # a training batch of 48 x 48 patches
        _norm("norm_patches_backward", "norm_bwd", 16, 48, 48, 64, "bf16", "bf16"),
        # gradients of a batch of frames at 256 features, trunk in single precision
        _norm("norm_batch_backward", "norm_bwd", 4, 256, 256, 256, "f16", "f32", kind="rms", gate="shared", bias=False),
        # one pooled vector through the block: weights are all there is to read
        _ffn("ffn_pixel", "ffn_fwd", 1, 1, 1, 256, 512, "f16", bias=True, res=False),
        # the video frame at 64 features
        _ffn("ffn_frame", "ffn_fwd", 1, 339, 510, 64, 128, "f16", act="gelu"),
        # a batch of 256 x 256 frames at 256 features: matrix products
        _ffn("ffn_batch", "ffn_fwd", 8, 256, 256, 256, 512, "bf16", bias=False),
        # the exact mode on one 256 x 256 frame
        _ffn("ffn_exact", "ffn_fwd", 1, 256, 256, 64, 256, "f32"),
        # a training batch of 48 x 48 patches
        _ffn("ffn_patches_backward", "ffn_bwd", 16, 48, 48, 64, 256, "bf16", act="gelu"),
        # odd sizes everywhere: channels and hidden units that fill no tile, images of 61 x 37
        _ffn("ffn_ragged_backward", "ffn_bwd", 7, 61, 37, 176, 464, "f16"),
        # the largest: two 256 x 256 frames at 256 features and a fourfold hidden layer
        _ffn("ffn_batch_backward", "ffn_bwd", 2, 256, 256, 256, 1024, "bf16", bias=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "ffn_fwd", "ffn_bwd"])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    unit = 8 if dtype == "f32" else 16
    c = unit * _log_int(rng, 16 // unit, 384 // unit)
    hidden = unit * _log_int(rng, 16 // unit, 1536 // unit)
    if op.startswith("norm"):
        most = (1 << 26) // c
    else:
        most = int((1.5e11 if dtype != "f32" else 1.5e10) / ((6 if op == "ffn_fwd" else 16) * c * hidden))
    pixels = _log_int(rng, 1, max(1, min(most, 1 << 18)))
    n = min(pixels, rng.choice([1, 1, 2, 3, 5, 8]))
    h = max(1, int(math.sqrt(pixels / n) * math.exp(rng.uniform(-0.7, 0.0))))
    w = max(1, pixels // (n * h))
    case = dict(op=op, n=n, h=h, w=w, c=c, dtype=dtype)
    if op.startswith("norm"):
        case.update(trunk=rng.choice([dtype, "f32"]), kind=rng.choice(["layer", "rms"]), gate=rng.choice(["image", "shared", "none"]),
                    bias=rng.choice([True, False]), post=rng.choice([True, True, False]), pre=True)
    else:
        case.update(hidden=hidden, act=rng.choice(["silu", "gelu", "relu", "none"]), bias=rng.choice([True, False]), res=rng.choice([True, False]))
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _planes(values, dtype):
    """[n][h][w][c] -> [n][c / cpb][h][w][cpb] of the type."""
    n, h, w, c = values.shape
    cpb = 8 if dtype == torch.float32 else 16
    return values.to(dtype).reshape(n, h, w, c // cpb, cpb).permute(0, 3, 1, 2, 4).contiguous()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, h, w, c = case["n"], case["h"], case["w"], case["c"]
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * scale

    def features(scale, dtype):  # activations of a trained network: channels of unequal mean and spread
        v = normal(n, h, w, c).mul_(normal(c, scale=0.3).exp_()).add_(normal(c, scale=0.5)).mul_(scale)
        return _planes(v, dtype)

    s = {"case": case}
    if case["op"].startswith("norm"):
        trunk = DTYPES[case["trunk"]]
        s["x"], s["y"] = features(2.0, trunk), features(1.0, dt)
        for side in ("post", "pre"):
            s[side] = (1.0 + normal(c, scale=0.1), normal(c, scale=0.1) if case["bias"] else None) if case[side] else None
        shape = {"image": (n, c), "shared": (c,), "none": None}[case["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(normal(*shape))
        s["res_scale"] = 0.1 if case["kind"] == "layer" else 1.0
        if case["op"] == "norm_bwd":
            s["d_sum"], s["d_out"] = _planes(normal(n, h, w, c, scale=0.02), trunk), _planes(normal(n, h, w, c, scale=0.02), dt)
    else:
        f = case["hidden"]
        s["x"] = features(1.0, dt)
        s["w_gate"], s["w_up"] = (normal(f, c, scale=c ** -0.5).to(dt) for _ in range(2))
        s["w_down"] = normal(c, f, scale=f ** -0.5).to(dt)
        s["b_gate"], s["b_up"], s["b_down"] = (normal(k, scale=0.1) if case["bias"] else None for k in (f, f, c))
        s["res_scale"] = 0.2 if case["res"] else 1.0
        if case["op"] == "ffn_bwd":
            s["d_out"] = _planes(normal(n, h, w, c, scale=0.02), dt)
        else:
            s["res"] = features(2.0, dt) if case["res"] else None
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    return {"norm_fwd": _norm_forward, "norm_bwd": _norm_backward, "ffn_fwd": _ffn_forward, "ffn_bwd": _ffn_backward}[s["case"]["op"]](s)


def _rows(buf):
    """A plane tensor's pixels as rows of 32-bit values, [n][h * w][c]."""
    n, p, h, w, k = buf.shape
    return buf.permute(0, 2, 3, 1, 4).reshape(n, h * w, p * k).float()


def _back(rows, like, dtype=None):
    n, _, h, w, _ = like.shape
    return _planes(rows.reshape(n, h, w, rows.shape[-1]), dtype or like.dtype)


def _normalise(v, kind):
    """(v - mean) / std over the channels, and 1 / std."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    return v * r, r


def _affine(vhat, wb):
    return vhat * wb[0] if wb[1] is None else vhat * wb[0] + wb[1]


def _normalise_grad(d_hat, vhat, r, kind):
    """The gradient of _normalise's input."""
    d = d_hat - vhat * (d_hat * vhat).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - d_hat.mean(-1, keepdim=True)
    return d * r


def _gate_rows(s):
    return None if s["gate"] is None else s["gate"] if s["gate"].dim() == 1 else s["gate"][:, None, :]


def _norm_forward(s):
    case = s["case"]
    if own:
        from superresolution_amd import _lib, ops
        total, out = ops.block_norm(ops.Planes.wrap(s["x"]), ops.Planes.wrap(s["y"]), post=s["post"], pre=s["pre"], gate=s["gate"],
                                    res_scale=s["res_scale"], eps=EPS, kind=_lib.NORM_LAYER if case["kind"] == "layer" else _lib.NORM_RMS)
        return {"sum": total.buf, "out": out.buf}
    x, v = _rows(s["x"]), _rows(s["y"])
    if s["post"]:
        v = _affine(_normalise(v, case["kind"])[0], s["post"])
    g = _gate_rows(s)
    total = x + s["res_scale"] * (v if g is None else g * v)
    out = _affine(_normalise(total, case["kind"])[0], s["pre"])
    return {"sum": _back(total, s["x"]), "out": _back(out, s["y"])}


def _norm_backward(s):
    case = s["case"]
    if own:
        from superresolution_amd import _lib, ops
        g = ops.block_norm_backward(ops.Planes.wrap(s["x"]), ops.Planes.wrap(s["y"]), d_sum=ops.Planes.wrap(s["d_sum"]), d_out=ops.Planes.wrap(s["d_out"]),
                                    post=s["post"], pre=s["pre"], gate=s["gate"], res_scale=s["res_scale"], eps=EPS,
                                    kind=_lib.NORM_LAYER if case["kind"] == "layer" else _lib.NORM_RMS)
        return {k: v.buf if isinstance(v, ops.Planes) else v for k, v in g.items() if v is not None}
    kind, scale, gate = case["kind"], s["res_scale"], _gate_rows(s)
    x, v = _rows(s["x"]), _rows(s["y"])
    if s["post"]:
        yhat, ry = _normalise(v, kind)
        v = _affine(yhat, s["post"])
    that, rt = _normalise(x + scale * (v if gate is None else gate * v), kind)
    d_out, found = _rows(s["d_out"]), {}
    d = _rows(s["d_sum"]) + _normalise_grad(d_out * s["pre"][0], that, rt, kind)
    dv = scale * (d if gate is None else gate * d)
    dy = _normalise_grad(dv * s["post"][0], yhat, ry, kind) if s["post"] else dv
    found["dx"], found["dy"] = _back(d, s["x"]), _back(dy, s["y"])
    if gate is not None:
        found["d_gate"] = scale * (d * v).sum(1 if s["gate"].dim() == 2 else (0, 1))
    if s["post"]:
        found["d_post_weight"] = (dv * yhat).sum((0, 1))
        if s["post"][1] is not None:
            found["d_post_bias"] = dv.sum((0, 1))
    found["d_pre_weight"] = (d_out * that).sum((0, 1))
    if s["pre"][1] is not None:
        found["d_pre_bias"] = d_out.sum((0, 1))
    return found


def _act(a, act):
    """act(a) and its derivative."""
    if act == "silu":
        t = torch.sigmoid(a)
        return a * t, t * (1.0 + a * (1.0 - t))
    if act == "gelu":
        p = 0.5 * (1.0 + torch.erf(a * math.sqrt(0.5)))
        return a * p, p + a * torch.exp(-0.5 * a.square()) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "relu":
        return a.clamp_min(0.0), (a > 0).to(a.dtype)
    return a, torch.ones_like(a)


def _linear(v, w, b=None):
    r = v @ w.float().t()
    return r if b is None else r + b


def _ffn_forward(s):
    if own:
        from superresolution_amd import ops
        res = None if s["res"] is None else ops.Planes.wrap(s["res"])
        return ops.gated_ffn(ops.Planes.wrap(s["x"]), s["w_gate"], s["w_up"], s["w_down"], b_gate=s["b_gate"], b_up=s["b_up"], b_down=s["b_down"],
                             act=_own_act(s), res=res, res_scale=s["res_scale"]).buf
    x = _rows(s["x"]).flatten(0, 1)
    hid = _act(_linear(x, s["w_gate"], s["b_gate"]), s["case"]["act"])[0] * _linear(x, s["w_up"], s["b_up"])
    y = s["res_scale"] * _linear(hid, s["w_down"], s["b_down"])
    if s["res"] is not None:
        y = _rows(s["res"]).flatten(0, 1) + y
    return _back(y, s["x"])


def _ffn_backward(s):
    if own:
        from superresolution_amd import ops
        g = ops.gated_ffn_backward(ops.Planes.wrap(s["x"]), ops.Planes.wrap(s["d_out"]), s["w_gate"], s["w_up"], s["w_down"], b_gate=s["b_gate"],
                                   b_up=s["b_up"], b_down=s["b_down"], act=_own_act(s), res_scale=s["res_scale"])
        return {k: v.buf if isinstance(v, ops.Planes) else v for k, v in g.items() if v is not None}
    x, dy = _rows(s["x"]).flatten(0, 1), s["res_scale"] * _rows(s["d_out"]).flatten(0, 1)
    u = _linear(x, s["w_up"], s["b_up"])
    act, slope = _act(_linear(x, s["w_gate"], s["b_gate"]), s["case"]["act"])
    dh = dy @ s["w_down"].float()
    dg, du = dh * u * slope, dh * act
    dt = s["x"].dtype
    found = {"dx": _back(dg @ s["w_gate"].float() + du @ s["w_up"].float(), s["x"]), "d_w_gate": (dg.t() @ x).to(dt), "d_w_up": (du.t() @ x).to(dt),
             "d_w_down": (dy.t() @ (act * u)).to(dt)}
    if s["b_gate"] is not None:
        found.update(d_b_gate=dg.sum(0), d_b_up=du.sum(0), d_b_down=dy.sum(0))
    return found


def _own_act(s):
    from superresolution_amd import _lib
    return {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "relu": _lib.ACT_RELU, "none": _lib.ACT_NONE}[s["case"]["act"]]


# ---- what a pass has to read, write and compute -----------------------------------------------------------------------
def work(case):
    m, c = case["n"] * case["h"] * case["w"], case["c"]
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("norm"):
        ts = 4 if case["trunk"] == "f32" else 2
        # forward: x, y -> sum, out; backward: x, y, d_sum, d_out -> dx, dy
        if case["op"] == "norm_fwd":
            return {"bytes": m * c * 2 * (es + ts), "flops": m * c * 16}
        return {"bytes": m * c * 3 * (es + ts), "flops": m * c * 40}
    f = case["hidden"]
    if case["op"] == "ffn_fwd":
        return {"bytes": m * c * es * (3 if case["res"] else 2) + 3 * c * f * es, "flops": 6 * m * c * f}
    # the gate, up and down products again, then the gradients of the inputs and of the three weights
    return {"bytes": m * c * es * 3 + 6 * c * f * es, "flops": 16 * m * c * f}


# ---- the same from the definition, in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    n, h, w, c = case["n"], case["h"], case["w"], case["c"]

    def wide(t):
        return None if t is None else t.double()

    def pixels(buf):  # [n][h][w][c]
        return wide(buf).movedim(1, 3).reshape(n, h, w, c)

    def stored(v, like):
        k = like.shape[-1]
        return v.reshape(n, h, w, c // k, k).movedim(3, 1)

    if case["op"].startswith("norm"):
        def norm(v, wb):
            if case["kind"] == "layer":
                v = v - v.sum(-1, keepdim=True) / c
            v = v / torch.sqrt((v * v).sum(-1, keepdim=True) / c + EPS) * wb["weight"]
            return v if wb["bias"] is None else v + wb["bias"]

        leaf = {"x": pixels(s["x"]), "y": pixels(s["y"]), "gate": wide(s["gate"])}
        for side in ("post", "pre"):
            leaf[side + "_weight"], leaf[side + "_bias"] = (None, None) if s[side] is None else (wide(s[side][0]), wide(s[side][1]))
        if case["op"] == "norm_bwd":
            leaf = {k: None if v is None else v.requires_grad_() for k, v in leaf.items()}
        v = leaf["y"]
        if s["post"] is not None:
            v = norm(v, {"weight": leaf["post_weight"], "bias": leaf["post_bias"]})
        if leaf["gate"] is not None:
            v = v * (leaf["gate"] if leaf["gate"].dim() == 1 else leaf["gate"].reshape(n, 1, 1, c))
        total = leaf["x"] + s["res_scale"] * v
        out = norm(total, {"weight": leaf["pre_weight"], "bias": leaf["pre_bias"]})
        if case["op"] == "norm_fwd":
            return {"sum": stored(total, s["x"]), "out": stored(out, s["y"])}
        torch.autograd.backward([total, out], [pixels(s["d_sum"]), pixels(s["d_out"])])
        names = {"gate": "d_gate", "post_weight": "d_post_weight", "post_bias": "d_post_bias", "pre_weight": "d_pre_weight", "pre_bias": "d_pre_bias"}
        found = {"dx": stored(leaf["x"].grad, s["x"]), "dy": stored(leaf["y"].grad, s["y"])}
        found.update({v: leaf[k].grad for k, v in names.items() if leaf[k] is not None})
        return found

    names = ("w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")
    leaf = {k: wide(s[k]) for k in names}
    leaf["x"] = pixels(s["x"]).reshape(-1, c)
    if case["op"] == "ffn_bwd":
        leaf = {k: None if v is None else v.requires_grad_() for k, v in leaf.items()}

    def layer(v, which):
        r = torch.mm(v, leaf["w_" + which].T)
        return r if leaf["b_" + which] is None else r + leaf["b_" + which]

    a = layer(leaf["x"], "gate")
    act = {"silu": lambda t: t / (1.0 + torch.exp(-t)), "gelu": lambda t: t * torch.special.erfc(-t / math.sqrt(2.0)) / 2.0,
           "relu": lambda t: torch.where(t > 0, t, torch.zeros_like(t)), "none": lambda t: t}[case["act"]]
    y = s["res_scale"] * layer(act(a) * layer(leaf["x"], "up"), "down")
    if case["op"] == "ffn_fwd":
        if s["res"] is not None:
            y = y + pixels(s["res"]).reshape(-1, c)
        return stored(y, s["x"])
    y.backward(pixels(s["d_out"]).reshape(-1, c))
    found = {"dx": stored(leaf["x"].grad, s["x"])}
    found.update({"d_" + k: leaf[k].grad for k in names if leaf[k] is not None})
    return found
