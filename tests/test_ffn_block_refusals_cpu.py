"""What block_norm and gated_ffn refuse.  The C entry points check everything before they touch the GPU, so their refusals run
here on made-up addresses; the reference form's gradients are checked against differences as well."""
import ctypes as C

import pytest
import torch

from superresolution_amd import _lib, ops
from tests import ffn_block_ref as R

F32, F16, BF16, I8 = _lib.F32, _lib.F16, _lib.BF16, _lib.I8
L = _lib.lib()


def view(ptr, dt, c=64, hw=64):
    t = _lib.Tensor()
    cpb = ops.cpb(dt)
    t.ptr, t.dtype, t.plane_stride, t.img_stride = ptr, dt, hw * cpb, hw * c
    return t


def norm_desc(grad=False):
    d = _lib.BlockNormGradDesc() if grad else _lib.BlockNormDesc()
    d.n, d.h, d.w, d.c, d.kind, d.gate_per_image, d.eps, d.res_scale = 2, 8, 8, 64, _lib.NORM_LAYER, 1, 1e-5, 1.0
    d.x, d.y = view(0x1000, F16), view(0x2000, F16)
    d.post_weight, d.post_bias, d.pre_weight, d.pre_bias, d.gate = 0x5000, 0x6000, 0x7000, 0x8000, 0x9000
    if grad:
        d.d_sum, d.d_out, d.dx, d.dy = (view(p, F16) for p in (0x3000, 0x4000, 0xa000, 0xb000))
        d.d_post_weight, d.d_post_bias, d.d_pre_weight, d.d_pre_bias, d.d_gate = 0xc000, 0xd000, 0xe000, 0xf000, 0x10000
    else:
        d.sum, d.out = view(0x3000, F16), view(0x4000, F16)
    return d


def refused(rc, words):
    assert rc == -1
    msg = L.srmi_last_error().decode()
    assert words in msg, msg


NORM_BAD = [(dict(n=0), "bad shape"), (dict(h=-1), "bad shape"), (dict(c=0), "bad shape"), (dict(c=20), "bad shape"), (dict(c=1040), "bad shape"),
            (dict(c=24), "plane width"), (dict(n=1 << 16, h=1 << 8, w=1 << 8), "2^31"), (dict(kind=2), "kind"), (dict(eps=-1.0), "eps"),
            (dict(eps=float("nan")), "eps"), (dict(x=_lib.Tensor()), "no x"), (dict(x=view(0x1008, F16)), "16 bytes"), (dict(y=view(0x2002, F16)), "16 bytes"),
            (dict(y=view(0x2000, F32)), "type"), (dict(x=view(0x1000, BF16)), "type"), (dict(y=_lib.Tensor()), "not there"),
            (dict(post_weight=None), "post_bias without"), (dict(pre_weight=None), "pre_bias without")]


@pytest.mark.parametrize("change,words", NORM_BAD, ids=lambda v: str(v) if isinstance(v, str) else ",".join(v))
@pytest.mark.parametrize("grad", [False, True])
def test_block_norm_refuses(change, words, grad):
    d = norm_desc(grad)
    for k, v in change.items():
        setattr(d, k, v)
    ws = C.c_void_p(0x100000)
    refused(L.srmi_block_norm_backward(C.byref(d), ws, 1 << 40, None) if grad else L.srmi_block_norm(C.byref(d), None), words)


@pytest.mark.parametrize("change,words", [(dict(out=_lib.Tensor()), "out goes with"), (dict(sum=view(0x3000, F32)), "trunk"), (dict(out=view(0x4000, BF16)), "one type"),
                                          (dict(out=view(0x4000, I8)), "one type"), (dict(out=view(0x4004, F16)), "16 bytes")])
def test_block_norm_forward_refuses(change, words):
    d = norm_desc()
    for k, v in change.items():
        setattr(d, k, v)
    refused(L.srmi_block_norm(C.byref(d), None), words)


def test_block_norm_refuses_without_a_body():
    d = norm_desc()
    d.y, d.gate, d.post_weight, d.post_bias = _lib.Tensor(), None, None, None
    refused(L.srmi_block_norm(C.byref(d), None), "the sum is x")
    d.pre_weight = d.pre_bias = None
    refused(L.srmi_block_norm(C.byref(d), None), "neither")
    d = norm_desc()
    d.x = d.y = d.sum = d.out = view(0x1000, I8)
    refused(L.srmi_block_norm(C.byref(d), None), "f32, f16 or bf16")
    refused(L.srmi_block_norm(None, None), "null")


@pytest.mark.parametrize("change,words", [(dict(dx=_lib.Tensor()), "dx"), (dict(dy=_lib.Tensor()), "dx"), (dict(d_gate=None), "gradient's place"),
                                          (dict(d_pre_bias=None), "gradient's place"), (dict(d_out=_lib.Tensor()), "d_out goes with"),
                                          (dict(dx=view(0xa000, F32)), "trunk"), (dict(dy=view(0xb000, F32)), "one type")])
def test_block_norm_backward_refuses(change, words):
    d = norm_desc(True)
    for k, v in change.items():
        setattr(d, k, v)
    refused(L.srmi_block_norm_backward(C.byref(d), C.c_void_p(0x100000), 1 << 40, None), words)


def test_block_norm_backward_refuses_a_short_workspace():
    d = norm_desc(True)
    need = L.srmi_block_norm_backward_workspace(C.byref(d))
    assert need > 0
    refused(L.srmi_block_norm_backward(C.byref(d), C.c_void_p(0x100000), need - 1, None), "workspace")
    refused(L.srmi_block_norm_backward(C.byref(d), None, need, None), "workspace")
    refused(L.srmi_block_norm_backward(C.byref(d), C.c_void_p(0x100008), need, None), "workspace")
    d.c = 7
    assert L.srmi_block_norm_backward_workspace(C.byref(d)) == 0 and L.srmi_block_norm_backward_workspace(None) == 0


def ffn_desc(grad=False):
    d = _lib.GatedFfnGradDesc() if grad else _lib.GatedFfnDesc()
    d.dtype, d.n, d.h, d.w, d.c, d.hidden, d.act, d.res_scale = F16, 2, 8, 8, 64, 128, _lib.ACT_SILU, 1.0
    d.x = view(0x1000, F16)
    d.w_gate, d.w_up, d.w_down, d.b_gate, d.b_up, d.b_down = 0x4000, 0x5000, 0x6000, 0x7000, 0x8000, 0x9000
    if grad:
        d.d_out, d.dx = view(0x2000, F16), view(0x3000, F16)
        d.d_w_gate, d.d_w_up, d.d_w_down, d.d_b_gate, d.d_b_up, d.d_b_down = 0xa000, 0xb000, 0xc000, 0xd000, 0xe000, 0xf000
    else:
        d.res, d.out = view(0x2000, F16), view(0x3000, F16)
    return d


def ffn_call(d, ws=0x100000, size=1 << 40):
    f = L.srmi_gated_ffn_backward if isinstance(d, _lib.GatedFfnGradDesc) else L.srmi_gated_ffn
    return f(C.byref(d), C.c_void_p(ws), size, None)


@pytest.mark.parametrize("change,words", [(dict(dtype=I8), "compute type"), (dict(n=0), "bad shape"), (dict(w=-3), "bad shape"), (dict(c=72), "bad shape"),
                                          (dict(hidden=100), "bad shape"), (dict(c=4112), "bad shape"), (dict(hidden=16400), "bad shape"),
                                          (dict(n=1 << 15, h=1 << 8, w=1 << 8), "bad shape"), (dict(act=5), "activation"), (dict(act=-1), "activation"),
                                          (dict(x=_lib.Tensor()), "no x"), (dict(x=view(0x1000, F32)), "compute type"), (dict(x=view(0x1004, F16)), "16 bytes"),
                                          (dict(w_up=None), "null weight"), (dict(w_down=0x6008), "multiples of 16")])
@pytest.mark.parametrize("grad", [False, True])
def test_gated_ffn_refuses(change, words, grad):
    d = ffn_desc(grad)
    for k, v in change.items():
        setattr(d, k, v)
    refused(ffn_call(d), words)


def test_gated_ffn_refuses_outputs():
    for change, words in ((dict(out=_lib.Tensor()), "no out"), (dict(out=view(0x3000, BF16)), "compute type"), (dict(res=view(0x2000, F32)), "compute type"),
                          (dict(out=view(0x1000, F16)), "must not be x")):
        d = ffn_desc()
        for k, v in change.items():
            setattr(d, k, v)
        refused(ffn_call(d), words)
    for change, words in ((dict(dx=_lib.Tensor()), "no dx"), (dict(d_out=_lib.Tensor()), "no d_out"), (dict(d_w_up=None), "null weight"),
                          (dict(d_b_up=None), "gradient's place"), (dict(b_down=None), "gradient's place"), (dict(dx=view(0x2000, F16)), "must not be")):
        d = ffn_desc(True)
        for k, v in change.items():
            setattr(d, k, v)
        refused(ffn_call(d), words)


@pytest.mark.parametrize("grad", [False, True])
def test_gated_ffn_refuses_a_short_workspace(grad):
    d = ffn_desc(grad)
    d.n, d.h, d.w, d.c, d.hidden = 1, 64, 64, 512, 1024
    d.x = view(0x1000, F16, 512, 4096)
    need = (L.srmi_gated_ffn_backward_workspace if grad else L.srmi_gated_ffn_workspace)(C.byref(d))
    assert need > 0
    refused(ffn_call(d, size=need - 1), "workspace")
    refused(ffn_call(d, ws=0x100004, size=need), "workspace")
    refused(ffn_call(d, ws=0, size=need), "workspace")


def test_convolutions_refuse_the_block_activations():
    d = _lib.ConvDesc()
    d.dtype, d.n, d.h, d.w, d.cin, d.cout, d.cout_tile, d.act, d.ps_r = F16, 1, 8, 8, 64, 64, 64, _lib.ACT_SILU, 1
    d.inp, d.out, d.wpk, d.bias = view(0x1000, F16), view(0x2000, F16), 0x3000, 0x4000
    refused(L.srmi_conv3x3(C.byref(d), None), "activation")


# ---- the Python surface's own checks ------------------------------------------------------------------------------------
def test_python_checks():
    x = ops.Planes(1, 32, 4, 4, F16, device="cpu")
    w = torch.zeros(48, 32, dtype=torch.float16)
    down = torch.zeros(32, 48, dtype=torch.float16)
    with pytest.raises(_lib.SrmiError, match="on a GPU"):
        ops.gated_ffn(x, w, w, down)
    with pytest.raises(_lib.SrmiError, match="w_up"):
        ops.gated_ffn(x, w, w[:16], down)
    with pytest.raises(_lib.SrmiError, match="w_down"):
        ops.gated_ffn(x, w, w, w)
    with pytest.raises(_lib.SrmiError, match="w_gate"):
        ops.gated_ffn(x, w.float(), w, down)
    with pytest.raises(_lib.SrmiError, match="w_gate"):
        ops.gated_ffn(x, torch.zeros(32, 48, dtype=torch.float16).t(), w, down)
    with pytest.raises(_lib.SrmiError, match="b_gate"):
        ops.gated_ffn(x, w, w, down, b_gate=torch.zeros(47))
    one = torch.ones(32)
    with pytest.raises(_lib.SrmiError, match="on a GPU"):
        ops.block_norm(x, pre=(one, None))
    with pytest.raises(_lib.SrmiError, match="pre_weight"):
        ops.block_norm(x, pre=(one.half(), None))
    with pytest.raises(_lib.SrmiError, match="gate"):
        ops.block_norm(x, x, gate=torch.ones(2, 32))
    with pytest.raises(_lib.SrmiError, match="y is"):
        ops.block_norm(x, ops.Planes(1, 32, 4, 5, F16, device="cpu"))
    with pytest.raises(_lib.SrmiError, match="plane buffer"):
        ops.Planes.wrap(torch.zeros(1, 2, 4, 4, 8, dtype=torch.float16))
    with pytest.raises(_lib.SrmiError, match="plane buffer"):
        ops.Planes.wrap(torch.zeros(1, 2, 4, 4, 32, dtype=torch.float16)[..., ::2])
    p = ops.Planes.wrap(x.buf)
    assert (p.n, p.c, p.h, p.w, p.dtype) == (1, 32, 4, 4, F16) and p.buf is x.buf


def test_structs_have_the_size_of_the_header(tmp_path):
    import os
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"srmi_block_norm_desc_t": _lib.BlockNormDesc, "srmi_block_norm_grad_desc_t": _lib.BlockNormGradDesc,
             "srmi_gated_ffn_desc_t": _lib.GatedFfnDesc, "srmi_gated_ffn_grad_desc_t": _lib.GatedFfnGradDesc}
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "srmi355.h"\nint main(void){' + "".join(f'printf("%zu\\n", sizeof({n}));' for n in names) + "return 0;}")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    sizes = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in sizes] == [C.sizeof(t) for t in names.values()]


def test_packed_descriptors_fill_their_structs():
    for packed, t in ((ops._NORM, _lib.BlockNormDesc), (ops._NORM_GRAD, _lib.BlockNormGradDesc), (ops._FFN, _lib.GatedFfnDesc), (ops._FFN_GRAD, _lib.GatedFfnGradDesc)):
        assert packed.size == C.sizeof(t)
    x = ops.Planes(2, 32, 4, 5, F16, device="cpu")
    for c0 in (0, 16):
        v = x.view(c0)
        assert (v.ptr, v.img_stride, v.plane_stride, v.dtype, v.flags, v.qscale, v.reserved) == x.fields(c0)
    d = _lib.GatedFfnDesc.from_buffer_copy(ops._FFN.pack(F16, 2, 4, 5, 32, 48, _lib.ACT_GELU, 0.5, *x.fields(), *ops._NONE, *x.fields(), 1, 2, 3, 4, 5, 6))
    assert (d.dtype, d.n, d.h, d.w, d.c, d.hidden, d.act, d.res_scale) == (F16, 2, 4, 5, 32, 48, _lib.ACT_GELU, 0.5)
    assert d.x.ptr == x.buf.data_ptr() and d.res.ptr is None and d.out.plane_stride == 320
    assert (d.w_gate, d.w_up, d.w_down, d.b_gate, d.b_up, d.b_down) == (1, 2, 3, 4, 5, 6)


def test_reference_gradients_against_differences():
    """The plain forms the GPU tests trust: autograd's gradients along a direction against central differences in 64 bits."""
    gen = torch.Generator().manual_seed(0)
    x, y = R.rnd(gen, 2, 3, 16), R.rnd(gen, 2, 3, 16)
    w, g = 1 + R.rnd(gen, 16, scale=0.1), torch.sigmoid(R.rnd(gen, 2, 16))
    for kind in (_lib.NORM_LAYER, _lib.NORM_RMS):
        f = lambda x, y, w, g: (R.block_norm(x, y, (w, None), (w, w), g, 0.3, 1e-5, kind)[1] ** 2).sum()  # noqa: E731
        assert torch.autograd.gradcheck(f, [t.clone().requires_grad_() for t in (x, y, w, g)])
    wg, wu, wd = R.rnd(gen, 8, 16, scale=0.25), R.rnd(gen, 8, 16, scale=0.25), R.rnd(gen, 16, 8, scale=0.3)
    for act in (_lib.ACT_SILU, _lib.ACT_GELU, _lib.ACT_LRELU, _lib.ACT_NONE):
        f = lambda x, a, b, c: R.gated_ffn(x.reshape(-1, 16), a, b, c, None, None, None, act, None, 0.5)  # noqa: E731
        assert torch.autograd.gradcheck(f, [t.clone().requires_grad_() for t in (x, wg, wu, wd)])
