"""Host side of layer_norm, gated_linear and the 8-bit activations (no GPU needed): the oracle's pins, schemas, refusals of the
torch ops and of the C ABI, workspace sizes."""
import ctypes as C

import pytest
import torch

import recsdk_amd  # noqa: F401
from oracle import ffn_oracle as FO
from recsdk_amd import _capi

M = torch.ops.mxrec


def _g(seed=0):
    return torch.Generator().manual_seed(seed)


# ---- oracle pins -------------------------------------------------------------------------------------------------------

def test_oracle_layer_norm_is_the_library_function_and_its_gradient():
    g = _g()
    x = torch.randn(7, 33, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(33, generator=g, dtype=torch.float64, requires_grad=True)
    b = torch.randn(33, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(7, 33, generator=g, dtype=torch.float64)
    y, mean, rstd = FO.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5)
    ref = torch.nn.functional.layer_norm(x, (33,), w, b, 1e-5)
    assert torch.allclose(y, ref, rtol=0, atol=1e-13)
    want = torch.autograd.grad(ref, (x, w, b), dy)
    got = FO.layer_norm_backward(dy, x.detach(), w.detach(), mean, rstd)
    for a, c in zip(got, want):
        assert torch.allclose(a, c, rtol=0, atol=1e-12)


@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_oracle_gated_linear_is_autograd_and_differences(name):
    g = _g(1)
    x = torch.randn(5, 9, generator=g, dtype=torch.float64)
    w = torch.randn(14, 9, generator=g, dtype=torch.float64)
    b = torch.randn(14, generator=g, dtype=torch.float64)
    do = torch.randn(5, 7, generator=g, dtype=torch.float64)
    lib = torch.nn.functional.silu if name == "silu" else torch.nn.functional.gelu

    def f(x, w, b):
        z = torch.nn.functional.linear(x, w, b)
        return lib(z[:, :7]) * z[:, 7:]

    out, z = FO.gated_linear(x, w, b, name)
    assert torch.allclose(out, f(x, w, b), rtol=0, atol=1e-13)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(f(*leaves), leaves, do)
    got = FO.gated_linear_backward(do, x, w, z, name)
    for a, c in zip(got, want):
        assert torch.allclose(a, c, rtol=0, atol=1e-12)
    # central differences of the scalar sum(out * do) in a few directions
    for k, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        lo, hi = [(x, w, b)[i] if i != k else t - h * d for i in range(3)], [(x, w, b)[i] if i != k else t + h * d for i in range(3)]
        num = float(((FO.gated_linear(*hi, name)[0] - FO.gated_linear(*lo, name)[0]) * do).sum()) / (2 * h)
        # third derivatives of order 100 at h^2 = 1e-10, rounding 1e-16 * 100 / h
        assert abs(num - float((got[k] * d).sum())) < 1e-7


def test_oracle_pack8_is_torchs_float8_under_a_power_of_two():
    g = _g(2)
    x = torch.randn(40, 75, generator=g) * torch.exp(4 * torch.randn(40, 1, generator=g))
    x[0], x[1, :32], x[2, 3], x[3, 70] = 0.0, 448.0 * 2.0 ** -7, float("inf"), float("nan")
    x[4] = 2.0 ** -140
    x[5, :] = torch.finfo(torch.float32).max
    vals, exps = FO.pack8(x)
    for gi in range(3):
        v, e = x[:, 32 * gi:32 * gi + 32], exps[:, gi].to(torch.int64) - 127
        top = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dim=1).double()
        unit = torch.ldexp(torch.ones(40, dtype=torch.float64), e)
        assert bool((top <= 448 * unit).all()) and bool(((top > 224 * unit) | (e == -126)).all())
        scaled = torch.where(torch.isfinite(v), v.double() / unit[:, None], torch.full_like(v, float("nan"), dtype=torch.float64))
        want = scaled.float().to(torch.float8_e4m3fn).double()
        assert torch.equal(vals[:, 32 * gi:32 * gi + 32].nan_to_num(777.0), want.nan_to_num(777.0))
    back = FO.unpack8(vals, exps, torch.float32)
    fin = torch.isfinite(x)
    unit = torch.ldexp(torch.ones(exps.shape, dtype=torch.float64), exps.to(torch.int64) - 127).repeat_interleave(32, dim=1)[:, :75]
    assert bool(((back - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, unit * 2.0 ** -10))[fin].all())
    assert bool(torch.isnan(back[~fin]).all())
    # again: nothing changes
    again = FO.pack8(back)
    assert torch.equal(FO.unpack8(*again, torch.float32).nan_to_num(777.0), back.nan_to_num(777.0))


# ---- schemas and refusals of the torch ops ---------------------------------------------------------------------------------

def test_schemas():
    assert str(M.layer_norm.default._schema) == "mxrec::layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps=1.0000000000000001e-05) -> Tensor"
    assert str(M.gated_linear.default._schema).startswith("mxrec::gated_linear(Tensor x, Tensor weight, Tensor? bias=None, str activation=")
    assert str(M.activation_pack8.default._schema) == "mxrec::activation_pack8(Tensor x) -> Tensor[]"
    assert str(M.activation_unpack8.default._schema) == "mxrec::activation_unpack8(Tensor codes, Tensor exponents, ScalarType dtype) -> Tensor"


def test_layer_norm_refusals():
    x, w = torch.zeros(8, 48, dtype=torch.float16), torch.zeros(48, dtype=torch.float16)
    run = lambda x_=x, w_=w, b_=w, eps=1e-5: M.layer_norm(x_, w_, b_, eps)
    for kw, text in ((dict(x_=torch.zeros((), dtype=torch.float16)), "at least 1 dimension"), (dict(x_=x.int()), "dtype expect float32, float16 or bfloat16"),
                     (dict(x_=torch.zeros(2, 16385, dtype=torch.float16)), "last dimension of x must in range"), (dict(x_=torch.zeros(2, 0, dtype=torch.float16)), "must in range"),
                     (dict(w_=w[:40]), "weight must be 1D"), (dict(b_=w[None]), "bias must be 1D"), (dict(w_=w.double()), "weight dtype expect"),
                     (dict(w_=w.bfloat16(), b_=w.bfloat16()), "weight dtype expect"), (dict(w_=w.float()), "must have one dtype"), (dict(eps=0.0), "eps must be positive"),
                     (dict(eps=-1.0), "eps must be positive"), (dict(eps=float("nan")), "eps must be positive"), (dict(eps=1e-60), "eps must be positive"),
                     (dict(eps=float("inf")), "eps must be positive"), (dict(), "no CPU implementation"), (dict(w_=None, b_=None), "no CPU implementation")):
        with pytest.raises(RuntimeError, match=text):
            run(**kw)
    with pytest.raises(RuntimeError, match="d_out must have the shape"):
        M.layer_norm_backward(x[:4], x, w, torch.zeros(8), torch.zeros(8))
    with pytest.raises(RuntimeError, match="mean and rstd must be float32"):
        M.layer_norm_backward(x, x, w, torch.zeros(7), torch.zeros(8))


def test_gated_linear_refusals():
    x, w, b = torch.zeros(6, 24, dtype=torch.bfloat16), torch.zeros(20, 24, dtype=torch.bfloat16), torch.zeros(20, dtype=torch.bfloat16)
    run = lambda x_=x, w_=w, b_=b, act="silu", c8=False: M.gated_linear(x_, w_, b_, act, c8)
    for kw, text in ((dict(x_=x[0, 0]), "at least 1 dimension"), (dict(x_=x.long()), "dtype expect"), (dict(w_=w[0]), "weight must be 2D"),
                     (dict(w_=w[:, :16]), "weight dim\\[1\\] must equal"), (dict(w_=w[:19]), "twice a number"), (dict(w_=w[:0]), "twice a number"),
                     (dict(w_=w.half()), "weight must have the dtype of x"), (dict(b_=b[:10]), "bias must be 1D"), (dict(b_=b.half()), "bias dtype expect"),
                     (dict(act="relu"), "activation expect 'silu' or 'gelu'"), (dict(x_=x.float(), w_=w.float(), b_=b.float(), c8=True), "checkpoint8 needs"),
                     (dict(x_=torch.zeros(2, 16385, dtype=torch.bfloat16), w_=torch.zeros(2, 16385, dtype=torch.bfloat16)), "last dimension of x must in range"),
                     (dict(), "no CPU implementation"), (dict(b_=None), "no CPU implementation"), (dict(b_=b.float()), "no CPU implementation")):
        with pytest.raises(RuntimeError, match=text):
            run(**kw)
    z = torch.zeros(6, 1, 2, 32, dtype=torch.bfloat16)             # what the forward keeps: a block of 2 x 32 columns for f = 10
    c = torch.zeros(6, 2, 32).to(torch.float8_e4m3fn)
    do = torch.zeros(6, 10, dtype=torch.bfloat16)
    for args, text in (((do[:5], x, w, z), "d_out must have"), ((do.float(), x, w, z), "d_out must have"), ((do, x, w, z[:5]), "z must be"),
                       ((do, x, w, z.float()), "z must be"), ((do, x, w, z), "z_aux must be"), ((do, x, w, z, torch.zeros(6, 2, 1, dtype=torch.uint8)), "z_aux must be"),
                       ((do, x, w, z, torch.zeros(6, 2, 32)), "z_aux must be"), ((do, x, w, c, torch.zeros(6, 1, dtype=torch.uint8)), "z_aux must be"),
                       ((do, x, w, z, torch.zeros(6, 2, 32, dtype=torch.uint8)), "no CPU implementation"),
                       ((do, x, w, c, torch.zeros(6, 2, 1, dtype=torch.uint8)), "no CPU implementation"),
                       ((do.float(), x.float(), w.float(), c.float()), "no CPU implementation")):
        with pytest.raises(RuntimeError, match=text):
            M.gated_linear_backward(*args)


def test_pack8_refusals():
    x = torch.zeros(4, 40, dtype=torch.float16)
    for t, text in ((x[0, 0], "at least 1 dimension"), (x.int(), "dtype expect"), (torch.zeros(1, 65537, dtype=torch.float16), "must in range"), (x, "no CPU implementation")):
        with pytest.raises(RuntimeError, match=text):
            M.activation_pack8(t)
    c, e = x.to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8)
    for args, text in (((x, e, torch.float16), "codes must be float8_e4m3fn"), ((c, e[:, :1], torch.float16), "exponents must be uint8"), ((c, e.int(), torch.float16), "exponents must be uint8"),
                       ((c, e, torch.float64), "dtype expect"), ((c, e, torch.float16), "no CPU implementation")):
        with pytest.raises(RuntimeError, match=text):
            M.activation_unpack8(*args)


# ---- C ABI -----------------------------------------------------------------------------------------------------------------

def _fill(cls, **over):
    p = cls()
    p.struct_size = C.sizeof(cls)
    base = dict(dtype=_capi.HSTU_BF16, param_dtype=_capi.HSTU_BF16, grad_dtype=_capi.HSTU_BF16, bias_dtype=_capi.HSTU_BF16, grad_bias_dtype=_capi.HSTU_BF16,
                rows=100, cols=512, x_stride=512, dy_stride=512, eps=1e-5, m=100, k=512, f=256, dout_stride=256, act=0, keep=1)
    for name, typ in cls._fields_:
        if name in over:
            setattr(p, name, over[name])
        elif typ is C.c_void_p:
            setattr(p, name, 0x10000)
        elif name in base:
            setattr(p, name, base[name])
    return p


def _err():
    return _capi.lib().hstu_hip_last_error().decode()


def test_c_abi_layer_norm():
    L, P, B = _capi.lib(), _capi.HstuLayerNormParams, _capi.HstuLayerNormBwdParams
    assert L.hstu_hip_layer_norm(None, None) == -1 and "NULL" in _err()
    for over, rc, text in ((dict(struct_size=3), -1, "size mismatch"), (dict(dtype=3), -1, "dtype expect"), (dict(param_dtype=_capi.HSTU_F16), -1, "param_dtype expect"),
                           (dict(rows=-1), -1, "rows must in range"), (dict(rows=(1 << 30) + 1), -1, "rows must in range"), (dict(cols=0), -1, "cols must in range"),
                           (dict(cols=16385), -1, "cols must in range"), (dict(eps=0.0), -1, "eps must be positive"), (dict(eps=float("nan")), -1, "eps must be positive"),
                           (dict(eps=float("inf")), -1, "eps must be positive"), (dict(x_stride=-1), -1, "x_stride"), (dict(mean=None), -1, "mean and rstd"),
                           (dict(x=None), -1, "must not be NULL"), (dict(y=None), -1, "must not be NULL"), (dict(x=0x10001), -2, "aligned"),
                           (dict(param_dtype=0, weight=0x10002), -2, "aligned"), (dict(rows=0, x=None, y=None), 0, "")):
        p = _fill(P, **over)
        assert L.hstu_hip_layer_norm(C.byref(p), None) == rc and text in (_err() if rc else ""), (over, _err())
    n = C.c_uint64(0)
    for over, rc, text in ((dict(grad_dtype=_capi.HSTU_F16), -1, "grad_dtype expect"), (dict(dy_stride=-1), -1, "dy_stride"), (dict(d_y=None), -1, "must not be NULL"),
                           (dict(d_x=0x10001), -2, "aligned")):
        p = _fill(B, **over)
        assert L.hstu_hip_layer_norm_backward_get_workspace_size(C.byref(p), C.byref(n)) == rc and text in _err(), (over, _err())
        assert L.hstu_hip_layer_norm_backward(C.byref(p), 0x10000, 1 << 30, None) == rc
    p = _fill(B)
    assert L.hstu_hip_layer_norm_backward_get_workspace_size(C.byref(p), None) == -1
    assert L.hstu_hip_layer_norm_backward_get_workspace_size(C.byref(p), C.byref(n)) == 0 and n.value == 7 * 2 * 512 * 4   # 16 rows a workgroup
    assert L.hstu_hip_layer_norm_backward(C.byref(p), None, 0, None) == -3 and "workspace" in _err()
    assert L.hstu_hip_layer_norm_backward(C.byref(p), 0x10004, 1 << 30, None) == -3
    p = _fill(B, d_weight=None, d_bias=None)
    assert L.hstu_hip_layer_norm_backward_get_workspace_size(C.byref(p), C.byref(n)) == 0 and n.value == 0
    p = _fill(B, d_weight=None, d_bias=None, d_x=None)
    assert L.hstu_hip_layer_norm_backward(C.byref(p), None, 0, None) == 0      # nothing wanted, nothing launched


def test_c_abi_gated_linear():
    L, P, B = _capi.lib(), _capi.HstuGatedParams, _capi.HstuGatedBwdParams
    n = C.c_uint64(0)
    for over, rc, text in ((dict(struct_size=3), -1, "size mismatch"), (dict(dtype=3), -1, "dtype expect"), (dict(bias_dtype=_capi.HSTU_F16), -1, "bias_dtype expect"),
                           (dict(act=2), -1, "act expect"), (dict(keep=3), -1, "keep expect"), (dict(keep=2, dtype=0, bias_dtype=0), -1, "8-bit checkpoints need"),
                           (dict(m=-1), -1, "x dim0"), (dict(k=0), -1, "x dim1"), (dict(k=16385), -1, "x dim1"), (dict(f=0), -1, "weight dim0"), (dict(f=32769), -1, "weight dim0"),
                           (dict(x_stride=-1), -1, "x_stride"), (dict(x=None), -1, "must not be NULL"), (dict(z=None), -1, "z (and z_aux"),
                           (dict(keep=2, z_aux=None), -1, "z (and z_aux"), (dict(z_aux=None), -1, "z (and z_aux"), (dict(out=0x10001), -2, "aligned"), (dict(m=0, x=None), 0, "")):
        p = _fill(P, **over)
        assert L.hstu_hip_gated_linear_get_workspace_size(C.byref(p), C.byref(n)) == rc and (rc == 0 or text in _err()), (over, _err())
        assert L.hstu_hip_gated_linear(C.byref(p), 0x10000, 1 << 40, None) == rc
    p = _fill(P)
    assert L.hstu_hip_gated_linear_get_workspace_size(C.byref(p), C.byref(n)) == 0 and n.value == 0
    # rows that do not lie on 16-byte boundaries are brought there in the workspace
    p = _fill(P, k=509, x_stride=509)
    assert L.hstu_hip_gated_linear_get_workspace_size(C.byref(p), C.byref(n)) == 0 and n.value >= (100 + 512) * 512 * 2
    assert L.hstu_hip_gated_linear(C.byref(p), 0x10000, n.value - 1, None) == -3 and "workspace" in _err()
    for over, rc, text in ((dict(keep=0), -1, "keep expect 1 or 2"), (dict(grad_bias_dtype=_capi.HSTU_F16), -1, "grad_bias_dtype expect"), (dict(dout_stride=-1), -1, "dout_stride"),
                           (dict(d_out=None), -1, "must not be NULL"), (dict(x=None), -1, "for d_weight"), (dict(weight=None), -1, "for d_x"), (dict(d_x=0x10001), -2, "aligned")):
        p = _fill(B, **over)
        assert L.hstu_hip_gated_linear_backward_get_workspace_size(C.byref(p), C.byref(n)) == rc and text in _err(), (over, _err())
        assert L.hstu_hip_gated_linear_backward(C.byref(p), 0x10000, 1 << 40, None) == rc
    p = _fill(B)
    assert L.hstu_hip_gated_linear_backward_get_workspace_size(C.byref(p), C.byref(n)) == 0 and n.value >= 100 * 512 * 2
    assert L.hstu_hip_gated_linear_backward(C.byref(p), None, 0, None) == -3
    p = _fill(B, d_x=None, d_weight=None, d_bias=None)
    assert L.hstu_hip_gated_linear_backward_get_workspace_size(C.byref(p), C.byref(n)) == 0 and n.value == 0
    assert L.hstu_hip_gated_linear_backward(C.byref(p), None, 0, None) == 0


def test_c_abi_pack8():
    L, P = _capi.lib(), _capi.HstuPack8Params
    for fn in (L.hstu_hip_activation_pack8, L.hstu_hip_activation_unpack8):
        for over, rc, text in ((dict(struct_size=3), -1, "size mismatch"), (dict(dtype=3), -1, "dtype expect"), (dict(rows=-1), -1, "rows must in range"), (dict(cols=0), -1, "cols must in range"),
                               (dict(cols=65537), -1, "cols must in range"), (dict(x_stride=-1), -1, "x_stride"), (dict(codes=None), -1, "must not be NULL"), (dict(x=0x10001), -2, "aligned")):
            p = _fill(P, **over)
            assert fn(C.byref(p), None) == rc and text in _err(), (over, _err())
        p = _fill(P, rows=0, x=None)
        assert fn(C.byref(p), None) == 0
    p = _fill(P, x_stride=511)
    assert L.hstu_hip_activation_unpack8(C.byref(p), None) == -1 and "at least cols" in _err()


def test_c_abi_refuses_what_one_launch_does_not_hold():
    """A launch holds less than 2^32 threads: the largest rows by the largest columns are refused before anything is launched."""
    L = _capi.lib()
    rows = 1 << 30
    for fn in (L.hstu_hip_activation_pack8, L.hstu_hip_activation_unpack8):
        p = _fill(_capi.HstuPack8Params, rows=rows, cols=65536, x_stride=65536)
        assert fn(C.byref(p), None) == -2 and "too large for one launch" in _err()
    p = _fill(_capi.HstuGatedParams, m=rows, k=512, x_stride=512, f=32768)
    assert L.hstu_hip_gated_linear(C.byref(p), 0x10000, 1 << 62, None) == -2 and "too large for one launch" in _err()
    p = _fill(_capi.HstuGatedBwdParams, m=rows, k=16384, x_stride=16384, f=32, dout_stride=32)
    assert L.hstu_hip_gated_linear_backward(C.byref(p), 0x10000, 1 << 62, None) == -2 and "too large for one launch" in _err()
