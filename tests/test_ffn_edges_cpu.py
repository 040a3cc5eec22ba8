"""Host side of layer_norm, gated_linear and the 8-bit activations where it can go wrong (no GPU needed)."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

import recsdk_amd  # noqa: F401
from oracle import ffn_oracle as FO
from recsdk_amd import _capi
from tests.ffn_cases import INSTANCES, described

M = torch.ops.mxrec
BF = torch.bfloat16


def test_forward_mode_tangents_are_refused():
    """A result without a tangent would count as a constant: every op refuses an input that carries one, with and without gradients
    being recorded, and serves it where forward mode is switched off (which here ends at the missing CPU implementation)."""
    x, w, one = torch.randn(8, 64).to(BF), torch.randn(64, 64).to(BF), torch.ones(64, dtype=BF)
    do, stat = torch.randn(8, 32).to(BF), torch.ones(8)
    z, low = torch.zeros(8, 1, 2, 32, dtype=BF), torch.zeros(8, 2, 32, dtype=torch.uint8)
    with fwd_ad.dual_level():
        d = lambda t: fwd_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: M.layer_norm(d(x), one, one), lambda: M.layer_norm(x, d(one), None), lambda: M.layer_norm(x, None, d(one)),
                 lambda: M.layer_norm(d(x.clone().requires_grad_(True)), one, one), lambda: M.layer_norm_forward(d(x), one, one),
                 lambda: M.layer_norm_backward(d(x), x, one, stat, stat), lambda: M.layer_norm_backward(x, d(x), one, stat, stat),
                 lambda: M.layer_norm_backward(x, x, one, d(stat), stat), lambda: M.gated_linear(d(x), w), lambda: M.gated_linear(x, d(w)),
                 lambda: M.gated_linear(x, w, d(one), "gelu", True), lambda: M.gated_linear_forward(x, d(w)),
                 lambda: M.gated_linear_backward(d(do), x, w, z, low), lambda: M.gated_linear_backward(do, x, w, d(z), low), lambda: M.activation_pack8(d(x))]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
                call()
        dual = d(x)
        with fwd_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="no CPU implementation"):
            M.layer_norm(dual, one, one)
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            M.layer_norm(x, one, one)


def test_the_sizes_of_the_gpu_tests_reach_every_instance():
    """Every kernel that a product can take: forward, d_x and d_weight in each tile and type, the backward's with one share of the
    contraction and with more (fp32 has no 128 x 128 with four buffers, and its 256 x 256 no shares), few rows in each number of row blocks."""
    for code, name in ((_capi.HSTU_BF16, "bf16"), (_capi.HSTU_F16, "f16"), (_capi.HSTU_F32, "f32")):
        tiles = ["256x256", "128x128", "256x128", "64x128"] + ["128x128_deep"] * (name != "f32")
        want = {f"rows_{name}_{r}" for r in (16, 32, 48, 64)} | {f"tiles_{name}_{t}" for t in tiles}
        want |= {f"{op}_{name}_{t}_{s}" for op in ("dx", "dw") for t in tiles for s in "1n" if not (name == "f32" and t == "256x256" and s == "n")}
        assert want == {d for size in INSTANCES for d in described(*size, code)}


def test_described_kernels():
    L = _capi.lib()
    assert described(16384, 1024, 4096, _capi.HSTU_BF16) == ("tiles_bf16_256x256", "dx_bf16_256x256_1", "dw_bf16_256x256_n")
    assert described(1, 512, 2048, _capi.HSTU_BF16)[0] == "rows_bf16_16" and described(48, 1024, 4096, _capi.HSTU_F16)[0] == "rows_f16_48"
    p = _capi.HstuGatedParams(struct_size=C.sizeof(_capi.HstuGatedParams), dtype=0, bias_dtype=0, k=8, f=8, m=1, x_stride=8, x=16, weight=16, out=16)
    buf = C.create_string_buffer(8)
    assert L.hstu_hip_gated_linear_describe_kernel(C.byref(p), buf, 8) == 0 and buf.value == b"rows_f3"      # cut, and ended
    assert L.hstu_hip_gated_linear_describe_kernel(C.byref(p), None, 8) == -1 and L.hstu_hip_gated_linear_describe_kernel(None, buf, 8) == -1
    assert L.hstu_hip_gated_linear_backward_describe_kernel(None, buf, 8) == -1
    p.k = 0
    assert L.hstu_hip_gated_linear_describe_kernel(C.byref(p), buf, 8) == -1


def test_packing_again_changes_no_value_but_may_change_the_codes():
    """225 rounds down to 224 = 448 / 2, which the next exponent below holds."""
    x = torch.tensor([[225.0, -13.0, 0.3, 2.0 ** -9, 100.0]])
    vals, exps = FO.pack8(x)
    back = FO.unpack8(vals, exps, torch.float32)
    again, exps2 = FO.pack8(back)
    assert float(vals[0, 0]) == 224.0 and int(exps[0, 0]) == 127 and float(again[0, 0]) == 448.0 and int(exps2[0, 0]) == 126
    assert torch.equal(FO.unpack8(again, exps2, torch.float32), back) and torch.equal(again, 2 * vals)
