"""Host side of layer_norm, gated_linear and the 8-bit activations where it can go wrong (no GPU needed)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

import recsdk_amd  # noqa: F401

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
