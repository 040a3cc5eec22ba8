"""layer_norm, gated_linear and the 8-bit activations where they can go wrong: extreme rows, what lies behind the last column,
forward-mode tangents, every instance of the products, missing parameters, far offsets.  Tolerances as in test_ffn_gpu.py."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

import recsdk_amd  # noqa: F401
from tests.test_ffn_gpu import BF, EPS, M, say

pytestmark = pytest.mark.gpu


# ---- forward-mode tangents ---------------------------------------------------------------------------------------------------

def test_forward_mode_tangents_are_refused_not_lost():
    x, w = torch.randn(8, 64, device="cuda", dtype=BF), torch.randn(64, 64, device="cuda", dtype=BF)
    one = torch.ones(64, device="cuda", dtype=BF)
    y, mean, rstd = M.layer_norm_forward(x, one, one, EPS)
    out, *kept = M.gated_linear_forward(x, w)
    codes, exps = M.activation_pack8(x)
    with fwd_ad.dual_level():
        d = lambda t: fwd_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: M.layer_norm(d(x), one, one, EPS), lambda: M.layer_norm(x, d(one), None, EPS), lambda: M.layer_norm(x, None, d(one), EPS),
                 lambda: M.layer_norm_forward(d(x), one, one, EPS), lambda: M.layer_norm_backward(d(y), x, one, mean, rstd),
                 lambda: M.layer_norm_backward(y, x, one, d(mean), rstd), lambda: M.layer_norm(d(x.clone().requires_grad_(True)), one, one, EPS),
                 lambda: M.gated_linear(d(x), w), lambda: M.gated_linear(x, d(w)), lambda: M.gated_linear(x, w, d(one), "gelu", True),
                 lambda: M.gated_linear_forward(x, d(w)), lambda: M.gated_linear_backward(d(out), x, w, *kept), lambda: M.activation_pack8(d(x)),
                 lambda: M.gated_linear(d(x.clone().requires_grad_(True)), w)]
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
                say("not refused", i)           # (the call before this line is the one that raises)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
                say("not refused without gradients", i)
        # of an upstream gradient
        for fn in (lambda t: M.layer_norm(t, one, one, EPS), lambda t: M.gated_linear(t, w)):
            leaf = x.clone().requires_grad_(True)
            r = fn(leaf)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(r, leaf, d(torch.ones_like(r)))
        # tensors without a tangent are served as ever, and a dual tensor where the mode is off
        assert torch.equal(M.layer_norm(x, one, one, EPS), y) and torch.equal(M.gated_linear(x, w), out)
        dual = d(x)
        with fwd_ad._set_fwd_grad_enabled(False):
            assert torch.equal(M.layer_norm(dual, one, one, EPS), y) and torch.equal(M.gated_linear(dual, w), out)
    for fn in (lambda t: M.layer_norm(t, one, one, EPS), lambda t: M.gated_linear(t, w)):
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(fn, (x,), (torch.ones_like(x),))
    assert torch.equal(M.activation_unpack8(codes, exps, BF), M.activation_unpack8(codes.clone(), exps, BF))
