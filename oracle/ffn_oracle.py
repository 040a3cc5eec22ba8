"""CPU oracle for ``mxrec::layer_norm``, ``mxrec::gated_linear`` and ``mxrec::activation_pack8`` in 64 bits.  TEST INFRASTRUCTURE ONLY.

The formulas of ``include/hstu_ffn.h`` restated; pinned in ``tests/test_ffn_cpu.py`` against torch's library functions,
autograd and central differences, and the 8-bit format against torch's own float8 conversion.
"""
from __future__ import annotations

import math

import torch

GROUP = 32


def layer_norm(x, weight, bias, eps):
    """(y, mean, rstd) over the last axis."""
    x = x.double()
    mean = x.mean(dim=-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(dim=-1, keepdim=True) + eps)
    y = (x - mean) * rstd
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    return y, mean[..., 0], rstd[..., 0]


def layer_norm_backward(dy, x, weight, mean, rstd):
    """(d_x, d_weight, d_bias)."""
    dy, x = dy.double(), x.double()
    rstd = rstd.double()[..., None]
    xh = (x - mean.double()[..., None]) * rstd
    a = dy if weight is None else dy * weight.double()
    dx = rstd * (a - a.mean(dim=-1, keepdim=True) - xh * (a * xh).mean(dim=-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    return dx, (dy * xh).sum(dim=rows) if rows else dy * xh, dy.sum(dim=rows) if rows else dy.clone()


def act(z, name):
    z = z.double()
    if name == "silu":
        return z * torch.sigmoid(z)
    return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))


def act_grad(z, name):
    z = z.double()
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)


def gated_linear(x, weight, bias, name):
    """(out, z)."""
    z = x.double() @ weight.double().t()
    if bias is not None:
        z = z + bias.double()
    f = weight.shape[0] // 2
    return act(z[..., :f], name) * z[..., f:], z


def gated_linear_backward(dout, x, weight, z, name):
    """(d_x, d_weight, d_bias, dz) for a given z."""
    f = weight.shape[0] // 2
    dout, z = dout.double(), z.double()
    dz = torch.cat([dout * z[..., f:] * act_grad(z[..., :f], name), dout * act(z[..., :f], name)], dim=-1)
    d2, x2 = dz.reshape(-1, 2 * f), x.double().reshape(-1, x.shape[-1])
    return dz @ weight.double(), d2.t() @ x2, d2.sum(dim=0), dz


def pack8(x):
    """(code values before the exponent, exponent bytes) of ``[rows, cols]``: by search, one group at a time in 64 bits."""
    x = x.double()
    rows, cols = x.shape
    groups = (cols + GROUP - 1) // GROUP
    vals, exps = torch.zeros_like(x), torch.zeros(rows, groups, dtype=torch.uint8)
    for gi in range(groups):
        v = x[:, gi * GROUP:(gi + 1) * GROUP]
        top = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dim=1)
        e = torch.full((rows,), -126, dtype=torch.int64)
        while bool((top > 448.0 * torch.ldexp(torch.ones_like(top), e)).any()):
            e = torch.where(top > 448.0 * torch.ldexp(torch.ones_like(top), e), e + 1, e)
        s = torch.ldexp(torch.where(torch.isfinite(v), v, torch.full_like(v, float("nan"))), -e[:, None])
        # nearest multiple of the step of the binade (2^-9 at the smallest), ties to even
        _, ex = torch.frexp(s)
        step = torch.ldexp(torch.ones_like(s), (ex.to(torch.int64) - 1).clamp(min=-6) - 3)
        vals[:, gi * GROUP:(gi + 1) * GROUP] = torch.round(s / step) * step
        exps[:, gi] = (e + 127).to(torch.uint8)
    return vals, exps


def unpack8(vals, exps, dtype):
    """What codes and exponents stand for in ``dtype``, in 64 bits (rounded to ``dtype`` where its precision or range asks for it)."""
    cols = vals.shape[-1]
    e = (exps.to(torch.int64) - 127).repeat_interleave(GROUP, dim=-1)[..., :cols]
    top = torch.finfo(dtype).max
    return torch.ldexp(vals.double(), e).clamp(-top, top)
