"""Measured cases of the feed-forward half of a layer: ``layer_norm``, ``gated_linear`` (both projections, activation and
product) and 8-bit activation checkpoints.

Kinds of a case:

``norm_fwd``     y = LayerNorm(x) w + b over the last axis (serving)
``norm_train``   the same, then d_x, d_weight, d_bias for a given d_y
``gated_fwd``    h = act(x Wg^T + bg) * (x Wu^T + bu), W = (Wg | Wu) as one [2 f, k] matrix (serving)
``gated_train``  the same, then d_x, d_weight (, d_bias) for a given d_h; with ``ckpt8`` the backward reads the
                 pre-activations back from 8 bits
``pack``         an activation to 8 bits (e4m3 codes, one power-of-two exponent for 32 columns) and back
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
GROUP = 32


def listed():
    return [
        # the norm in front of a layer, for one token of one user: latency
        dict(name="norm_fwd_one_token", kind="norm_fwd", rows=1, cols=512, dtype="bf16"),
        # a training step over 262144 packed tokens at the layer's width
        dict(name="norm_train_512", kind="norm_train", rows=262144, cols=512, dtype="bf16"),
        # a norm over the head dim: 4 heads of 128 for each of 65536 tokens
        dict(name="norm_train_heads", kind="norm_train", rows=262144, cols=128, dtype="fp16"),
        # full precision, an odd number of rows, a width that is no multiple of a wave
        dict(name="norm_train_fp32_odd", kind="norm_train", rows=7687, cols=1000, dtype="fp32"),
        # one token: the weights are all there is to read
        dict(name="gated_fwd_one_token", kind="gated_fwd", m=1, k=512, f=2048, dtype="bf16", act="silu", bias=True, ckpt8=False),
        # the candidates of a small scoring request
        dict(name="gated_fwd_few_rows", kind="gated_fwd", m=48, k=1024, f=4096, dtype="fp16", act="silu", bias=False, ckpt8=False),
        # a prompt batch of packed histories
        dict(name="gated_fwd_batch", kind="gated_fwd", m=8192, k=1024, f=4096, dtype="bf16", act="silu", bias=False, ckpt8=False),
        # the training step of the block
        dict(name="gated_train", kind="gated_train", m=16384, k=1024, f=4096, dtype="bf16", act="silu", bias=False, ckpt8=False),
        # the same block with its pre-activations kept in 8 bits
        dict(name="gated_train_ckpt8", kind="gated_train", m=16384, k=512, f=2048, dtype="bf16", act="silu", bias=True, ckpt8=True),
        # ragged in every size: rows of x, W and h at any 2-byte boundary
        dict(name="gated_train_odd", kind="gated_train", m=2789, k=1001, f=2731, dtype="fp16", act="gelu", bias=True, ckpt8=False),
        # a small full-precision model
        dict(name="gated_train_fp32", kind="gated_train", m=1123, k=240, f=960, dtype="fp32", act="silu", bias=True, ckpt8=False),
        # an activation of a training batch put aside in 8 bits
        dict(name="pack_batch", kind="pack", rows=16384, cols=8192, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_fwd", "norm_train", "gated_fwd", "gated_train", "gated_train", "gated_train", "pack"])
    if kind in ("norm_fwd", "norm_train", "pack"):
        while True:
            rows, cols = _log_int(rng, 1, 262144), _log_int(rng, 16, 8192)
            if rng.random() < 0.5:
                cols = max(8, cols // 8 * 8)
            if rows * cols <= 16384 * 8192:
                break
        dtype = rng.choice(["bf16", "fp16"]) if kind == "pack" else rng.choice(["bf16", "fp16", "fp32"])
        return dict(kind=kind, rows=rows, cols=cols, dtype=dtype)
    while True:
        m, k, f = _log_int(rng, 1, 16384), _log_int(rng, 32, 2048), _log_int(rng, 32, 8192)
        if rng.random() < 0.6:
            k, f = max(16, k // 16 * 16), max(16, f // 16 * 16)
        if m * k * f <= 16384 * 1024 * 4096:
            break
    ckpt8 = kind == "gated_train" and rng.random() < 0.4
    dtype = rng.choice(["bf16", "fp16"]) if ckpt8 or m * k * f > 2048 * 1024 * 1024 else rng.choice(["bf16", "fp16", "fp32"])
    return dict(kind=kind, m=m, k=k, f=f, dtype=dtype, act=rng.choice(["silu", "silu", "gelu"]), bias=rng.random() < 0.5, ckpt8=ckpt8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std + mean).to(t)

    state = dict(case=dict(case))
    if case["kind"] in ("norm_fwd", "norm_train", "pack"):
        rows, cols = case["rows"], case["cols"]
        # a residual stream: channels of unequal scale and offset, a few large ones
        scale = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
        shift = 0.3 * torch.randn(cols, generator=g, device="cuda")
        state["x"] = (torch.randn(rows, cols, generator=g, device="cuda") * scale + shift).to(t)
        if case["kind"] != "pack":
            state["weight"], state["bias"] = normal(cols, std=0.2, mean=1.0), normal(cols, std=0.1)
        if case["kind"] == "norm_train":
            state["dy"] = normal(rows, cols)
            for n in ("x", "weight", "bias"):
                state[n].requires_grad_(True)
    else:
        m, k, f = case["m"], case["k"], case["f"]
        state["x"] = normal(m, k)
        state["weight"] = normal(2 * f, k, std=k ** -0.5)
        state["bias"] = normal(2 * f, std=0.1) if case["bias"] else None
        if case["kind"] == "gated_train":
            state["dh"] = normal(m, f)
            for n in ("x", "weight", "bias"):
                if state[n] is not None:
                    state[n].requires_grad_(True)
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------------

def _plain_norm(s, train):
    x, w, b = s["x"].detach(), s["weight"].detach().float(), s["bias"].detach().float()
    t, x = x.dtype, x.float()
    mean = x.mean(dim=1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(dim=1, keepdim=True) + EPS)
    xh = d * rstd
    y = (xh * w + b).to(t)
    if not train:
        return y
    dy = s["dy"].float()
    a = dy * w
    dx = (a - a.mean(dim=1, keepdim=True) - xh * (a * xh).mean(dim=1, keepdim=True)) * rstd
    return y, dx.to(t), (dy * xh).sum(dim=0).to(t), dy.sum(dim=0).to(t)


def _pow2(e):
    """2^e in 32 bits, exactly, for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_pack(v):
    """fp32 values -> the fp32 values that their 8-bit form stands for; groups of 32 along the last axis."""
    rows, cols = v.shape
    pad = (cols + GROUP - 1) // GROUP * GROUP
    wide = torch.zeros(rows, pad, dtype=torch.float32, device=v.device)
    wide[:, :cols] = v
    wide = wide.reshape(rows, pad // GROUP, GROUP)
    finite = torch.isfinite(wide)
    top = torch.where(finite, wide.abs(), 0.0).amax(dim=2, keepdim=True)
    frac, ex = torch.frexp(top)
    e = torch.where(top > 0, ex - 9 + (frac > 0.875).to(ex.dtype), -126).clamp(min=-126)
    scaled = torch.where(finite, wide, float("nan")) * _pow2(-e)
    back = scaled.to(torch.float8_e4m3fn).float() * _pow2(e)
    return back.reshape(rows, pad)[:, :cols]


def _plain_act(z, act):
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))


def _plain_act_grad(z, act):
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-z))
        return sg * (1.0 + z * (1.0 - sg))
    return 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5


def _plain_gated(s, case):
    t, f, act = s["x"].dtype, case["f"], case["act"]
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    zg, zu = z[:, :f], z[:, f:]
    h = (_plain_act(zg, act) * zu).to(t)
    if case["kind"] == "gated_fwd":
        return h
    if case["ckpt8"]:
        zg, zu = _plain_pack(zg), _plain_pack(zu)
    dh = s["dh"].float()
    dz = torch.cat([dh * zu * _plain_act_grad(zg, act), dh * _plain_act(zg, act)], dim=1)
    out = (h, (dz @ w).to(t), (dz.t() @ x).to(t))
    return out if s["bias"] is None else out + (dz.sum(dim=0).to(t),)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        import recsdk_amd  # noqa: F401

        ops = torch.ops.mxrec
        if kind == "norm_fwd":
            return ops.layer_norm(state["x"], state["weight"], state["bias"], EPS)
        if kind == "norm_train":
            leaves = [state["x"], state["weight"], state["bias"]]
            y = ops.layer_norm(*leaves, EPS)
            return (y.detach(),) + torch.autograd.grad(y, leaves, state["dy"])
        if kind == "pack":
            codes, exponents = ops.activation_pack8(state["x"])
            return ops.activation_unpack8(codes, exponents, state["x"].dtype)
        if kind == "gated_fwd":
            return ops.gated_linear(state["x"], state["weight"], state["bias"], case["act"])
        leaves = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
        h = ops.gated_linear(state["x"], state["weight"], state["bias"], case["act"], case["ckpt8"])
        return (h.detach(),) + torch.autograd.grad(h, leaves, state["dh"])
    if kind in ("norm_fwd", "norm_train"):
        return _plain_norm(state, kind == "norm_train")
    if kind == "pack":
        t = state["x"].dtype
        top = torch.finfo(t).max
        return _plain_pack(state["x"].float()).clamp(-top, top).to(t)
    return _plain_gated(state, case)


def work(case):
    e = _BYTES[case["dtype"]]
    if case["kind"] in ("norm_fwd", "norm_train", "pack"):
        rows, cols = case["rows"], case["cols"]
        n = rows * cols
        if case["kind"] == "norm_fwd":
            return {"bytes": (2 * n + 2 * cols) * e, "flops": 8 * n}
        if case["kind"] == "norm_train":
            return {"bytes": (4 * n + 4 * cols) * e, "flops": 20 * n}
        held = n + rows * ((cols + GROUP - 1) // GROUP)      # codes and exponents: written, and read again
        return {"bytes": 2 * n * e + 2 * held, "flops": 4 * n}
    m, k, f = case["m"], case["k"], case["f"]
    b = 2 * f if case["bias"] else 0
    if case["kind"] == "gated_fwd":
        return {"bytes": (m * k + 2 * f * k + b + m * f) * e, "flops": 4 * m * k * f}
    return {"bytes": (2 * m * k + 4 * f * k + 2 * b + 2 * m * f) * e, "flops": 12 * m * k * f}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------

def _pow2_exact(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _round_e4m3(y):
    """Nearest e4m3 value (ties to even) of |y| <= 448, in 64 bits: three mantissa bits, exponents from -6."""
    _, ex = torch.frexp(y)
    step = _pow2_exact((ex - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def _pack_exact(v):
    rows, cols = v.shape
    out = torch.empty_like(v)
    whole = cols // GROUP * GROUP
    for lo, hi, width in ((0, whole, GROUP), (whole, cols, cols - whole)):
        if hi == lo:
            continue
        part = v[:, lo:hi].reshape(rows, (hi - lo) // width, width)
        top = part.abs().amax(dim=2, keepdim=True)
        e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)).clamp(min=-126)
        # log2 may land on either side of a whole number: settle on the smallest exponent that holds the group
        e = torch.where(top <= 448.0 * _pow2_exact(e - 1), e - 1, e)
        e = torch.where(top > 448.0 * _pow2_exact(e), e + 1, e).clamp(min=-126)
        out[:, lo:hi] = (_round_e4m3(part * _pow2_exact(-e)) * _pow2_exact(e)).reshape(rows, hi - lo)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "pack":
        top = torch.finfo(s["x"].dtype).max
        return _pack_exact(s["x"].double()).clamp(-top, top)
    leaves = [s[n].detach().double().requires_grad_(kind.endswith("train")) for n in ("x", "weight", "bias") if s[n] is not None]
    if kind in ("norm_fwd", "norm_train"):
        x, w, b = leaves
        var = x.var(dim=1, keepdim=True, unbiased=False)
        y = (x - x.mean(dim=1, keepdim=True)) / torch.sqrt(var + EPS) * w + b
        if kind == "norm_fwd":
            return y
        return (y.detach(),) + torch.autograd.grad(y, leaves, s["dy"].double())

    def gated(z):
        g, u = z[:, :case["f"]], z[:, case["f"]:]
        return (g * torch.sigmoid(g) if case["act"] == "silu" else g * torch.special.ndtr(g)) * u

    z = torch.mm(leaves[0], leaves[1].t())
    if len(leaves) == 3:
        z = z + leaves[2]
    if kind == "gated_fwd":
        return gated(z)
    if not case["ckpt8"]:
        h = gated(z)
        return (h.detach(),) + torch.autograd.grad(h, leaves, s["dh"].double())
    held = z.detach()
    f = case["f"]
    held = torch.cat([_pack_exact(held[:, :f]), _pack_exact(held[:, f:])], dim=1).requires_grad_(True)
    dz = torch.autograd.grad(gated(held), held, s["dh"].double())[0]
    return (gated(z.detach()),) + torch.autograd.grad(z, leaves, dz)
