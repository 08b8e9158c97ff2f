"""Float64 restatement of the residual join with the norms around it (no reference code).

  u = N_post(o);  t = sigmoid(gate) * u;  r = x + a * t;  h = N_pre(r)

N a LayerNorm or ("rms") an RMS norm over the last axis. The backward starts from r.
"""

import numpy as np

__all__ = ["norm", "norm_bwd", "residual_norm", "residual_norm_bwd"]


def _sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


def _f64(x):
    return None if x is None else np.asarray(x, np.float64)


def _hat(v, kind, eps):
    mean = v.mean(-1, keepdims=True) if kind == "layer" else 0.0
    rstd = 1.0 / np.sqrt(((v - mean) ** 2).mean(-1, keepdims=True) + eps)
    return (v - mean) * rstd, rstd


def norm(v, pair, kind="layer", eps=1e-5):
    scale, offset = (_f64(p) for p in pair)
    y = _hat(_f64(v), kind, eps)[0] * scale
    return y if offset is None else y + offset


def norm_bwd(v, pair, dy, kind="layer", eps=1e-5):
    """(dv, dscale, doffset)"""
    hat, rstd = _hat(_f64(v), kind, eps)
    g = dy * _f64(pair[0])
    dv = g - hat * (g * hat).mean(-1, keepdims=True)
    if kind == "layer":
        dv = dv - g.mean(-1, keepdims=True)
    axes = tuple(range(dy.ndim - 1))
    return rstd * dv, (dy * hat).sum(axes), dy.sum(axes)


def residual_norm(x, o, gate=None, post=None, res_scale=None, pre=None, kind="layer", eps=1e-5):
    """(r, h), r not rounded; h None without pre."""
    t = _f64(o) if post is None else norm(o, post, kind, eps)
    if gate is not None:
        t = _sigmoid(_f64(gate)) * t
    r = _f64(x) + (t if res_scale is None else _f64(res_scale) * t)
    return r, None if pre is None else norm(r, pre, kind, eps)


def residual_norm_bwd(r, o, gate, post, res_scale, pre, dr, dh, kind="layer", eps=1e-5):
    """(dx, do, dgate, dpost_scale, dpost_offset, dres_scale, dpre_scale, dpre_offset); None for
    what is not there."""
    o = _f64(o)
    d = np.zeros_like(o) if dr is None else _f64(dr)
    dpre = [None, None]
    if pre is not None:
        back, *dpre = norm_bwd(r, pre, _f64(dh), kind, eps)
        d = d + back
    u = o if post is None else norm(o, post, kind, eps)
    sig = np.ones_like(o) if gate is None else _sigmoid(_f64(gate))
    dt = d if res_scale is None else d * _f64(res_scale)
    axes = tuple(range(o.ndim - 1))
    dres = None if res_scale is None else (d * sig * u).sum(axes)
    dgate = None if gate is None else dt * u * sig * (1.0 - sig)
    do, dpost = dt * sig, [None, None]
    if post is not None:
        do, *dpost = norm_bwd(o, post, do, kind, eps)
    for pair, grads in ((post, dpost), (pre, dpre)):
        if pair is not None and pair[1] is None:
            grads[1] = None
    return d, do, dgate, dpost[0], dpost[1], dres, dpre[0], dpre[1]
