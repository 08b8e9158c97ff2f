"""AdamW steps (no reference code): in float64, and the 8-bit states' codes in float32.

  g = grad * grad_scale;  m = b1*m + (1 - b1)*g;  v = b2*v + (1 - b2)*g*g
  p = p*(1 - lr*decay) - lr/(1 - b1^t) * m / (sqrt(v)/sqrt(1 - b2^t) + eps)

encode and decode are the definition of the 8-bit states, operation by operation in float32 (each
rounded once, as the codes next to a border depend on it), over blocks of 256 elements.
"""

import numpy as np

__all__ = ["BLOCK", "moments32", "step", "encode", "decode"]

BLOCK = 256
_f32 = np.float32


def step(p, grad, m, v, t, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0,
         grad_scale=1.0):
    """(p, m, v) after the t-th step, float64."""
    p, grad, m, v = (np.asarray(a, np.float64) for a in (p, grad, m, v))
    g = grad * grad_scale
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    denom = np.sqrt(v) / np.sqrt(1 - beta2 ** t) + eps
    return p * (1 - lr * weight_decay) - lr / (1 - beta1 ** t) * m / denom, m, v


def moments32(grad, m, v, beta1=0.9, beta2=0.999, grad_scale=1.0):
    """(m, v) in float32, each operation rounded once."""
    g = np.asarray(grad, _f32) * _f32(grad_scale)
    m = np.asarray(m, _f32) * _f32(beta1) + g * _f32(1 - beta1)
    v = np.asarray(v, _f32) * _f32(beta2) + (g * _f32(1 - beta2)) * g
    return m, v


def _blocks(x):
    n = -(-x.size // BLOCK) * BLOCK
    return np.concatenate([x.reshape(-1), np.zeros(n - x.size, x.dtype)]).reshape(-1, BLOCK)


def encode(m, v):
    """(int8 codes, uint8 codes, float32 scales [blocks, 2]) of flat float32 states."""
    size = m.size
    m, v = _blocks(np.asarray(m, _f32)), _blocks(np.asarray(v, _f32))
    scales = np.stack([np.abs(m).max(1), v.max(1)], 1)
    over = np.where(scales > 0, scales, _f32(1))
    qm = np.sign(m) * np.rint(np.sqrt(np.abs(m) / over[:, :1]) * _f32(127))
    qv = np.rint(np.sqrt(np.sqrt(v / over[:, 1:])) * _f32(255))
    qv = np.where(v > 0, np.maximum(qv, 1), qv)
    return (qm.astype(np.int8).reshape(-1)[:size], qv.astype(np.uint8).reshape(-1)[:size], scales)


def decode(qm, qv, scales):
    """(m, v) float32 that the codes stand for."""
    size = qm.size
    rm = _blocks(qm).astype(_f32) * _f32(1 / 127)
    rv = _blocks(qv).astype(_f32) * _f32(1 / 255)
    rv = rv * rv
    return ((rm * np.abs(rm)) * scales[:, :1]).reshape(-1)[:size], (
        (rv * rv) * scales[:, 1:]).reshape(-1)[:size]
