"""Plain 64-bit restatement of the operators of a deployed W8A8 decoder block (test infrastructure): the per-token
8-bit quantisation, the integer product, the residual add between two norms, the rotary embedding."""
import math

import torch


def quant_rows(v, sym=True):
    """v (rows, K) -> (codes int64, scales fp32 (rows,), zeros int64 (rows,)).  Scale and reciprocal are fp32 numbers by
    definition; the product with the reciprocal is formed exactly (fp64) and rounded half to even.  Rows that are not
    finite: scale NaN, codes 0, zero 0."""
    v32 = v.float()
    if sym:
        wide = v32.abs().amax(1).clamp(min=1e-5)
        s, r = wide / torch.tensor(127.0), torch.tensor(127.0) * (torch.tensor(1.0) / wide)
        z = torch.zeros(v.shape[0], dtype=torch.float64)
        low, high = -127, 127
    else:
        lo, hi = v32.amin(1).clamp(max=0), v32.amax(1).clamp(min=0)
        wide = (hi - lo).clamp(min=1e-5)
        s, r = wide / torch.tensor(255.0), torch.tensor(255.0) * (torch.tensor(1.0) / wide)
        z = -128 - torch.round(lo.double() * r.double())
        low, high = -128, 127
    bad = ~torch.isfinite(wide)
    q = (torch.round(v32.double() * r.double()[:, None]) + z[:, None]).clamp(low, high)
    q[bad], z[bad], s[bad] = 0, 0, float('nan')
    return q.long(), s, z.long()


def act(x, kind):
    """in fp64"""
    x = x.double()
    if kind == 'silu':
        return x / (1 + torch.exp(-x))
    if kind == 'gelu':
        return x * (1 + torch.erf(x / math.sqrt(2))) / 2
    return x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))) / 2


def int8_product(a, a_s, b, b_s, bias=None, a_z=None, out_dtype=torch.float32):
    """The integer product with its three fp32 operations and one rounding, each as the kernel documents it."""
    q = a.double() if a_z is None else a.double() - a_z.reshape(-1, 1).double()
    total = q @ b.double().t()                       # whole numbers below 2^53: exact
    y = total.float() * a_s.reshape(-1, 1).float() * b_s.reshape(1, -1).float()
    if bias is not None:
        y = y + bias.float()
    return y.to(out_dtype)


def rms(v, weight, eps, offset=0.0):
    v = v.double()
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * (weight.double() + offset)


def residual(x, res=None, post_weight=None, gate=None, scale=1.0, eps=1e-6, offset=0.0):
    """h before its rounding, in fp64"""
    t = x.double()
    if post_weight is not None:
        t = rms(t, post_weight, eps, offset)
    if gate is not None:
        t = t * gate.double()
    t = t * scale
    return t if res is None else res.double() + t


def rotary(x, positions, inv_freq, interleaved=False, scale=1.0):
    """x (B, H, T, D), in fp64"""
    r = 2 * inv_freq.numel()
    pos = positions if positions.dim() == 2 else positions[None]
    angle = pos.double()[:, None, :, None] * inv_freq.double()
    cos, sin = angle.cos() * scale, angle.sin() * scale
    out = x.double().clone()
    if interleaved:
        a, b = x[..., 0:r:2].double(), x[..., 1:r:2].double()
        out[..., 0:r:2], out[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :r // 2].double(), x[..., r // 2:r].double()
        out[..., :r // 2], out[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return out
