"""Products of tokens in 8-bit integers, in 64 bits on the CPU (not collected by
pytest).

Codes are defined by fp32 steps, which numpy rounds one at a time; the sum of
their products is exact; what follows is fp32: e = 2^-24 a rounding."""
import numpy as np
import torch

from token_reference import E, SUBNORMAL, UNIT


def codes(x):
    """x [rows, k] of any type -> (codes int64 [rows, k], scale float32 [rows]); finite rows."""
    x = x.detach().cpu().float().numpy()
    most = np.abs(x).max(1) if x.shape[1] else np.zeros(len(x), np.float32)
    scale = np.where(most > 0, np.maximum(most * np.float32(1 / 127), np.float32(2.0 ** -126)), np.float32(0))
    inv = np.where(scale > 0, np.float32(1) / np.where(scale > 0, scale, np.float32(1)), np.float32(0))
    q = x * inv[:, None]
    assert q.dtype == np.float32
    q = np.trunc(q + np.copysign(np.float32(0.5), q)).clip(-127, 127).astype(np.int64)
    return torch.from_numpy(q), torch.from_numpy(scale)


def product(x, w, ws, bias, act):
    """x [rows, k], w int8 [n, k], ws [n], bias [n] or None -> (y, bound) in 64 bits.

    (float)sum, s * ws, their product and the bias's addition: four roundings, of the product's size but the last.
    SiLU is at most 1.1 steep; exp of |y| has a relative error of some 2 + 1.5 |y| roundings (its argument's times its
    size), the sum and quotient two more."""
    q, s = codes(x)
    p = (q.double() @ w.cpu().double().t()) * s.double()[:, None] * ws.cpu().double()
    b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.cpu().double()
    y = p + b
    off = 4 * E * (p.abs() + b.abs())
    u = UNIT[x.dtype]
    if act == "silu":
        z = y * torch.sigmoid(y)
        off = 1.1 * off + (6 + 2 * y.abs()) * E * z.abs() + 1e-36
    else:
        z = y.clamp_min(0) if act == "relu" else y
    return z, off * (1 + u) + u * z.abs() + SUBNORMAL[x.dtype]
