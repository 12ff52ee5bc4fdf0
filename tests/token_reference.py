"""The token operators in 64 bits on the CPU, written from their formulas, and
the rounding bounds that go with them (not collected by pytest).

Units: u = half an ulp of the output's type relative to its value; e = 2^-24,
an fp32 rounding."""
import numpy as np
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SUBNORMAL = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
E = 2.0 ** -24


def f64(t):
    return t.detach().cpu().to(torch.float64)


def group_norm(x, groups, gamma, beta, eps, act):
    """x [n, pixels, c] -> (y, bound)."""
    dtype, x = x.dtype, f64(x)
    n, p, c = x.shape
    g = x.view(n, p, groups, c // groups)
    mean = g.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(g.var((1, 3), correction=0, keepdim=True) + eps)
    gamma = torch.ones(c, dtype=torch.float64) if gamma is None else torch.as_tensor(gamma, dtype=torch.float64)
    beta = torch.zeros(c, dtype=torch.float64) if beta is None else torch.as_tensor(beta, dtype=torch.float64)
    scale = (rstd * gamma.view(1, 1, groups, -1)).expand(n, 1, groups, -1).reshape(n, 1, c)
    xhat = ((g - mean) * rstd).reshape(n, p, c) * gamma
    y = xhat + beta
    # rounding of the mean (a few fp32 roundings of its size), of the spread (relative), and of the last steps
    off = 8 * E * mean.abs().expand(n, 1, groups, c // groups).reshape(n, 1, c) * scale.abs() + 16 * E * (xhat.abs() + beta.abs())
    if act == "silu":
        # |silu'| <= 1.1; exp and the reciprocal in fp32
        return y * torch.sigmoid(y), 1.1 * off + 16 * E * y.abs() + UNIT[dtype] * (y * torch.sigmoid(y)).abs() + SUBNORMAL[dtype]
    y = y.clamp_min(0) if act == "relu" else y
    return y, off + UNIT[dtype] * y.abs() + SUBNORMAL[dtype]


def rotary(x, positions, sections, inv_freq, neighbours, inverse=False):
    """x [b, n, h, d], positions [b or 1, n, axes] -> (y, bound)."""
    dtype, x = x.dtype, f64(x)
    pairs = sum(sections)
    pos = positions.cpu().numpy().astype(np.longdouble)
    axis = np.repeat(np.arange(len(sections)), sections)
    two_pi = np.longdouble("6.283185307179586476925286766559")
    turn = pos[..., axis] * (np.asarray(inv_freq, np.float32).astype(np.longdouble) / two_pi)
    angle = torch.from_numpy(((turn - np.floor(turn)) * two_pi).astype(np.float64))[:, :, None]
    cos, sin = torch.cos(angle), torch.sin(angle) * (-1 if inverse else 1)
    y = x.clone()
    i = torch.arange(pairs)
    a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + pairs)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    bound = UNIT[dtype] * y.abs() + SUBNORMAL[dtype]
    both = (x[..., a].abs() + x[..., b].abs()) * 8 * E
    bound[..., a] += both
    bound[..., b] += both
    return y, bound


def attention(q, k, v, keep, scale, dtype=None):
    """q [b, lq, h, d], k and v [b, lk, hkv, d], keep bool [b, lq, lk] ->
    (out, bound).  Keys that nobody keeps take no part whatever they hold."""
    dtype = dtype or q.dtype
    q, k, v, keep = f64(q), f64(k), f64(v), keep.cpu()
    b, lq, h, d = q.shape
    lk, hkv = k.shape[1:3]
    used = keep.any(1)[:, :, None, None]
    k, v = torch.where(used, k, 0.0), torch.where(used, v, 0.0)
    q = q.view(b, lq, hkv, h // hkv, d).permute(0, 2, 3, 1, 4)
    k, v = k.permute(0, 2, 3, 1)[:, :, None], v.permute(0, 2, 1, 3)[:, :, None]
    s = q @ k * scale
    s = torch.where(keep[:, None, None], s, -torch.inf)
    top = s.amax(-1, keepdim=True) if lk else torch.zeros(s.shape[:-1] + (1,), dtype=s.dtype)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out, spread = p @ v, p @ v.abs()
    # A score's error: d products and sums, and the factor; twice, for the score and the largest one.  The
    # probability's: exp2 of a rounded argument.  The sums': one rounding a key.  Then the probability's and the
    # result's rounding to the type.
    reach = (q.abs() @ k.abs() * abs(scale)).amax(-1, keepdim=True) if lk else total
    score = 2 * (d + 8) * E * reach + 2 * E * s.masked_fill(torch.isinf(s), 0).abs().amax(-1, keepdim=True) * 4 if lk else total
    rel = score + (lk + 16) * E + 2 * UNIT[dtype]
    bound = rel * spread + UNIT[dtype] * out.abs() + SUBNORMAL[dtype] * 2
    back = lambda t: t.permute(0, 3, 1, 2, 4).reshape(b, lq, h, d)  # noqa: E731
    return back(out), back(bound)


def assert_within(got, want, bound, what=""):
    got = f64(got)
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} != {tuple(want.shape)}"
    off = (got - want).abs()
    bad = ~(off <= bound)  # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst {float((off / bound.clamp_min(1e-300)).nan_to_num(9e9).max()):.2f} of it"


def append(codes, scales, x, table, starts, counts, block):
    """The cache's append, fp32 step by step on the CPU: codes int8 [pages,
    heads, block, d], scales [pages, heads], x [b, tokens, heads, d]; returns
    new arrays."""
    codes, scales = codes.cpu().numpy().copy(), scales.cpu().numpy().copy()
    x, table = x.detach().cpu().float().numpy(), table.cpu().numpy()
    f = np.float32

    def steps(v, inv):
        with np.errstate(invalid="ignore", over="ignore"):
            s = (v * inv).astype(f)
            q = np.trunc((s + np.copysign(f(0.5), s)).astype(f))
        return np.clip(np.nan_to_num(q, nan=0.0, posinf=127, neginf=-127), -127, 127).astype(np.int8)

    for b in range(x.shape[0]):
        start, count = int(starts[b]), min(int(counts[b]), x.shape[1])
        if start < 0:
            continue
        for page in range(start // block, (start + max(count, 0) + block - 1) // block):
            lo, hi = max(start, page * block), min(start + count, (page + 1) * block)
            if lo >= hi or page >= table.shape[1] or not 0 <= table[b, page] < codes.shape[0]:
                continue
            i, had = table[b, page], lo - page * block
            for h in range(x.shape[2]):
                new = x[b, lo - start:hi - start, h]
                fin = np.abs(new[np.isfinite(new)])
                most = fin.max() if fin.size else f(0)
                want = max(f(most) * f(1 / 127), f(2.0 ** -126)) if most > 0 else f(0)
                was = scales[i, h] if had else f(0)
                now = max(f(want), was)
                inv = f(1) / now if now > 0 else f(0)
                if now != was:
                    codes[i, h, :had] = steps(codes[i, h, :had].astype(f), f(was * inv))
                codes[i, h, had:had + hi - lo] = steps(new, inv)
                scales[i, h] = now
    return codes, scales
