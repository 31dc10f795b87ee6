"""The channels-last operators in 64 bits (torch on the CPU or the GPU), from
their formulas, and the error bounds the tests hold the kernels to.

Bounds. u is half a step of the output's type (2^-9 relative for bf16 counted
as finfo.eps/2, and so on): the one rounding at the end. The rest is float32
arithmetic: E = 2^-24 times a count of roundings times the magnitudes that are
added, never the (possibly cancelled) result. The two-byte types evaluate
exponentials and reciprocals on the special-function unit; for |z| <= 16 the
argument z*log2(e) of exp2 carries 2^-24 * 23 and the unit 2 ulp, so sigmoid
and Phi are within 2^-19 relative, plus 1.5e-7 absolute for Phi's polynomial.
"""
import math

import torch

F64 = torch.float64
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (F64, torch.float32, torch.bfloat16, torch.float16)}
TINY = {F64: 0.0, torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def act(z, kind, t=1.0):
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2))
    if kind == "softclip":
        o = torch.relu(z.abs() - t)
        return torch.where(o > 0, torch.sign(z) * (t + o / (1 + o)), z)
    return z


def dact(z, kind, t=1.0):
    if kind == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "softclip":
        return (1 + torch.relu(z.abs() - t)) ** -2
    return torch.ones_like(z)


# Largest |act'| and |act''|.
SLOPE, CURVE = 1.13, 2.0


def spread(v, d):
    return v.repeat_interleave(d, -1)


def statistics(x, groups, eps, lens):
    n, s, c = x.shape
    mean = torch.zeros(n, groups, dtype=F64, device=x.device)
    rstd = torch.full((n, groups), 1 / math.sqrt(eps), dtype=F64, device=x.device)
    for i in range(n):
        if lens[i]:
            v = x[i, :lens[i]].to(F64).reshape(lens[i], groups, c // groups)
            mean[i] = v.mean((0, 2))
            var = ((v - mean[i][None, :, None]) ** 2).mean((0, 2))
            rstd[i] = (var + eps) ** -0.5
    return mean, rstd


def group_norm(x, w, b, groups, eps, kind, t, lens):
    """y (zeros where padded), mean, rstd, and a bound on y's error."""
    n, s, c = x.shape
    d = c // groups
    mean, rstd = statistics(x, groups, eps, lens)
    w = torch.ones(c, dtype=F64, device=x.device) if w is None else w.to(F64)
    b = torch.zeros(c, dtype=F64, device=x.device) if b is None else b.to(F64)
    y = torch.zeros(n, s, c, dtype=F64, device=x.device)
    bound = torch.zeros_like(y)
    fast = x.dtype != torch.float32
    for i in range(n):
        v = x[i, :lens[i]].to(F64)
        mu, r = spread(mean[i], d), spread(rstd[i], d)
        xh = (v - mu) * r
        z = xh * w + b
        y[i, :lens[i]] = act(z, kind, t)
        # mean = K + offset. The offset is a mean of differences x - K, each at
        # most 2 max|x|, whose partial sums carry rounding errors of their own
        # size: a thread's few values in order and then a tree, 8 roundings of
        # 2 max|x| together, whether or not the mean itself cancels to nothing;
        # and the mean's own rounding. rstd and the products: 16 roundings; the
        # bias's addition: 1.
        size = v.abs().max() if lens[i] else 0.0
        dz = 2.0 ** -24 * ((16 * size + mu.abs()) * r * w.abs() + 16 * (xh * w).abs() + z.abs()
                           + b.abs())
        ev = (2.0 ** -19 if fast else 2.0 ** -21) * z.abs()
        bound[i, :lens[i]] = SLOPE * dz + ev + HALF_STEP[x.dtype] * y[i, :lens[i]].abs()
    return y, mean, rstd, bound + TINY[x.dtype]


def group_norm_backward(dy, xv, mean, rstd, w, b, groups, kind, t, lens, dtype):
    """dx (zeros where padded), dw, db and bounds on their errors; xv holds the
    input (or what its checkpoint stands for) in 64 bits, mean and rstd what
    the kernel is given."""
    n, s, c = dy.shape
    d = c // groups
    w = torch.ones(c, dtype=F64, device=dy.device) if w is None else w.to(F64)
    b = torch.zeros(c, dtype=F64, device=dy.device) if b is None else b.to(F64)
    dx = torch.zeros(n, s, c, dtype=F64, device=dy.device)
    bx = torch.zeros_like(dx)
    dw, db, bw, bb = torch.zeros(4, c, dtype=F64, device=dy.device)
    fast = dtype != torch.float32
    for i in range(n):
        if not lens[i]:
            continue
        v, g = xv[i, :lens[i]].to(F64), dy[i, :lens[i]].to(F64)
        mu, r = spread(mean[i].to(F64), d), spread(rstd[i].to(F64), d)
        xh = (v - mu) * r
        z = xh * w + b
        dz = g * dact(z, kind, t)
        # xh: its subtraction is of values the size of |v| + |mu|; z: 4
        # roundings more; the slope moves by CURVE times z's error.
        exh = 2.0 ** -24 * (2 * xh.abs() + (v.abs() + mu.abs()) * r)
        ez = exh * w.abs() + 2.0 ** -24 * 4 * (z.abs() + b.abs())
        ev = 2.0 ** -18 if fast else 2.0 ** -21
        edz = g.abs() * (CURVE * ez + ev * (1 + z.abs()))
        # Sums: a thread adds at most 256 rows in order, the joins add 64.
        roundings = 2.0 ** -24 * (min(256, lens[i]) + 64)
        dw += (dz * xh).sum(0)
        db += dz.sum(0)
        ebw = edz * xh.abs() + dz.abs() * exh + roundings * (dz * xh).abs()
        bw += ebw.sum(0)
        bb += (edz + roundings * dz.abs()).sum(0)

        def mean_of(q):
            return spread(q.reshape(lens[i], groups, d).mean((0, 2)), d)

        s1, s2 = mean_of(dz * w), mean_of(dz * w * xh)
        e1 = mean_of((edz + roundings * dz.abs()) * w.abs())
        e2 = mean_of(ebw * w.abs())
        dx[i, :lens[i]] = r * (dz * w - s1 - xh * s2)
        bx[i, :lens[i]] = (r * (edz * w.abs() + e1 + xh.abs() * e2 + exh * s2.abs()
                                + 2.0 ** -24 * 6 * ((dz * w).abs() + s1.abs() + (xh * s2).abs()))
                           + HALF_STEP[dtype] * dx[i, :lens[i]].abs() + TINY[dtype])
    return dx, dw, db, bx, bw + 2.0 ** -126, bb + 2.0 ** -126


def pack(x, block):
    """(codes, scales) of a matrix, each float32 step of the format rounded."""
    r, c = x.shape
    codes = torch.zeros(r, c, dtype=torch.int8, device=x.device)
    scales = torch.zeros(r, -(-c // block), dtype=torch.float32, device=x.device)
    for k, lo in enumerate(range(0, c, block)):
        part = x[:, lo:lo + block].to(F64)
        bad = ~torch.isfinite(part).all(1, keepdim=True)
        top = part.abs().max(1, keepdim=True).values.clamp(min=2.0 ** -100)
        inverse = (127 / top).float().to(F64)
        q = torch.round((part * inverse).float().to(F64))
        codes[:, lo:lo + block] = torch.where(bad, 0.0, q).to(torch.int8)
        scales[:, k] = torch.where(bad, math.nan, top / 127)[:, 0].float()
    return codes, scales


def restore(codes, scales, block):
    """What they stand for, in 64 bits (each value a float32)."""
    c = codes.shape[1]
    s = scales.repeat_interleave(block, 1)[:, :c]
    return (codes.float() * s).to(F64)


def assert_within(name, got, want, bound):
    g = got.to(F64)
    assert g.shape == want.shape, (name, g.shape, want.shape)
    bad = ~((g - want).abs() <= bound)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{name}{list(i)}: got {float(g[i])!r}, want {float(want[i])!r}, "
                             f"off {float((g - want)[i].abs()):g}, bound {float(bound[i]):g}; "
                             f"{int(bad.sum())} of {bad.numel()} outside")
