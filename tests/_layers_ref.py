"""Plain 64-bit forms of the layers with dropout and gradients, on the CPU, with bounds on what 32-bit arithmetic and
the rounding to the tensors' type may do to them.

Bounds: ``u`` = 2^-24 is half a step of fp32; a sum of n products in fp32 in any order is off by at most n u times the
sum of the products' magnitudes; a value rounded to type t by finfo(t).eps / 2 of itself (plus half the smallest
denormal).  The activations' and their derivatives' own error is ``ACT_ERR`` per unit of max(1, |z|): the 16-bit path
takes Abramowitz & Stegun 7.1.26 (1.5e-7) with a hardware exponential and reciprocal of about 2^-22; 2e-6 covers the sum.
Slopes: |silu'|, |gelu'|, |quick_gelu'| <= 1.13, second derivatives <= 0.86 (quick GELU: 1.702 / 2)."""
import math

import numpy as np
import torch

U = 2.0 ** -24
ACT_ERR = 2e-6


def philox(ctr, key):
    """Philox4x32-10 (Salmon et al. 2011) over arrays of 32-bit words."""
    c = [np.asarray(v, np.uint64) for v in np.broadcast_arrays(*ctr)]
    k0, k1 = (int(v) for v in key)
    m = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def keep_scale(shape, p, seed, offset, row0=0):
    """The mask times its scale, fp64; rows numbered from row0."""
    shape = tuple(shape) or (1,)
    t = int(np.rint(p * 65536))
    if t == 0:
        return torch.ones(shape, dtype=torch.float64)
    if t == 65536:
        return torch.zeros(shape, dtype=torch.float64)
    cols = shape[-1]
    rows = int(np.prod(shape[:-1], dtype=np.int64))
    n8 = (cols + 7) // 8
    r = (np.arange(rows, dtype=np.uint64) + np.uint64(row0))[:, None]
    seed &= (1 << 64) - 1
    w = philox((np.arange(n8, dtype=np.uint64)[None], r & np.uint64(0xFFFFFFFF), r >> np.uint64(32), np.uint64(offset)),
               (seed & 0xFFFFFFFF, seed >> 32))
    num = np.stack([h for v in w for h in (v & np.uint64(0xFFFF), v >> np.uint64(16))], axis=2).reshape(rows, n8 * 8)
    keep = torch.from_numpy(num[:, :cols].astype(np.int64) >= t)
    return (keep.double() * (65536.0 / (65536 - t))).reshape(shape)


def act(z, name):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "quick_gelu":
        return z * torch.sigmoid(1.702 * z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    return z


def act_grad(z, name):
    if name is None:
        return torch.ones_like(z)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    a = 1.702 if name == "quick_gelu" else 1.0
    s = torch.sigmoid(a * z)
    return s + a * z * s * (1 - s)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(ref, err, dtype):
    """Bound of a value with error ``err`` behind its rounding to dtype."""
    return err + half(dtype) * (ref.abs() + err) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def check(name, got, ref, bound):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.isfinite(got).all(), name
    over = (got - ref).abs() - bound
    worst = float(over.max()) if over.numel() else 0.0
    if worst > 0:
        i = int(over.argmax())
        raise AssertionError(f"{name}: {float(got.flatten()[i])} for {float(ref.flatten()[i])}, bound "
                             f"{float(bound.expand_as(ref).flatten()[i]):.3e} (element {i} of {tuple(ref.shape)})")


def d(t):
    return None if t is None else t.detach().double().cpu()


def linear_ref(x, w, bias, resid, dy, name, p, seed, offset, dtype):
    """(values, bounds) of y, dx, dw, db for inputs of any type (taken as they are)."""
    x, w, bias, resid, dy = d(x), d(w), d(bias), d(resid), d(dy)
    k, n = w.shape[1], w.shape[0]
    lead = x.shape[:-1]
    x = x.reshape(-1, k)
    m = x.shape[0]
    s = keep_scale((m, n), p, seed, offset)
    z, za = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, za = z + bias, za + bias.abs()
    ez = (k + 2) * U * za
    one = torch.ones_like(z)
    ea = (1.13 * ez + ACT_ERR * torch.maximum(one, z.abs())) if name else ez
    y = s * act(z, name)
    ey = s * ea + 4 * U * y.abs()
    if resid is not None:
        r = resid.reshape(m, n)
        y, ey = y + r, ey + U * (y.abs() + r.abs())
    out = {"y": (y.reshape(lead + (n,)), rounded(y, ey, dtype).reshape(lead + (n,)))}
    if dy is None:
        return out
    g = dy.reshape(m, n)
    dz = g * s * act_grad(z, name)
    edz = 4 * U * dz.abs()
    if name:
        edz = edz + (g * s).abs() * (0.86 * ez + ACT_ERR * torch.maximum(one, z.abs()))
    out["db"] = (dz.sum(0), edz.sum(0) + (m + 2) * U * dz.abs().sum(0))
    edr = rounded(dz, edz, dtype)            # dz goes through the products in the tensors' type
    dx = dz @ w
    edx = edr @ w.abs() + (n + 2) * U * ((dz.abs() + edr) @ w.abs())
    out["dx"] = (dx.reshape(lead + (k,)), rounded(dx, edx, dtype).reshape(lead + (k,)))
    dw = dz.t() @ x
    edw = edr.t() @ x.abs() + (m + 2) * U * ((dz.abs() + edr).t() @ x.abs())
    out["dw"] = (dw, rounded(dw, edw, dtype))
    return out


def groupnorm_ref(x, x1, gamma, beta, dy, eps, name, groups, p, seed, offset, dtype):
    """(values, bounds) of y, dx, dx1, dgamma, dbeta.  A statistic's sum is off by at most 200 u of its magnitudes: a
    thread adds at most about 100 values one after the other, the rest are folds of a few dozen (then doubles)."""
    x, x1, gamma, beta, dy = d(x), d(x1), d(gamma), d(beta), d(dy)
    c0 = x.shape[-1]
    shape = x.shape if x1 is None else x.shape[:-1] + (c0 + x1.shape[-1],)
    x = x if x1 is None else torch.cat([x, x1], dim=-1)
    b, c = x.shape[0], x.shape[-1]
    cpg = c // groups
    S = 200 * U
    v = x.reshape(b, -1, groups, cpg)
    mean = v.mean((1, 3), keepdim=True)
    t = v - mean
    var = (t * t).mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    hw = v.shape[1]                                                       # sums are taken about the middle of three values
    if hw:
        about = torch.stack([v[:, 0, :, 0], v[:, hw // 2, :, cpg // 2], v[:, -1, :, -1]]).median(0).values[:, None, :, None]
        off = (v - about).abs()
    else:
        off = t.abs()
    emean = S * off.mean((1, 3), keepdim=True) + U * mean.abs()
    evar = S * ((off * off).mean((1, 3), keepdim=True) + 2 * (mean - about if hw else mean).abs() * off.mean((1, 3), keepdim=True))
    ers = 0.5 * rstd ** 2 * evar * (1 + evar * rstd ** 2) + 4 * U         # relative
    xh = t * rstd
    exh = rstd * (emean + U * v.abs()) + xh.abs() * (ers + 3 * U)
    ga, be = gamma.reshape(groups, cpg), beta.reshape(groups, cpg)
    u = xh * ga + be
    eu = ga.abs() * exh + 2 * U * (xh.abs() * ga.abs() + be.abs())
    s = keep_scale(shape, p, seed, offset).reshape(v.shape)
    one = torch.ones_like(u)
    y = s * act(u, name)
    ey = s * (1.13 * eu + (ACT_ERR * torch.maximum(one, u.abs()) if name else 0)) + 4 * U * y.abs()
    out = {"y": (y.reshape(shape), rounded(y, ey, dtype).reshape(shape))}
    if dy is None:
        return out
    g = dy.reshape(v.shape) * s
    du = g * act_grad(u, name)
    edu = 4 * U * du.abs()
    if name:
        edu = edu + g.abs() * (0.86 * eu + ACT_ERR * torch.maximum(one, u.abs()))
    h, eh = du * ga, edu * ga.abs() + U * (du * ga).abs()
    a, q = h.mean((1, 3), keepdim=True), (h * xh).mean((1, 3), keepdim=True)
    ea = eh.mean((1, 3), keepdim=True) + S * h.abs().mean((1, 3), keepdim=True)
    eq = (eh * xh.abs() + h.abs() * exh).mean((1, 3), keepdim=True) + S * (h * xh).abs().mean((1, 3), keepdim=True)
    dx = rstd * (h - a - xh * q)
    edx = rstd * (eh + ea + xh.abs() * eq + exh * q.abs()) + (ers + 8 * U) * rstd * (h.abs() + a.abs() + (xh * q).abs())
    dxb = rounded(dx, edx, dtype).reshape(shape)
    dx = dx.reshape(shape)
    out["dx"] = (dx[..., :c0], dxb[..., :c0])
    if x1 is not None:
        out["dx1"] = (dx[..., c0:], dxb[..., c0:])
    n = 400 * U
    out["dgamma"] = ((du * xh).sum((0, 1)).reshape(c),
                     ((edu * xh.abs() + du.abs() * exh) + n * (du * xh).abs()).sum((0, 1)).reshape(c))
    out["dbeta"] = (du.sum((0, 1)).reshape(c), (edu + n * du.abs()).sum((0, 1)).reshape(c))
    return out
