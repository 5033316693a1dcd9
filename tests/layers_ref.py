"""Plain 64-bit forms of the network's layers (Engine.rotary, group_norm, gated, Plan.mask_head)
with, for each output, a bound on how far a float computation with one rounding at the end may be
from it. Half a unit of the last place of a type is torch.finfo(t).eps / 2 relative to the value;
F32 is that of float. The constants of the bounds count roundings:

* a product or sum of floats is off by F32 of its value, a sum of n products taken in order by
  (n + 1) F32 of the sum of their sizes; tensor cores may cut instead of round, twice that;
* CUDA's expf, erfcf, sincospif and the division are within 4 units of the last place; the fast
  exponential and division of the 16-bit paths are within 2^-21 relative plus 2^-22 times the
  exponent, 2^-17 at the largest exponent a test reaches (|z| <= 32).
"""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24
FAST = {torch.float32: 16 * F32, torch.float16: 2.0 ** -17, torch.bfloat16: 2.0 ** -17}


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the spacing of the subnormal numbers: what rounding may lose near zero."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def act(kind, z):
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if kind == "sigmoid":
        return torch.sigmoid(z)
    if kind == "relu":
        return torch.clamp_min(z, 0)
    return z


def act_grad(kind, z):
    if kind == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "sigmoid":
        s = torch.sigmoid(z)
        return s * (1 - s)
    if kind == "relu":
        return (z > 0).to(z.dtype)
    return torch.ones_like(z)


def worst(got, want, bound):
    """The largest |got - want| / bound; inf where the two disagree on what is finite."""
    got = got.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    if not got.numel():
        return 0.0
    same = torch.isnan(got) == torch.isnan(want)
    inf = torch.isinf(want) | torch.isinf(got)
    same &= ~inf | (got == want)
    if not bool(same.all()):
        return math.inf
    fine = torch.isfinite(want)
    return float(((got - want).abs() / bound)[fine].max()) if bool(fine.any()) else 0.0


def rotary(x, pos, freq, mag, rotary_dim, layout, inverse=False):
    """x [B][T][H][D], pos [T] or [B][T]: (y, bound)."""
    d, half = x.double(), rotary_dim // 2
    a = pos.double()[..., None] * torch.as_tensor(freq, device=x.device)
    a = (a if a.dim() == 3 else a[None])[:, :, None] * (-1 if inverse else 1)
    c, s = mag * torch.cos(a), mag * torch.sin(a)
    if layout == "interleaved":
        i0, i1 = torch.arange(0, rotary_dim, 2), torch.arange(1, rotary_dim, 2)
    else:
        i0, i1 = torch.arange(half), torch.arange(half, rotary_dim)
    y = d.clone()
    x0, x1 = d[..., i0], d[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    # cos and sin to 4 units, two products and a sum; the double angle's own 2^-52 of it
    size = torch.zeros_like(d)
    size[..., i0] = size[..., i1] = (x0.abs() + x1.abs()) * mag * (8 * F32 + 2.0 ** -51 * a.abs())
    return y, size + half_ulp(x.dtype) * y.abs() + tiny(x.dtype)


def group_norm(x, groups, gamma, beta, eps, kind):
    """x [B][L][C]: (y, bound, mean, rstd)."""
    d = x.double()
    b, n, ch = d.shape
    g = d.reshape(b, n, groups, -1)
    mean = g.mean((1, 3), keepdim=True)
    var = (g - mean).square().mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    ga = torch.ones(ch, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    be = torch.zeros(ch, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    xh = ((g - mean) * rstd).reshape(b, n, ch)
    z = xh * ga + be
    y = act(kind, z)
    # the mean is off by at most 32 F32 of the largest |x - pivot|, below twice the spread plus
    # its own rounding; rstd by 64 F32; the affine map by 4 F32 of its terms; slopes are below 1.2
    spread = (g - mean).abs().amax((1, 3), keepdim=True)
    dz = ((32 * 2 * spread + 4 * (g.abs() + mean.abs())) * rstd * F32).expand_as(g).reshape(b, n, ch) * ga.abs()
    dz = dz + (64 + 4) * F32 * ((xh * ga).abs() + be.abs())
    return y, 1.2 * dz + (FAST[x.dtype] + half_ulp(x.dtype)) * y.abs() + tiny(x.dtype), mean.flatten(1), rstd.flatten(1)


def group_norm_backward(dy, x, groups, gamma, beta, mean, rstd, kind):
    """((dx, dgamma, dbeta), their bounds), mean and rstd [B][G] as the call is given them."""
    d, b, n, ch = x.double(), *x.shape
    ga = torch.ones(ch, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    be = torch.zeros(ch, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    mu, rs = mean.double()[:, None, :, None], rstd.double()[:, None, :, None]
    per = lambda t: t.reshape(b, n, groups, -1)  # noqa: E731
    xh = ((per(d) - mu) * rs).reshape(b, n, ch)
    exh = ((per(d).abs() + mu.abs()) * rs * 3 * F32).reshape(b, n, ch)      # difference and product
    z = xh * ga + be
    ez = exh * ga.abs() + 2 * F32 * (z.abs() + be.abs())
    slope, w = act_grad(kind, z), dy.double()
    eslope = (0 if kind == "none" else 1.0) * ez + FAST[x.dtype] * (1 + z.abs()) * (kind != "none")   # second derivatives below 1
    if kind == "relu":
        eslope = eslope * 0 + (z.abs() <= ez).double()      # either side of the corner
    dz = w * slope
    edz = w.abs() * eslope + 2 * F32 * dz.abs()
    terms, eterms = dz * xh, edz * xh.abs() + dz.abs() * exh
    dgamma, dbeta = terms.sum((0, 1)), dz.sum((0, 1))
    # sums in order of at most 1024 terms a thread, then joined: 1100 roundings of the sizes
    egamma = eterms.sum((0, 1)) + 1100 * F32 * terms.abs().sum((0, 1))
    ebeta = edz.sum((0, 1)) + 1100 * F32 * dz.abs().sum((0, 1))
    dd, m = dz * ga, n * (ch // groups)
    first, second = per(dd).sum((1, 3), keepdim=True) / m, per(dd * xh).sum((1, 3), keepdim=True) / m
    efirst = per(edz * ga.abs() + 1200 * F32 * dd.abs()).sum((1, 3), keepdim=True) / m
    esecond = per((eterms + 1200 * F32 * terms.abs()) * ga.abs()).sum((1, 3), keepdim=True) / m
    dx = rs * (per(dd) - first - per(xh) * second)
    size = per(dd).abs() + first.abs() + (per(xh) * second).abs()
    edx = rs * (per(edz * ga.abs()) + efirst + per(xh).abs() * esecond + per(exh) * second.abs() + 4 * F32 * size)
    dx, edx = dx.reshape(b, n, ch), edx.reshape(b, n, ch)
    pt = gamma.dtype if gamma is not None else torch.float32
    return ((dx, dgamma, dbeta), (edx + half_ulp(x.dtype) * dx.abs() + tiny(x.dtype), egamma + half_ulp(pt) * dgamma.abs() + tiny(pt),
                                  ebeta + half_ulp(pt) * dbeta.abs() + tiny(pt)))


def _projection(x, w, b):
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b, size + b.abs()
    return z, 2 * (x.shape[-1] + 2) * F32 * size


def gated(x, wg, wu, bg, bu, kind):
    """x [m][k]: (y, bound)."""
    t = x.dtype
    d = [None if v is None else v.double() for v in (x, wg, wu, bg, bu)]
    (g, eg), (u, eu) = _projection(d[0], d[1], d[3]), _projection(d[0], d[2], d[4])
    a = act(kind, g)
    ea = 1.2 * eg + FAST[t] * a.abs()
    y = a * u
    return y, ea * (u.abs() + eu) + a.abs() * eu + (half_ulp(t) + 2 * F32) * y.abs() + tiny(t)


def gated_backward(dy, x, wg, wu, bg, bu, kind):
    """((dx, dwg, dwu, dbg, dbu), their bounds): the projections' gradients are rounded to the
    type between the products, everything else once."""
    t = x.dtype
    d = [None if v is None else v.double() for v in (x, wg, wu, bg, bu)]
    (g, eg), (u, eu) = _projection(d[0], d[1], d[3]), _projection(d[0], d[2], d[4])
    w = dy.double()
    a, s = act(kind, g), act_grad(kind, g)
    ea = 1.2 * eg + FAST[t] * a.abs()
    es = (kind != "none") * (eg + FAST[t] * (1 + g.abs()))
    if kind == "relu":
        es = (g.abs() <= eg).double()
    dg, du = w * u * s, w * a
    edg = w.abs() * (eu * s.abs() + u.abs() * es + eu * es) + 2 * F32 * dg.abs()
    edu = w.abs() * ea + F32 * du.abs()
    rdg, rdu = edg + half_ulp(t) * (dg.abs() + edg) + tiny(t), edu + half_ulp(t) * (du.abs() + edu) + tiny(t)   # as the next product sees them
    n, m = dg.shape[1], dg.shape[0]
    dx = dg @ d[1] + du @ d[2]
    edx = rdg @ d[1].abs() + rdu @ d[2].abs() + 2 * (2 * n + 2) * F32 * ((dg.abs() + rdg) @ d[1].abs() + (du.abs() + rdu) @ d[2].abs())
    out, err = [dx], [edx]
    for v, ev in ((dg, rdg), (du, rdu)):
        out.append(v.t() @ d[0])
        err.append(ev.t() @ d[0].abs() + 2 * (m + 2) * F32 * ((v.abs() + ev).t() @ d[0].abs()))
    # the tensor cores sum the rounded gradients, the CUDA cores (float32) the ones before rounding
    for v, ev in ((dg, edg if t == torch.float32 else rdg), (du, edu if t == torch.float32 else rdu)):
        out.append(v.sum(0))
        err.append(ev.sum(0) + 2 * (m + 2) * F32 * (v.abs() + ev).sum(0))
    return out, [e + half_ulp(t) * o.abs() + tiny(t) for o, e in zip(out, err)]


def mask_head(hidden, weight, bias, din):
    """hidden [n][S][bands][T][K]: (masks [n][..], bound)."""
    t = hidden.dtype
    h, w = hidden.double(), weight.double()
    masks, bounds = [], []
    for c in range(h.shape[0]):
        for s in range(h.shape[1]):
            at = 0
            for band, d in enumerate(din):
                b = None if bias is None else bias[s].double()
                v, ev = _projection(h[c, s, band], w[s, at:at + d], None if b is None else b[at:at + d])
                g, eg = _projection(h[c, s, band], w[s, at + d:at + 2 * d], None if b is None else b[at + d:at + 2 * d])
                q = torch.sigmoid(g)
                eq = 0.3 * eg + FAST[t] * q      # the sigmoid's slope is at most 1/4
                masks.append((v * q).flatten())
                bounds.append((ev * (q + eq) + v.abs() * eq + 2 * F32 * (v * q).abs() + 1e-40).flatten())
                at += 2 * d
    n = h.shape[0]
    return torch.cat(masks).view(n, -1), torch.cat(bounds).view(n, -1)
