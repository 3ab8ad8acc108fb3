"""Plain 64-bit forms of the channels-last operators, and how far a kernel may be from them.

The bounds count roundings.  A sum of n terms in fp32 is off by at most n 2^-23 times the sum of the terms' magnitudes (one
step a term; 2^-23 and not 2^-24 because the tensor cores' additions do not round to nearest).  A result that is stored in a
type is off by half a step more: finfo.eps / 2 relative, and half the smallest step near zero.  The activations' exponential and
division are good to (16 + |z|) 2^-23 relative.  Errors of the inputs of a product or an activation go through by the
product rule and by the activation's largest slopes; what is of second order is covered by 5 per cent."""
import math

import torch

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -23
# largest |act'| and |act''|
SLOPES = {"none": (1, 0), "relu": (1, 0), "silu": (1.1, 0.5), "gelu": (1.13, 0.8), "gelu_tanh": (1.13, 0.8), "sigmoid": (0.25, 0.1)}


def act(z, kind):
    """act(z), act'(z)"""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), (z > 0).to(z.dtype)
    s = torch.sigmoid(z)
    if kind == "sigmoid":
        return s, s * (1 - s)
    if kind == "silu":
        return z * s, s + z * s * (1 - s)
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * a * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1 - s) * 2 * a * (1 + 3 * 0.044715 * z * z)


def stored(value, err, dtype):
    """The bound of `value` once it is stored."""
    f = torch.finfo(DTYPES[dtype])
    return 1.05 * err + f.eps / 2 * (value.abs() + err) + f.smallest_normal * f.eps


def act_error(z, ez, kind):
    """bounds of act and act' where z is off by up to ez"""
    a, d = act(z, kind)
    s1, s2 = SLOPES[kind]
    own = (16 + z.abs()) * U
    ed = s2 * ez + own * 1.2 + (z.abs() <= ez).double() * (1.0 if kind == "relu" else 0.0)
    return s1 * ez + own * torch.maximum(a.abs(), z.abs()) * (kind != "relu" and kind != "none"), ed


def check(got, want, err, dtype, what):
    bound = stored(want, err, dtype)
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1, f"{what}: {worst:.3g} times the bound"


# ---- group norm -----------------------------------------------------------------------------------------------------

def norm(x, groups, eps, gamma, beta, kind, dtype, dy=None):
    """{name: (value, bound before storing)} of y, mean, rstd and, with dy, of dx, dgamma, dbeta.  All [n][p][c], 64 bits."""
    n, p, c = x.shape
    m = p * (c // groups)
    xg = x.reshape(n, p, groups, -1)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    var = ((xg - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    # sums run in parts of at most a few hundred terms that are joined: log-like, 64 steps are ample for the mean of |x|
    e_mean = 64 * U * xg.abs().mean(dim=(1, 3), keepdim=True)
    e_rstd = rstd * (64 * U + (e_mean * rstd) ** 2)
    xhat = (xg - mean) * rstd
    e_xhat = (e_mean + U * (xg.abs() + mean.abs())) * rstd + xhat.abs() * (e_rstd / rstd + 2 * U)
    flat = lambda t: t.reshape(n, p, c)  # noqa: E731
    z = flat(xhat) * gamma + beta
    ez = flat(e_xhat) * gamma.abs() + 2 * U * (z.abs() + beta.abs())
    y, slope = act(z, kind)
    ey, e_slope = act_error(z, ez, kind)
    out = {"y": (y, ey), "mean": (mean.reshape(n, groups), e_mean.reshape(n, groups)),
           "rstd": (rstd.reshape(n, groups), e_rstd.reshape(n, groups))}
    if dy is not None:
        dz, edz = dy * slope, dy.abs() * e_slope
        terms, eterms = dz * flat(xhat), edz * flat(xhat).abs() + dz.abs() * flat(e_xhat)
        out["dgamma"] = terms.sum((0, 1)), (eterms + 128 * U * terms.abs()).sum((0, 1))
        out["dbeta"] = dz.sum((0, 1)), (edz + 128 * U * dz.abs()).sum((0, 1))
        w, ew = (dz * gamma).reshape(xg.shape), (edz * gamma.abs()).reshape(xg.shape)
        mean_of = lambda t: t.mean(dim=(1, 3), keepdim=True)  # noqa: E731
        a, ea = mean_of(w), mean_of(ew) + 128 * U * mean_of(w.abs())
        b, eb = mean_of(w * xhat), mean_of(ew * xhat.abs() + w.abs() * e_xhat) + 128 * U * mean_of((w * xhat).abs())
        dx = rstd * (w - a - xhat * b)
        size = rstd * (w.abs() + a.abs() + (xhat * b).abs())
        edx = rstd * (ew + ea + xhat.abs() * eb + e_xhat * b.abs()) + size * (4 * U + e_rstd / rstd)
        out["dx"] = flat(dx), flat(edx)
    assert m > 0
    return out


# ---- gated feed-forward block ---------------------------------------------------------------------------------------

def ff(t, kind, dtype, dy=None):
    """The block on the 64-bit tensors of `t` (x, w_gate, w_up, w_down, b_gate, b_up, b_down; the biases may be None)."""
    half = torch.finfo(DTYPES[dtype]).eps / 2
    tiny = float(torch.finfo(DTYPES[dtype]).smallest_normal) * half * 2
    x, wg, wu, wd = t["x"], t["w_gate"], t["w_up"], t["w_down"]
    mag = lambda a, b: a.abs() @ b.abs()  # noqa: E731

    def project(v, w, b, ev=None):
        value, size = v @ w.t(), mag(v, w.t())
        err = (v.shape[1] + 4) * U * (size if b is None else size + b.abs())
        if ev is not None:
            err = err + ev @ w.t().abs()
        return (value if b is None else value + b), err

    g, eg = project(x, wg, t["b_gate"])
    u, eu = project(x, wu, t["b_up"])

    def gated(g, eg, u, eu):
        a, _ = act(g, kind)
        ea, _ = act_error(g, eg, kind)
        h = a * u
        err = 1.05 * (ea * u.abs() + a.abs() * eu + ea * eu)
        return h, err + half * (h.abs() + err) + tiny

    h, eh = gated(g, eg, u, eu)
    y, ey = project(h, wd, t["b_down"], eh)
    out = {"y": (y, ey), "gate": (g, eg), "up": (u, eu)}
    if dy is None:
        return out
    a, d = act(g, kind)
    ea, ed = act_error(g, eg, kind)
    dh, edh = dy @ wd, (dy.shape[1] + 4) * U * mag(dy, wd)

    def three(p, ep, q, eq, r, er):
        v = p * q * r
        err = 1.05 * (ep * (q * r).abs() + eq * (p * r).abs() + er * (p * q).abs() + ep * eq * r.abs() + ep * q.abs() * er
                      + p.abs() * eq * er)
        return v, err + half * (v.abs() + err) + tiny

    one, zero = torch.ones_like(g), torch.zeros_like(g)
    dg, edg = three(dh, edh, u, eu, d, ed)
    du, edu = three(dh, edh, a, ea, one, zero)
    h, eh = gated(g, eg, u, eu)
    steps = lambda k: (k + 4) * U  # noqa: E731
    out["dx"] = dg @ wg + du @ wu, (edg @ wg.abs() + edu @ wu.abs()) + steps(2 * g.shape[1]) * (mag(dg, wg) + mag(du, wu))
    rows = x.shape[0]
    for name, p, ep, q in (("dw_gate", dg, edg, x), ("dw_up", du, edu, x)):
        out[name] = p.t() @ q, ep.t() @ q.abs() + steps(rows) * mag(p.t(), q)
    out["dw_down"] = dy.t() @ h, dy.t().abs() @ eh + steps(rows) * mag(dy.t(), h)
    out["db_gate"] = dg.sum(0), edg.sum(0) + steps(rows) * dg.abs().sum(0)
    out["db_up"] = du.sum(0), edu.sum(0) + steps(rows) * du.abs().sum(0)
    out["db_down"] = dy.sum(0), steps(rows) * dy.abs().sum(0)
    return out
